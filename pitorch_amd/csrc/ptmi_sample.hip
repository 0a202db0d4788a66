// Sampling of one token per row of logits: one workgroup a row.
//
// A row's order is that of its logits, larger first, equal ones by index, and
// every filter keeps a beginning of it: what stays is known by the smallest
// logit that stays and how many of its equals do.  top_k looks for the logit
// at which a count, top_p for the one at which a sum of weights reaches its
// mark: a histogram of the logits between two bounds in kBins bins of equal
// width, the bin that holds the mark, and so on in that bin; once few enough
// logits are left in it they are compared with each other.  A step is two
// passes over the row (one that fills the bins, one that takes out the
// members of the bin found), and of a language model's logits one step is
// enough.  The row is read from memory once, into shared memory (up to 32768
// logits; longer rows are read again, from the caches, for every pass).
//
// Weights are whole multiples of 2^-44 in 64 bits: sums of them are exact and
// the same in any order, so the atomics of the bins leave the result as it is.
//
// A row is one compute unit's work.  Of the 49 thousand cycles of a row of
// 32000 under top_p alone, the load takes 4, the pass that fills the bins (a
// weight each, some 35 instructions) 19, the search behind it 9, the draw 12;
// the count under top_k 10, as the bins' atomics go.  That row: 20.4 us; 64 rows
// of it with all sets of filters: 29.5; 509 rows of 50259, two rows on a unit:
// 90 (simple form, a bisection over the row: 177, 223, 535).
#include "ptmi_paged.h"

#include <cfloat>
#include <climits>

namespace ptmi {

namespace {

typedef unsigned long long u64;
typedef float f4v __attribute__((ext_vector_type(4)));

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2 * kThreads;
constexpr int kList = 256;           // logits of a bin that are compared with each other, by kThreads / kList threads each
static_assert(kSampleVocab <= 64 * 4 * kThreads - 4, "64 turns of a block, wherever in a float4 a row starts");

struct SampleArgs {
    const float *logits; long ld;
    int vocab;
    const float *temperature; const int *top_k; const float *top_p, *min_p, *u;
    int *token;
};

// ── weights ──────────────────────────────────────────────────────────────
// The coefficients of exp2_weight's polynomial, in scalar registers (as
// literals each would first be copied into a vector register for its fma:
// half as many instructions again).
struct Exp2Poly {
    double c[10];
    __device__ __forceinline__ Exp2Poly()
        : c{1.0000000000000135, 0.6931471805599462, 0.2402265069564034, 0.05550410866465167, 0.009618129193934313,
            0.0013333558200794592, 0.0001540343375125101, 1.5252672924850737e-05, 1.325964524488711e-06,
            1.0205905413765595e-07} {
#pragma unroll
        for (int i = 0; i < 10; i++) asm("" : "+s"(c[i]));
    }
};
// 2^y for y in (-1000, 0]: 2^n p(f), n the nearest integer, p of degree 9
// through 2^f at the Chebyshev nodes of [-1/2, 1/2] (relative error 1.9e-14,
// a third of 2^-44).  y + 1.5 2^52 has n as its last bits.
__device__ __forceinline__ double exp2_weight(const Exp2Poly &q, double y) {
    constexpr double kShift = 6755399441055744.0;
    const double n = y + kShift, f = y - (n - kShift);
    double p = q.c[9];
#pragma unroll
    for (int i = 8; i >= 0; i--) p = fma(p, f, q.c[i]);
    return __builtin_amdgcn_ldexp(p, (int)__double_as_longlong(n));
}
// To the nearest multiple of 2^-44, as their number: w + 2^8 has them as its last bits.
__device__ __forceinline__ u64 fixed(double w) {
    return (u64)(__double_as_longlong(w + 256.0) - __double_as_longlong(256.0));
}

// What a search adds up: counts, or weights.
struct CountOf {
    __device__ __forceinline__ u64 operator()(float) const { return 1; }
};
struct WeightOf {
    Exp2Poly poly;
    float top;
    double scale, min_p;             // log2(e) / temperature
    __device__ __forceinline__ u64 operator()(float x) const {
        const double w = exp2_weight(poly, fmax(((double)x - (double)top) * scale, -60.0));   // (x = top: 1 to the nearest 2^-44)
        return w >= min_p ? fixed(w) : 0;
    }
};

// ── sums over waves and the block ────────────────────────────────────────
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_add(u64 v) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_scan(u64 v) {          // inclusive
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}

// Lane i's value, i the same in all lanes.
__device__ __forceinline__ u64 lane_value(u64 v, int i) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, i);
}

constexpr int kQueue = 64 + 4 * 64;  // logits a wave has picked out: under 64, and what its next turn adds

struct SampleLds {
    union {
        u64 bins[kBins];
        float queue[kWaves][kQueue]; // of the draw
    };
    u64 wave[kWaves];
    float list_x[kList];
    u64 list_w[kList], above[kList], equal[kList];
    unsigned lo, hi;                 // of a bin's members, as ordered bits
    int members, bin, index;
    u64 before, sum;
    float value;
    u64 turn_sum[64];
};

// Floats as integers in the same order (-0 below 0).
__device__ __forceinline__ unsigned ordered(float x) {
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Sums over the waves, from every wave's sums over its lanes: lane w gets that of waves 0..w, from 15 on the whole
// one.  (s.wave is not to be written again before another barrier.)
__device__ __forceinline__ u64 sum_waves(u64 scanned, SampleLds &s, int wave) {
    const int lane = threadIdx.x & 63;
    if (lane == 63) s.wave[wave] = scanned;
    __syncthreads();
    return wave_scan(lane < kWaves ? s.wave[lane] : 0);
}

// ── a row ────────────────────────────────────────────────────────────────
__device__ __forceinline__ f4v only_infinite(f4v v) {
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = v[e] == INFINITY ? 0.0f : -INFINITY;
    return v;
}

// The row's logits in float4s of 16 aligned bytes: wave w has a run of 64
// `turns` of them, and in turn j its lane l float4 64 (w turns + j) + l.  What
// stands before and behind the row in its first and last float4 counts as
// -infinity, as NaN does; among infinite maxima only they count, as 0.  LOCAL:
// `at` is a copy in shared memory, else the row.
template <bool LOCAL>
struct Row {
    static constexpr int AHEAD = LOCAL ? 1 : 4;            // turns whose loads are on their way at once
    const f4v *at;
    int wave, skip, vocab, turns;    // skip: floats before the row in its first float4
    bool top_inf;

    __device__ __forceinline__ int place(int w, int j) const { return (w * turns + j) * 64 + ((int)threadIdx.x & 63); }
    __device__ __forceinline__ int index(int q) const { return 4 * q - skip; }       // of float4 q's first logit
    __device__ __forceinline__ f4v fetch(int w, int j) const {                       // from memory
        const int q = place(w, j), q0 = (w * turns + j) * 64;
        f4v v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (index(q0) >= 0 && index(q0 + 64) <= vocab) {                             // uniform: all inside
            v = at[q];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = fmaxf(v[e] + 0.0f, -INFINITY);        // (-0 as 0, NaN as -infinity)
        } else if (index(q) < vocab) {
            const f4v x = at[q];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if ((unsigned)(index(q) + e) < (unsigned)vocab) v[e] = fmaxf(x[e] + 0.0f, -INFINITY);
        }
        return v;
    }
    __device__ __forceinline__ f4v get(int w, int j) const {
        if constexpr (LOCAL) return at[place(w, j)];
        f4v v = fetch(w, j);
        if (top_inf) {
            asm("");                                         // (a branch, not six more instructions for every four)
            v = only_infinite(v);
        }
        return v;
    }
    // f(four logits, their place) for all of this thread's
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        for (int j0 = 0; j0 < turns; j0 += AHEAD) {
            f4v v[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; j++) v[j] = get(wave, min(j0 + j, turns - 1));
#pragma unroll
            for (int j = 0; j < AHEAD; j++)
                if (j0 + j < turns) f(v[j], place(wave, j0 + j));
        }
    }
};

// The logit at which the running sum of `measure` over the logits in [lo, hi],
// in their order, reaches need(their whole sum), which is more than 0 and at
// most that sum: its value, the sum before it and the sum of its equals.
// logits: how many lie in the bounds, or more.
struct Mark { float value; u64 before, equals, need; };

template <bool LOCAL, typename M, typename F>
__device__ __forceinline__ Mark find_mark(const Row<LOCAL> &row, SampleLds &s, float lo, float hi, int logits, const M &measure, F &&need_of) {
    const int t = threadIdx.x, lane = t & 63;
    Mark k = {hi, 0, 0, 0};
    bool first = true;
    for (int step = 0; step < 64; step++) {                  // (each takes 11 bits of the bounds' distance: under 40)
        // Bins of (hi - x)/2, which no pair of floats overflows.  lo < hi fall into different ones, so the bounds
        // close in; where even half their distance is nothing (subnormals next to each other), hi alone is a bin.
        const float half = 0.5f * hi, range = half - 0.5f * lo;
        const bool apart = range > 0.0f, normal = range >= 1e-20f;
        const float pre = normal ? 1.0f : 0x1p100f, inv = apart ? (float)kBins / (range * pre) : 0.0f;   // (finite)
        auto bin_of = [&](float x) {
            const int b = min((int)(fmaf(-0.5f, x, half) * pre * inv), kBins - 1);
            return apart || x == hi ? b : 1;
        };
        if (t < kList) s.above[t] = s.equal[t] = 0;
        if (t == 0) { s.members = 0; s.lo = 0xFFFFFFFFu; s.hi = 0; }
        int bin = -1;                                        // none: all in [lo, hi], which are few
        if (logits > kList) {
            s.bins[t] = s.bins[t + kThreads] = 0;
            __syncthreads();
            if (first && normal && logits > row.vocab / 32) {   // (as below, but hi is the largest and pre 1)
                row.each([&](const f4v &x, int) {
                    u64 w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = measure(x[e]);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (x[e] >= lo && w[e]) atomicAdd(&s.bins[min((int)(fmaf(-0.5f, x[e], half) * inv), kBins - 1)], w[e]);
                });
            } else {
                row.each([&](const f4v &x, int) {
                    if (!__any(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= lo)) return;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (!(x[e] >= lo && x[e] <= hi)) continue;
                        const u64 w = measure(x[e]);
                        if (w) atomicAdd(&s.bins[bin_of(x[e])], w);
                    }
                });
            }
            __syncthreads();
            const u64 b0 = s.bins[2 * t], b1 = s.bins[2 * t + 1], scanned = wave_scan(b0 + b1), sums = sum_waves(scanned, s, row.wave);
            const u64 c1 = scanned + (row.wave ? lane_value(sums, row.wave - 1) : 0), c0 = c1 - b1, cb = c0 - b0;
            if (first) k.need = need_of(lane_value(sums, 63));
            first = false;
            if (k.before + cb < k.need && k.need <= k.before + c0) { s.bin = 2 * t; s.before = k.before + cb; s.sum = b0; }
            if (k.before + c0 < k.need && k.need <= k.before + c1) { s.bin = 2 * t + 1; s.before = k.before + c0; s.sum = b1; }
            __syncthreads();
            bin = s.bin;
            k.before = s.before;
            k.equals = s.sum;
            k.value = hi;
            if (!(lo < hi)) return k;                            // all equal
        } else {
            __syncthreads();
        }
        // Bounds a little outside of the bin's (its border is off by a few roundings of bin/inv and of hi, and half of
        // a subnormal hi by one of its own) spare most logits the rest.  In halves, as the bins: finite, up to `from`,
        // which may be -infinity.
        float from = lo, to = hi;
        if (normal && bin >= 0) {
            const float width = range / kBins, off = 1e-6f * fabsf(half) + 1e-37f;
            if (bin < kBins - 1) from = fmaxf(lo, 2.0f * (half - (float)(bin + 1) * width * 1.00001f - off));
            to = fminf(hi, 2.0f * (half - (float)bin * width * 0.99999f + off));
        }
        float least = INFINITY, most = -INFINITY;
        row.each([&](const f4v &x, int) {
            bool in[4], some = false;
#pragma unroll
            for (int e = 0; e < 4; e++) some |= in[e] = x[e] >= from && x[e] <= to;
            if (!__any(some)) return;
            u64 mask[4];
            int n = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                in[e] &= x[e] >= lo && x[e] <= hi && (bin < 0 || bin_of(x[e]) == bin);
                mask[e] = __ballot(in[e]);
                n += __popcll(mask[e]);
                least = fminf(least, in[e] ? x[e] : INFINITY);
                most = fmaxf(most, in[e] ? x[e] : -INFINITY);
            }
            if (n == 0) return;
            int at = lane == 0 ? atomicAdd(&s.members, n) : 0;
            at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int mine = (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask[e] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask[e], at));
                if (in[e] && mine < kList) s.list_x[mine] = x[e];
                at += __popcll(mask[e]);
            }
        });
        __syncthreads();
        const int n = s.members;
        if (n <= kList) {
            // All pairs of them, each member's by as many threads as there are.
            const u64 own = t < n ? measure(s.list_x[t]) : 0;
            if (t < n) s.list_w[t] = own;
            const u64 sums = sum_waves(wave_scan(own), s, row.wave);
            if (first) k.need = need_of(lane_value(sums, 63));
            const int width = n <= 64 ? 64 : kList, i = t % width;
            if (i < n) {
                const float x = s.list_x[i];
                u64 above = 0, equal = 0;
                for (int j = t / width; j < n; j += kThreads / width) {
                    const float y = s.list_x[j];
                    const u64 w = s.list_w[j];
                    above += y > x ? w : 0;
                    equal += y == x ? w : 0;
                }
                if (above) atomicAdd(&s.above[i], above);
                if (equal) atomicAdd(&s.equal[i], equal);
            }
            __syncthreads();
            if (t < n) {
                const u64 above = k.before + s.above[t], equal = s.equal[t];
                if (above < k.need && k.need <= above + equal) { s.value = s.list_x[t]; s.before = above; s.sum = equal; }   // equals agree
            }
            __syncthreads();
            k.value = s.value;
            k.before = s.before;
            k.equals = s.sum;
            return k;
        }
        least = -group_max<64>(-least);
        most = group_max<64>(most);
        if (lane == 0 && least <= most) {
            atomicMin(&s.lo, ordered(least));
            atomicMax(&s.hi, ordered(most));
        }
        __syncthreads();
        lo = from_ordered(s.lo);
        hi = from_ordered(s.hi);
        __syncthreads();
    }
    return k;
}

// CAP: logits that the copy in shared memory holds; 0: no copy.  Where two
// rows fit a compute unit's shared memory the registers are held to it, some
// spilled: 509 rows of 50259 took 139 us so, 162 at one row a unit.
template <int CAP>
__global__ __launch_bounds__(kThreads, CAP == 0 || CAP == 8192 ? 8 : 4) void k_sample(SampleArgs a) {
    __shared__ SampleLds s;
    __shared__ f4v copy[CAP ? CAP / 4 : 1];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = blockIdx.x;
    const float *base = a.logits + (long)r * a.ld;
    Row<(CAP > 0)> row;
    row.skip = (int)((uintptr_t)base >> 2 & 3);
    row.at = reinterpret_cast<const f4v *>(base - row.skip);
    row.wave = wave;
    row.vocab = a.vocab;
    row.turns = (a.vocab + row.skip + 4 * kThreads - 1) / (4 * kThreads);
    row.top_inf = false;
    const float temp = a.temperature ? a.temperature[r] : 1.0f;
    const int top_k = a.top_k ? a.top_k[r] : 0;
    const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_pf = a.min_p ? a.min_p[r] : 0.0f;
    float u = a.u ? a.u[r] : 0.0f;
    // the largest logit
    float top = -INFINITY;
#pragma unroll 8
    for (int j = 0; j < row.turns; j++) {
        const f4v v = row.fetch(wave, j);
        if constexpr (CAP > 0) copy[row.place(wave, j)] = v; // (a wave reads another's only behind a barrier)
        top = fmaxf(fmaxf(top, fmaxf(v[0], v[1])), fmaxf(v[2], v[3]));
    }
    if constexpr (CAP > 0) row.at = copy;
    top = group_max<64>(top);
    if (lane == 0) s.list_x[wave] = top;
    if (t == 0) s.index = a.vocab;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; w++) top = fmaxf(top, s.list_x[w]);
    if (top == -INFINITY) {
        if (t == 0) a.token[r] = -1;
        return;
    }
    if (top == INFINITY) {                                   // uniform
        row.top_inf = true;
        top = 0.0f;
        if constexpr (CAP > 0)
            for (int j = 0; j < row.turns; j++) copy[row.place(wave, j)] = only_infinite(copy[row.place(wave, j)]);
    }
    if (!(temp > 0.0f) || top_k == 1) {                      // the first index of the maximum
        int i = a.vocab;
        row.each([&](const f4v &v, int q) {
#pragma unroll
            for (int e = 3; e >= 0; e--) i = v[e] == top ? min(i, row.index(q) + e) : i;
        });
        for (int d = 32; d; d >>= 1) i = min(i, __shfl_xor(i, d));
        if (lane == 0) atomicMin(&s.index, i);
        __syncthreads();
        if (t == 0) a.token[r] = s.index;
        return;
    }
    const double scale = 1.4426950408889634 / (double)temp;
    const WeightOf weight = {Exp2Poly(), top, scale, min_pf > 1.0f ? 1.0 : min_pf > 0.0f ? (double)min_pf : 0.0};
    // Logits under floor_ weigh nothing (2^-46 is 0, of 2^-44), whatever stays.
    const double reach = (double)top - 46.0 / scale;
    const float floor_ = reach > -(double)FLT_MAX ? (float)reach - fabsf((float)reach) * 1e-6f : -FLT_MAX;
    // stays: logits above `last`, and the first `ties` of its `equals`
    float last = floor_;
    u64 ties = (u64)a.vocab, equals = 0;
    int logits = a.vocab;            // from `last` on, or more
    if (top_k > 0 && top_k < a.vocab) {
        const Mark k = find_mark(row, s, floor_, top, a.vocab, CountOf(), [&](u64 weigh) { return min((u64)top_k, weigh); });
        last = k.value;
        equals = k.equals;
        ties = k.need - k.before;
        logits = (int)(k.before + k.equals);
    }
    if (!(top_p >= 1.0f)) {
        const u64 dropped = equals > ties ? (equals - ties) * weight(last) : 0;
        // stays: sums before it under top_p * total, so the last is where the sum reaches it
        const Mark k = find_mark(row, s, last, top, logits, weight, [&](u64 sum) {
            const double lim = top_p > 0.0f ? (double)top_p * (double)(sum - dropped) : 0.0;
            u64 need = (u64)lim;
            if ((double)need < lim) need++;
            return max(need, (u64)1);
        });
        // how many equals it has, and how many of them until the mark (of numbers under 2^18 a quotient is near enough)
        const u64 each = weight(k.value), rest = k.need - k.before;
        const double one = 1.0 / (double)each;
        u64 n = (u64)((double)rest * one);
        n += n * each < rest ? 1 : 0;                        // (rest/each a little under a whole number: one more than its floor)
        equals = (u64)((double)k.equals * one + 0.5);
        ties = k.value > last ? n : min(ties, n);
        last = k.value;
    }
    // more equals of the last than stay: the index of the last that does
    int cut = INT_MAX;
    if (equals > ties) {                                     // uniform
        auto equal = [&](const f4v &v) { return (v[0] == last) + (v[1] == last) + (v[2] == last) + (v[3] == last); };
        u64 seen = 0;
        row.each([&](const f4v &v, int) { seen += equal(v); });
        const u64 sums = sum_waves(wave_scan(seen), s, wave);
        seen = wave ? lane_value(sums, wave - 1) : 0;        // before this wave's run
        row.each([&](const f4v &v, int q) {
            const u64 mine = equal(v), upto = seen + wave_scan(mine), from = upto - mine;
            int k = (int)(ties - from), at = 0;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (v[e] == last && --k == 0) at = e;
            if (from < ties && ties <= upto) s.index = row.index(q) + at;
            seen = lane_value(upto, 63);
        });
        __syncthreads();
        cut = s.index;
    }
    // The draw, in the order of indices: sums of the waves' runs, then of the turns of the run that holds the mark, a
    // turn a wave.  Behind a filter few logits stay: they are picked out first, and their weights taken 64 at a time.
    const bool tied = cut != INT_MAX;                        // uniform, and hardly ever so
    const float above = tied ? last : last == 0.0f ? -0x1p-149f : from_ordered(ordered(last) - 1);   // (the next float below)
    auto stays = [&](float x, int i) { return x > above || (tied && x == last && i <= cut); };
    u64 w = 0;
    {
        // (a wave's accesses to shared memory are in order)
        int n = 0;                                           // in the wave's queue, under 64 between turns of the loop
        row.each([&](const f4v &v, int q) {
            if (!__any(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= last)) return;
            bool in[4];
            u64 mask[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                in[e] = stays(v[e], row.index(q) + e);
                mask[e] = __ballot(in[e]);
            }
            if (!~(mask[0] & mask[1] & mask[2] & mask[3])) { // none to pick out
#pragma unroll
                for (int e = 0; e < 4; e++) w += weight(v[e]);
                return;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask[e] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask[e], n));
                if (in[e]) s.queue[wave][at] = v[e];
                n += __popcll(mask[e]);
            }
            __builtin_amdgcn_wave_barrier();
            while (n >= 64) {                                // (under kQueue)
                n -= 64;
                w += weight(s.queue[wave][n + lane]);
            }
            __builtin_amdgcn_wave_barrier();
        });
        if (n > 0) {
            const u64 one = weight(s.queue[wave][min(lane, n - 1)]);
            w += lane < n ? one : 0;
        }
    }
    w = sum_waves(wave_scan(w), s, wave);
    const u64 total = lane_value(w, 63);
    u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    const u64 target = min((u64)((double)u * (double)total), total - 1);
    const int run = max(__ffsll((unsigned long long)__ballot(w > target)) - 1, 0);   // (under kWaves: from lane 15 on w is total)
    const u64 before = run > 0 ? lane_value(w, run - 1) : 0;
    f4v v;
    auto four = [&](int j) -> u64 {                          // this lane's weights of turn j of the run
        v = row.get(run, j);
        u64 w = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const u64 one = weight(v[e]);
            w += stays(v[e], row.index(row.place(run, j)) + e) ? one : 0;
        }
        return w;
    };
    for (int j = wave; j < row.turns; j += kWaves) {
        const u64 upto = wave_scan(four(j));
        if (lane == 63) s.turn_sum[j] = upto;
    }
    __syncthreads();
    const u64 mine = lane < row.turns ? s.turn_sum[lane] : 0, upto = before + wave_scan(mine), past = __ballot(upto > target);
    if (!past) return;                                       // (never: the run holds the mark)
    const int j = __ffsll((unsigned long long)past) - 1;
    if (wave != j % kWaves) return;
    w = four(j);
    u64 c = __shfl(upto - mine, j) + wave_scan(w) - w;
    if (c <= target && target < c + w) {
        bool done = false;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = row.index(row.place(run, j)) + e;
            if (stays(v[e], i)) c += weight(v[e]);
            if (!done && c > target) { a.token[r] = i; done = true; }
        }
    }
}

}  // namespace

}  // namespace ptmi

using namespace ptmi;

extern "C" int ptmi_sample_dev(const float *logits, long ld, int rows, int vocab, const float *temperature,
                               const int *top_k, const float *top_p, const float *min_p, const float *u, int *token,
                               void *stream) {
    if (rows < 0 || vocab < 1 || vocab > kSampleVocab || ld < vocab)
        return set_error(PTMI_ERR_ARG, "ptmi_sample: rows=%d vocab=%d (1..%d) ld=%ld", rows, vocab, kSampleVocab, ld);
    if (rows == 0) return PTMI_OK;
    if (!logits || !token) return set_error(PTMI_ERR_ARG, "ptmi_sample: NULL argument");
    if ((uintptr_t)logits & 3) return set_error(PTMI_ERR_ARG, "ptmi_sample: logits not 4-byte aligned");
    int st = ensure_init();
    if (st) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    const SampleArgs a = {logits, ld, vocab, temperature, top_k, top_p, min_p, u, token};
    const int n = vocab + (ld % 4 || (uintptr_t)logits & 15 ? 3 : 0);    // logits of the longest copy
    hipLaunchKernelGGL(n <= 8192 ? k_sample<8192> : n <= 16384 ? k_sample<16384> : n <= 32768 ? k_sample<32768> : k_sample<0>,
                       dim3(rows), dim3(kThreads), 0, stream ? (hipStream_t)stream : lib_stream(), a);
    PTMI_HIP(hipGetLastError());
    return PTMI_OK;
}
