// Attention of new rows over a paged cache.
//
// For one key head of one request, M = new tokens x query heads that share
// it are the rows of two products over the keys, joined by a softmax that
// runs along with them (running maximum m, sum l, weighted values o):
//   m' = max(m, s), l' = l 2^(m - m') + sum 2^(s - m'), o' = o 2^(m - m') + sum 2^(s - m') v
// with scores s = (scale log2(e) q).k, so that every e^x is one 2^x.
//
// Four kernels, by M and the type of the pages.  Up to 16 rows (single tokens, a few tokens) are bound
// by the bytes of the cache: k_attn_stream for up to 4, on the vector units,
// k_attn_few through the fp32 matrix instructions, k_attn_few_b16 through the
// bf16 ones.  More rows are bound by the products: k_attn_tile, on the 16-bit
// matrix cores.  Against the simple form
// (a wave a row, a key at a time): 64 requests of one token and 12 heads of 64,
// 617 -> 40 us; 2 of 70 to 131 thousand positions, 32 heads on 8 of 128 in
// bf16, 115600 -> 180; 16 chunks of 512 tokens, 12 heads of 64, 23100 -> 330.
//
// Lengths are known on the device alone, so the launch does not depend on
// them: the work of all requests is one axis of units of 64 keys (request by
// request, head by head, tile of rows by tile), and every workgroup takes an
// equal stretch of it.  A stretch that ends inside a head leaves its part
// (m, l, o) in the workspace, and k_attn_join adds such parts up in order.
#include "ptmi_paged.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <unordered_map>

namespace ptmi {

namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f2v __attribute__((ext_vector_type(2)));

constexpr int kUnit = 64;            // keys of a unit
constexpr int kFewRows = 16;         // rows of k_attn_few
constexpr int kTileRows = 128;       // least rows of a tile of k_attn_tile
constexpr int kThreads = 256;

// An item whose units several workgroups take: its first part is slot 1 of
// the workgroup it begins in, the others slot 0 of the next ones.
struct Cut {
    int parts;                       // 0: none
    int row0, n, kvh, tile;
    int pad[3];
};

struct AttnArgs {
    const void *k, *v;
    long page_stride, pos_stride, head_stride;
    int n_pages;
    FastDiv page;
    const int *table; int width;
    const int *row_start, *kv_len; int n_req;
    const float *q; long ldq;
    float *out; long ldo;
    int rows, kv_heads, hd;
    FastDiv group;                   // query heads of a key head
    int tile_tokens;                 // tokens of a tile: those whose rows it holds whole
    int few_rows;                    // most rows of a request of the kernel for few
    float qscale;                    // scale * log2(e)
    float minus_one;
    float *parts;                    // parts of items cut between workgroups
    Cut *cuts;                       // by workgroup: the cut item that begins in its stretch
};

// ── the axis of units ────────────────────────────────────────────────────
struct Request { int n, row0, len; };

__device__ __forceinline__ Request request(const AttnArgs &a, int s) {
    Request r;
    r.row0 = a.row_start[s];
    r.n = min(max(a.row_start[s + 1] - r.row0, 0), a.rows);
    r.len = (int)min((long)max(a.kv_len[s], 0), (long)a.width * a.page.d);
    return r;
}

__device__ __forceinline__ long quotient(long a, long b) { // 32 bits where they do
    return (a | b) < UINT_MAX ? (long)((unsigned)a / (unsigned)b) : a / b;
}

// Units of one key head of a request; 0: the other kernel's.  Tile i of rows
// has floor((b + i tt)/64) of them, tt its tokens: the keys its last whole
// token would see, at most a unit or two too many at the request's end, which
// find no key and cost nothing.  64 tiles on, a tile has tt units more.
__device__ __forceinline__ unsigned tile_keys0(const AttnArgs &a, const Request &r) {
    return (unsigned)max(r.len - r.n, 0) + a.tile_tokens + kUnit - 1;
}
// Units of the 64 k tiles before block k of 64, if block 0 has s.
__device__ __forceinline__ long blocks_before(long k, long s, int tt) { return k * s + 32 * tt * k * (k - 1); }

template <bool TILE>
__device__ __forceinline__ long head_units(const AttnArgs &a, const Request &r) {
    const bool few = (long)r.n * a.group.d <= a.few_rows;
    if (r.n == 0 || few == TILE) return 0;
    if constexpr (TILE) {
        const int tt = a.tile_tokens, tiles = (r.n + tt - 1) / tt, k = tiles >> 6, rest = tiles & 63;
        const unsigned b0 = tile_keys0(a, r);
        long s = 0, s_rest = 0;
        for (int i = 0; i < (k ? 64 : rest); i++) {
            s += (b0 + (unsigned)(i * tt)) / kUnit;
            if (i + 1 == rest) s_rest = s;
        }
        return blocks_before(k, s, tt) + s_rest + (long)rest * tt * k;
    } else {
        return max(1, (r.len + kUnit - 1) / kUnit);
    }
}

// The units of 256 requests at a time, as sums in shared memory, and the requests.
struct Axis {
    long pre[kThreads + 1];          // units before request c0 + i
    Request req[kThreads];
    long wsum[kThreads / 64];
    int c0;
};

// Inclusive sums over the wave by DPP: within rows of 16 lanes, then each
// row's (half's) last lane to the next row (half).
template <int CTRL, int ROWS>
__device__ __forceinline__ long dpp_add(long v) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + (long)((unsigned long)hi << 32 | lo);
}
__device__ __forceinline__ long wave_scan(long v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}

// Fills x for requests [c0, c0 + 256) after `before` units; all threads of
// the block take part, the first 256 hold a request each.
template <bool TILE>
__device__ void axis_fill(const AttnArgs &a, Axis &x, int c0, long before) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const bool mine = t < kThreads;
    long v = 0;
    Request r = {0, 0, 0};
    if (mine && c0 + t < a.n_req) {
        r = request(a, c0 + t);
        v = head_units<TILE>(a, r) * a.kv_heads;
    }
    const long incl = wave_scan(v);
    __syncthreads();
    if (mine) {
        x.req[t] = r;
        if (lane == 63) x.wsum[w] = incl;
    }
    __syncthreads();
    if (mine) {
        for (int i = 0; i < w; i++) before += x.wsum[i];
        x.pre[t + 1] = before + incl;
        if (t == 0) { x.pre[0] = before; x.c0 = c0; }
    }
    __syncthreads();
}

// Counts all units; x then holds the requests' first 256.
template <bool TILE>
__device__ long axis_init(const AttnArgs &a, Axis &x) {
    long total = 0;
    if (a.n_req > kThreads)
        for (int c0 = 0; c0 < a.n_req; c0 += kThreads) {
            axis_fill<TILE>(a, x, c0, total);
            total = x.pre[kThreads];
        }
    axis_fill<TILE>(a, x, 0, 0);
    return a.n_req > kThreads ? total : x.pre[kThreads];
}

// The request that holds unit u < total (refills x as needed).
template <bool TILE>
__device__ int axis_find(const AttnArgs &a, Axis &x, long u) {
    while (u >= x.pre[kThreads]) axis_fill<TILE>(a, x, x.c0 + kThreads, x.pre[kThreads]);
    int lo = 0, hi = kThreads;                              // pre[lo] <= u < pre[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (x.pre[mid] <= u) lo = mid;
        else hi = mid;
    }
    return x.c0 + lo;
}

// The stretches: workgroup g of n takes units [first(g), first(g + 1)).
struct Split {
    long each, more;                 // the first `more` take each + 1
    __device__ Split(long total, int n) : each(quotient(total, n)), more(total - each * n) {}
    __device__ long first(int g) const { return g * each + min((long)g, more); }
    __device__ int of(long u) const {                      // the workgroup that takes unit u
        const long longer = more * (each + 1);
        return (int)(u < longer ? quotient(u, each + 1) : more + quotient(u - longer, each));
    }
};

// Lane i's value, i the same in all lanes.
__device__ __forceinline__ long lane_value(long v, int i) {
    return (long)((unsigned long)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 |
                  (unsigned)__builtin_amdgcn_readlane((int)v, i));
}

// One item of the axis: a head's keys for one tile of rows, units [a, b).
struct Item {
    int s, kvh, tile;
    long a, b;
    Request r;
};
template <bool TILE>
__device__ Item axis_item(const AttnArgs &a, Axis &x, long u) {
    Item it;
    it.s = axis_find<TILE>(a, x, u);
    it.r = x.req[it.s - x.c0];
    const long per = head_units<TILE>(a, it.r), base = x.pre[it.s - x.c0];
    it.kvh = (int)quotient(u - base, per);
    it.a = base + it.kvh * per;
    it.b = it.a + per;
    it.tile = 0;
    if constexpr (TILE) {                                  // lane i: tile 64 k + i
        const int tt = a.tile_tokens, lane = threadIdx.x & 63;
        const long mine = (tile_keys0(a, it.r) + (unsigned)(lane * tt)) / kUnit, upto = wave_scan(mine);
        const long s = lane_value(upto, 63);
        long k = 0, w = u - it.a;
        while (blocks_before(k + 1, s, tt) <= w) k++;
        w -= blocks_before(k, s, tt);
        const long end = upto + (long)(lane + 1) * tt * k;
        const int i = __popcll(__ballot(end <= w));         // (under 64: w lies in block k)
        it.tile = (int)(64 * k) + i;
        it.b = it.a + blocks_before(k, s, tt) + lane_value(end, i);
        it.a = it.b - lane_value(mine, i) - tt * k;
    }
    return it;
}

// What a workgroup whose stretch ended in `it` tells k_attn_join.
__device__ __forceinline__ void note_cut(const AttnArgs &a, int wg, const Split &split, const Item &it, long u, long ue) {
    if (threadIdx.x) return;
    const int parts = u == it.a && ue < it.b ? split.of(it.b - 1) - wg + 1 : 0;
    a.cuts[wg] = Cut{parts, it.r.row0, it.r.n, it.kvh, it.tile, {0, 0, 0}};
}

// XCD x runs every eighth workgroup: give each XCD neighbouring stretches,
// so that the tiles of one head find its keys in that XCD's L2.
__device__ __forceinline__ int stretch_of_block() {
    const int n = gridDim.x, b = blockIdx.x;               // (n a multiple of 8)
    return (b & 7) * (n >> 3) + (b >> 3);
}

// ── loads ────────────────────────────────────────────────────────────────
template <bool BF16> struct Raw4 { float4 x; };
template <> struct Raw4<true> { uint2 x; };

template <bool BF16>
__device__ __forceinline__ Raw4<BF16> raw_load(const void *base, long at) {
    Raw4<BF16> r;
    if constexpr (BF16) r.x = *reinterpret_cast<const uint2 *>(static_cast<const unsigned short *>(base) + at);
    else r.x = *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
    return r;
}
template <bool BF16>
__device__ __forceinline__ Raw4<BF16> raw_zero() {
    Raw4<BF16> r;
    if constexpr (BF16) r.x = make_uint2(0, 0);
    else r.x = make_float4(0.f, 0.f, 0.f, 0.f);
    return r;
}
__device__ __forceinline__ f4v widen(const Raw4<false> &r) { return f4v{r.x.x, r.x.y, r.x.z, r.x.w}; }
__device__ __forceinline__ f4v widen(const Raw4<true> &r) {
    return f4v{__uint_as_float(r.x.x << 16), __uint_as_float(r.x.x & 0xFFFF0000u), __uint_as_float(r.x.y << 16),
               __uint_as_float(r.x.y & 0xFFFF0000u)};
}

// Element offset of a key's position from its page number; -1: not there.
__device__ __forceinline__ long key_offset(const AttnArgs &a, int key, int limit, int pg, int kvh) {
    if (key >= limit || (unsigned)pg >= (unsigned)a.n_pages) return -1;
    return pg * a.page_stride + (long)(key - a.page.quot(key) * a.page.d) * a.pos_stride + kvh * a.head_stride;
}
__device__ __forceinline__ int page_of(const AttnArgs &a, int s, int key, int limit) {
    return key < limit ? a.table[(long)s * a.width + a.page.quot(key)] : -1;
}

__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
// Values that are not finite as 0.
__device__ __forceinline__ void drop_odd(Raw4<false> &r) {
    r.x = make_float4(finite_bits(r.x.x) ? r.x.x : 0.f, finite_bits(r.x.y) ? r.x.y : 0.f,
                      finite_bits(r.x.z) ? r.x.z : 0.f, finite_bits(r.x.w) ? r.x.w : 0.f);
}
__device__ __forceinline__ void drop_odd(Raw4<true> &r) {
    const f4v x = widen(r);
    if (!finite_bits(x.x)) r.x.x &= 0xFFFF0000u;
    if (!finite_bits(x.y)) r.x.x &= 0x0000FFFFu;
    if (!finite_bits(x.z)) r.x.y &= 0xFFFF0000u;
    if (!finite_bits(x.w)) r.x.y &= 0x0000FFFFu;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// ── few rows ─────────────────────────────────────────────────────────────
// v_mfma_f32_16x16x4_f32: lane l supplies A[l%16][l/16] and B[l/16][l%16];
// result register r of lane l is C[4*(l/16) + r][l%16].  S^T = K.Q^T: a
// lane's four scores are keys 4g..4g+3 of row l%16, the operands of
// O^T += V^T.P^T as they stand.  The contraction over head_dim may take its
// index in any order that q and k share (lane group g takes float4s g, g+4,
// ...), and the rows of V^T too: lane li loads float4s li, li+16 of a value
// row, whose component e is row li of result tile e.  So K and V both come as
// 16-byte loads of whole rows.  16 rows is what one such tile holds, and what
// the bytes pay for: 64 requests of 8 new tokens, 12 heads of 64 behind up to
// 2048 positions: 90 us, 4.5 TB/s.
__device__ __forceinline__ f4v mfma4(float a, float b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Floats of a part: o [16][pitch], then (m, l) [16] (dt = head_dim / 32, rounded up).
constexpr int few_pitch(int dt) { return dt > 2 ? 128 : 64; }
constexpr int few_part(int dt) { return kFewRows * few_pitch(dt) + 2 * kFewRows; }

template <int HQ, bool BF16>
struct FewBlock {                    // 16 keys of one head
    Raw4<BF16> k[HQ], v[4][HQ > 4 ? 2 : 1];
    long off;                        // lane's key li; -1: not there
};

template <int HQ, bool PAD, bool BF16>
__device__ __forceinline__ void few_load(const AttnArgs &a, FewBlock<HQ, BF16> &b, int n4) {
    constexpr int C4 = HQ > 4 ? 2 : 1;
    const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < HQ; j++) {
        const int i = 4 * j + g;
        b.k[j] = raw_zero<BF16>();
        if (b.off >= 0 && (!PAD || i < n4)) b.k[j] = raw_load<BF16>(a.k, b.off + 4 * i);
    }
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const long off = __shfl(b.off, 4 * g + s);
#pragma unroll
        for (int c = 0; c < C4; c++) {
            const int i = li + 16 * c;
            b.v[s][c] = raw_zero<BF16>();
            if (off >= 0 && (!PAD || i < n4)) b.v[s][c] = raw_load<BF16>(a.v, off + 4 * i);
        }
    }
}

struct FewLds {
    static constexpr int NW = kThreads / 64;
    float m[NW][kFewRows], l[NW][kFewRows];
};

// Joins the four waves' (m, l, acc) of a key head's stretch [u, ue): to the output, or to the workgroup's part.
template <int HQ>
__device__ __forceinline__ void few_out(const AttnArgs &a, const Item &it, int wg, long u, long ue, const f4v (&acc)[HQ > 4 ? 8 : 4],
                                        float m, float l, int hd, float *red, FewLds &st) {
    constexpr int C4 = HQ > 4 ? 2 : 1, FP = few_pitch(HQ / 2), PITCH = FP + 4, NW = FewLds::NW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
    const int n4 = hd >> 2, G = a.group.d, M = it.r.n * G;
    // the four waves' sums, one maximum for all
    l = xsum32(xsum16(l));
    if (g == 0) { st.m[wave][li] = m; st.l[wave][li] = l; }
    __syncthreads();
    float gm = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; w++) gm = fmaxf(gm, st.m[w][li]);
    const float ref = gm == -INFINITY ? 0.0f : gm, f = exp2_hw(m - ref);
    if (li < M) {
#pragma unroll
        for (int c = 0; c < C4; c++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const f4v o = {acc[4 * c][r], acc[4 * c + 1][r], acc[4 * c + 2][r], acc[4 * c + 3][r]};
                *reinterpret_cast<f4v *>(red + (wave * kFewRows + li) * PITCH + 4 * (16 * c + 4 * g + r)) = o * f;
            }
    }
    __syncthreads();
    const bool whole = u == it.a && ue == it.b;
    float *part = a.parts + (long)(2 * wg + (u == it.a)) * few_part(HQ / 2);
    for (int e = threadIdx.x; e < M * n4; e += kThreads) {
        const int i = e / n4, c = e - i * n4;
        f4v o = *reinterpret_cast<const f4v *>(red + i * PITCH + 4 * c);
#pragma unroll
        for (int w = 1; w < NW; w++) o += *reinterpret_cast<const f4v *>(red + (w * kFewRows + i) * PITCH + 4 * c);
        float im = -INFINITY, il = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) im = fmaxf(im, st.m[w][i]);
        const float iref = im == -INFINITY ? 0.0f : im;
#pragma unroll
        for (int w = 0; w < NW; w++) il += st.l[w][i] * exp2_hw(st.m[w][i] - iref);
        if (whole) {
            const int t = a.group.quot(i), r = it.r.row0 + t;
            if ((unsigned)r < (unsigned)a.rows)
                *reinterpret_cast<f4v *>(a.out + r * a.ldo + (long)(it.kvh * G + i - t * G) * hd + 4 * c) =
                    o * (il == 0.0f ? 0.0f : 1.0f / il);
        } else {
            *reinterpret_cast<f4v *>(part + i * FP + 4 * c) = o;
            if (c == 0) {
                part[kFewRows * FP + 2 * i] = im;
                part[kFewRows * FP + 2 * i + 1] = il;
            }
        }
    }
}

template <int HQ, bool PAD>
__global__ __launch_bounds__(kThreads, 2) void k_attn_few(AttnArgs a) {
    constexpr int C4 = HQ > 4 ? 2 : 1, NC = 4 * C4, NW = kThreads / 64;
    __shared__ Axis axis;
    __shared__ __align__(16) float red[NW * kFewRows * (few_pitch(HQ / 2) + 4)];
    __shared__ FewLds st;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
    const int hd = PAD ? a.hd : 16 * HQ, n4 = hd >> 2, G = a.group.d;
    const Split split(axis_init<false>(a, axis), gridDim.x);
    const int wg = stretch_of_block();
    const long u1 = split.first(wg + 1);
    if (threadIdx.x == 0 && split.first(wg) == u1) a.cuts[wg].parts = 0;
    for (long u = split.first(wg); u < u1;) {
        const Item it = axis_item<false>(a, axis, u);
        const long ue = min(u1, it.b);
        const int M = it.r.n * G, len = it.r.len;
        // this lane's row: token li / G, query head li % G
        const int tok = a.group.quot(li), row = it.r.row0 + tok;
        const bool live = li < M && (unsigned)row < (unsigned)a.rows;
        const float *qrow = a.q + row * a.ldq + (long)(it.kvh * G + li - tok * G) * hd;
        f4v qf[HQ];
#pragma unroll
        for (int j = 0; j < HQ; j++) {
            const int i = 4 * j + g;
            qf[j] = f4v{0.f, 0.f, 0.f, 0.f};
            if (live && (!PAD || i < n4)) qf[j] = *reinterpret_cast<const f4v *>(qrow + 4 * i) * a.qscale;
        }
        const int see = len - it.r.n + tok + 1;             // keys [0, see)
        const int see0 = len - it.r.n + 1;                  // of the first row
        f4v acc[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) acc[c] = f4v{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.0f;
        // this wave's 16 keys of every unit; two blocks of keys and one more of page numbers in flight
        int kb = (int)(u - it.a) * 4 + wave;
        const int kend = (int)(ue - it.a) * 4;
        FewBlock<HQ, false> cur, nxt;
        cur.off = key_offset(a, kb * 16 + li, len, page_of(a, it.s, kb * 16 + li, len), it.kvh);
        int pg = page_of(a, it.s, (kb + NW) * 16 + li, len);
        few_load<HQ, PAD>(a, cur, n4);
        for (; kb < kend; kb += NW) {
            nxt.off = kb + NW < kend ? key_offset(a, (kb + NW) * 16 + li, len, pg, it.kvh) : -1;
            few_load<HQ, PAD>(a, nxt, n4);
            pg = page_of(a, it.s, (kb + 2 * NW) * 16 + li, len);
            f4v s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
            for (int j = 0; j < HQ; j++) {
                const f4v x = widen(cur.k[j]);
                s0 = mfma4(x.x, qf[j].x, s0);
                s1 = mfma4(x.y, qf[j].y, s1);
                s0 = mfma4(x.z, qf[j].z, s0);
                s1 = mfma4(x.w, qf[j].w, s1);
            }
            const f4v s = s0 + s1;
            const unsigned there = (unsigned)__ballot(cur.off >= 0) >> (4 * g);   // bit r: key 4g + r
            const int key = kb * 16 + 4 * g;
            bool use[4];
            float bm = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                use[r] = (there >> r & 1) && key + r < see;
                bm = use[r] ? fmaxf(bm, s[r]) : bm;
            }
            LanePair pr = pl16(bm);
            bm = fmaxf(pr.lo, pr.hi);
            pr = pl32(bm);
            const float mn = fmaxf(m, fmaxf(pr.lo, pr.hi)), ref = mn == -INFINITY ? 0.0f : mn;
            if (__any(mn > m)) {
                const float f = exp2_hw(m - ref);
                l *= f;
                m = mn;
#pragma unroll
                for (int c = 0; c < NC; c++) acc[c] *= f;
            }
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float e = exp2_hw(s[r] - ref);
                p[r] = use[r] ? e : 0.0f;
                l += p[r];
            }
            f4v v[4][C4];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int c = 0; c < C4; c++) v[t][c] = widen(cur.v[t][c]);
            if (max(kb * 16, see0) < min(kb * 16 + 16, len)) {
                // rows that do not see a key must not meet its value if that is not finite (0 * NaN):
                // it leaves the product, and the rows that see it get a NaN in its place
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int c = 0; c < C4; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const unsigned long bad = __ballot(!finite_bits(v[t][c][e]));
                            if (!bad) continue;
                            if (!finite_bits(v[t][c][e])) v[t][c][e] = 0.0f;
#pragma unroll
                            for (int h = 0; h < 4; h++)
#pragma unroll
                                for (int r = 0; r < 4; r++)
                                    if ((bad >> (16 * h + 4 * g + r) & 1) && kb * 16 + 4 * h + t < see)
                                        acc[4 * c + e][r] = NAN;
                        }
            }
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int c = 0; c < NC; c++) acc[c] = mfma4(v[t][c >> 2][c & 3], p[t], acc[c]);
            cur = nxt;
        }
        few_out<HQ>(a, it, wg, u, ue, acc, m, l, hd, red, st);
        if (ue == u1) note_cut(a, wg, split, it, u, ue);
        __syncthreads();
        u = ue;
    }
}

// bf16 pages: v_mfma_f32_16x16x32_bf16, whose operands are eight elements of a
// lane, takes keys and values as they are.  A query or weight is three of
// them, its leading 8 bits, the next 8 and the rest (cut off, not rounded:
// nothing overflows, and the three are all 24), so a product is as exact as in
// fp32.  Two blocks of 16 keys are one contraction: slot 4 x + s of lane group
// g is key 4g + s of block x, so P^T stands as S^T left it and lane li's
// values of eight keys are picked apart into V^T's rows.
// The fp32 instructions would bound bf16 pages: 64 requests of one token at
// 8192, 32 heads on 4 of 128, took 277 us, now 220 (1.07 GB, 4.9 TB/s); 20 on 4
// of 80, 248 -> 170; 8 new tokens of 12 heads of 64 at 4096, 213 -> 180.  (One
// request at 100: 12.7 -> 13.8, for the thirds.)  The queries' thirds in
// registers spill what is on its way: 352 us for the first.  Three workgroups a
// unit where heads are small: 123 us for the last with heads of 32, 175 with two.
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f4v mfma_b16(u4v a, u4v b, f4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}
// The upper (lower) halves of a and b side by side, a's first.
__device__ __forceinline__ unsigned upper_halves(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }
__device__ __forceinline__ unsigned lower_halves(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100); }

struct Thirds {                      // of eight floats
    u4v h, m, l;
    __device__ __forceinline__ void set(int i, float x, float y) {   // elements 2 i and 2 i + 1
        const unsigned xb = __float_as_uint(x), yb = __float_as_uint(y);
        h[i] = upper_halves(xb, yb);
        const float x1 = x - __uint_as_float(xb & 0xFFFF0000u), y1 = y - __uint_as_float(yb & 0xFFFF0000u);
        const unsigned x1b = __float_as_uint(x1), y1b = __float_as_uint(y1);
        m[i] = upper_halves(x1b, y1b);
        l[i] = upper_halves(__float_as_uint(x1 - __uint_as_float(x1b & 0xFFFF0000u)),
                            __float_as_uint(y1 - __uint_as_float(y1b & 0xFFFF0000u)));
    }
};

template <int HQ, bool PAD>
__global__ __launch_bounds__(kThreads, HQ <= 4 ? 3 : 2) void k_attn_few_b16(AttnArgs a) {
    constexpr int C4 = HQ > 4 ? 2 : 1, NC = 4 * C4, NW = kThreads / 64;
    __shared__ Axis axis;
    __shared__ __align__(16) float red[NW * kFewRows * (few_pitch(HQ / 2) + 4)];
    __shared__ FewLds st;
    __shared__ u4v qs[HQ / 2][3][64];                        // the queries' thirds (registers hold keys and values on their way)
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
    const int hd = PAD ? a.hd : 16 * HQ, n4 = hd >> 2, G = a.group.d;
    const Split split(axis_init<false>(a, axis), gridDim.x);
    const int wg = stretch_of_block();
    const long u1 = split.first(wg + 1);
    if (threadIdx.x == 0 && split.first(wg) == u1) a.cuts[wg].parts = 0;
    for (long u = split.first(wg); u < u1;) {
        const Item it = axis_item<false>(a, axis, u);
        const long ue = min(u1, it.b);
        const int M = it.r.n * G, len = it.r.len;
        const int tok = a.group.quot(li), row = it.r.row0 + tok;             // this lane's row
        const bool live = li < M && (unsigned)row < (unsigned)a.rows;
        const float *qrow = a.q + row * a.ldq + (long)(it.kvh * G + li - tok * G) * hd;
        // this wave's 16 keys of two units at a time; two pairs of blocks and one more of page numbers in flight
        int kb = (int)(u - it.a) * 4 + wave;
        const int kend = (int)(ue - it.a) * 4;
        auto key_of = [&](int b) { return b * 16 + li; };
        auto page_at = [&](int b) { return b < kend ? page_of(a, it.s, key_of(b), len) : -1; };
        FewBlock<HQ, true> cur[2], nxt[2];
        int pg[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            cur[x].off = key_offset(a, key_of(kb + x * NW), len, page_at(kb + x * NW), it.kvh);
            pg[x] = page_at(kb + (2 + x) * NW);
        }
#pragma unroll
        for (int x = 0; x < 2; x++) few_load<HQ, PAD>(a, cur[x], n4);
        f4v qx[HQ];
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < HQ; j++) {
            const int i = 4 * j + g;
            qx[j] = f4v{0.f, 0.f, 0.f, 0.f};
            if (live && (!PAD || i < n4)) qx[j] = *reinterpret_cast<const f4v *>(qrow + 4 * i) * a.qscale;
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(qx[j][e]));
        }
        LanePair pr = pl16(top);
        pr = pl32(fmaxf(pr.lo, pr.hi));
        // a third under 2^-126 would lose bits: rows that are all small count in 2^-64
        const bool small = fmaxf(pr.lo, pr.hi) < 0x1p-80f;
        const float up = small ? 0x1p64f : 1.0f, down = small ? 0x1p-64f : 1.0f;
        static_assert(HQ / 2 <= NW, "a wave's share of the row: elements of float4s 8 j + g and 8 j + 4 + g");
#pragma unroll
        for (int j = 0; j < HQ / 2; j++) {
            if (j != wave) continue;
            Thirds q;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const f4v x = qx[2 * j + s] * up;
                q.set(2 * s, x.x, x.y);
                q.set(2 * s + 1, x.z, x.w);
            }
            qs[j][0][lane] = q.h;
            qs[j][1][lane] = q.m;
            qs[j][2][lane] = q.l;
        }
        __syncthreads();
        const int see = len - it.r.n + tok + 1;             // keys [0, see)
        const int see0 = len - it.r.n + 1;                  // of the first row
        f4v acc[NC];
#pragma unroll
        for (int c = 0; c < NC; c++) acc[c] = f4v{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.0f;
        for (; kb < kend; kb += 2 * NW) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                nxt[x].off = key_offset(a, key_of(kb + (2 + x) * NW), len, pg[x], it.kvh);
                few_load<HQ, PAD>(a, nxt[x], n4);
            }
#pragma unroll
            for (int x = 0; x < 2; x++) pg[x] = page_at(kb + (4 + x) * NW);
            asm volatile("" ::: "memory");                   // (queries are read again, not kept)
            f4v s[2];
            bool use[2][4];
            float bm = -INFINITY;
            s[0] = s[1] = f4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < HQ / 2; j++) {
                const u4v qh = qs[j][0][lane], qm = qs[j][1][lane], ql = qs[j][2][lane];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const u4v k = {cur[x].k[2 * j].x.x, cur[x].k[2 * j].x.y, cur[x].k[2 * j + 1].x.x, cur[x].k[2 * j + 1].x.y};
                    s[x] = mfma_b16(k, ql, s[x]);
                    s[x] = mfma_b16(k, qm, s[x]);
                    s[x] = mfma_b16(k, qh, s[x]);
                }
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                s[x] *= down;
                const unsigned there = (unsigned)(__ballot(cur[x].off >= 0) >> (4 * g));   // bit r: key 4g + r
                const int key = (kb + x * NW) * 16 + 4 * g;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    use[x][r] = (there >> r & 1) && key + r < see;
                    bm = use[x][r] ? fmaxf(bm, s[x][r]) : bm;
                }
            }
            pr = pl16(bm);
            bm = fmaxf(pr.lo, pr.hi);
            pr = pl32(bm);
            const float mn = fmaxf(m, fmaxf(pr.lo, pr.hi)), ref = mn == -INFINITY ? 0.0f : mn;
            if (__any(mn > m)) {
                const float f = exp2_hw(m - ref);
                l *= f;
                m = mn;
#pragma unroll
                for (int c = 0; c < NC; c++) acc[c] *= f;
            }
            Thirds p;
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float e0 = exp2_hw(s[x][r] - ref), e1 = exp2_hw(s[x][r + 1] - ref);
                    const float p0 = use[x][r] ? e0 : 0.0f, p1 = use[x][r + 1] ? e1 : 0.0f;
                    l += p0;
                    l += p1;
                    p.set(2 * x + r / 2, p0, p1);
                }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int k0 = (kb + x * NW) * 16;
                if (max(k0, see0) >= min(k0 + 16, len)) continue;
                // rows that do not see a key must not meet its value if that is not finite (0 * NaN):
                // it leaves the product, and the rows that see it get a NaN in its place
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int c = 0; c < C4; c++) {
                        const f4v v = widen(cur[x].v[t][c]);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const unsigned long bad = __ballot(!finite_bits(v[e]));
                            if (!bad) continue;
#pragma unroll
                            for (int h = 0; h < 4; h++)
#pragma unroll
                                for (int r = 0; r < 4; r++)
                                    if ((bad >> (16 * h + 4 * g + r) & 1) && k0 + 4 * h + t < see) acc[4 * c + e][r] = NAN;
                        }
                        drop_odd(cur[x].v[t][c]);
                    }
            }
#pragma unroll
            for (int c = 0; c < C4; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    u4v v;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint2 y = cur[i >> 1].v[2 * (i & 1)][c].x, z = cur[i >> 1].v[2 * (i & 1) + 1][c].x;
                        v[i] = e & 1 ? upper_halves(e & 2 ? y.y : y.x, e & 2 ? z.y : z.x)
                                     : lower_halves(e & 2 ? y.y : y.x, e & 2 ? z.y : z.x);
                    }
                    f4v &o = acc[4 * c + e];
                    o = mfma_b16(v, p.l, o);
                    o = mfma_b16(v, p.m, o);
                    o = mfma_b16(v, p.h, o);
                }
#pragma unroll
            for (int x = 0; x < 2; x++) cur[x] = nxt[x];
        }
        few_out<HQ>(a, it, wg, u, ue, acc, m, l, hd, red, st);
        if (ue == u1) note_cut(a, wg, split, it, u, ue);
        __syncthreads();
        u = ue;
    }
}

// ── one to four rows ─────────────────────────────────────────────────────
// So few rows leave the matrix units' 16 idle; here the vector units do both
// products.  Lane (g, li) of a wave takes keys 4g..4g+3 of 16 and float4s of
// their rows: 16 lanes read a whole row of K or V side by side.  Scores are
// summed over the 16 lanes; each lane group keeps a maximum and sums of its
// own, and all 16 of the block's meet at the end.  Bound by the bytes of the
// cache: 64 requests of 12 heads of 64, 180 MB of fp32 in 35.5 us, 5.1 TB/s (55
// us through the matrix instructions); 954 MB of bf16, 4 heads of 128 on each
// key head: 172 us, 5.5 TB/s.
constexpr float kLazyFew = 8.0f;     // a maximum up to 2^8 above m does not move m

// FAST: four keys from a multiple of 4 on share a page, and bf16 rows may be
// read 16 bytes at a time (page sizes of 4; head_dim and strides of 8).
template <int C4, bool FAST, bool BF16>
struct StreamBlock {                 // a lane's keys of 16
    Raw4<BF16> k[4][C4], v[4][C4];
    unsigned there;                  // bit s: key 4g + s is
};

// The float4 c of lane li's share of a row.
template <int C4, bool BF16>
__device__ __forceinline__ int stream_chunk(int li, int c) { return BF16 && C4 == 2 ? 2 * li + c : li + 16 * c; }

template <int C4, bool FAST, bool BF16>
__device__ __forceinline__ void stream_row(Raw4<BF16> (&r)[C4], const void *base, long at, int li, int n4) {
    if constexpr (BF16 && C4 == 2 && FAST) {
        const int i = min(2 * li, n4 - 2);
        const uint4 x = *reinterpret_cast<const uint4 *>(static_cast<const unsigned short *>(base) + at + 4 * i);
        r[0].x = make_uint2(x.x, x.y);
        r[1].x = make_uint2(x.z, x.w);
    } else {
#pragma unroll
        for (int c = 0; c < C4; c++) r[c] = raw_load<BF16>(base, at + 4 * min(stream_chunk<C4, BF16>(li, c), n4 - 1));
    }
}

// Page numbers of the lane's keys (FAST: of the first).
template <bool FAST>
struct StreamPages { int pg[FAST ? 1 : 4]; };
template <bool FAST>
__device__ __forceinline__ StreamPages<FAST> stream_pages(const AttnArgs &a, int s, int key, int len) {
    StreamPages<FAST> p;
#pragma unroll
    for (int i = 0; i < (FAST ? 1 : 4); i++) p.pg[i] = page_of(a, s, key + i, len);
    return p;
}

template <int C4, bool FAST, bool BF16>
__device__ __forceinline__ void stream_load(const AttnArgs &a, StreamBlock<C4, FAST, BF16> &b, int key, int len,
                                            const StreamPages<FAST> &p, int kvh, int li, int n4) {
    // keys that are not there read the cache's first row
    const long first = key_offset(a, key, len, p.pg[0], kvh);
    b.there = 0;
#pragma unroll
    for (int s = 0; s < 4; s++) {
        long off;
        if constexpr (FAST) off = first >= 0 && key + s < len ? first + s * a.pos_stride : -1;
        else off = s == 0 ? first : key_offset(a, key + s, len, p.pg[FAST ? 0 : s], kvh);
        if (off >= 0) b.there |= 1u << s;
        off = max(off, 0l);
        stream_row<C4, FAST, BF16>(b.k[s], a.k, off, li, n4);
        stream_row<C4, FAST, BF16>(b.v[s], a.v, off, li, n4);
    }
}

__device__ __forceinline__ float dot4(const f4v &x, const f4v &y, float s) {
    return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, s))));
}

template <int MR, int C4, bool FAST, bool BF16>
__global__ __launch_bounds__(kThreads) void k_attn_stream(AttnArgs a) {
    constexpr int NW = kThreads / 64, NP = 4 * NW, FP = few_pitch(2 * C4);
    __shared__ Axis axis;
    __shared__ __align__(16) float red[NP][MR][64 * C4];
    __shared__ float st_m[NP][MR], st_l[NP][MR];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, g = lane >> 4;
    const int hd = a.hd, n4 = hd >> 2, G = a.group.d;
    const Split split(axis_init<false>(a, axis), gridDim.x);
    const int wg = stretch_of_block();
    const long u1 = split.first(wg + 1);
    if (threadIdx.x == 0 && split.first(wg) == u1) a.cuts[wg].parts = 0;
    for (long u = split.first(wg); u < u1;) {
        const Item it = axis_item<false>(a, axis, u);
        const long ue = min(u1, it.b);
        const int M = it.r.n * G, len = it.r.len;
        int kb = (int)(u - it.a) * 4 + wave;
        const int kend = (int)(ue - it.a) * 4;
        StreamPages<FAST> pg = stream_pages<FAST>(a, it.s, kb * 16 + 4 * g, len);
        f4v q[MR][C4];
        int see[MR];
#pragma unroll
        for (int i = 0; i < MR; i++) {
            const int tok = a.group.quot(i), row = it.r.row0 + tok;
            see[i] = len - it.r.n + tok + 1;
#pragma unroll
            for (int c = 0; c < C4; c++) {
                const int at = stream_chunk<C4, BF16>(li, c);
                q[i][c] = f4v{0.f, 0.f, 0.f, 0.f};
                if (i < M && (unsigned)row < (unsigned)a.rows && at < n4)
                    q[i][c] = *reinterpret_cast<const f4v *>(a.q + row * a.ldq + (long)(it.kvh * G + i - tok * G) * hd + 4 * at) *
                              a.qscale;
            }
        }
        f4v acc[MR][C4];
        float m[MR], l[MR];
#pragma unroll
        for (int i = 0; i < MR; i++) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < C4; c++) acc[i][c] = f4v{0.f, 0.f, 0.f, 0.f};
        }
        StreamBlock<C4, FAST, BF16> cur, nxt;
        stream_load(a, cur, kb * 16 + 4 * g, len, pg, it.kvh, li, n4);
        pg = stream_pages<FAST>(a, it.s, (kb + NW) * 16 + 4 * g, len);
        for (; kb < kend; kb += NW) {
            stream_load(a, nxt, (kb + NW) * 16 + 4 * g, kb + NW < kend ? len : 0, pg, it.kvh, li, n4);
            pg = stream_pages<FAST>(a, it.s, (kb + 2 * NW) * 16 + 4 * g, len);
            float s[MR][4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                f4v x[C4];
#pragma unroll
                for (int c = 0; c < C4; c++) x[c] = widen(cur.k[t][c]);
#pragma unroll
                for (int i = 0; i < MR; i++) {
                    float d = dot4(x[0], q[i][0], 0.0f);
                    if constexpr (C4 == 2) d = dot4(x[1], q[i][1], d);
                    s[i][t] = group_sum<16>(d);
                }
            }
            const int key = kb * 16 + 4 * g;
            // every row sees all 16 keys
            const bool full = __all(cur.there == 15u) && kb * 16 + 16 <= see[0];
            if (!full) {
#pragma unroll
                for (int i = 0; i < MR; i++)
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        if (!(cur.there >> t & 1) || key + t >= see[i]) s[i][t] = -INFINITY;
            }
            bool move = false;
#pragma unroll
            for (int i = 0; i < MR; i++) move |= fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])) > m[i] + kLazyFew;
            if (__any(move)) {
#pragma unroll
                for (int i = 0; i < MR; i++) {
                    const float mn = fmaxf(m[i], fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
                    const float f = exp2_hw(m[i] - (mn == -INFINITY ? 0.0f : mn));
                    m[i] = mn;
                    l[i] *= f;
#pragma unroll
                    for (int c = 0; c < C4; c++) acc[i][c] *= f;
                }
            }
#pragma unroll
            for (int i = 0; i < MR; i++) {
                const float ref = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
                for (int t = 0; t < 4; t++) s[i][t] = exp2_hw(s[i][t] - ref);
                l[i] += (s[i][0] + s[i][1]) + (s[i][2] + s[i][3]);
            }
            if (full) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int c = 0; c < C4; c++) {
                        const f4v v = widen(cur.v[t][c]);
#pragma unroll
                        for (int i = 0; i < MR; i++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[i][c][e] = fmaf(s[i][t], v[e], acc[i][c][e]);
                    }
            } else {                                         // an unseen value may be a NaN: it is not multiplied
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int c = 0; c < C4; c++) {
                        const f4v v = widen(cur.v[t][c]);
#pragma unroll
                        for (int i = 0; i < MR; i++)
                            if ((cur.there >> t & 1) && key + t < see[i])
#pragma unroll
                                for (int e = 0; e < 4; e++) acc[i][c][e] = fmaf(s[i][t], v[e], acc[i][c][e]);
                    }
            }
            cur = nxt;
        }
        const int part_i = 4 * wave + g;
        if (li < MR) {
            st_m[part_i][li] = MR == 1 ? m[0] : li == 0 ? m[0] : li == 1 ? m[1 % MR] : li == 2 ? m[2 % MR] : m[3 % MR];
            st_l[part_i][li] = MR == 1 ? l[0] : li == 0 ? l[0] : li == 1 ? l[1 % MR] : li == 2 ? l[2 % MR] : l[3 % MR];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MR; i++) {
            float gm = -INFINITY;
#pragma unroll
            for (int p = 0; p < NP; p++) gm = fmaxf(gm, st_m[p][i]);
            const float f = exp2_hw(m[i] - (gm == -INFINITY ? 0.0f : gm));
#pragma unroll
            for (int c = 0; c < C4; c++)
                *reinterpret_cast<f4v *>(&red[part_i][i][4 * stream_chunk<C4, BF16>(li, c)]) = acc[i][c] * f;
        }
        __syncthreads();
        const bool whole = u == it.a && ue == it.b;
        float *part = a.parts + (long)(2 * wg + (u == it.a)) * few_part(2 * C4);
        for (int e = threadIdx.x; e < min(M, MR) * n4; e += kThreads) {
            const int i = e / n4, c = e - i * n4;
            float im = -INFINITY, il = 0.0f;
#pragma unroll
            for (int p = 0; p < NP; p++) im = fmaxf(im, st_m[p][i]);
            const float iref = im == -INFINITY ? 0.0f : im;
            f4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int p = 0; p < NP; p++) {
                o += *reinterpret_cast<const f4v *>(&red[p][i][4 * c]);
                il += st_l[p][i] * exp2_hw(st_m[p][i] - iref);
            }
            if (whole) {
                const int t = a.group.quot(i), r = it.r.row0 + t;
                if ((unsigned)r < (unsigned)a.rows)
                    *reinterpret_cast<f4v *>(a.out + r * a.ldo + (long)(it.kvh * G + i - t * G) * hd + 4 * c) =
                        o * (il == 0.0f ? 0.0f : 1.0f / il);
            } else {
                *reinterpret_cast<f4v *>(part + i * FP + 4 * c) = o;
                if (c == 0) *reinterpret_cast<f2v *>(part + kFewRows * FP + 2 * i) = f2v{im, il};
            }
        }
        if (ue == u1) note_cut(a, wg, split, it, u, ue);
        __syncthreads();
        u = ue;
    }
}

// ── many rows ────────────────────────────────────────────────────────────
// fp32 products on the 16-bit matrix cores: x = 2^e (h + l) with h the
// nearest fp16 of x 2^-e and l that of the rest, 22 bits of x; of the four
// products of two such numbers l.l, under 2^-22 of the whole, is left out.
// e is the tile's (a row of q's) largest exponent less kTop, so h and l keep
// all their bits down to 2^-16 of the largest value, and below that an error
// of 2^-39 of it.  Three v_mfma_f32_32x32x16_f16 per product run at a third of
// 1180 TFLOP/s (what a large fp16 product reaches here), the fp32 matrix
// instructions at 154.  bf16 keys and values are h alone: two products.
// 16 chunks of 512 behind up to 3584 positions, 12 heads of 64: 300 us, 210
// TFLOP/s of the 390 that three products allow (bf16, 8 chunks behind 2048, 32
// heads on 8 of 128: 370 of 590).  What bounds it is the issue of both kinds of
// instruction: 48 matrix and some 480 vector ones (split, softmax, addresses)
// per 64 keys of a wave's 32 rows hardly overlap, and under both the clock
// falls to 1.55 GHz.  Measured and left: 8 waves a workgroup for heads up to 64
// (370 us to 350 then), three waves a SIMD (453, spills), wave priorities and
// scheduling groups (no difference).
//
// Wave w holds rows 32w.. of the tile as columns: S^T = K.Q^T leaves a lane
// with 32 of the unit's scores of its row l%32 and its partner l^32 with the
// others; its result registers, split, are the operand of O^T += V^T.P^T, if
// V^T's columns (keys) stand in the same order: registers 4b..4b+3 of half h
// are keys 8b + 4h.. of a 32-key block.
constexpr int kTop = 14;             // largest |h| < 2^15
constexpr int kBias = 9;             // weights are held times 2^9:
constexpr float kLazy = 6.0f;        // a maximum up to 2^6 above m does not move m (2^15 < 65504)


__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(min(max(e, -126), 127) + 127) << 23); }

__device__ __forceinline__ f16v mfma16(h8v a, h8v b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ h2v cvt2(float x, float y) {
    const f2v v = {x, y};
    return __builtin_convertvector(v, h2v);
}
// (x, y) s as h + l.  minus_one: -1, of a value the compiler does not know, so
// that each l is one fused operation on both precisions (a subtraction would
// be two and a packing).
__device__ __forceinline__ void split2(float x, float y, float minus_one, h2v &h, h2v &l) {
    h = cvt2(x, y);
    l = h2v{(_Float16)fmaf((float)h.x, minus_one, x), (_Float16)fmaf((float)h.y, minus_one, y)};
}
__device__ __forceinline__ void split4(const f4v &x, float minus_one, h4v &h, h4v &l) {
    h2v h0, h1, l0, l1;
    split2(x.x, x.y, minus_one, h0, l0);
    split2(x.z, x.w, minus_one, h1, l1);
    h = h4v{h0.x, h0.y, h1.x, h1.y};
    l = h4v{l0.x, l0.y, l1.x, l1.y};
}
// The largest magnitude seen, of any bits: the largest bits as unsigned (of
// the negative ones, if any) and as signed (of the positive ones, if any).
struct TopBits {
    unsigned u = 0;
    int i = 0;
    __device__ __forceinline__ void add(const f4v &x) {
        u = max(max(u, __float_as_uint(x.x)), max(max(__float_as_uint(x.y), __float_as_uint(x.z)), __float_as_uint(x.w)));
        i = max(max(i, __float_as_int(x.x)), max(max(__float_as_int(x.y), __float_as_int(x.z)), __float_as_int(x.w)));
    }
    __device__ __forceinline__ unsigned bits() const { return max(u & 0x7FFFFFFFu, (unsigned)i & 0x7FFFFFFFu); }
};
// The upper halves of two magnitudes' bits, and the wave's largest of each
// (enough for the exponent, and to tell infinities and NaN).
typedef unsigned short u2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u2v top_halves(unsigned k, unsigned v) {
    return __builtin_bit_cast(u2v, (k >> 16) | (v & 0xFFFF0000u));
}
template <int CTRL>
__device__ __forceinline__ u2v dpp_max(u2v x) {
    const unsigned o = __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true);
    return __builtin_elementwise_max(x, __builtin_bit_cast(u2v, o));
}
__device__ __forceinline__ u2v wave_top(u2v x) {
    x = dpp_max<0xB1>(x);
    x = dpp_max<0x4E>(x);
    x = dpp_max<0x141>(x);
    x = dpp_max<0x140>(x);
    int hi, lo = pl16i(__builtin_bit_cast(int, x), hi);
    x = __builtin_elementwise_max(__builtin_bit_cast(u2v, lo), __builtin_bit_cast(u2v, hi));
    lo = pl32i(__builtin_bit_cast(int, x), hi);
    return __builtin_elementwise_max(__builtin_bit_cast(u2v, lo), __builtin_bit_cast(u2v, hi));
}
constexpr unsigned kNotFinite = 0x7F80;                     // upper half of an infinity's bits
__device__ __forceinline__ unsigned finite_top(unsigned top, const f4v &x) {
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (finite_bits(x[e])) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
    return top;
}

// Waves of a tile of heads up to 32 dt: small ones leave room for two workgroups of four (12 heads of 64: 350 us, 370
// with one of eight); for large ones keys are split for twice the rows (32 heads on 8 of 128, bf16: 417 us, 617 with four).
constexpr int tile_waves(int dt) { return dt <= 2 ? 4 : 8; }
constexpr int tile_part(int dt) { return 32 * tile_waves(dt) * (32 * dt + 2); }   // floats

template <int DT, bool BF16>
struct TileLds {
    static constexpr int HP = 32 * DT, KP = HP + 8, VP = kUnit + 8;      // pitches in halves
    static constexpr int PL = BF16 ? 1 : 2;                              // planes: h, l
    _Float16 k[2][PL][kUnit * KP], v[2][PL][HP * VP];                    // units b and b + 1
    long off[4][kUnit];              // units b..b+3: offsets of their keys, -1: not there
    int all[4];                      // whether all 64 are
    unsigned top[2][tile_waves(DT)]; // each wave's top_halves of the unit in flight
    int odd[4];                      // whether one of their values is not finite
};

// Where in its 64 keys a value row keeps quad `place`: rows 16 apart, whose
// writes would meet in one bank, use different 16-key groups.
__device__ __forceinline__ int vplace(int row, int place) { return place ^ ((row >> 4 & 3) << 2); }

// NW waves of 32 rows; PAD: head_dim is not 32 DT (slots past it are zero).
// While unit b's products run, unit b + 1 is split into shared memory (its
// other half) and unit b + 2 is on its way to registers: one barrier a unit.
template <int DT, bool PAD, bool BF16>
__global__ __launch_bounds__(64 * tile_waves(DT), 2) void k_attn_tile(AttnArgs a) {
    typedef TileLds<DT, BF16> Lds;
    constexpr int HP = Lds::HP, KP = Lds::KP, VP = Lds::VP, PL = Lds::PL, KS = HP / 16, NW = tile_waves(DT), NT = 64 * NW;
    constexpr int C = 8 * DT;                                            // float4s of a row
    constexpr int KL = NT / kUnit, KT = (C + KL - 1) / KL;               // threads of a key row, float4s of each
    constexpr int VT = (16 * C + NT - 1) / NT;                           // value tasks of a thread: 4 keys x 4 columns
    static_assert(C % KL == 0, "every key thread has the same float4s");
    __shared__ Axis axis;
    __shared__ __align__(16) Lds lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const int hd = PAD ? a.hd : HP, n4 = hd >> 2, G = a.group.d;
    const float m1 = a.minus_one;
    const Split split(axis_init<true>(a, axis), gridDim.x);
    const int wg = stretch_of_block();
    const long u1 = split.first(wg + 1);
    if (threadIdx.x == 0 && split.first(wg) == u1) a.cuts[wg].parts = 0;
    for (long u = split.first(wg); u < u1;) {
        const Item it = axis_item<true>(a, axis, u);
        const long ue = min(u1, it.b);
        const int tt = a.tile_tokens, t0 = it.tile * tt;
        const int end = min(max(it.r.len - it.r.n + min(it.r.n, t0 + tt), 0), it.r.len);   // keys the tile sees
        // this lane's row of the tile
        const int mrow = wave * 32 + col, tok = t0 + a.group.quot(mrow), row = it.r.row0 + tok;
        const bool live = mrow < tt * G && tok < it.r.n && (unsigned)row < (unsigned)a.rows;
        const bool busy = __any(live);                       // this wave has rows
        const long head = it.kvh * G + mrow - (tok - t0) * G;
        const int see = it.r.len - it.r.n + tok + 1;        // its keys: [0, see)
        const int see0 = it.r.len - it.r.n + t0 + 1;        // of the tile's first row
        const int b0 = (int)(u - it.a), b1 = (int)min((long)(end + kUnit - 1) / kUnit, ue - it.a);   // units of keys
        // Offsets of unit b's keys go to slot b & 3 a barrier ahead of their use.  Wave b % NW does unit b, with
        // page numbers that it asked for NW units before.
        auto put_off = [&](int b, int pg) {
            const long off = b < b1 ? key_offset(a, b * kUnit + lane, end, pg, it.kvh) : -1;
            lds.off[b & 3][lane] = off;
            const bool all = __all(off >= 0);
            if (lane == 0) lds.all[b & 3] = all;
        };
        auto page_at = [&](int b) { return b < b1 ? page_of(a, it.s, b * kUnit + lane, end) : -1; };
        const int turn = (wave - b0) & (NW - 1);             // this wave's first unit, from b0
        int pg = page_at(b0 + turn);
        // q: columns 16 ks + 8 half .. of the row (on its way while the page numbers are)
        f4v qx[KS][2];
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int d = 16 * ks + 8 * half + 4 * j;
                qx[ks][j] = f4v{0.f, 0.f, 0.f, 0.f};
                if (live && (!PAD || d < hd)) qx[ks][j] = *reinterpret_cast<const f4v *>(a.q + row * a.ldq + head * hd + d);
            }
        __syncthreads();                                     // the last item's readers are done
        if (turn < 3) {
            put_off(b0 + turn, pg);
            pg = page_at(b0 + turn + NW);
        }
        if (tid < 4) lds.odd[tid] = 0;
        __syncthreads();
        // a unit's keys and values as they come: K thread (key, i): float4s i, i + KL, ..; V task (quad, c):
        // keys 4 quad.., float4 c
        typedef Raw4<BF16> RawK[KT], RawV[VT][4];
        RawK rk;
        RawV rv;
        const int kkey = tid / KL, ki = tid % KL;
        auto load = [&](int b, RawK &rk, RawV &rv) {
            const long *off = lds.off[b & 3];
            const bool all = lds.all[b & 3];
            const long ko = off[kkey];
#pragma unroll
            for (int j = 0; j < KT; j++) {
                const int i = ki + KL * j;
                const bool in = !PAD || i < n4;
                rk[j] = raw_load<BF16>(a.k, max(ko, 0l) + 4 * (in ? i : 0));
                if (PAD && !in) rk[j] = raw_zero<BF16>();
            }
#pragma unroll
            for (int t = 0; t < VT; t++) {
                const int task = tid + t * NT, quad = min(task / C, 15), c = task % C;
                const bool in = !PAD || c < n4;
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    rv[t][s] = raw_load<BF16>(a.v, max(off[4 * quad + s], 0l) + 4 * (in ? c : 0));
                    if (PAD && !in) rv[t][s] = raw_zero<BF16>();
                }
            }
            if (!all) {
                if (ko < 0)
#pragma unroll
                    for (int j = 0; j < KT; j++) rk[j] = raw_zero<BF16>();
#pragma unroll
                for (int t = 0; t < VT; t++)
#pragma unroll
                    for (int s = 0; s < 4; s++)
                        if (off[4 * min((tid + t * NT) / C, 15) + s] < 0) rv[t][s] = raw_zero<BF16>();
            }
        };
        // its largest exponents, for all waves; values that are not finite leave it (the rows that see them get NaN)
        auto tops = [&](int b, RawK &rk, RawV &rv) {
            TopBits kb, vb;
#pragma unroll
            for (int j = 0; j < KT; j++) kb.add(widen(rk[j]));
#pragma unroll
            for (int t = 0; t < VT; t++)
#pragma unroll
                for (int s = 0; s < 4; s++) vb.add(widen(rv[t][s]));
            u2v top = wave_top(top_halves(kb.bits(), vb.bits()));
            if (top.x >= kNotFinite || top.y >= kNotFinite) {
                if (top.y >= kNotFinite) {
                    if (lane == 0) lds.odd[b & 3] = 1;
#pragma unroll
                    for (int t = 0; t < VT; t++)
#pragma unroll
                        for (int s = 0; s < 4; s++) drop_odd(rv[t][s]);
                }
                unsigned km = 0, vm = 0;
#pragma unroll
                for (int j = 0; j < KT; j++) km = finite_top(km, widen(rk[j]));
#pragma unroll
                for (int t = 0; t < VT; t++)
#pragma unroll
                    for (int s = 0; s < 4; s++) vm = finite_top(vm, widen(rv[t][s]));
                top = wave_top(top_halves(km, vm));
            }
            if (lane == 0) lds.top[b & 1][wave] = __builtin_bit_cast(unsigned, top);
        };
        // exponents of the unit in LDS (k_e, v_e) and of the next; v_e only grows
        int k_e = 0, v_e = -1000, k_n = 0, v_n = -1000;
        auto next_exponents = [&](int b) {
            u2v top = {0, 0};
#pragma unroll
            for (int w = 0; w < NW; w++) top = __builtin_elementwise_max(top, __builtin_bit_cast(u2v, lds.top[b & 1][w]));
            k_n = max((int)(top.x >> 7) - 127, -100) - kTop;
            v_n = max(v_e, max((int)(top.y >> 7) - 127, -100) - kTop);
        };
        auto split_unit = [&](int b, RawK &rk, RawV &rv) {
            const float ks_ = pow2(-k_n), vs_ = pow2(-v_n);
#pragma unroll
            for (int j = 0; j < KT; j++) {
                h4v h, r;
                split4(widen(rk[j]) * ks_, m1, h, r);
                const int at = kkey * KP + 4 * (ki + KL * j);
                *reinterpret_cast<h4v *>(&lds.k[b & 1][0][at]) = h;
                if constexpr (PL == 2) *reinterpret_cast<h4v *>(&lds.k[b & 1][PL - 1][at]) = r;
            }
#pragma unroll
            for (int t = 0; t < VT; t++) {
                const int task = tid + t * NT, quad = task / C, c = task % C;
                f4v x[4];
#pragma unroll
                for (int s = 0; s < 4; s++) x[s] = widen(rv[t][s]) * vs_;
                // quad 4 st + 2 b + h stands at place 4 st + 2 h + b
                const int place = vplace(4 * c, (quad & ~3) | (quad & 1) << 1 | (quad >> 1 & 1));
                if ((16 * C) % NT == 0 || quad < 16)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        h4v h, r;
                        split4(f4v{x[0][e], x[1][e], x[2][e], x[3][e]}, m1, h, r);
                        const int at = (4 * c + e) * VP + 4 * place;
                        *reinterpret_cast<h4v *>(&lds.v[b & 1][0][at]) = h;
                        if constexpr (PL == 2) *reinterpret_cast<h4v *>(&lds.v[b & 1][PL - 1][at]) = r;
                    }
            }
        };
        f16v acc[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[d][r] = 0.0f;
        float m = -INFINITY, l = 0.0f;
        int acc_e = -1000;                                   // acc counts in 2^acc_e
        RawK rk0;
        RawV rv0;
        if (b0 < b1) {                                       // unit b0 to LDS, b0 + 1 to registers
            load(b0, rk0, rv0);
            load(b0 + 1, rk, rv);
        }
        h8v qh[KS], ql[KS];
        int qe;
        {
            unsigned top = 0;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    qx[ks][j] *= a.qscale;
                    top = finite_top(top, qx[ks][j]);
                }
            const LanePair pr = pl32(__uint_as_float(top));
            qe = max((int)(__float_as_uint(fmaxf(pr.lo, pr.hi)) >> 23) - 127, -100) - kTop;
            const float sc = pow2(-qe);
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    h4v h, r;
                    split4(qx[ks][j] * sc, m1, h, r);
#pragma unroll
                    for (int e = 0; e < 4; e++) { qh[ks][4 * j + e] = h[e]; ql[ks][4 * j + e] = r[e]; }
                }
        }
        if (b0 < b1) {
            tops(b0, rk0, rv0);
            tops(b0 + 1, rk, rv);
            __syncthreads();
            next_exponents(b0);
            split_unit(b0, rk0, rv0);
            k_e = k_n;
            v_e = v_n;
            __syncthreads();
        }
        for (int b = b0; b < b1; b++) {
            const bool odd = lds.odd[b & 3];
            next_exponents(b + 1);
            f16v s[2];
            if (busy) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[0][r] = s[1][r] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++)
#pragma unroll
                    for (int kh = 0; kh < 2; kh++) {
                        const int at = (kh * 32 + col) * KP + 16 * ks + 8 * half;
                        const h8v h = *reinterpret_cast<const h8v *>(&lds.k[b & 1][0][at]);
                        s[kh] = mfma16(h, qh[ks], s[kh]);
                        s[kh] = mfma16(h, ql[ks], s[kh]);
                        if constexpr (PL == 2)
                            s[kh] = mfma16(*reinterpret_cast<const h8v *>(&lds.k[b & 1][PL - 1][at]), qh[ks], s[kh]);
                    }
                split_unit(b + 1, rk, rv);
            } else {
                split_unit(b + 1, rk, rv);
            }
            load(b + 2, rk, rv);
            if (((wave - b - 3) & (NW - 1)) == 0) {
                put_off(b + 3, pg);
                pg = page_at(b + 3 + NW);
                if (lane == 0) lds.odd[(b + 3) & 3] = 0;
            }
            if (busy) {
                const float c = pow2(k_e + qe);              // scores are s * c
                if (!lds.all[b & 3] || b * kUnit + kUnit > see0) {
#pragma unroll
                    for (int kh = 0; kh < 2; kh++)
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const int key = 32 * kh + 8 * (r >> 2) + 4 * half + (r & 3);
                            if (lds.off[b & 3][key] < 0 || b * kUnit + key >= see) s[kh][r] = -INFINITY;
                        }
                }
                float top = s[0][0];                         // (in a chain: two values an instruction)
#pragma unroll
                for (int r = 1; r < 32; r++) top = fmaxf(top, s[r >> 4][r & 15]);
                const LanePair pr = pl32(top);
                top = fmaxf(pr.lo, pr.hi) * c;
                // the accumulated values follow m and v_e
                if (__any(top > m + kLazy) || v_e != acc_e) {
                    const float mn = top > m + kLazy ? top : m;
                    const float f = exp2_hw(m - (mn == -INFINITY ? 0.0f : mn));
                    l *= f;
                    m = mn;
                    const float fv = f * (v_e - acc_e > 126 ? 0.0f : pow2(acc_e - v_e));
                    acc_e = v_e;
#pragma unroll
                    for (int d = 0; d < DT; d++) acc[d] *= fv;
                }
                const float nm = (m == -INFINITY ? 0.0f : -m) + kBias;
                float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
                for (int kh = 0; kh < 2; kh++) {
#pragma unroll
                    for (int st = 0; st < 2; st++) {         // 16 keys
                        h8v ph, pl;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const float p0 = exp2_hw(fmaf(s[kh][8 * st + 2 * j], c, nm));
                            const float p1 = exp2_hw(fmaf(s[kh][8 * st + 2 * j + 1], c, nm));
                            sum0 += p0;
                            sum1 += p1;
                            h2v h, r;
                            split2(p0, p1, m1, h, r);
                            ph[2 * j] = h.x; ph[2 * j + 1] = h.y;
                            pl[2 * j] = r.x; pl[2 * j + 1] = r.y;
                        }
#pragma unroll
                        for (int d = 0; d < DT; d++) {
                            const int at = (32 * d + col) * VP + 4 * vplace(32 * d + col, 8 * kh + 4 * st + 2 * half);
                            const h8v h = *reinterpret_cast<const h8v *>(&lds.v[b & 1][0][at]);
                            acc[d] = mfma16(h, ph, acc[d]);
                            acc[d] = mfma16(h, pl, acc[d]);
                            if constexpr (PL == 2)
                                acc[d] = mfma16(*reinterpret_cast<const h8v *>(&lds.v[b & 1][PL - 1][at]), ph, acc[d]);
                        }
                    }
                }
                l += sum0 + sum1;
                if (odd) {                                   // rows that see a value that is not finite
                    for (int key = 0; key < kUnit; key++) {
                        const long off = lds.off[b & 3][key];
                        if (off < 0 || b * kUnit + key >= see) continue;
#pragma unroll
                        for (int d = 0; d < DT; d++)
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                const int at = 32 * d + 8 * q + 4 * half;
                                if (PAD && at >= hd) continue;
                                const f4v x = widen(raw_load<BF16>(a.v, off + at));
#pragma unroll
                                for (int e = 0; e < 4; e++) acc[d][4 * q + e] = finite_bits(x[e]) ? acc[d][4 * q + e] : NAN;
                            }
                    }
                }
            }
            k_e = k_n;
            v_e = v_n;
            tops(b + 2, rk, rv);
            __syncthreads();
        }
        {
            const LanePair pr = pl32(l);
            l = (pr.lo + pr.hi) * pow2(-kBias);
        }
        const float unit = pow2(acc_e) * pow2(-kBias);       // what acc counts in
        if (u == it.a && ue == it.b) {
            if (live) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                float *o = a.out + row * a.ldo + head * hd;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const int at = 32 * d + 8 * b + 4 * half;
                        const f4v x = {acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]};
                        if (!PAD || at < hd) *reinterpret_cast<f4v *>(o + at) = x * unit * inv;
                    }
            }
        } else if (busy) {
            // [wave][4 d + b][lane] of float4, then (m, l) of every row
            float *part = a.parts + (long)(2 * wg + (u == it.a)) * tile_part(DT);
            f4v *po = reinterpret_cast<f4v *>(part) + (long)wave * 4 * DT * 64 + lane;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int b = 0; b < 4; b++)
                    po[(4 * d + b) * 64] = f4v{acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]} * unit;
            if (half == 0)
                *reinterpret_cast<f2v *>(part + 32 * NW * 32 * DT + 2 * mrow) = f2v{m, l};
        }
        if (ue == u1) note_cut(a, wg, split, it, u, ue);
        u = ue;
    }
}

// ── joining parts ────────────────────────────────────────────────────────
// Reads what the cut items left: 5 us behind k_attn_stream (latency), 15 behind
// 512 workgroups of k_attn_tile, each of whose two parts is 34 KB (head_dim 64).
// A running (m, l, o) over parts.
struct Join {
    float m, l;
    f4v o;
    __device__ __forceinline__ void add(float pm, float pl, const f4v &po) {
        const float mn = fmaxf(m, pm), ref = mn == -INFINITY ? 0.0f : mn;
        const float f = exp2_hw(m - ref), pf = exp2_hw(pm - ref);
        l = l * f + pl * pf;
        o = o * f + po * pf;
        m = mn;
    }
};
// Adds parts first, first + step, .. < n, AHEAD of them on their way at once: their (m, l) `ml` floats and their
// values `at` floats into each.
template <int AHEAD, typename F>
__device__ __forceinline__ void join_parts(Join &j, int first, int step, int n, long ml, long at, F &&part_of) {
    for (int p0 = first; p0 < n; p0 += AHEAD * step) {
        f2v pml[AHEAD];
        f4v po[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const float *p = part_of(min(p0 + i * step, n - 1));
            pml[i] = *reinterpret_cast<const f2v *>(p + ml);
            po[i] = *reinterpret_cast<const f4v *>(p + at);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (p0 + i * step < n) j.add(pml[i].x, pml[i].y, po[i]);
    }
}

// Block w joins the item that workgroup w of k_attn_few or k_attn_stream
// noted; blocks from n_few on those of k_attn_tile.  Its threads share the
// item's float4s and, where those are few, its parts.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_attn_join(AttnArgs a, int n_few, const Cut *tile_cuts, const float *tile_parts) {
    constexpr int NW = tile_waves(DT), FR = kFewRows * few_pitch(DT);
    __shared__ Join part[kThreads];
    const int hd = a.hd, n4 = hd >> 2, G = a.group.d, tid = threadIdx.x;
    if ((int)blockIdx.x < n_few) {
        const int w = blockIdx.x;
        const Cut c = a.cuts[w];
        if (c.parts == 0) return;
        auto part_of = [&](int p) { return a.parts + (long)(2 * (w + p) + (p == 0)) * few_part(DT); };
        const int n = c.n * G * n4, slices = max(1, kThreads / n), lanes = min(n, kThreads);   // slices of parts
        for (int e0 = 0; e0 < n; e0 += kThreads) {
            const int e = e0 + tid % lanes, slice = tid / lanes, i = e / n4, col = e - i * n4;
            Join j = {-INFINITY, 0.0f, {0.f, 0.f, 0.f, 0.f}};
            if (e < n && slice < slices)
                join_parts<8>(j, slice, slices, c.parts, FR + 2 * i, i * few_pitch(DT) + 4 * col, part_of);
            part[tid] = j;
            __syncthreads();
            if (slice == 0 && e < n) {
                for (int s = 1; s < slices; s++) {
                    const Join &o = part[tid + s * lanes];
                    j.add(o.m, o.l, o.o);
                }
                const int t = a.group.quot(i), r = c.row0 + t;
                if ((unsigned)r < (unsigned)a.rows)
                    *reinterpret_cast<f4v *>(a.out + r * a.ldo + (long)(c.kvh * G + i - t * G) * hd + 4 * col) =
                        j.o * (j.l == 0.0f ? 0.0f : 1.0f / j.l);
            }
            __syncthreads();
        }
        return;
    }
    // four blocks an item: float4 q of every fourth
    const int w = ((int)blockIdx.x - n_few) >> 2, q0 = (int)blockIdx.x - n_few & 3;
    const Cut c = tile_cuts[w];
    if (c.parts == 0) return;
    auto part_of = [&](int p) { return tile_parts + (long)(2 * (w + p) + (p == 0)) * tile_part(DT); };
    const int tt = a.tile_tokens, t0 = c.tile * tt;
    constexpr int NE = 64 * NW * DT / kThreads;              // float4s of a thread
    Join j[NE];
    float *to[NE];
    long ml[NE], at[NE];
#pragma unroll
    for (int i = 0; i < NE; i++) {                           // as the lanes of the tile's waves
        const int e = tid + i * kThreads, lane = e & 63, wave = (e >> 6) % NW, q = 4 * (e / (64 * NW)) + q0;
        const int mrow = wave * 32 + (lane & 31), col = 8 * q + 4 * (lane >> 5);
        const int tok = t0 + a.group.quot(mrow), row = c.row0 + tok;
        const bool live = mrow < tt * G && tok < c.n && (unsigned)row < (unsigned)a.rows && col < hd;
        to[i] = live ? a.out + row * a.ldo + (c.kvh * G + mrow - (tok - t0) * G) * (long)hd + col : nullptr;
        ml[i] = 32 * NW * 32 * DT + 2 * mrow;
        at[i] = 4l * ((wave * 4 * DT + q) * 64 + lane);
        j[i] = Join{-INFINITY, 0.0f, {0.f, 0.f, 0.f, 0.f}};
    }
    for (int p0 = 0; p0 < c.parts; p0 += 2) {
        const float *p[2] = {part_of(p0), part_of(min(p0 + 1, c.parts - 1))};
        f2v pml[2][NE];
        f4v po[2][NE];
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < NE; i++) {
                if (!to[i]) continue;
                pml[s][i] = *reinterpret_cast<const f2v *>(p[s] + ml[i]);
                po[s][i] = *reinterpret_cast<const f4v *>(p[s] + at[i]);
            }
#pragma unroll
        for (int s = 0; s < 2; s++)
            if (p0 + s < c.parts)
#pragma unroll
                for (int i = 0; i < NE; i++)
                    if (to[i]) j[i].add(pml[s][i].x, pml[s][i].y, po[s][i]);
    }
#pragma unroll
    for (int i = 0; i < NE; i++)
        if (to[i]) *reinterpret_cast<f4v *>(to[i]) = j[i].o * (j[i].l == 0.0f ? 0.0f : 1.0f / j[i].l);
}

// ── launch ───────────────────────────────────────────────────────────────
// Workgroups: what the chip holds at once.  More would split heads further
// and start anew (64 requests of 32 heads on 4, 1024 bf16 positions of 128,
// through the fp32 instructions: 104 us on 1024 workgroups, 54 on the 512 that
// fit), fewer leave it idle
// (1024 requests of 12 heads, 100 positions of 64: 168 us on 512, 133 on 1024).
constexpr int kFewGroups = 1024;                            // the most for few rows
constexpr int kTileGroups = 512;
constexpr int tile_groups(int dt) { return 2048 / tile_waves(dt); }

int tile_dt(int hd) { return (hd + 31) / 32; }

typedef void (*Fn)(AttnArgs);
typedef void (*JoinFn)(AttnArgs, int, const Cut *, const float *);

template <int HQ>
Fn few_fn(int hd, bool b16) {
    return hd == 16 * HQ ? (b16 ? k_attn_few_b16<HQ, false> : k_attn_few<HQ, false>)
                         : (b16 ? k_attn_few_b16<HQ, true> : k_attn_few<HQ, true>);
}
template <int MR, int C4>
Fn stream_fn2(bool fast, bool b16) {
    return fast ? (b16 ? k_attn_stream<MR, C4, true, true> : k_attn_stream<MR, C4, true, false>)
                : (b16 ? k_attn_stream<MR, C4, false, true> : k_attn_stream<MR, C4, false, false>);
}
Fn stream_fn(int rows, const ptmi_pages_t &p) {
    const bool b16 = p.type == PTMI_BF16, wide = p.head_dim > 64;
    const bool fast = p.page_size % 4 == 0 &&
                      !(b16 && (p.head_dim | p.page_stride | p.pos_stride | p.head_stride) % 8);
    return rows == 1 ? (wide ? stream_fn2<1, 2>(fast, b16) : stream_fn2<1, 1>(fast, b16))
         : rows == 2 ? (wide ? stream_fn2<2, 2>(fast, b16) : stream_fn2<2, 1>(fast, b16))
                     : (wide ? stream_fn2<4, 2>(fast, b16) : stream_fn2<4, 1>(fast, b16));
}
template <int DT>
Fn tile_fn(int hd, bool b16) {
    return hd == 32 * DT ? (b16 ? k_attn_tile<DT, false, true> : k_attn_tile<DT, false, false>)
                         : (b16 ? k_attn_tile<DT, true, true> : k_attn_tile<DT, true, false>);
}

int few_groups(Fn fn) {
    static std::unordered_map<Fn, int> known;
    int &n = known[fn];
    if (n == 0) {
        int per_cu = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, (const void *)fn, kThreads, 0) != hipSuccess) per_cu = 2;
        n = std::min(kFewGroups, 256 * std::max(1, per_cu));
    }
    return n;
}

// Which kernels a call runs.
struct Plan {
    bool few, tile;
    int stream;                      // rows of k_attn_stream in k_attn_few's place; 0: not
    size_t few_at, tile_at, floats;  // of the workspace (the cuts come first)
};
Plan attn_plan(const ptmi_pages_t &p, int n_heads, int max_new) {
    const int group = n_heads / p.n_kv_heads;
    Plan c = {};
    c.few = group <= kFewRows;
    c.tile = max_new == 0 || (long)max_new * group > kFewRows;
    if (max_new > 0 && (long)max_new * group <= 4) c.stream = max_new * group == 3 ? 4 : max_new * group;
    c.tile_at = (kFewGroups + kTileGroups) * sizeof(Cut) / sizeof(float);
    c.few_at = c.tile_at;
    c.tile_at += c.few ? (size_t)2 * kFewGroups * few_part(tile_dt(p.head_dim)) : 0;
    c.floats = c.tile_at;
    if (c.tile) c.floats += (size_t)2 * tile_groups(tile_dt(p.head_dim)) * tile_part(tile_dt(p.head_dim));
    return c;
}

int check_heads(const char *who, const ptmi_pages_t *pages, int n_heads, int max_new) {
    int st = check_pages(who, pages);
    if (st) return st;
    if (n_heads < 1 || n_heads % pages->n_kv_heads || n_heads / pages->n_kv_heads > kTileRows)
        return set_error(PTMI_ERR_ARG, "%s: n_heads=%d for n_kv_heads=%d", who, n_heads, pages->n_kv_heads);
    if (max_new < 0) return set_error(PTMI_ERR_ARG, "%s: max_new=%d", who, max_new);
    return PTMI_OK;
}

}  // namespace

}  // namespace ptmi

using namespace ptmi;

extern "C" {

size_t ptmi_paged_attention_work(const ptmi_pages_t *pages, int n_heads, int max_new) {
    if (check_heads("ptmi_paged_attention_work", pages, n_heads, max_new)) return 0;
    return attn_plan(*pages, n_heads, max_new).floats * sizeof(float);
}

int ptmi_paged_attention_dev(const ptmi_pages_t *pages, const int *block_table, int table_width,
                             const int *row_start, const int *kv_len, int n_requests, int max_new, const float *q,
                             long ldq, float *out, long ldo, int rows, int n_heads, float scale, void *work,
                             size_t work_bytes, void *stream) {
    int st = check_heads("ptmi_paged_attention", pages, n_heads, max_new);
    if (st) return st;
    const ptmi_pages_t &p = *pages;
    if (n_requests < 0 || table_width < 1 || rows < 0 || !std::isfinite(scale * 1.44269504f))
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: n_requests=%d table_width=%d rows=%d scale=%g", n_requests,
                         table_width, rows, (double)scale);
    if ((long long)table_width * p.page_size > INT_MAX - 4096)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: %d pages of %d positions a request", table_width, p.page_size);
    if (n_requests == 0 || rows == 0) return PTMI_OK;
    if (!block_table || !row_start || !kv_len || !q || !out || !work)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: NULL argument");
    const long w = (long)n_heads * p.head_dim;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15 || ldq % 4 || ldo % 4 || ldq < w || ldo < w)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: rows must be 16-byte aligned and hold %d heads (ldq=%ld ldo=%ld)",
                         n_heads, ldq, ldo);
    if (q == out) return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: out must not be q");
    const Plan plan = attn_plan(p, n_heads, max_new);
    if (work_bytes < plan.floats * sizeof(float))
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: work holds %zu bytes, %zu needed", work_bytes,
                         plan.floats * sizeof(float));
    if ((st = ensure_init())) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    const int group = n_heads / p.n_kv_heads;
    AttnArgs a = {p.k, p.v, p.page_stride, p.pos_stride, p.head_stride, p.n_pages, FastDiv(p.page_size), block_table,
                  table_width, row_start, kv_len, n_requests, q, ldq, out, ldo, rows, p.n_kv_heads, p.head_dim,
                  FastDiv(group), 32 * tile_waves(tile_dt(p.head_dim)) / group, plan.stream ? plan.stream : kFewRows,
                  scale * 1.44269504088896341f,
                  -1.0f, (float *)work + plan.few_at, (Cut *)work};
    hipStream_t s = stream ? (hipStream_t)stream : lib_stream();
    const bool b16 = p.type == PTMI_BF16;
    const int hd = p.head_dim;
    const int dt = tile_dt(hd), n_tile = plan.tile ? tile_groups(dt) : 1;
    int n_few = 1;
    if (plan.few) {
        const Fn fn = plan.stream ? stream_fn(plan.stream, p) : dt == 1 ? few_fn<2>(hd, b16) : dt == 2 ? few_fn<4>(hd, b16) : dt == 3 ? few_fn<6>(hd, b16)
                    : few_fn<8>(hd, b16);
        n_few = few_groups(fn);
        hipLaunchKernelGGL(fn, dim3(n_few), dim3(kThreads), 0, s, a);
    }
    if (plan.tile) {
        const Fn fn = dt == 1 ? tile_fn<1>(hd, b16) : dt == 2 ? tile_fn<2>(hd, b16) : dt == 3 ? tile_fn<3>(hd, b16)
                    : tile_fn<4>(hd, b16);
        AttnArgs b = a;
        b.parts = (float *)work + plan.tile_at;
        b.cuts = a.cuts + kFewGroups;
        hipLaunchKernelGGL(fn, dim3(n_tile), dim3(64 * tile_waves(dt)), 0, s, b);
    }
    // One unit a head and nothing but single rows: nothing is ever cut.
    if (plan.tile || (long)table_width * p.page_size > kUnit) {
        // (the last workgroup's stretch ends with an item)
        const int n_join = 4 * (n_tile - 1);
        const JoinFn join = dt == 1 ? k_attn_join<1> : dt == 2 ? k_attn_join<2> : dt == 3 ? k_attn_join<3> : k_attn_join<4>;
        hipLaunchKernelGGL(join, dim3(n_few - 1 + n_join), dim3(kThreads), 0, s, a, n_few - 1, a.cuts + kFewGroups,
                           (const float *)work + plan.tile_at);
    }
    PTMI_HIP(hipGetLastError());
    return PTMI_OK;
}

}  // extern "C"
