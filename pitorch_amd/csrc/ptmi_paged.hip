// A step's bookkeeping over a paged cache, and the write of its new keys and
// values.
#include "ptmi_paged.h"

#include <algorithm>
#include <climits>

namespace ptmi {

namespace {

// ── bookkeeping ──────────────────────────────────────────────────────────
// Exclusive sums over the requests of the pages that each takes and gives and
// of its rows; then every page that moves and every row is found by its rank
// in them, independently of the others.  The pool's entry i is, after the
// ended requests' pages went onto it, pool[i] below the old count and above
// it the (i - count)-th given page, read where it comes from: so nothing that
// is written here is read here.
// A step's rows bound it: few fit one workgroup; for many, workgroups that
// each hold all sums share the rows and pages.  The first one also writes the
// lengths; only where these stand in the place of the cached lengths, which
// other workgroups still read, does a launch of its own (k_paged_plan_end).
// 16 requests of one token: 14.6 -> 4.9 us a call (sums of 1024 in 20 steps
// with a barrier each before, now in two); 1021 requests, 44 thousand rows,
// 14 thousand pages: 150 -> 8.7 us, and 3.5 for the second launch where there is
// one (one workgroup, a request's pages and rows by one thread each before).
// Both are latency: a handful of dependent loads, and 0.4 MB written.
constexpr int kPlanThreads = 1024;
constexpr int kPlanSmall = 1024, kPlanMost = 8192;          // requests whose sums fit in shared memory
constexpr int kPlanOneRows = 4096;                          // rows that one workgroup writes
constexpr int kPlanLimit = 1 << 24;                         // a request's new tokens, and its pages

struct PlanArgs {
    const int *past, *fresh;
    int n;
    int *pool;
    const int *pool_count;
    int n_pages;
    FastDiv page;
    int *table;
    int width;
    int *kv_len, *pool_left, *row_start, *row_pos, *row_slot;
    int max_rows;
    int *status;
    bool end;                        // the first workgroup writes the lengths as well
};

// Sums over the requests before i; entry n: of all.
template <int CAP>
struct PlanLds {
    int past[CAP], take[CAP + 1], give[CAP + 1], row[CAP + 1];
    long wave[3][kPlanThreads / 64];
    int bad;
};
struct PlanTotals { long take, give, rows; int refused; };

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {           // inclusive
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    return dpp_add<0x143, 0xC>(v);
}

__device__ __forceinline__ int pages_of(const PlanArgs &a, int len) { return len > 0 ? a.page.quot(len - 1) + 1 : 0; }

template <int CAP>
__device__ PlanTotals plan_sums(const PlanArgs &a, PlanLds<CAP> &s, int count) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    if (t == 0) s.bad = count < 0 || count > a.n_pages ? 8 : 0;
    long take = 0, give = 0, rows = 0;                       // before this turn's requests
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
        const int i = i0 + t;
        int p = 0, f = 0;
        if (i < a.n) { p = a.past[i]; f = a.fresh[i]; }
        int bad = 0, tk = 0, gv = 0;
        // (kPlanLimit: sums of a wave's 64 stay under 2^31)
        if (p < 0 || f < -1 || f > kPlanLimit || f > INT_MAX - p || pages_of(a, p) > kPlanLimit) {
            bad = 8;
            p = f = 0;
        } else {
            const int now = pages_of(a, p + max(f, 0)), old = pages_of(a, p);
            if (now > a.width) bad = 2;
            tk = f < 0 ? 0 : now - old;
            gv = f < 0 ? old : 0;
            f = max(f, 0);
        }
        const int st = wave_scan(tk), sg = wave_scan(gv), sr = wave_scan(f);
        __syncthreads();
        if (bad) atomicOr(&s.bad, bad);
        if (lane == 63) { s.wave[0][w] = st; s.wave[1][w] = sg; s.wave[2][w] = sr; }
        __syncthreads();
        long bt = take, bg = give, br = rows;
        for (int k = 0; k < kPlanThreads / 64; k++) {
            if (k == w) {
                if (i < a.n) {
                    s.past[i] = p;
                    s.take[i] = (int)(bt + st - tk);
                    s.give[i] = (int)(bg + sg - gv);
                    s.row[i] = (int)(br + sr - f);
                }
            }
            bt += s.wave[0][k];
            bg += s.wave[1][k];
            br += s.wave[2][k];
        }
        take = bt;
        give = bg;
        rows = br;
    }
    __syncthreads();
    if (t == 0) {
        s.take[a.n] = (int)take;
        s.give[a.n] = (int)give;
        s.row[a.n] = (int)rows;
    }
    __syncthreads();
    int refused = s.bad;
    if (count + give > a.n_pages) refused |= 8;
    if (take > count + give) refused |= 1;
    if (rows > a.max_rows) refused |= 4;
    return {take, give, rows, refused};
}

// The last request whose sum before it is at most x (x < sum[n]).
__device__ __forceinline__ int plan_find(const int *sum, int n, int x) {
    int lo = 0, hi = n;                                     // sum[lo] <= x < sum[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sum[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int CAP>
__device__ void plan_end(const PlanArgs &a, const PlanLds<CAP> &s, const PlanTotals &all, int count) {
    for (int i = threadIdx.x; i <= a.n; i += kPlanThreads) {
        a.row_start[i] = all.refused ? 0 : s.row[i];
        if (i < a.n) a.kv_len[i] = all.refused ? a.past[i] : a.fresh[i] < 0 ? 0 : s.past[i] + (s.row[i + 1] - s.row[i]);
    }
    if (threadIdx.x == 0) {
        *a.pool_left = all.refused ? count : (int)(count + all.give - all.take);
        *a.status = all.refused;
    }
}

template <int CAP>
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PlanArgs a) {
    __shared__ PlanLds<CAP> s;
    const int P = a.page.d, count = *a.pool_count;
    const PlanTotals all = plan_sums(a, s, count);
    const int first = (int)blockIdx.x * kPlanThreads + threadIdx.x, step = (int)gridDim.x * kPlanThreads;
    if (!all.refused) {
        auto given = [&](int g) {                            // the g-th given page
            const int i = plan_find(s.give, a.n, g);
            return a.table[(long)i * a.width + (g - s.give[i])];
        };
        auto taken = [&](int k) {                            // the k-th taken page
            const int at = count + (int)all.give - 1 - k;
            return at < count ? a.pool[at] : given(at - count);
        };
        for (int g = first; g < all.give; g += step) a.pool[count + g] = given(g);
        for (int k = first; k < all.take; k += step) {
            const int i = plan_find(s.take, a.n, k);
            a.table[(long)i * a.width + pages_of(a, s.past[i]) + (k - s.take[i])] = taken(k);
        }
        for (int r = first; r < all.rows; r += step) {
            const int i = plan_find(s.row, a.n, r), pos = s.past[i] + (r - s.row[i]), j = a.page.quot(pos);
            const int old = pages_of(a, s.past[i]);
            const int page = j < old ? a.table[(long)i * a.width + j] : taken(s.take[i] + j - old);
            a.row_pos[r] = pos;
            a.row_slot[r] = (unsigned)page < (unsigned)a.n_pages ? page * P + (pos - j * P) : -1;
        }
    }
    for (int r = (all.refused ? 0 : (int)all.rows) + first; r < a.max_rows; r += step) a.row_pos[r] = a.row_slot[r] = -1;
    if (a.end && blockIdx.x == 0) plan_end(a, s, all, count);
}

template <int CAP>
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan_end(PlanArgs a) {
    __shared__ PlanLds<CAP> s;
    const int count = *a.pool_count;
    const PlanTotals all = plan_sums(a, s, count);
    plan_end(a, s, all, count);
}

// ── store ────────────────────────────────────────────────────────────────
struct StoreArgs {
    const float *q; long ldq;
    float *q_out; long ldo;
    const float *k, *v; long ldkv;
    const int *pos, *slot;
    const float *rope;
    int rows, rope_len, n_heads, kv_heads, hd4;
    void *kc, *vc;
    long page_stride, pos_stride, head_stride;
    int slots;
    FastDiv page;
};

// Nearest bf16, ties to even; NaN stays NaN.
__device__ __forceinline__ unsigned bf16_bits(float x) {
    const unsigned u = __float_as_uint(x);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (u >> 16) | 0x40u;
    return (u + 0x7FFFu + (u >> 16 & 1u)) >> 16;
}

template <bool BF16>
__device__ __forceinline__ void put4(void *base, long at, float4 x) {
    if constexpr (BF16) {
        const uint2 w = {bf16_bits(x.x) | bf16_bits(x.y) << 16, bf16_bits(x.z) | bf16_bits(x.w) << 16};
        *reinterpret_cast<uint2 *>(static_cast<unsigned short *>(base) + at) = w;
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(base) + at) = x;
    }
}

// One thread per float4 of a row's [q | k | v] heads: both halves of two pairs
// of RoPE, and nothing is read twice but the row's angles (from the caches, by
// its heads).  Bound by the bytes: 8190 rows of 32 + 8 + 8 heads of 128, bf16
// pages, 373 MB in 70 us, 5.3 TB/s (a large copy: 5.2); 64 rows of 12 + 12 +
// 12 heads of 64: 3 us, the latency of a slot, a row and a store.
template <bool BF16>
__global__ __launch_bounds__(256) void k_paged_store(StoreArgs a) {
    const int r = blockIdx.y, slot = a.slot[r];
    if ((unsigned)slot >= (unsigned)a.slots) return;
    const int pos = a.rope ? a.pos[r] : 0;
    if (a.rope && (unsigned)pos >= (unsigned)a.rope_len) return;
    const int nq = a.q ? a.n_heads : 0, items = (nq + 2 * a.kv_heads) * a.hd4;
    const int e = blockIdx.x * 256 + threadIdx.x;
    if (e >= items) return;
    const int head = e / a.hd4, c = (e - head * a.hd4) * 4;
    const int kvh = head - nq;                              // < 0: a query head; then keys, then values
    const bool is_v = kvh >= a.kv_heads;
    const float *src = kvh < 0 ? a.q + r * a.ldq + (long)head * a.hd4 * 4
                     : is_v ? a.v + r * a.ldkv + (long)(kvh - a.kv_heads) * a.hd4 * 4
                            : a.k + r * a.ldkv + (long)kvh * a.hd4 * 4;
    float4 x = *reinterpret_cast<const float4 *>(src + c);
    if (a.rope && !is_v) {
        const float4 t = *reinterpret_cast<const float4 *>(a.rope + (long)pos * a.hd4 * 4 + c);
        x = make_float4(x.x * t.x - x.y * t.y, x.x * t.y + x.y * t.x, x.z * t.z - x.w * t.w, x.z * t.w + x.w * t.z);
    }
    if (kvh < 0) {
        *reinterpret_cast<float4 *>(a.q_out + r * a.ldo + (long)head * a.hd4 * 4 + c) = x;
        return;
    }
    const int pg = a.page.quot(slot);
    const long at = pg * a.page_stride + (long)(slot - pg * a.page.d) * a.pos_stride +
                    (long)(is_v ? kvh - a.kv_heads : kvh) * a.head_stride + c;
    put4<BF16>(is_v ? a.vc : a.kc, at, x);
}

}  // namespace

int check_pages(const char *who, const ptmi_pages_t *p) {
    if (!p || !p->k || !p->v) return set_error(PTMI_ERR_ARG, "%s: NULL cache", who);
    if (((uintptr_t)p->k | (uintptr_t)p->v) & 15) return set_error(PTMI_ERR_ARG, "%s: cache not 16-byte aligned", who);
    if (p->type != PTMI_F32 && p->type != PTMI_BF16) return set_error(PTMI_ERR_ARG, "%s: cache type %d", who, p->type);
    if (p->n_pages < 1 || p->page_size < 1 || (long long)p->n_pages * p->page_size > INT_MAX)
        return set_error(PTMI_ERR_ARG, "%s: %d pages of %d positions", who, p->n_pages, p->page_size);
    if (p->n_kv_heads < 1 || p->head_dim < 4 || p->head_dim % 4 || p->head_dim > 128)
        return set_error(PTMI_ERR_ARG, "%s: n_kv_heads=%d head_dim=%d (a multiple of 4 up to 128)", who, p->n_kv_heads,
                         p->head_dim);
    const long st[] = {p->page_stride, p->pos_stride, p->head_stride};
    for (long v : st)
        if (v < p->head_dim || v % 4)
            return set_error(PTMI_ERR_ARG, "%s: cache strides %ld %ld %ld (multiples of 4, at least head_dim)", who,
                             st[0], st[1], st[2]);
    return PTMI_OK;
}

}  // namespace ptmi

using namespace ptmi;

extern "C" {

int ptmi_paged_plan_dev(const int *past, const int *fresh, int n_requests, int *pool, const int *pool_count,
                        int n_pages, int page_size, int *block_table, int table_width, int *kv_len,
                        int *pool_left, int *row_start, int *row_pos, int *row_slot, int max_rows, int *status,
                        void *stream) {
    if (n_requests < 0 || n_requests > kPlanMost || max_rows < 0 || n_pages < 1 || page_size < 1 || table_width < 1 ||
        (long long)n_pages * page_size > INT_MAX)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_plan: n_requests=%d n_pages=%d page_size=%d table_width=%d max_rows=%d",
                         n_requests, n_pages, page_size, table_width, max_rows);
    if (!pool || !pool_count || !pool_left || !row_start || !status ||
        (n_requests && (!past || !fresh || !block_table || !kv_len)) || (max_rows && (!row_pos || !row_slot)))
        return set_error(PTMI_ERR_ARG, "ptmi_paged_plan: NULL argument");
    int st = ensure_init();
    if (st) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    const bool one = max_rows <= kPlanOneRows;
    const PlanArgs a = {past, fresh, n_requests, pool, pool_count, n_pages, FastDiv(page_size), block_table,
                        table_width, kv_len, pool_left, row_start, row_pos, row_slot, max_rows, status,
                        one || (kv_len != past && pool_left != pool_count)};
    hipStream_t s = stream ? (hipStream_t)stream : lib_stream();
    const bool small = n_requests <= kPlanSmall;
    const int groups = one ? 1 : std::min(256, (max_rows + kPlanThreads - 1) / kPlanThreads);
    hipLaunchKernelGGL(small ? k_paged_plan<kPlanSmall> : k_paged_plan<kPlanMost>, dim3(groups), dim3(kPlanThreads), 0, s, a);
    if (!a.end)
        hipLaunchKernelGGL(small ? k_paged_plan_end<kPlanSmall> : k_paged_plan_end<kPlanMost>, dim3(1), dim3(kPlanThreads),
                           0, s, a);
    PTMI_HIP(hipGetLastError());
    return PTMI_OK;
}

int ptmi_paged_store_dev(const ptmi_pages_t *pages, const float *q, long ldq, float *q_out, long ldo, int n_heads,
                         const float *k, const float *v, long ldkv, const int *row_pos, const int *row_slot,
                         int rows, const float *rope, int rope_len, void *stream) {
    int st = check_pages("ptmi_paged_store", pages);
    if (st) return st;
    const ptmi_pages_t &p = *pages;
    if (rows < 0 || n_heads < (q ? 1 : 0) || n_heads > (1 << 20) || p.n_kv_heads > (1 << 20))
        return set_error(PTMI_ERR_ARG, "ptmi_paged_store: rows=%d n_heads=%d n_kv_heads=%d", rows, n_heads, p.n_kv_heads);
    if (rows == 0) return PTMI_OK;
    if (!k || !v || !row_slot || (q && !q_out) || (rope && (!row_pos || rope_len < 1)))
        return set_error(PTMI_ERR_ARG, "ptmi_paged_store: NULL argument");
    const long qw = (long)n_heads * p.head_dim, kw = (long)p.n_kv_heads * p.head_dim;
    if (((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)rope) & 15 ||
        (q && (ldq % 4 || ldo % 4 || ldq < qw || ldo < qw)) || ldkv % 4 || ldkv < kw)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_store: rows must be 16-byte aligned and hold their heads (ldq=%ld ldo=%ld ldkv=%ld)",
                         ldq, ldo, ldkv);
    if (q && q_out == q && ldo != ldq)                       // (a row would be written over another)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_store: q_out is q, with another row stride (ldq=%ld ldo=%ld)", ldq, ldo);
    if ((st = ensure_init())) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    StoreArgs a = {q, ldq, q_out, ldo, k, v, ldkv, row_pos, row_slot, rope, rows, rope_len, n_heads, p.n_kv_heads,
                   p.head_dim / 4, p.k, p.v, p.page_stride, p.pos_stride, p.head_stride, p.n_pages * p.page_size,
                   FastDiv(p.page_size)};
    const int items = ((q ? n_heads : 0) + 2 * p.n_kv_heads) * a.hd4;
    hipStream_t s = stream ? (hipStream_t)stream : lib_stream();
    for (int r0 = 0; r0 < rows; r0 += 65535) {              // the grid's y extent
        StoreArgs b = a;
        const int n = rows - r0 < 65535 ? rows - r0 : 65535;
        if (q) { b.q += r0 * ldq; b.q_out += r0 * ldo; }
        b.k += r0 * ldkv; b.v += r0 * ldkv; b.slot += r0;
        if (rope) b.pos += r0;
        hipLaunchKernelGGL(p.type == PTMI_BF16 ? k_paged_store<true> : k_paged_store<false>,
                           dim3((items + 255) / 256, n), dim3(256), 0, s, b);
        PTMI_HIP(hipGetLastError());
    }
    return PTMI_OK;
}

}  // extern "C"
