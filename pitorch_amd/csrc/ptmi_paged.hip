// A step's bookkeeping over a paged cache, and the write of its new keys and
// values.
#include "ptmi_paged.h"

#include <climits>

namespace ptmi {

namespace {

// ── bookkeeping ──────────────────────────────────────────────────────────
// Page counts of a request before and after its new tokens, and sums of
// them over the requests before it.  All of it is a scan over the requests
// and look-ups by rank; the lengths stay on the device.
constexpr int kPlanThreads = 1024;

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
};

struct PlanSums { long long take, give, rows; };

__device__ __forceinline__ PlanSums operator+(PlanSums a, PlanSums b) {
    return {a.take + b.take, a.give + b.give, a.rows + b.rows};
}

// Exclusive sums over the block's threads; *total gets the block's.
__device__ PlanSums block_scan(PlanSums v, PlanSums *lds, PlanSums *total) {
    const int t = threadIdx.x;
    lds[t] = v;
    __syncthreads();
    for (int d = 1; d < kPlanThreads; d <<= 1) {
        PlanSums o = {0, 0, 0};
        if (t >= d) o = lds[t - d];
        __syncthreads();
        lds[t] = lds[t] + o;
        __syncthreads();
    }
    const PlanSums incl = lds[t];
    *total = lds[kPlanThreads - 1];
    __syncthreads();
    return {incl.take - v.take, incl.give - v.give, incl.rows - v.rows};
}

__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PlanArgs a) {
    __shared__ PlanSums lds[kPlanThreads];
    __shared__ int bad;
    const int t = threadIdx.x, P = a.page.d;
    const int count = *a.pool_count;
    if (t == 0) bad = count < 0 || count > a.n_pages ? 8 : 0;
    __syncthreads();
    auto pages = [&](int len) { return len > 0 ? a.page.quot(len - 1) + 1 : 0; };
    auto sums = [&](int i) -> PlanSums {
        if (i >= a.n) return {0, 0, 0};
        const int p = a.past[i], f = a.fresh[i];
        if (p < 0 || f < -1 || f > INT_MAX - p) return {0, 0, 0};
        if (f < 0) return {0, pages(p), 0};
        return {pages(p + f) - pages(p), 0, f};
    };
    // totals, and what refuses the step
    PlanSums all = {0, 0, 0}, part;
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
        const int i = i0 + t;
        if (i < a.n) {
            const int p = a.past[i], f = a.fresh[i];
            if (p < 0 || f < -1 || f > INT_MAX - p) atomicOr(&bad, 8);
            else if (pages(p + (f > 0 ? f : 0)) > a.width) atomicOr(&bad, 2);
            else if (f < 0)
                for (int j = 0; j < pages(p); j++)
                    if ((unsigned)a.table[(long)i * a.width + j] >= (unsigned)a.n_pages) { atomicOr(&bad, 8); break; }
        }
        block_scan(sums(i), lds, &part);
        all = all + part;
    }
    if (t == 0) {
        if (count + all.give > a.n_pages) atomicOr(&bad, 8);
        if (all.take > count + all.give) atomicOr(&bad, 1);
        if (all.rows > a.max_rows) atomicOr(&bad, 4);
    }
    __syncthreads();
    const long top = count + all.give;
    if (!bad)                                              // pages that the pool held before this step
        for (long j = t; j < all.take; j += kPlanThreads) {
            const long at = top - 1 - j;
            if (at < count && (unsigned)a.pool[at] >= (unsigned)a.n_pages) atomicOr(&bad, 8);
        }
    __syncthreads();
    const int refused = bad;
    __syncthreads();
    if (refused) {
        for (int i = t; i < a.n; i += kPlanThreads) a.kv_len[i] = a.past[i];
        for (int i = t; i <= a.n; i += kPlanThreads) a.row_start[i] = 0;
        for (int r = t; r < a.max_rows; r += kPlanThreads) a.row_pos[r] = a.row_slot[r] = -1;
        if (t == 0) { *a.pool_left = count; *a.status = refused; }
        return;
    }
    PlanSums before = {0, 0, 0};
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {       // ended requests give their pages back
        const int i = i0 + t;
        const PlanSums v = sums(i), at = before + block_scan(v, lds, &part);
        for (int j = 0; j < v.give; j++) a.pool[count + at.give + j] = a.table[(long)i * a.width + j];
        before = before + part;
    }
    __syncthreads();
    before = {0, 0, 0};
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {       // the others take theirs
        const int i = i0 + t;
        const PlanSums v = sums(i), at = before + block_scan(v, lds, &part);
        if (i < a.n) {
            const int p = a.past[i], f = a.fresh[i], old = pages(p);
            for (int j = 0; j < v.take; j++) a.table[(long)i * a.width + old + j] = a.pool[top - 1 - (at.take + j)];
            for (int r = 0; r < f; r++) {
                const int pos = p + r, j = a.page.quot(pos);
                const int page = j < old ? a.table[(long)i * a.width + j] : a.pool[top - 1 - (at.take + j - old)];
                a.row_pos[at.rows + r] = pos;
                a.row_slot[at.rows + r] = page * P + (pos - j * P);
            }
            a.row_start[i] = (int)at.rows;
            a.kv_len[i] = f < 0 ? 0 : p + f;
        }
        before = before + part;
    }
    for (long r = all.rows + t; r < a.max_rows; r += kPlanThreads) a.row_pos[r] = a.row_slot[r] = -1;
    if (t == 0) {
        a.row_start[a.n] = (int)all.rows;
        *a.pool_left = (int)(top - all.take);
        *a.status = 0;
    }
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

// One thread per float4 of a row's [q | k | v] heads.
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
    if (n_requests < 0 || max_rows < 0 || n_pages < 1 || page_size < 1 || table_width < 1 ||
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
    const PlanArgs a = {past, fresh, n_requests, pool, pool_count, n_pages, FastDiv(page_size), block_table,
                        table_width, kv_len, pool_left, row_start, row_pos, row_slot, max_rows, status};
    hipLaunchKernelGGL(k_paged_plan, dim3(1), dim3(kPlanThreads), 0, stream ? (hipStream_t)stream : lib_stream(), a);
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
