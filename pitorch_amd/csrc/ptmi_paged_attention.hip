// Attention of new rows over a paged cache.
//
// One wave per row and head takes 64 keys at a time, one per lane, with a
// running maximum m and sum l of the softmax:
//   m' = max(m, s), l' = l e^(m - m') + sum e^(s - m'), o' = o e^(m - m') + sum e^(s - m') v.
#include "ptmi_paged.h"

#include <climits>
#include <cmath>

namespace ptmi {

namespace {

struct AttnArgs {
    const void *k, *v;
    long page_stride, pos_stride, head_stride;
    int n_pages;
    FastDiv page;
    const int *table; int width;
    const int *row_start, *kv_len; int n_req;
    const float *q; long ldq;
    float *out; long ldo;
    int rows, heads, kv_heads, hd;
    float scale;
};

template <bool BF16>
__device__ __forceinline__ float4 get4(const void *base, long at) {
    if constexpr (BF16) {
        const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const unsigned short *>(base) + at);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xFFFF0000u));
    } else {
        return *reinterpret_cast<const float4 *>(static_cast<const float *>(base) + at);
    }
}

template <bool BF16>
__global__ __launch_bounds__(64) void k_attn_simple(AttnArgs a) {
    __shared__ float qs[128], ps[64];
    __shared__ long at[64];
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    // the request whose rows hold r
    int lo = 0, hi = a.n_req;                               // row_start[lo] <= r < row_start[hi]
    if (r < a.row_start[0] || r >= a.row_start[a.n_req]) return;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.row_start[mid] <= r) lo = mid;
        else hi = mid;
    }
    const int n = a.row_start[lo + 1] - a.row_start[lo];
    const int len = min(max(a.kv_len[lo], 0), (int)min((long)a.width * a.page.d, (long)INT_MAX));
    const int keys = min(len, len - n + (r - a.row_start[lo]) + 1);
    const int kvh = h / (a.heads / a.kv_heads);
    for (int d = lane; d < a.hd; d += 64) qs[d] = a.q[r * a.ldq + (long)h * a.hd + d];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (int k0 = 0; k0 < keys; k0 += 64) {
        const int key = k0 + lane;
        float s = -INFINITY;
        long off = -1;
        if (key < keys) {
            const int j = a.page.quot(key), pg = a.table[(long)lo * a.width + j];
            if ((unsigned)pg < (unsigned)a.n_pages) {
                off = pg * a.page_stride + (long)(key - j * a.page.d) * a.pos_stride + kvh * a.head_stride;
                s = 0.0f;
                for (int d = 0; d < a.hd; d += 4) {
                    const float4 x = get4<BF16>(a.k, off + d);
                    s = fmaf(x.x, qs[d], s); s = fmaf(x.y, qs[d + 1], s);
                    s = fmaf(x.z, qs[d + 2], s); s = fmaf(x.w, qs[d + 3], s);
                }
                s *= a.scale;
            }
        }
        const float mn = fmaxf(m, group_max<64>(s)), ref = mn == -INFINITY ? 0.0f : mn;
        const float f = expf(m - ref), p = expf(s - ref);
        l = l * f + group_sum<64>(p);
        m = mn;
        ps[lane] = p;
        at[lane] = off;
        __syncthreads();
        o[0] *= f; o[1] *= f;
        for (int j = 0; j < 64; j++) {
            if (at[j] < 0) continue;
            for (int t = 0; t < 2; t++) {
                const int d = lane + 64 * t;
                if (d >= a.hd) continue;
                const float4 x = get4<BF16>(a.v, at[j] + (d & ~3));
                const float v = d & 2 ? (d & 1 ? x.w : x.z) : (d & 1 ? x.y : x.x);
                o[t] = fmaf(ps[j], v, o[t]);
            }
        }
        __syncthreads();
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int t = 0; t < 2; t++)
        if (lane + 64 * t < a.hd) a.out[r * a.ldo + (long)h * a.hd + lane + 64 * t] = o[t] * inv;
}

int check_heads(const char *who, const ptmi_pages_t *pages, int n_heads, int max_new) {
    int st = check_pages(who, pages);
    if (st) return st;
    if (n_heads < 1 || n_heads % pages->n_kv_heads || n_heads > 65535)
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
    return 16;
}

int ptmi_paged_attention_dev(const ptmi_pages_t *pages, const int *block_table, int table_width,
                             const int *row_start, const int *kv_len, int n_requests, int max_new, const float *q,
                             long ldq, float *out, long ldo, int rows, int n_heads, float scale, void *work,
                             size_t work_bytes, void *stream) {
    int st = check_heads("ptmi_paged_attention", pages, n_heads, max_new);
    if (st) return st;
    const ptmi_pages_t &p = *pages;
    if (n_requests < 0 || table_width < 1 || rows < 0 || !std::isfinite(scale))
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: n_requests=%d table_width=%d rows=%d scale=%g", n_requests,
                         table_width, rows, (double)scale);
    if (n_requests == 0 || rows == 0) return PTMI_OK;
    if (!block_table || !row_start || !kv_len || !q || !out || !work)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: NULL argument");
    const long w = (long)n_heads * p.head_dim;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15 || ldq % 4 || ldo % 4 || ldq < w || ldo < w)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: rows must be 16-byte aligned and hold %d heads (ldq=%ld ldo=%ld)",
                         n_heads, ldq, ldo);
    if (q == out) return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: out must not be q");
    const size_t need = ptmi_paged_attention_work(pages, n_heads, max_new);
    if (work_bytes < need)
        return set_error(PTMI_ERR_ARG, "ptmi_paged_attention: work holds %zu bytes, %zu needed", work_bytes, need);
    if ((st = ensure_init())) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    const AttnArgs a = {p.k, p.v, p.page_stride, p.pos_stride, p.head_stride, p.n_pages, FastDiv(p.page_size),
                        block_table, table_width, row_start, kv_len, n_requests, q, ldq, out, ldo, rows, n_heads,
                        p.n_kv_heads, p.head_dim, scale};
    hipStream_t s = stream ? (hipStream_t)stream : lib_stream();
    hipLaunchKernelGGL(p.type == PTMI_BF16 ? k_attn_simple<true> : k_attn_simple<false>, dim3(rows, n_heads), dim3(64),
                       0, s, a);
    PTMI_HIP(hipGetLastError());
    return PTMI_OK;
}

}  // extern "C"
