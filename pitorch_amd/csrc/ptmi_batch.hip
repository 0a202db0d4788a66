// Many requests through one model: the layers of a step over the new rows of
// all of them, their keys and values in one paged cache.
//
// A step is what the prompt pass is (GEMMs over rows, ptmi_prefill.hip), with
// rows of different requests at different positions: RoPE and the cache write
// are an operator of their own instead of the QKV product's epilogue, the
// attention reads pages, and only the last row of a request meets the
// classifier.  The host knows every length (it hands them in), so it refuses
// a step before anything is enqueued; the device's own bookkeeping then never
// does.
#include "ptmi_model.h"
#include "ptmi_paged.h"

#include <algorithm>
#include <cstring>
#include <vector>

namespace ptmi {

namespace {

constexpr size_t kBatchWs = (size_t)8 << 20;       // split-K partials, floats (as the prompt pass)
constexpr size_t kInts = 4, kAlign = 256;

// rope[pos][i] = (cos, sin) of the pair (2i, 2i + 1), as the decode step computes them.
__global__ __launch_bounds__(256) void k_rope_table(float2 *rope, int n, int hd) {
    const int e = blockIdx.x * 256 + threadIdx.x, half = hd / 2;
    if (e >= n * half) return;
    float c, s;
    d_rope_cs(2 * (e % half), hd, e / half, &c, &s);
    rope[e] = make_float2(c, s);
}

__global__ __launch_bounds__(256) void k_take_rows(const float4 *in, const int *row, float4 *out, int d4) {
    const float4 *src = in + (long)row[blockIdx.x] * d4;
    for (int i = threadIdx.x; i < d4; i += 256) out[(long)blockIdx.x * d4 + i] = src[i];
}

// 0, 1, .. (the pool: every page, the last on top first)
__global__ __launch_bounds__(256) void k_iota(int *p, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = n - 1 - i;
}

}  // namespace

}  // namespace ptmi

// The step's inputs as the host packs them (S requests, R rows): counts of
// new tokens [S], tokens [R], last rows [S], then temperature, top_k, top_p,
// min_p and u [S] each, of the requests with new tokens in order.
struct ptmi_batch {
    ptmi::Resident *res = nullptr;
    ptmi::Config c{};
    int S = 0, R = 0, n_pages = 0, page = 0, width = 0;
    ptmi_pages_t pages{};            // of layer 0
    size_t layer_bytes = 0;          // of one layer's keys (or values)
    char *mem = nullptr;             // device
    float *x = nullptr, *xn = nullptr, *qkv = nullptr, *ao = nullptr, *sh = nullptr, *xl = nullptr, *logits = nullptr;
    float *ws = nullptr, *rope = nullptr;
    void *work = nullptr;
    size_t work_bytes = 0;
    int *in = nullptr, *kv_len = nullptr, *pool = nullptr, *count = nullptr, *table = nullptr, *row_start = nullptr,
        *row_pos = nullptr, *row_slot = nullptr, *status = nullptr, *token = nullptr;
    int *host = nullptr;             // pinned: the inputs, then the tokens and the status
    size_t in_ints = 0;
    std::vector<int> len;            // of every request
    std::vector<int> slot;           // its row of `logits` after the last step; -1: none
    int free_pages = 0;
};

using namespace ptmi;

namespace {

int pages_for(int len, int page) { return len / page + (len % page != 0); }

// The layers over rows [0, R) of the step: logits of `n_last` rows into b->logits.
int enqueue_layers(ptmi_batch *b, int R, int max_new, int n_last, hipStream_t s) {
    const Resident *r = b->res;
    const Config &c = b->c;
    const int D = c.dim, H = c.hidden, L = c.n_layers;
    const int *tokens = b->in + b->S, *last = tokens + b->R;
    SplitK pend = {};
    int st;
    for (int l = 0; l < L; l++) {
        launch_rmsnorm_rows(b->x, r->rms_att + (long)l * D, b->xn, R, D, pend, b->x, l == 0 ? tokens : nullptr, r->emb,
                            nullptr, s);
        PTMI_HIP(hipGetLastError());
        if ((st = launch_gemm(2, b->xn, D, r->wqkv + (long)l * 3 * D * D, D, b->qkv, 3 * D, R, 3 * D, D, 0, b->ws, kBatchWs, s)))
            return st;
        ptmi_pages_t p = b->pages;
        p.k = (char *)p.k + l * b->layer_bytes;
        p.v = (char *)p.v + l * b->layer_bytes;
        if ((st = ptmi_paged_store_dev(&p, b->qkv, 3 * D, b->qkv, 3 * D, c.n_heads, b->qkv + D, b->qkv + 2 * D, 3 * D, b->row_pos,
                                       b->row_slot, R, b->rope, c.seq_len, s)))
            return st;
        if ((st = ptmi_paged_attention_dev(&p, b->table, b->width, b->row_start, b->kv_len, b->S, max_new, b->qkv, 3 * D, b->ao, D,
                                           R, c.n_heads, host_att_scale(c.head_dim), b->work, b->work_bytes, s)))
            return st;
        if ((st = launch_gemm(2, b->ao, D, r->wo + (long)l * D * D, D, b->x, D, R, D, D, 1, b->ws, kBatchWs, s, b->x, &pend)))
            return st;
        const float *w13 = r->w13 + (long)l * 2 * H * D, *rms = r->rms_ffn + (long)l * D;
        GemmEpi swiglu = {GEMM_EPI_SWIGLU, b->sh, H, 0, 0};
        swiglu.only_out = 1;                                 // (C stands for the unstored h1 and h3)
        GemmNorm nm = {};
        nm.kind = GEMM_NORM_PLAIN;
        nm.w = rms;
        nm.xn_out = b->xn;
        if (pend.splits == 0 && gemm_norm_fusable(R, 2 * H, D, b->x, D, w13, D, swiglu.kind, nm)) {
            if ((st = launch_gemm(2, b->x, D, w13, D, b->sh, 2 * H, R, 2 * H, D, 0, nullptr, 0, s, nullptr, nullptr, &swiglu, &nm)))
                return st;
        } else {
            launch_rmsnorm_rows(b->x, rms, b->xn, R, D, pend, b->x, nullptr, r->emb, nullptr, s);
            PTMI_HIP(hipGetLastError());
            if ((st = launch_gemm(2, b->xn, D, w13, D, b->sh, 2 * H, R, 2 * H, D, 0, b->ws, kBatchWs, s, nullptr, nullptr, &swiglu)))
                return st;
        }
        if ((st = launch_gemm(2, b->sh, H, r->w2 + (long)l * D * H, H, b->x, D, R, D, H, 1, b->ws, kBatchWs, s, b->x, &pend)))
            return st;
    }
    launch_rmsnorm_rows(b->x, r->rms_final, b->xn, R, D, pend, b->x, nullptr, r->emb, nullptr, s);
    const float *rows = b->xn;
    if (n_last < R) {                                        // (else every row is a last one)
        hipLaunchKernelGGL(k_take_rows, dim3(n_last), dim3(256), 0, s, (const float4 *)b->xn, last, (float4 *)b->xl, D / 4);
        rows = b->xl;
    }
    PTMI_HIP(hipGetLastError());
    return launch_gemm(2, rows, D, r->wcls, D, b->logits, c.vocab, n_last, c.vocab, D, 0, b->ws, kBatchWs, s);
}

}  // namespace

extern "C" {

int ptmi_batch_create(ptmi_model_t *m, int max_requests, int max_rows, int n_pages, int page_size, int cache_type,
                      ptmi_batch_t **out) {
    if (!m || !out) return set_error(PTMI_ERR_ARG, "ptmi_batch_create: NULL argument");
    *out = nullptr;
    if (max_requests < 1 || max_requests > 8192 || max_rows < 1 || max_rows > (1 << 20) || n_pages < 1 || page_size < 1 ||
        (long long)n_pages * page_size > INT32_MAX || (cache_type != PTMI_F32 && cache_type != PTMI_BF16))
        return set_error(PTMI_ERR_ARG, "ptmi_batch_create: max_requests=%d max_rows=%d n_pages=%d page_size=%d cache_type=%d",
                         max_requests, max_rows, n_pages, page_size, cache_type);
    if (m->c.vocab > kSampleVocab)
        return set_error(PTMI_ERR_ARG, "ptmi_batch_create: vocab=%d (at most %d)", m->c.vocab, kSampleVocab);
    int st = ensure_init();
    if (st) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    ptmi_batch *b = new ptmi_batch();
    b->res = m->res;
    b->res->model_holds++;           // it holds the weights itself, and needs neither the model nor the blob any more
    b->c = m->c;
    const Config &c = b->c;
    b->S = max_requests;
    b->R = max_rows;
    b->n_pages = n_pages;
    b->page = page_size;
    b->width = pages_for(c.seq_len, page_size);
    const size_t S = max_requests, R = max_rows, D = c.dim, H = c.hidden, V = c.vocab, hd = c.head_dim, f = sizeof(float);
    const long row = (long)D;                                // (n_kv_heads == n_heads: the model has seen to it)
    b->pages = {nullptr, nullptr, cache_type, n_pages, page_size, c.n_heads, c.head_dim, row * page_size, row, (long)hd};
    b->layer_bytes = (size_t)n_pages * page_size * D * (cache_type == PTMI_BF16 ? 2 : 4);
    b->layer_bytes = (b->layer_bytes + kAlign - 1) / kAlign * kAlign;
    char align_to[16] __attribute__((aligned(16)));          // (a cache that stands somewhere, for the size alone)
    b->pages.k = b->pages.v = align_to;
    b->work_bytes = ptmi_paged_attention_work(&b->pages, c.n_heads, 0);
    b->in_ints = S + R + S + 5 * S;
    struct Piece { void **at; size_t bytes; };
    const Piece pieces[] = {
        {&b->pages.k, b->layer_bytes * c.n_layers}, {&b->pages.v, b->layer_bytes * c.n_layers},
        {(void **)&b->x, R * D * f}, {(void **)&b->xn, R * D * f}, {(void **)&b->qkv, R * 3 * D * f}, {(void **)&b->ao, R * D * f},
        {(void **)&b->sh, R * H * f}, {(void **)&b->xl, S * D * f}, {(void **)&b->logits, S * V * f}, {(void **)&b->ws, kBatchWs * f},
        {(void **)&b->rope, (size_t)c.seq_len * hd * f}, {&b->work, b->work_bytes}, {(void **)&b->in, b->in_ints * kInts},
        {(void **)&b->kv_len, S * kInts}, {(void **)&b->pool, (size_t)n_pages * kInts}, {(void **)&b->count, kInts},
        {(void **)&b->table, S * b->width * kInts}, {(void **)&b->row_start, (S + 1) * kInts}, {(void **)&b->row_pos, R * kInts},
        {(void **)&b->row_slot, R * kInts}, {(void **)&b->status, kInts}, {(void **)&b->token, S * kInts}};
    size_t total = 0;
    for (const Piece &p : pieces) total += (p.bytes + kAlign - 1) / kAlign * kAlign;
    hipError_t e = b->work_bytes ? hipMalloc(&b->mem, total) : hipErrorInvalidValue;
    if (e == hipSuccess) e = hipHostMalloc(&b->host, (b->in_ints + S + 1) * kInts, hipHostMallocDefault);
    hipStream_t s = lib_stream();
    if (e == hipSuccess) {
        size_t o = 0;
        for (const Piece &p : pieces) { *p.at = b->mem + o; o += (p.bytes + kAlign - 1) / kAlign * kAlign; }
        e = hipMemsetAsync(b->kv_len, 0, S * kInts, s);
        if (e == hipSuccess) e = hipMemsetAsync(b->table, 0xFF, S * b->width * kInts, s);
        if (e == hipSuccess) e = hipMemcpyAsync(b->count, &n_pages, kInts, hipMemcpyHostToDevice, s);
        hipLaunchKernelGGL(k_iota, dim3((n_pages + 255) / 256), dim3(256), 0, s, b->pool, n_pages);
        const int pairs = c.seq_len * (int)(hd / 2);
        hipLaunchKernelGGL(k_rope_table, dim3((pairs + 255) / 256), dim3(256), 0, s, (float2 *)b->rope, c.seq_len, (int)hd);
        if (e == hipSuccess) e = hipGetLastError();
        if (e == hipSuccess) e = hipStreamSynchronize(s);
    }
    if (e != hipSuccess) {
        st = hip_check(e, "ptmi_batch_create");
        ptmi_batch_destroy(b);
        return st;
    }
    b->len.assign(S, 0);
    b->slot.assign(S, -1);
    b->free_pages = n_pages;
    *out = b;
    return PTMI_OK;
}

void ptmi_batch_destroy(ptmi_batch_t *b) {
    if (!b) return;
    (void)hipStreamSynchronize(lib_stream());
    if (b->mem) (void)hipFree(b->mem);
    if (b->host) (void)hipHostFree(b->host);
    release_blob(b->res);
    delete b;
}

int ptmi_batch_length(const ptmi_batch_t *b, int request) {
    return b && request >= 0 && request < b->S ? b->len[request] : -1;
}

int ptmi_batch_free_pages(const ptmi_batch_t *b) { return b ? b->free_pages : -1; }

int ptmi_batch_step(ptmi_batch_t *b, const int *n_new, const int *tokens, const ptmi_sampling_t *sampling, int *next) {
    if (!b || !n_new) return set_error(PTMI_ERR_ARG, "ptmi_batch_step: NULL argument");
    const Config &c = b->c;
    long long rows = 0, need = 0, back = 0;
    int max_new = 0, active = 0;
    for (int i = 0; i < b->S; i++) {
        const int n = n_new[i], len = b->len[i];
        if (n < -1) return set_error(PTMI_ERR_ARG, "ptmi_batch_step: n_new[%d]=%d", i, n);
        if (n < 0) back += pages_for(len, b->page);
        if (n <= 0) continue;
        if (n > c.seq_len - len)
            return set_error(PTMI_ERR_STATE, "ptmi_batch_step: request %d has %d positions and %d new: seq_len is %d", i, len, n,
                             c.seq_len);
        rows += n;
        need += pages_for(len + n, b->page) - pages_for(len, b->page);
        max_new = std::max(max_new, n);
        active++;
    }
    if (rows > b->R) return set_error(PTMI_ERR_STATE, "ptmi_batch_step: %lld new tokens, room for %d", rows, b->R);
    if (need > b->free_pages + back)
        return set_error(PTMI_ERR_STATE, "ptmi_batch_step: %lld pages needed, %lld free", need, b->free_pages + back);
    if (rows && !tokens) return set_error(PTMI_ERR_ARG, "ptmi_batch_step: NULL tokens");
    for (long long i = 0; i < rows; i++)
        if (tokens[i] < 0 || tokens[i] >= c.vocab)
            return set_error(PTMI_ERR_ARG, "ptmi_batch_step: token %d outside [0, %d)", tokens[i], c.vocab);
    int st = ensure_init();
    if (st) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    // pack the inputs
    const size_t S = b->S, R = b->R;
    int *h = b->host, *last = h + S + R, *par = last + S;
    memcpy(h, n_new, S * kInts);
    if (rows) memcpy(h + S, tokens, rows * kInts);
    static const ptmi_sampling_t none = {};
    const ptmi_sampling_t &p = sampling ? *sampling : none;
    const void *arrays[5] = {p.temperature, p.top_k, p.top_p, p.min_p, p.u};
    int row = 0, k = 0;
    for (int i = 0; i < b->S; i++) {
        if (n_new[i] <= 0) continue;
        row += n_new[i];
        last[k] = row - 1;
        for (int j = 0; j < 5; j++)
            if (arrays[j]) memcpy(par + j * S + k, (const char *)arrays[j] + i * kInts, kInts);
        if (!arrays[0]) par[k] = 0;                          // no temperature: greedy
        k++;
    }
    hipStream_t s = lib_stream();
    PTMI_HIP(hipMemcpyAsync(b->in, h, b->in_ints * kInts, hipMemcpyHostToDevice, s));
    if ((st = ptmi_paged_plan_dev(b->kv_len, b->in, b->S, b->pool, b->count, b->n_pages, b->page, b->table, b->width, b->kv_len,
                                  b->count, b->row_start, b->row_pos, b->row_slot, b->R, b->status, s)))
        return st;
    int *got = h + b->in_ints;
    if (rows) {
        if ((st = enqueue_layers(b, (int)rows, max_new, active, s))) return st;
        const int *dp = b->in + S + R + S;
        const float *fp = (const float *)dp;
        if ((st = ptmi_sample_dev(b->logits, c.vocab, active, c.vocab, fp, arrays[1] ? dp + S : nullptr,
                                  arrays[2] ? fp + 2 * S : nullptr, arrays[3] ? fp + 3 * S : nullptr,
                                  arrays[4] ? fp + 4 * S : nullptr, b->token, s)))
            return st;
        PTMI_HIP(hipMemcpyAsync(got, b->token, active * kInts, hipMemcpyDeviceToHost, s));
    }
    PTMI_HIP(hipMemcpyAsync(got + S, b->status, kInts, hipMemcpyDeviceToHost, s));
    PTMI_HIP(hipStreamSynchronize(s));
    if (got[S]) return set_error(PTMI_ERR_STATE, "ptmi_batch_step: the device refused the step (%d)", got[S]);
    k = 0;
    for (int i = 0; i < b->S; i++) {
        if (n_new[i] < 0) b->len[i] = 0;
        else b->len[i] += n_new[i];
        b->slot[i] = n_new[i] > 0 ? k : -1;
        if (next) next[i] = n_new[i] > 0 ? got[k] : -1;
        if (n_new[i] > 0) k++;
    }
    b->free_pages += (int)(back - need);
    return PTMI_OK;
}

int ptmi_batch_logits(ptmi_batch_t *b, int request, float *out) {
    if (!b || !out || request < 0 || request >= b->S) return set_error(PTMI_ERR_ARG, "ptmi_batch_logits: request %d", request);
    if (b->slot[request] < 0) return set_error(PTMI_ERR_STATE, "ptmi_batch_logits: request %d had no tokens in the last step", request);
    hipStream_t s = lib_stream();
    PTMI_HIP(hipMemcpyAsync(out, b->logits + (size_t)b->slot[request] * b->c.vocab, (size_t)b->c.vocab * sizeof(float),
                            hipMemcpyDeviceToHost, s));
    PTMI_HIP(hipStreamSynchronize(s));
    return PTMI_OK;
}

}  // extern "C"
