// Sampling of one token per row of logits.
//
// A row's order is that of its keys: the logits' bits made monotone, larger
// logits first, equal ones by index.  Every filter keeps a beginning of that
// order, so what stays is known by one (key, number of that key's logits):
// found by rounds over the key's bits, each a histogram of what shares the
// bits found so far, of counts for top_k and of weights for top_p.  Weights
// are whole multiples of 2^-44 in 64 bits: their sums are exact and the same
// in any order, so shared-memory atomics leave the result unchanged.
#include "ptmi_paged.h"

namespace ptmi {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;

struct SampleArgs {
    const float *logits; long ld;
    int vocab;
    const float *temperature; const int *top_k; const float *top_p, *min_p, *u;
    int *token;
};

// Larger key = larger logit; 0 for NaN and -infinity (never chosen).
__device__ __forceinline__ unsigned key_of(float x) {
    if (!(x > -INFINITY)) return 0u;
    const unsigned b = __float_as_uint(x + 0.0f);           // -0 as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

struct Row { float top; double inv_t; };

__device__ __forceinline__ double weight(const Row &r, float x) {
    if (x == r.top) return 1.0;
    return exp(((double)x - (double)r.top) * r.inv_t);
}
__device__ __forceinline__ u64 fixed(double w) { return (u64)(w * 17592186044416.0 + 0.5); }   // 2^44

__global__ __launch_bounds__(kThreads) void k_sample_simple(SampleArgs a) {
    __shared__ u64 hist[256], part[kThreads];
    __shared__ unsigned red_k;
    __shared__ int red_i, s_bin;
    __shared__ u64 s_before;
    const int t = threadIdx.x, V = a.vocab;
    const float *x = a.logits + (long)blockIdx.x * a.ld;
    auto row_f = [&](const float *p, float off) { return p ? p[blockIdx.x] : off; };
    // the maximum and its first index
    unsigned bk = 0;
    for (int i = t; i < V; i += kThreads) bk = max(bk, key_of(x[i]));
    if (t == 0) { red_k = 0; red_i = V; }
    __syncthreads();
    atomicMax(&red_k, bk);
    __syncthreads();
    const unsigned kmax = red_k;
    const float temp = row_f(a.temperature, 1.0f);
    if (kmax == 0) { if (t == 0) a.token[blockIdx.x] = -1; return; }
    if (!(temp > 0.0f)) {
        for (int i = t; i < V; i += kThreads)
            if (key_of(x[i]) == kmax) { atomicMin(&red_i, i); break; }
        __syncthreads();
        if (t == 0) a.token[blockIdx.x] = red_i;
        return;
    }
    const Row row = {logit_of(kmax), 1.0 / (double)temp};
    int top_k = a.top_k ? a.top_k[blockIdx.x] : 0;
    const float top_p = row_f(a.top_p, 1.0f);
    float mp = row_f(a.min_p, 0.0f);
    const double min_p = mp > 1.0f ? 1.0 : mp > 0.0f ? (double)mp : 0.0;
    float uf = row_f(a.u, 0.0f);
    uf = uf > 0.0f ? fminf(uf, 0.99999994f) : 0.0f;
    // kept: key > tk, and the first tn (by index) of key == tk
    unsigned tk = 1;
    int tn = V;
    auto kept = [&](unsigned k) { return k >= tk; };
    // the first key, from the largest down, at which the running sum of `measure` exceeds `target`:
    // its key, and the sum before it
    auto find = [&](auto measure, u64 target, unsigned *key, u64 *before) {
        unsigned prefix = 0;
        u64 sum = 0;
        for (int sh = 24; sh >= 0; sh -= 8) {
            for (int b = t; b < 256; b += kThreads) hist[b] = 0;
            __syncthreads();
            for (int i = t; i < V; i += kThreads) {
                const unsigned k = key_of(x[i]);
                if (k && kept(k) && (sh == 24 || k >> (sh + 8) == prefix)) {
                    const u64 w = measure(i, k);
                    if (w) atomicAdd(&hist[k >> sh & 255], w);
                }
            }
            __syncthreads();
            if (t == 0) {
                int b = 255;
                u64 c = sum;
                while (b > 0 && c + hist[b] <= target) c += hist[b--];
                s_bin = b;
                s_before = c;
            }
            __syncthreads();
            prefix = prefix << 8 | (unsigned)s_bin;
            sum = s_before;
            __syncthreads();
        }
        *key = prefix;
        *before = sum;
    };
    if (top_k > 0 && top_k < V) {
        unsigned key;
        u64 before;
        find([&](int, unsigned) -> u64 { return 1; }, (u64)(top_k - 1), &key, &before);
        if (key > 0) { tk = key; tn = top_k - (int)before; }
    }
    // index order: the weight of i as it stays (ties of tk only the first tn)
    auto sum_all = [&](u64 w) -> u64 {                      // over the block
        part[t] = w;
        __syncthreads();
        for (int d = kThreads / 2; d > 0; d >>= 1) {
            if (t < d) part[t] += part[t + d];
            __syncthreads();
        }
        const u64 v = part[0];
        __syncthreads();
        return v;
    };
    auto mass = [&](unsigned k) -> u64 {
        if (!k) return 0;
        const double w = weight(row, logit_of(k));
        return w >= min_p ? fixed(w) : 0;
    };
    // ties of tk beyond tn do not count: there are `ties` of them in all
    auto count_ties = [&]() -> int {
        u64 c = 0;
        for (int i = t; i < V; i += kThreads) c += key_of(x[i]) == tk;
        return (int)sum_all(c);
    };
    if (top_p < 1.0f || !(top_p == top_p)) {
        const u64 wt = mass(tk);
        u64 w = 0;
        for (int i = t; i < V; i += kThreads) {
            const unsigned k = key_of(x[i]);
            if (k > tk) w += mass(k);
        }
        const int ties = min(count_ties(), tn);
        const u64 total = sum_all(w) + wt * ties;
        // stays: sum before it < p * total; the last of them is where the running sum reaches ceil(p * total)
        const double lim = top_p > 0.0f ? (double)top_p * (double)total : 0.0;
        u64 need = (u64)lim;
        if ((double)need < lim) need++;                     // before < lim  <=>  before < need
        if (need < 1) need = 1;
        unsigned key;
        u64 before;
        find([&](int, unsigned k) -> u64 { return mass(k); }, need - 1, &key, &before);
        if (key > tk) {
            tk = key;
            tn = V;
        }
        if (key >= tk) {
            const u64 w1 = mass(tk);
            const u64 n = w1 ? (need - before + w1 - 1) / w1 : 1;
            tn = (int)min((u64)tn, max(n, (u64)1));
        }
    }
    // the draw, in the order of indices: thread t takes a run of indices
    const int run = (V + kThreads - 1) / kThreads, i0 = min(t * run, V), i1 = min(i0 + run, V);
    u64 ties = 0;
    for (int i = i0; i < i1; i++) ties += key_of(x[i]) == tk;
    part[t] = ties;
    __syncthreads();
    u64 seen = 0;
    for (int j = 0; j < t; j++) seen += part[j];
    __syncthreads();
    u64 w = 0, c = seen;
    for (int i = i0; i < i1; i++) {
        const unsigned k = key_of(x[i]);
        if (k > tk || (k == tk && c++ < (u64)tn)) w += mass(k);
    }
    part[t] = w;
    __syncthreads();
    u64 before = 0, total = 0;
    for (int j = 0; j < kThreads; j++) {
        if (j == t) before = total;
        total += part[j];
    }
    const u64 target = (u64)((double)uf * (double)total);
    if (before <= target && target < before + w) {
        c = seen;
        for (int i = i0; i < i1; i++) {
            const unsigned k = key_of(x[i]);
            if (k > tk || (k == tk && c++ < (u64)tn)) before += mass(k);
            if (before > target) { a.token[blockIdx.x] = i; break; }
        }
    }
}

}  // namespace

}  // namespace ptmi

using namespace ptmi;

extern "C" int ptmi_sample_dev(const float *logits, long ld, int rows, int vocab, const float *temperature,
                               const int *top_k, const float *top_p, const float *min_p, const float *u, int *token,
                               void *stream) {
    if (rows < 0 || vocab < 1 || vocab > (1 << 18) || ld < vocab)
        return set_error(PTMI_ERR_ARG, "ptmi_sample: rows=%d vocab=%d (1..262144) ld=%ld", rows, vocab, ld);
    if (rows == 0) return PTMI_OK;
    if (!logits || !token) return set_error(PTMI_ERR_ARG, "ptmi_sample: NULL argument");
    if ((uintptr_t)logits & 3) return set_error(PTMI_ERR_ARG, "ptmi_sample: logits not 4-byte aligned");
    int st = ensure_init();
    if (st) return st;
    DeviceScope dev;
    if ((st = dev.enter())) return st;
    const SampleArgs a = {logits, ld, vocab, temperature, top_k, top_p, min_p, u, token};
    hipLaunchKernelGGL(k_sample_simple, dim3(rows), dim3(kThreads), 0, stream ? (hipStream_t)stream : lib_stream(), a);
    PTMI_HIP(hipGetLastError());
    return PTMI_OK;
}
