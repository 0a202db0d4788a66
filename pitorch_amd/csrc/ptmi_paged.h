// Shared by the units that serve many requests over one paged cache.
#pragma once

#include "ptmi_internal.h"

namespace ptmi {

// x / d for 0 <= x < 2^31 and 1 <= d < 2^31 by one multiplication: with
// m = floor(2^(31+s)/d) + 1 and 2^s >= d, x*m/2^(31+s) lies above x/d by
// x*(m*d - 2^(31+s))/(d*2^(31+s)) <= x/2^(31+s) < 1/d, so its floor is
// floor(x/d).
struct FastDiv {
    unsigned long long m;
    int sh, d;
    FastDiv() = default;
    explicit FastDiv(int div) : sh(31), d(div) {
        while ((1ll << (sh - 31)) < div) sh++;
        m = (1ull << sh) / (unsigned)div + 1;
    }
    __device__ __forceinline__ int quot(int x) const { return (int)((unsigned long long)(unsigned)x * m >> sh); }
};

// The calls of one process may come with another GPU current than the
// library's; this makes the library's current for the scope.
struct DeviceScope {
    int before = -1;
    int enter() {
        int cur = 0;
        PTMI_HIP(hipGetDevice(&cur));
        if (cur != lib_device()) {
            PTMI_HIP(hipSetDevice(lib_device()));
            before = cur;
        }
        return PTMI_OK;
    }
    ~DeviceScope() { if (before >= 0) (void)hipSetDevice(before); }
};

constexpr int kSampleVocab = (1 << 18) - 4;                 // the longest row of logits a token is sampled from

// PTMI_OK if the description of a paged cache is sound (host arithmetic).
int check_pages(const char *who, const ptmi_pages_t *pages);

}  // namespace ptmi
