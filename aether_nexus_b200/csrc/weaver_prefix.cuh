// weaver_prefix.cuh — lengths and causal limits of the shared-prefix attention's
// page lists, the same for all of its kernels.
#pragma once

#include "weaver_device.cuh"

namespace weaver {

// Tokens of `blocks` pages: the length on the device, at most the pages'
// capacity (a larger one is reported and cut).
__device__ __forceinline__ uint32_t page_len(const uint32_t* lens, uint32_t i, uint32_t blocks, uint32_t* status, bool report) {
    const uint32_t cap = blocks * kBlock;
    if (!lens || !blocks) return cap;
    const uint32_t n = lens[i];
    if (n > cap && report) atomicOr(status, DEVERR_REF_RANGE);
    return min(n, cap);
}
__device__ __forceinline__ uint32_t prefix_len(const PrefixArgs& a, const PrefixList& L, bool report) {
    return page_len(a.prefix_lens, L.pre_len, L.pre_blocks, a.status, report);
}
__device__ __forceinline__ uint32_t suffix_len(const PrefixArgs& a, const PrefixList& L, bool report) {
    return page_len(a.suffix_lens, L.suf_len, L.suf_blocks, a.status, report);
}

// Own tokens that query j of the list's ntok sees: all, or with the causal
// rule len - ntok + 1 + j of them.
__device__ __forceinline__ uint32_t suffix_limit(const PrefixList& L, uint32_t len, uint32_t j) {
    if (!L.causal) return len;
    const int64_t lim = static_cast<int64_t>(len) - L.ntok + 1 + j;
    return lim > 0 ? static_cast<uint32_t>(lim) : 0u;
}

}  // namespace weaver
