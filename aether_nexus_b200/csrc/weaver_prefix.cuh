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

// Own tokens that query j of ntok sees: all, or with the causal rule len -
// ntok + 1 + j of them.
__device__ __forceinline__ uint32_t suffix_limit(bool causal, uint32_t len, uint32_t ntok, uint32_t j) {
    if (!causal) return len;
    const int64_t lim = static_cast<int64_t>(len) - ntok + 1 + j;
    return lim > 0 ? static_cast<uint32_t>(lim) : 0u;
}

// Programmatic dependent launch: let the next kernel of the stream start / wait
// until the one before has completed and its writes are visible.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_prerequisites() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... Args>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, bool after, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = after ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// 1 / l; 0 for a row that saw nothing; NaN stays NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l); }

}  // namespace weaver
