// weaver_rope.cu — position rotation of query and key heads, with an optional
// RMS norm of each head first, and the append of keys and values into the
// paged hot pool that the decode step reads.  The reference rotates and
// appends in separate kernels of its full loop (ops.metal:107-160,
// inference.rs:504-562); the hot pool itself it only ever fills from the host.
//
//   n = x * rsqrt(mean(x^2) + eps) * w                 (only with a weight)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * f_i
//
// for pair i = (i, i + r/2) (half) or (2i, 2i+1) (interleaved) of the first r
// elements; the rest passes through.  All arithmetic in fp32, one rounding at
// the store.
//
// The angle: positions reach millions, where a 32-bit product position * f
// has lost the angle's leading digits.  f_i is kept as a 64-bit fixed-point
// fraction of a turn, so the low 64 bits of the integer product position *
// f_i ARE the angle modulo one turn, exact to position * 2^-64; its top 32
// bits, as a signed fraction in [-1/2, 1/2), go to sincospif.  No table, no
// range reduction.
//
// Bound by HBM: every element is read and written once.  A token's
// cosines and sines are computed once per CTA into shared memory and shared
// by all its heads (r/2 sincospif against (Hq + Hkv) * d elements).  D/16
// neighbouring threads own one head: each holds the two 16-byte chunks whose
// elements pair up, so the norm's sum is a shuffle over D/16 lanes and every
// access is 16 bytes wide.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "weaver_device.cuh"
#include "weaver_internal.hpp"

namespace weaver {
namespace {

constexpr uint32_t kRopeThreads = 256;
constexpr uint32_t kRopeMaxTokens = 4;  // tokens per CTA at most (shared-memory table)

__device__ __forceinline__ void unpack8(const uint4 raw, float f[8], __half) { h8_to_f8(raw, f); }
__device__ __forceinline__ void unpack8(const uint4 raw, float f[8], __nv_bfloat16) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __bfloat1622float2(h[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
__device__ __forceinline__ uint4 pack8(const float f[8], __half) {
    uint4 raw;
    __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    return raw;
}
__device__ __forceinline__ uint4 pack8(const float f[8], __nv_bfloat16) {
    uint4 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return raw;
}

// In: the activations' type, Out: the results' (the input's for the rotation
// alone, f16, the pool's type, for the append).
template <int D, typename In, typename Out, bool kAppend>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr uint32_t kLanes = D / 16;                   // threads per head
    constexpr uint32_t kGroups = kRopeThreads / kLanes;   // heads in flight per CTA
    constexpr uint32_t kUnroll = 2;                       // heads whose loads a thread issues together
    __shared__ float2 cs[kRopeMaxTokens][D / 2];

    const uint32_t tid = threadIdx.x, j = tid % kLanes, grp = tid / kLanes;
    const uint32_t t0 = blockIdx.x * a.tokens_per_cta;
    const uint32_t nt = min(a.tokens_per_cta, a.T - t0);
    const uint32_t U = a.Hq + a.Hkv + (kAppend && a.v ? a.Hkv : 0u);  // heads per token
    const uint32_t units = nt * U;
    const uint32_t nr = a.rot / 16, half = a.rot / 2;
    const bool turns = j < nr;
    // this thread's two chunks of 8 elements
    const uint32_t c0 = turns ? j : 2 * nr + 2 * (j - nr);
    const uint32_t c1 = turns ? j + nr : c0 + 1;

    struct Unit {
        uint4 lo, hi;
        uint32_t tok, head;  // token of the CTA; head in [q heads | k heads | v heads]
        int64_t slot;
        bool live;
    };
    auto fetch = [&](uint32_t u) {
        Unit x;
        x.live = u < units;
        x.tok = x.live ? u / U : 0u;
        x.head = x.live ? u - x.tok * U : 0u;
        x.slot = 0;
        x.lo = x.hi = make_uint4(0, 0, 0, 0);
        if (!x.live) return x;
        const uint64_t t = t0 + x.tok;
        if (kAppend) {
            x.slot = a.slots[t];
            // padding (negative) or beyond the pool: the token is skipped
            x.live = x.slot >= 0 && x.slot < static_cast<int64_t>(a.pool_rows);
            if (!x.live) {
                if (x.slot >= 0 && x.head == 0 && j == 0) atomicOr(a.bad, 1u);
                return x;
            }
        }
        const In* src;
        if (x.head < a.Hq) {
            src = static_cast<const In*>(a.q) + t * a.q_ts + x.head * a.q_hs;
        } else if (x.head < a.Hq + a.Hkv) {
            src = static_cast<const In*>(a.k) + t * a.k_ts + (x.head - a.Hq) * a.k_hs;
        } else {
            src = static_cast<const In*>(a.v) + t * a.v_ts + (x.head - a.Hq - a.Hkv) * a.v_hs;
        }
        x.lo = *reinterpret_cast<const uint4*>(src + c0 * 8);
        x.hi = *reinterpret_cast<const uint4*>(src + c1 * 8);
        return x;
    };

    // the first heads' loads are in flight while the table is computed
    Unit x[kUnroll];
#pragma unroll
    for (uint32_t i = 0; i < kUnroll; ++i) x[i] = fetch(grp + i * kGroups);
    for (uint32_t e = tid; e < nt * half; e += kRopeThreads) {
        const uint32_t t = e / half, i = e - t * half;
        const uint64_t turn = static_cast<uint64_t>(static_cast<int64_t>(a.positions[t0 + t])) * a.freq[i];
        float s, c;
        sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * 0x1p-31f, &s, &c);
        cs[t][i] = make_float2(c * a.amplitude, s * a.amplitude);
    }
    __syncthreads();

    for (uint32_t u = grp; u < units + grp; u += kGroups * kUnroll) {  // uniform trip count per warp
#pragma unroll
        for (uint32_t i = 0; i < kUnroll; ++i) {
            const Unit cur = x[i];
            x[i] = fetch(u + (kUnroll + i) * kGroups);
            float lo[8], hi[8];
            unpack8(cur.lo, lo, In());
            unpack8(cur.hi, hi, In());
            const bool is_q = cur.head < a.Hq, is_v = cur.head >= a.Hq + a.Hkv;
            const In* w = static_cast<const In*>(is_q ? a.q_weight : is_v ? nullptr : a.k_weight);
            if (a.q_weight || a.k_weight) {  // uniform over the launch: every lane takes the shuffles
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
                for (uint32_t o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (w) {
                    const float r = rsqrtf(ss * (1.0f / D) + a.eps);
                    float wl[8], wh[8];
                    unpack8(*reinterpret_cast<const uint4*>(w + c0 * 8), wl, In());
                    unpack8(*reinterpret_cast<const uint4*>(w + c1 * 8), wh, In());
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        lo[e] *= r * wl[e];
                        hi[e] *= r * wh[e];
                    }
                }
            }
            if (!cur.live) continue;
            if (turns && !is_v) {
                const float2* tab = cs[cur.tok];
                if (a.interleaved) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 p = tab[4 * c0 + e], r = tab[4 * c1 + e];
                        const float la = lo[2 * e], lb = lo[2 * e + 1], ha = hi[2 * e], hb = hi[2 * e + 1];
                        lo[2 * e] = la * p.x - lb * p.y;
                        lo[2 * e + 1] = lb * p.x + la * p.y;
                        hi[2 * e] = ha * r.x - hb * r.y;
                        hi[2 * e + 1] = hb * r.x + ha * r.y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 p = tab[8 * j + e];
                        const float la = lo[e], ha = hi[e];
                        lo[e] = la * p.x - ha * p.y;
                        hi[e] = ha * p.x + la * p.y;
                    }
                }
            }
            const uint64_t t = t0 + cur.tok;
            Out* dst;
            if (is_q) {
                dst = static_cast<Out*>(a.q_out) + t * a.qo_ts + cur.head * a.qo_hs;
            } else if (kAppend) {
                const uint32_t g = cur.head - a.Hq - (is_v ? a.Hkv : 0u);
                dst = static_cast<Out*>(is_v ? a.hot_v : a.hot_k) +
                      (static_cast<uint64_t>(cur.slot) * a.Hkv + g) * D;
            } else {
                dst = static_cast<Out*>(a.k_out) + t * a.ko_ts + (cur.head - a.Hq) * a.ko_hs;
            }
            *reinterpret_cast<uint4*>(dst + c0 * 8) = pack8(lo, Out());
            *reinterpret_cast<uint4*>(dst + c1 * 8) = pack8(hi, Out());
        }
    }
}

template <typename In, typename Out, bool kAppend>
cudaError_t launch_typed(const RopeArgs& a, cudaStream_t s) {
    const uint32_t grid = (a.T + a.tokens_per_cta - 1) / a.tokens_per_cta;
    if (a.D == 128)
        rope_kernel<128, In, Out, kAppend><<<grid, kRopeThreads, 0, s>>>(a);
    else
        rope_kernel<64, In, Out, kAppend><<<grid, kRopeThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope(RopeArgs a, bool append, cudaStream_t s) {
    if (a.T == 0) return cudaSuccess;
    a.tokens_per_cta = 1;
    if (append)
        return a.bf16 ? launch_typed<__nv_bfloat16, __half, true>(a, s) : launch_typed<__half, __half, true>(a, s);
    return a.bf16 ? launch_typed<__nv_bfloat16, __nv_bfloat16, false>(a, s) : launch_typed<__half, __half, false>(a, s);
}

}  // namespace weaver
