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
// Bound by HBM: every element is read and written once.  D/16 neighbouring
// threads own one head: each holds the two 16-byte chunks whose elements pair
// up, so the norm's sum is a shuffle over D/16 lanes and every access is 16
// bytes wide.  A warp stays with one token (1 to 8 warps share it): the token's
// cosines and sines are computed once, two pairs a lane, and handed round by
// shuffle into the registers of the lanes that use them, for all heads; so are
// the norms' weights.  With the table in shared memory and heads of several
// tokens mixed in a warp the kernel was bound by its instructions.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "weaver_device.cuh"
#include "weaver_internal.hpp"

namespace weaver {
namespace {

constexpr uint32_t kRopeThreads = 256;
constexpr uint32_t kRopeWarps = kRopeThreads / 32;

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
// Resident CTAs per SM: the append of a long prompt ran 85 us with three and 79
// with four (at 64 registers), the normed rotation of one 68 and 70.
template <int D, typename In, typename Out, bool kAppend>
__global__ void __launch_bounds__(kRopeThreads, kAppend ? 4 : 3) rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr uint32_t kLanes = D / 16;       // threads per head
    constexpr uint32_t kHeads = 32 / kLanes;  // heads per warp at a time
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t wpt = a.warps_per_token;
    const uint64_t t = static_cast<uint64_t>(blockIdx.x) * (kRopeWarps / wpt) + warp / wpt;
    if (t >= a.T) return;
    const uint32_t j = lane % kLanes, first = (warp % wpt) * kHeads + lane / kLanes, step = wpt * kHeads;
    int64_t slot = 0;
    if (kAppend) {
        slot = a.slots[t];
        if (slot < 0) return;  // padding
        if (slot >= static_cast<int64_t>(a.pool_rows)) {
            if (warp % wpt == 0 && lane == 0) atomicOr(a.bad, 1u);
            return;
        }
    }
    const uint32_t nr = a.rot / 16;
    const bool turns = j < nr;
    // this thread's two chunks of 8 elements
    const uint32_t c0 = turns ? j : 2 * nr + 2 * (j - nr);
    const uint32_t c1 = turns ? j + nr : c0 + 1;

    struct Raw {
        uint4 lo, hi;
    };
    auto load = [&](const In* src, bool in) {
        Raw x{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (in) {
            x.lo = *reinterpret_cast<const uint4*>(src + c0 * 8);
            x.hi = *reinterpret_cast<const uint4*>(src + c1 * 8);
        }
        return x;
    };
    const uint32_t n_kv = a.Hkv + (kAppend && a.v ? a.Hkv : 0u);  // key heads, then value heads
    auto load_q = [&](uint32_t h) { return load(static_cast<const In*>(a.q) + t * a.q_ts + h * a.q_hs, h < a.Hq); };
    auto load_kv = [&](uint32_t h) {
        const bool val = kAppend && h >= a.Hkv;
        const In* src = val ? static_cast<const In*>(a.v) + t * a.v_ts + (h - a.Hkv) * a.v_hs
                            : static_cast<const In*>(a.k) + t * a.k_ts + h * a.k_hs;
        return load(src, h < n_kv);
    };
    // the first heads are on their way while the angles are computed
    Raw q = load_q(first), q2 = q, kv = load_kv(first);
    if (!kAppend) q2 = load_q(first + step);

    // pairs 2 * lane, 2 * lane + 1 (the last lanes have none where rot < 128)
    const uint64_t pos = static_cast<uint64_t>(static_cast<int64_t>(a.positions[t]));
    float2 mine[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const uint32_t i = 2 * lane + e;
        const uint64_t turn = pos * a.freq[i < a.rot / 2 ? i : 0];
        float s, c;
        sincospif(static_cast<float>(static_cast<int32_t>(turn >> 32)) * 0x1p-31f, &s, &c);
        mine[e] = make_float2(c * a.amplitude, s * a.amplitude);
    }
    // half: element e of the low chunk pairs with e of the high one, pair 8 j + e;
    // interleaved: the low chunk holds pairs 4 c0 .., the high one 4 c1 ..
    float2 cs[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t pair = a.interleaved ? (e < 4 ? 4 * c0 + e : 4 * c1 + e - 4) : 8 * j + e;
        const uint32_t from = pair / 2 & 31;  // (a lane that does not turn asks for any)
        const float c = __shfl_sync(0xffffffffu, mine[e & 1].x, from), s = __shfl_sync(0xffffffffu, mine[e & 1].y, from);
        cs[e] = make_float2(c, s);
    }

    // norm (w: this kind's weights in registers, or none) and rotation of one head
    auto turn_head = [&](const Raw& x, bool norm, const float* w, float lo[8], float hi[8]) {
        unpack8(x.lo, lo, In());
        unpack8(x.hi, hi, In());
        if (norm) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
            for (uint32_t o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                lo[e] *= r * w[e];
                hi[e] *= r * w[8 + e];
            }
        }
        if (!turns) return;
        if (a.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float la = lo[2 * e], lb = lo[2 * e + 1], ha = hi[2 * e], hb = hi[2 * e + 1];
                lo[2 * e] = la * cs[e].x - lb * cs[e].y;
                lo[2 * e + 1] = lb * cs[e].x + la * cs[e].y;
                hi[2 * e] = ha * cs[e + 4].x - hb * cs[e + 4].y;
                hi[2 * e + 1] = hb * cs[e + 4].x + ha * cs[e + 4].y;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float la = lo[e], ha = hi[e];
                lo[e] = la * cs[e].x - ha * cs[e].y;
                hi[e] = ha * cs[e].x + la * cs[e].y;
            }
        }
    };
    auto store = [&](Out* dst, const float lo[8], const float hi[8]) {
        *reinterpret_cast<uint4*>(dst + c0 * 8) = pack8(lo, Out());
        *reinterpret_cast<uint4*>(dst + c1 * 8) = pack8(hi, Out());
    };
    auto weights = [&](const void* p, float w[16]) {
        if (!p) return;
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const In*>(p) + c0 * 8), w, In());
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const In*>(p) + c1 * 8), w + 8, In());
    };

    float w[16], lo[8], hi[8];
    weights(a.q_weight, w);
#pragma unroll 1
    for (uint32_t h = first; h < a.Hq + first % kHeads; h += step) {  // the same trips for every lane
        const Raw x = q;
        // the rotation alone has the registers to stay two heads ahead (8192 tokens
        // of 64 + 8 heads: 67 -> 59 us); the append at four CTAs does not gain
        q = kAppend ? load_q(h + step) : q2;
        if (!kAppend) q2 = load_q(h + 2 * step);
        turn_head(x, a.q_weight != nullptr, w, lo, hi);
        if (h < a.Hq) store(static_cast<Out*>(a.q_out) + t * a.qo_ts + h * a.qo_hs, lo, hi);
    }
    weights(a.k_weight, w);
#pragma unroll 1
    for (uint32_t h = first; h < n_kv + first % kHeads; h += step) {
        const Raw x = kv;
        kv = load_kv(h + step);
        turn_head(x, a.k_weight != nullptr, w, lo, hi);
        if (h >= n_kv) continue;
        if (kAppend) {
            const bool val = h >= a.Hkv;
            if (val) {  // values go as they are
                unpack8(x.lo, lo, In());
                unpack8(x.hi, hi, In());
            }
            store(static_cast<Out*>(val ? a.hot_v : a.hot_k) + (static_cast<uint64_t>(slot) * a.Hkv + h - (val ? a.Hkv : 0u)) * D,
                  lo, hi);
        } else {
            store(static_cast<Out*>(a.k_out) + t * a.ko_ts + h * a.ko_hs, lo, hi);
        }
    }
}

template <typename In, typename Out, bool kAppend>
cudaError_t launch_typed(const RopeArgs& a, cudaStream_t s) {
    const uint32_t per_cta = kRopeWarps / a.warps_per_token;
    const uint32_t grid = (a.T + per_cta - 1) / per_cta;
    if (a.D == 128)
        rope_kernel<128, In, Out, kAppend><<<grid, kRopeThreads, 0, s>>>(a);
    else
        rope_kernel<64, In, Out, kAppend><<<grid, kRopeThreads, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rope(RopeArgs a, bool append, cudaStream_t s) {
    if (a.T == 0) return cudaSuccess;
    // Warps per token: while the tokens do not fill the GPU, as many as have
    // heads to turn (latency); else as few as leave a warp eight rounds of heads,
    // since each of them computes the angles (64 query heads of 8192 tokens: 68 us
    // with two, 72 with one; 14 of 4099: 10 and 8).
    const uint32_t per_warp = 512 / a.D;  // heads a warp turns at a time
    const uint32_t rounds = (std::max(a.Hq, append && a.v ? 2 * a.Hkv : a.Hkv) + per_warp - 1) / per_warp;
    const uint32_t want = a.T <= 512 ? rounds : rounds / 8;
    a.warps_per_token = want >= 8 ? 8 : want >= 4 ? 4 : want >= 2 ? 2 : 1;
    if (append)
        return a.bf16 ? launch_typed<__nv_bfloat16, __half, true>(a, s) : launch_typed<__half, __half, true>(a, s);
    return a.bf16 ? launch_typed<__nv_bfloat16, __nv_bfloat16, false>(a, s) : launch_typed<__half, __half, false>(a, s);
}

}  // namespace weaver
