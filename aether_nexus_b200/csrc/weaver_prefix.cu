// weaver_prefix.cu — exact attention over the hot pool for a ragged batch whose
// sequences share prefixes: out = softmax over (the group's prefix tokens, the
// sequence's own tokens) of scale * q.K, times V.
//
// A page list (a group's prefix, or one sequence's own pages) is attended by a
// set of query rows: a prefix by the queries of all sequences of its group, a
// sequence's own pages by its own queries.  The rows of one kv head g are
// flattened as r = (token, q head of g), so K and V of a list are read once
// per row tile and not once per sequence: row r of a list is query token
// tok0 + r / G, q head g * G + r % G.  The log-sum-exp of the parts joins a
// row's prefix and own results:
//   M = max m_p,  out = sum o_p e^(m_p - M) / sum l_p e^(m_p - M).
//
// A plan cuts every (list, kv head, row tile) into items along the pages, so
// that there are enough CTAs however few rows there are; each item writes its
// rows' (m, l, o) and the merge joins them.  A row with a single item is
// written directly.
//
// prefix_rows16_kernel: tiles of 16 rows on mma.sync, as the multi-query
// attention of the flat caches: four warps take every fourth 16-token page of
// the item, each through its own two-stage cp.async ring; pages past the
// list's length and rows of the last page past it are written as zeros in
// shared memory, so what the pool holds there never enters a product.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "weaver_device.cuh"
#include "weaver_fa.cuh"
#include "weaver_internal.hpp"

namespace weaver {
namespace {

constexpr uint32_t kPxThreads = 128;

// Tokens of a list: its length on the device, at most its pages' capacity (a
// larger length is reported and cut).
__device__ __forceinline__ uint32_t list_len(const PrefixArgs& a, const PrefixList& L, uint32_t list, bool report) {
    const uint32_t cap = L.blocks * kBlock;
    const uint32_t* p = list < a.n_groups ? a.prefix_lens : a.suffix_lens;
    if (!p) return cap;
    const uint32_t n = p[list < a.n_groups ? list : list - a.n_groups];
    if (n > cap && report) atomicOr(a.status, DEVERR_REF_RANGE);
    return min(n, cap);
}

// Positions that query token j of the list's nq sees (all of them in a prefix).
__device__ __forceinline__ int32_t row_limit(const PrefixList& L, uint32_t len, uint32_t j) {
    if (!L.causal) return static_cast<int32_t>(len);
    const int64_t lim = static_cast<int64_t>(len) - L.ntok + 1 + j;
    return static_cast<int32_t>(lim > 0 ? lim : 0);
}

template <int D>
struct PxLayout {
    static constexpr uint32_t kTile = FaTile<D>::kTile;        // one page of K (or V) of one head
    static constexpr uint32_t kStage = 2 * kTile;
    static constexpr uint32_t kWarpRing = 2 * kStage;
    static constexpr uint32_t kRing = 4 * kWarpRing;
    static constexpr uint32_t kQ = 16 * D * 2;
    static constexpr uint32_t kRed = 4 * 16 * (D + 2) * 4;
    static constexpr uint32_t kBytes = (kRing > kRed ? kRing : kRed) + kQ;
};

template <int D>
__device__ __forceinline__ void px_issue(uint8_t* st, const PrefixArgs& a, uint64_t block, bool ok, uint32_t pos0,
                                         uint32_t len, uint32_t g, uint32_t lane) {
    constexpr uint32_t kChunks = D / 8;
#pragma unroll
    for (uint32_t i = lane; i < 16 * kChunks; i += 32) {
        const uint32_t row = i / kChunks, ch = i % kChunks;
        const bool valid = ok && pos0 + row < len;
        const uint64_t off = valid ? ((block * kBlock + row) * a.Hkv + g) * D + ch * 8 : 0ull;
        const uint32_t so = (ch >> 3) * FaTile<D>::kBox + swz128(row, ch & 7);
        cp_async16_zfill(st + so, a.k + off, valid);
        cp_async16_zfill(st + PxLayout<D>::kTile + so, a.v + off, valid);
    }
}

template <int D>
__global__ void __launch_bounds__(kPxThreads) prefix_rows16_kernel(const PrefixArgs a) {
    using L = PxLayout<D>;
    constexpr int KS = D / 16, NT = D / 8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __half* qs = reinterpret_cast<__half*>(smem + (L::kRing > L::kRed ? L::kRing : L::kRed));
    float* red = reinterpret_cast<float*>(smem);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2;
    const PrefixItem it = a.items[blockIdx.x];
    const PrefixTile tile = a.tiles[it.tile];
    const PrefixList list = a.lists[tile.list];
    const uint32_t g = tile.kvh, R = list.ntok * a.G;
    const uint32_t rows = min(16u, R - tile.row0);
    const uint32_t len = list_len(a, list, tile.list, tid == 0);
    const uint32_t* refs = (tile.list < a.n_groups ? a.prefix_refs : a.suffix_refs) + list.ref0;

    for (uint32_t i = tid; i < 16 * (D / 8); i += kPxThreads) {
        const uint32_t r = i / (D / 8), ch = i % (D / 8), rr = tile.row0 + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const uint64_t row = static_cast<uint64_t>(list.tok0 + rr / a.G) * a.Hq + g * a.G + rr % a.G;
            v = *reinterpret_cast<const uint4*>(a.q + row * D + ch * 8);
        }
        *reinterpret_cast<uint4*>(qs + r * D + ch * 8) = v;
    }
    __syncthreads();
    uint32_t qf[KS][4];
    fa_load_q<D>(qs, qf, lane);
    int32_t lim[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        const uint32_t r = gid + 8 * hh;
        lim[hh] = r < rows ? row_limit(list, len, (tile.row0 + r) / a.G) : 0;
    }
    // pages of this item below the tile's largest limit, every fourth of them
    const uint32_t top = static_cast<uint32_t>(row_limit(list, len, (tile.row0 + rows - 1) / a.G));
    const uint32_t b0 = it.blk0 + warp, b1 = min(it.blk1, (top + kBlock - 1) / kBlock);
    const uint32_t nb = b0 < b1 ? (b1 - b0 + 3) / 4 : 0;

    uint8_t* ring = smem + warp * L::kWarpRing;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;

    uint32_t valid = 0;  // bit k & 1: page k's reference is in the pool
    auto issue = [&](uint32_t k) {
        const uint32_t b = b0 + 4 * k;
        const uint32_t ref = refs[b] & 0x7FFFFFFFu;
        const bool ok = ref < a.pool_blocks;
        if (!ok && lane == 0) atomicOr(a.status, DEVERR_REF_RANGE);
        valid = (valid & ~(1u << (k & 1))) | (ok ? 1u << (k & 1) : 0u);
        px_issue<D>(ring + (k & 1) * L::kStage, a, ref, ok, b * kBlock, len, g, lane);
    };
    if (nb > 0) issue(0);
    cp_async_commit();
    for (uint32_t k = 0; k < nb; ++k) {
        const bool ok = (valid >> (k & 1)) & 1u;
        if (k + 1 < nb) issue(k + 1);
        cp_async_commit();
        cp_async_wait1();  // page k has landed (this lane's copies)
        __syncwarp();      // ... and every lane's
        const uint8_t* Ks = ring + (k & 1) * L::kStage;
        fa_block<D>(Ks, Ks + L::kTile, qf, lim, static_cast<int32_t>((b0 + 4 * k) * kBlock), a.scale, ok, m_run, l_run, o,
                    lane);
        __syncwarp();  // every lane done with the stage before it is refilled
    }
    cp_async_wait_all();
    __syncthreads();  // the rings are dead: reuse the space for the warps' partials
    fa_store_partial<D>(red + warp * 16 * (D + 2), m_run, l_run, o, lane);
    __syncthreads();
    for (uint32_t x = tid; x < 16 * D; x += kPxThreads) {
        const uint32_t r = x / D, d = x % D, rr = tile.row0 + r;
        if (r >= rows) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, red[(w * 16 + r) * (D + 2)]);
        float Lsum = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* pw = red + (w * 16 + r) * (D + 2);
            const float f = exp_shift(pw[0], M);
            Lsum += pw[1] * f;
            O += pw[2 + d] * f;
        }
        if (tile.direct) {
            const uint64_t row = static_cast<uint64_t>(list.tok0 + rr / a.G) * a.Hq + g * a.G + rr % a.G;
            a.out[row * D + d] = __float2half_rn(Lsum > 0.0f ? O / Lsum : 0.0f);
        } else {
            const uint64_t row = it.part_row + static_cast<uint64_t>(r);
            if (d == 0) a.part_ml[row] = make_float2(M, Lsum);
            a.part_o[row * D + d] = O;
        }
    }
}

// One warp per (query token, q head): the parts of its prefix tile and of its
// own tile.
template <int D>
__global__ void __launch_bounds__(256) prefix_merge_kernel(const PrefixArgs a) {
    constexpr int V = D / 32;  // elements per lane
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31;
    if (row >= static_cast<uint64_t>(a.n_tokens) * a.Hq) return;
    const uint32_t t = static_cast<uint32_t>(row / a.Hq), h = static_cast<uint32_t>(row % a.Hq), g = h / a.G;
    const uint32_t seq = a.tok_seq[t];
    const uint32_t ids[2] = {a.seq_group[seq], a.n_groups + seq};
    uint64_t base[2];
    uint32_t n[2], step[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const PrefixList L = a.lists[ids[s]];
        n[s] = 0;
        base[s] = 0;
        step[s] = 0;
        if (L.blocks == 0) continue;
        const uint32_t rr = (t - L.tok0) * a.G + h % a.G;
        const PrefixTile T = a.tiles[L.tile0 + g * L.n_tiles + rr / L.tile_rows];
        if (T.direct) return;  // its only item wrote the output
        n[s] = T.n_slots;
        step[s] = min(L.tile_rows, L.ntok * a.G - T.row0);
        base[s] = T.part_row0 + (rr - T.row0);
    }
    float M = -INFINITY;
#pragma unroll
    for (int s = 0; s < 2; ++s)
        for (uint32_t i = lane; i < n[s]; i += 32) M = fmaxf(M, a.part_ml[base[s] + static_cast<uint64_t>(i) * step[s]].x);
    M = warp_max(M);
    float Lsum = 0.0f, O[V];
#pragma unroll
    for (int v = 0; v < V; ++v) O[v] = 0.0f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll 4
        for (uint32_t i = 0; i < n[s]; ++i) {
            const uint64_t p = base[s] + static_cast<uint64_t>(i) * step[s];
            const float2 ml = a.part_ml[p];
            const float f = exp_shift(ml.x, M);
            Lsum += ml.y * f;
            if (V == 4) {
                const float4 x = *reinterpret_cast<const float4*>(a.part_o + p * D + lane * 4);
                O[0] += x.x * f, O[1] += x.y * f, O[2 % V] += x.z * f, O[3 % V] += x.w * f;
            } else {
                const float2 x = *reinterpret_cast<const float2*>(a.part_o + p * D + lane * 2);
                O[0] += x.x * f, O[1] += x.y * f;
            }
        }
    }
    if (a.out_m) {
        if (lane == 0) {
            a.out_m[row] = M;
            a.out_l[row] = Lsum;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) a.out_o[row * D + lane * V + v] = O[v];
        return;
    }
    const float inv = Lsum > 0.0f ? 1.0f / Lsum : 0.0f;
#pragma unroll
    for (int v = 0; v < V; v += 2)
        *reinterpret_cast<__half2*>(a.out + row * D + lane * V + v) = __floats2half2_rn(O[v] * inv, O[v + 1] * inv);
}

template <typename K>
cudaError_t with_smem(K kernel, size_t smem) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
}

}  // namespace

void plan_prefix(const PrefixGeometry& geo, uint32_t n_sm, PrefixTables* t) {
    const uint32_t G = geo.Hq / geo.Hkv, NG = geo.n_groups, B = geo.n_seqs;
    t->lists.resize(NG + B);
    t->seq_group.resize(B);
    for (uint32_t i = 0; i < NG; ++i) {
        const uint32_t s0 = geo.group_indptr[i], s1 = geo.group_indptr[i + 1];
        for (uint32_t b = s0; b < s1; ++b) t->seq_group[b] = i;
        PrefixList& L = t->lists[i];
        L = PrefixList{};
        L.tok0 = geo.q_indptr[s0];
        L.ntok = geo.q_indptr[s1] - L.tok0;
        L.ref0 = geo.prefix_indptr[i];
        L.blocks = geo.prefix_indptr[i + 1] - L.ref0;
    }
    t->tok_seq.resize(geo.q_indptr[B]);
    for (uint32_t b = 0; b < B; ++b) {
        for (uint32_t q = geo.q_indptr[b]; q < geo.q_indptr[b + 1]; ++q) t->tok_seq[q] = b;
        PrefixList& L = t->lists[NG + b];
        L = PrefixList{};
        L.tok0 = geo.q_indptr[b];
        L.ntok = geo.q_indptr[b + 1] - L.tok0;
        L.ref0 = geo.suffix_indptr[b];
        L.blocks = geo.suffix_indptr[b + 1] - L.ref0;
        L.causal = geo.causal ? 1u : 0u;
    }
    // a group's rows are written directly when nothing else adds to them
    auto alone = [&](uint32_t l) {
        if (geo.partials) return false;
        if (l >= NG) return t->lists[t->seq_group[l - NG]].blocks == 0;
        for (uint32_t b = geo.group_indptr[l]; b < geo.group_indptr[l + 1]; ++b)
            if (t->lists[NG + b].ntok && t->lists[NG + b].blocks) return false;
        return true;
    };
    // 16-row tiles: about three CTAs fit an SM; items of whole multiples of
    // four pages (one per warp), as long as that still gives two full waves
    uint64_t work = 0;
    for (const PrefixList& L : t->lists) work += static_cast<uint64_t>(L.blocks) * geo.Hkv * ((L.ntok * static_cast<uint64_t>(G) + 15) / 16);
    const uint64_t target = 6ull * n_sm;
    const uint64_t per = std::max<uint64_t>(4, ((work + target - 1) / target + 3) / 4 * 4);
    t->needs_merge = false;
    uint64_t part_rows = 0;
    for (uint32_t l = 0; l < NG + B; ++l) {
        PrefixList& L = t->lists[l];
        const uint64_t R = static_cast<uint64_t>(L.ntok) * G;
        L.tile_rows = 16;
        L.n_tiles = static_cast<uint32_t>((R + 15) / 16);
        L.tile0 = static_cast<uint32_t>(t->tiles.size());
        if (L.blocks == 0 || R == 0) continue;
        const uint32_t n_slots = static_cast<uint32_t>((L.blocks + per - 1) / per);
        const bool direct = n_slots == 1 && alone(l);
        for (uint32_t g = 0; g < geo.Hkv; ++g)
            for (uint32_t r = 0; r < L.n_tiles; ++r) {
                PrefixTile T{};
                T.list = l;
                T.kvh = g;
                T.row0 = r * 16;
                T.n_slots = n_slots;
                T.direct = direct ? 1u : 0u;
                T.part_row0 = part_rows;
                const uint64_t rows = std::min<uint64_t>(16, R - T.row0);
                for (uint32_t s = 0; s < n_slots; ++s) {
                    PrefixItem it{};
                    it.tile = static_cast<uint32_t>(t->tiles.size());
                    it.blk0 = static_cast<uint32_t>(static_cast<uint64_t>(s) * per);
                    it.blk1 = static_cast<uint32_t>(std::min<uint64_t>(L.blocks, (s + 1ull) * per));
                    it.part_row = part_rows + s * rows;
                    t->items16.push_back(it);
                }
                if (!direct) part_rows += n_slots * rows;
                t->tiles.push_back(T);
            }
        if (!direct) t->needs_merge = true;
    }
    // rows with nothing to attend to get their zeros from the merge
    for (uint32_t b = 0; b < B; ++b)
        if (t->lists[NG + b].ntok && !t->lists[NG + b].blocks && !t->lists[t->seq_group[b]].blocks) t->needs_merge = true;
    if (geo.partials && geo.q_indptr[B]) t->needs_merge = true;
    t->part_rows = part_rows;
}

cudaError_t launch_prefix(const PrefixArgs& a, uint32_t n_items16, bool merge, cudaStream_t s) {
    cudaError_t e;
    if (n_items16) {
        if (a.D == 128) {
            const size_t smem = 1024 + PxLayout<128>::kBytes;
            if ((e = with_smem(prefix_rows16_kernel<128>, smem)) != cudaSuccess) return e;
            prefix_rows16_kernel<128><<<n_items16, kPxThreads, smem, s>>>(a);
        } else {
            const size_t smem = 1024 + PxLayout<64>::kBytes;
            if ((e = with_smem(prefix_rows16_kernel<64>, smem)) != cudaSuccess) return e;
            prefix_rows16_kernel<64><<<n_items16, kPxThreads, smem, s>>>(a);
        }
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    if (merge) {
        const uint64_t rows = static_cast<uint64_t>(a.n_tokens) * a.Hq;
        const uint32_t grid = static_cast<uint32_t>((rows + 7) / 8);
        if (a.D == 128)
            prefix_merge_kernel<128><<<grid, 256, 0, s>>>(a);
        else
            prefix_merge_kernel<64><<<grid, 256, 0, s>>>(a);
        return cudaGetLastError();
    }
    return cudaSuccess;
}

}  // namespace weaver
