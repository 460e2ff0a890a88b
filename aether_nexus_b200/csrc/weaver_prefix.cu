// weaver_prefix.cu — exact attention over the hot pool for a ragged batch whose
// sequences share prefixes: out = softmax over (the group's prefix tokens, the
// sequence's own tokens) of scale * q.K, times V.
//
// Sequences with few queries pool them: the group's prefix is attended by the
// queries of all of its pooled sequences together, so its pages are read once
// per row tile and not once per sequence; a sequence's own pages are attended
// by its own queries.  The log-sum-exp of the parts joins a query's two results:
//   M = max m_p,  out = sum o_p e^(m_p - M) / sum l_p e^(m_p - M).
// A sequence with enough queries to fill tiles of its own (a prompt chunk), or
// alone in its group, attends to prefix and own pages in one run and needs no
// joining.
//
// A plan cuts every (list, kv head, row tile) into items along the pages, so
// that there are enough CTAs however few rows there are; each item writes its
// rows' (m, l, o) and the merge joins them.  A tile with one item whose rows
// get nothing from elsewhere is written directly.  Lists of more than 16 rows
// per kv head run on tcgen05 (weaver_prefix_tc.cu), the others here:
//
// prefix_rows16_kernel: tiles of 16 rows on mma.sync, as the multi-query
// attention of the flat caches: four warps take every fourth 16-token page of
// the item, each through its own two-stage cp.async ring; rows past a length
// are written as zeros in shared memory, so what the pool holds there never
// enters a product.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "weaver_device.cuh"
#include "weaver_fa.cuh"
#include "weaver_internal.hpp"
#include "weaver_prefix.cuh"

namespace weaver {
namespace {

constexpr uint32_t kPxThreads = 128;

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

// 1 / l; 0 for a row that saw nothing; NaN stays NaN.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l); }

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
    const uint32_t pre_len = prefix_len(a, list, tid == 0), suf_len = suffix_len(a, list, tid == 0);
    auto out_row = [&](uint32_t r) {  // row r of the tile in q and out
        const uint32_t rr = tile.row0 + r, j = rr / a.G;
        return static_cast<uint64_t>(a.row_tok[list.tok0 + j]) * a.Hq + g * a.G + (rr - j * a.G);
    };

    for (uint32_t i = tid; i < 16 * (D / 8); i += kPxThreads) {
        const uint32_t r = i / (D / 8), ch = i % (D / 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) v = *reinterpret_cast<const uint4*>(a.q + out_row(r) * D + ch * 8);
        *reinterpret_cast<uint4*>(qs + r * D + ch * 8) = v;
    }
    __syncthreads();
    uint32_t qf[KS][4];
    fa_load_q<D>(qs, qf, lane);
    int32_t lim_pre[2], lim_suf[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        const uint32_t r = gid + 8 * hh;
        lim_pre[hh] = r < rows ? static_cast<int32_t>(pre_len) : 0;
        lim_suf[hh] = r < rows ? static_cast<int32_t>(suffix_limit(list, suf_len, (tile.row0 + r) / a.G)) : 0;
    }
    // the item's pages below the lengths and the tile's largest limit: n_pre of
    // the prefix from blk0, then own ones from suf0; this warp takes every fourth
    const uint32_t top = suffix_limit(list, suf_len, (tile.row0 + rows - 1) / a.G);
    const uint32_t p1 = min(it.blk1, (pre_len + kBlock - 1) / kBlock);
    const uint32_t n_pre = p1 > it.blk0 ? p1 - it.blk0 : 0;
    const uint32_t suf0 = it.blk0 > list.pre_blocks ? it.blk0 - list.pre_blocks : 0;
    const uint32_t s1 = min(it.blk1 > list.pre_blocks ? it.blk1 - list.pre_blocks : 0, (top + kBlock - 1) / kBlock);
    const uint32_t n = n_pre + (s1 > suf0 ? s1 - suf0 : 0);
    const uint32_t nb = warp < n ? (n - warp + 3) / 4 : 0;

    uint8_t* ring = smem + warp * L::kWarpRing;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;

    uint32_t valid = 0;  // bit k & 1: page k's reference is in the pool
    auto own = [&](uint32_t k) { return warp + 4 * k >= n_pre; };
    auto page = [&](uint32_t k) { return own(k) ? suf0 + (warp + 4 * k - n_pre) : it.blk0 + warp + 4 * k; };
    auto issue = [&](uint32_t k) {
        const uint32_t b = page(k);
        const uint32_t ref = (own(k) ? a.suffix_refs[list.suf_ref0 + b] : a.prefix_refs[list.pre_ref0 + b]) & kRefMask;
        const bool ok = ref < a.pool_blocks;
        if (!ok && lane == 0) atomicOr(a.status, DEVERR_REF_RANGE);
        valid = (valid & ~(1u << (k & 1))) | (ok ? 1u << (k & 1) : 0u);
        px_issue<D>(ring + (k & 1) * L::kStage, a, ref, ok, b * kBlock, own(k) ? suf_len : pre_len, g, lane);
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
        fa_block<D>(Ks, Ks + L::kTile, qf, own(k) ? lim_suf : lim_pre, static_cast<int32_t>(page(k) * kBlock), a.scale, ok,
                    m_run, l_run, o, lane);
        __syncwarp();  // every lane done with the stage before it is refilled
    }
    cp_async_wait_all();
    __syncthreads();  // the rings are dead: reuse the space for the warps' partials
    fa_store_partial<D>(red + warp * 16 * (D + 2), m_run, l_run, o, lane);
    __syncthreads();
    for (uint32_t x = tid; x < 16 * D; x += kPxThreads) {
        const uint32_t r = x / D, d = x % D;
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
            a.out[out_row(r) * D + d] = __float2half_rn(O * inverse_sum(Lsum));
        } else {
            const uint64_t row = it.part_row + static_cast<uint64_t>(r);
            if (d == 0) a.part_ml[row] = make_float2(M, Lsum);
            a.part_o[row * D + d] = O;
        }
    }
}

// One warp per (query token, q head): the parts of its pooled tile and of its
// own tile.
template <int D>
__global__ void __launch_bounds__(256) prefix_merge_kernel(const PrefixArgs a) {
    constexpr int V = D / 32;  // elements per lane
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31;
    if (row >= static_cast<uint64_t>(a.n_tokens) * a.Hq) return;
    const uint32_t t = static_cast<uint32_t>(row / a.Hq), h = static_cast<uint32_t>(row % a.Hq), g = h / a.G;
    const uint4 at = a.tok_lists[t];
    uint64_t base[2];
    uint32_t n[2], step[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        n[s] = 0;
        base[s] = 0;
        step[s] = 0;
        const uint32_t list = s ? at.z : at.x;
        if (list == ~0u) continue;
        const PrefixList L = a.lists[list];
        if (L.pre_blocks + L.suf_blocks == 0) continue;
        const uint32_t rr = (s ? at.w : at.y) * a.G + h % a.G;
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
    const float inv = inverse_sum(Lsum);
#pragma unroll
    for (int v = 0; v < V; v += 2)
        *reinterpret_cast<__half2*>(a.out + row * D + lane * V + v) = __floats2half2_rn(O[v] * inv, O[v + 1] * inv);
}

}  // namespace

// A sequence whose own queries fill this many rows of a kv head gets tiles of
// its own over prefix and own pages: its padding to 128 rows is at most a
// quarter then, and it saves writing and reading two partials a row.
constexpr uint32_t kOwnRows = 512;
// Up to 16 rows a 16-row tile costs one pass over the pages either way.
constexpr uint32_t kRows16 = 16;

void plan_prefix(const PrefixGeometry& geo, uint32_t n_sm, PrefixTables* t) {
    const uint32_t G = geo.Hq / geo.Hkv, NG = geo.n_groups, B = geo.n_seqs, none = ~0u;
    t->tok_lists.assign(geo.q_indptr[B], uint4{none, 0, none, 0});
    for (uint32_t i = 0; i < NG; ++i) {
        const uint32_t s0 = geo.group_indptr[i], s1 = geo.group_indptr[i + 1];
        const uint32_t pre0 = geo.prefix_indptr[i], pre_blocks = geo.prefix_indptr[i + 1] - pre0;
        auto queries = [&](uint32_t b) { return geo.q_indptr[b + 1] - geo.q_indptr[b]; };
        auto few = [&](uint32_t b) { return queries(b) > 0 && static_cast<uint64_t>(queries(b)) * G < kOwnRows; };
        uint32_t n_few = 0;
        for (uint32_t b = s0; b < s1; ++b) n_few += few(b);
        const bool pool = pre_blocks > 0 && n_few > 1;
        if (pool) {
            PrefixList L{};
            L.tok0 = static_cast<uint32_t>(t->row_tok.size());
            L.pre_ref0 = pre0;
            L.pre_blocks = pre_blocks;
            L.pre_len = i;
            for (uint32_t b = s0; b < s1; ++b)
                if (few(b))
                    for (uint32_t q = geo.q_indptr[b]; q < geo.q_indptr[b + 1]; ++q) {
                        t->tok_lists[q].x = static_cast<uint32_t>(t->lists.size());
                        t->tok_lists[q].y = L.ntok++;
                        t->row_tok.push_back(q);
                    }
            t->lists.push_back(L);
        }
        for (uint32_t b = s0; b < s1; ++b) {
            if (!queries(b)) continue;
            PrefixList L{};
            L.tok0 = static_cast<uint32_t>(t->row_tok.size());
            if (!(pool && few(b))) {
                L.pre_ref0 = pre0;
                L.pre_blocks = pre_blocks;
                L.pre_len = i;
            }
            L.suf_ref0 = geo.suffix_indptr[b];
            L.suf_blocks = geo.suffix_indptr[b + 1] - L.suf_ref0;
            L.suf_len = b;
            L.causal = geo.causal ? 1u : 0u;
            for (uint32_t q = geo.q_indptr[b]; q < geo.q_indptr[b + 1]; ++q) {
                t->tok_lists[q].z = static_cast<uint32_t>(t->lists.size());
                t->tok_lists[q].w = L.ntok++;
                t->row_tok.push_back(q);
            }
            t->lists.push_back(L);
        }
    }
    const uint32_t n_lists = static_cast<uint32_t>(t->lists.size());
    auto pages = [&](uint32_t l) { return t->lists[l].pre_blocks + t->lists[l].suf_blocks; };
    auto rows_of = [&](uint32_t l) { return static_cast<uint64_t>(t->lists[l].ntok) * G; };
    // lists whose rows get something from another list too
    std::vector<uint8_t> joined(n_lists, geo.partials ? 1 : 0);
    t->needs_merge = geo.partials && geo.q_indptr[B];
    for (const uint4& x : t->tok_lists) {
        const bool p = x.x != none && pages(x.x), o = x.z != none && pages(x.z);
        if (p && o) joined[x.x] = joined[x.z] = 1;
        if (!p && !o) t->needs_merge = true;  // its zeros come from the merge
    }

    // tiles, and the work of either kind
    struct TcTile { uint32_t tile, n, cost; };
    std::vector<TcTile> tc;
    uint64_t work16 = 0, cost_tc = 0, n_tc = 0;
    for (uint32_t l = 0; l < n_lists; ++l) {
        PrefixList& L = t->lists[l];
        const bool small = rows_of(l) <= kRows16;
        L.tile_rows = small ? 16 : 256;
        L.n_tiles = static_cast<uint32_t>((rows_of(l) + L.tile_rows - 1) / L.tile_rows);
        L.tile0 = static_cast<uint32_t>(t->tiles.size());
        if (!pages(l)) continue;
        if (t->tiles.size() + static_cast<uint64_t>(geo.Hkv) * L.n_tiles > 0x7FFFFFFFull) throw std::length_error("too many tiles");
        for (uint32_t g = 0; g < geo.Hkv; ++g)
            for (uint32_t r = 0; r < L.n_tiles; ++r) {
                PrefixTile T{};
                T.list = l;
                T.kvh = g;
                T.row0 = r * L.tile_rows;
                if (small) {
                    work16 += pages(l);
                } else {
                    // 128-token tiles below the causal limit of the tile's last
                    // row, the pages taken as full
                    const uint64_t rows = std::min<uint64_t>(256, rows_of(l) - T.row0);
                    uint64_t own = static_cast<uint64_t>(L.suf_blocks) * kBlock;
                    if (L.causal) {
                        const int64_t lim = static_cast<int64_t>(own) - L.ntok + 1 + (T.row0 + rows - 1) / G;
                        own = lim > 0 ? std::min<uint64_t>(own, lim) : 0;
                    }
                    const uint32_t n = static_cast<uint32_t>((L.pre_blocks + 7) / 8 + (own + 127) / 128);
                    // a token tile of 256 rows keeps the exponentials busy for two
                    // tiles of 128, one of fewer rows waits for HBM
                    const uint32_t cost = rows > 128 ? 8 : 5;
                    tc.push_back(TcTile{static_cast<uint32_t>(t->tiles.size()), std::max(n, 1u), cost});
                    cost_tc += static_cast<uint64_t>(tc.back().n) * cost;
                    n_tc += tc.back().n;
                }
                t->tiles.push_back(T);
            }
    }
    uint64_t part_rows = 0;
    auto tile_rows = [&](const PrefixTile& T) {
        const PrefixList& L = t->lists[T.list];
        return std::min<uint64_t>(L.tile_rows, rows_of(T.list) - T.row0);
    };

    // 16-row tiles: about three CTAs fit an SM; items of whole multiples of
    // four pages (one per warp), as long as that still gives two full waves
    const uint64_t target = 6ull * n_sm;
    const uint64_t per = std::max<uint64_t>(4, ((work16 + target - 1) / target + 3) / 4 * 4);
    for (uint32_t ti = 0; ti < t->tiles.size(); ++ti) {
        PrefixTile& T = t->tiles[ti];
        if (t->lists[T.list].tile_rows != 16) continue;
        const uint64_t n = pages(T.list), rows = tile_rows(T);
        T.n_slots = static_cast<uint32_t>((n + per - 1) / per);
        T.direct = T.n_slots == 1 && !joined[T.list];
        T.part_row0 = part_rows;
        for (uint32_t s = 0; s < T.n_slots; ++s) {
            PrefixItem it{};
            it.tile = ti;
            it.blk0 = static_cast<uint32_t>(s * per);
            it.blk1 = static_cast<uint32_t>(std::min<uint64_t>(n, (s + 1) * per));
            it.part_row = part_rows + s * rows;
            t->items16.push_back(it);
        }
        if (T.direct) continue;
        part_rows += T.n_slots * rows;
        t->needs_merge = true;
    }

    // tensor-memory tiles: one CTA per SM, each with an equal share of the
    // cost along the list of tiles, so a tile is cut only where a share ends
    const uint32_t n_ctas = static_cast<uint32_t>(std::min<uint64_t>(n_sm, n_tc));
    t->tc_ptr.assign(1, 0);
    uint64_t spent = 0;
    uint32_t cta = 0;
    for (const TcTile& x : tc) {
        PrefixTile& T = t->tiles[x.tile];
        const uint64_t rows = tile_rows(T);
        T.part_row0 = part_rows;
        for (uint32_t b = 0; b < x.n;) {
            const uint64_t end = cost_tc * (cta + 1) / n_ctas;  // this CTA's share ends here
            uint64_t take = (end > spent ? end - spent : 0) / x.cost;
            if (cta + 1 == n_ctas) take = x.n - b;
            if (take == 0) take = t->items_tc.size() == t->tc_ptr.back() ? 1 : 0;  // at least one token tile each
            if (take == 0) {
                t->tc_ptr.push_back(static_cast<uint32_t>(t->items_tc.size()));
                ++cta;
                continue;
            }
            take = std::min<uint64_t>(take, x.n - b);
            PrefixItem it{};
            it.tile = x.tile;
            it.blk0 = b;
            it.blk1 = static_cast<uint32_t>(b + take);
            it.two = rows <= 128 && take > 1;
            it.part_row = part_rows + T.n_slots * rows;
            T.n_slots += it.two ? 2 : 1;
            t->items_tc.push_back(it);
            b += static_cast<uint32_t>(take);
            spent += take * x.cost;
        }
        T.direct = T.n_slots == 1 && !joined[T.list];
        if (T.direct) continue;
        part_rows += T.n_slots * rows;
        t->needs_merge = true;
    }
    if (!tc.empty()) t->tc_ptr.push_back(static_cast<uint32_t>(t->items_tc.size()));
    t->part_rows = part_rows;
}

namespace {

template <int D>
cudaError_t rows16(const PrefixArgs& a, uint32_t n_items, cudaStream_t s) {
    const size_t smem = 1024 + PxLayout<D>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(prefix_rows16_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    prefix_rows16_kernel<D><<<n_items, kPxThreads, smem, s>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_prefix_rows16(const PrefixArgs& a, uint32_t n_items, cudaStream_t s) {
    return a.D == 128 ? rows16<128>(a, n_items, s) : rows16<64>(a, n_items, s);
}

cudaError_t launch_prefix_merge(const PrefixArgs& a, cudaStream_t s) {
    const uint32_t grid = static_cast<uint32_t>((static_cast<uint64_t>(a.n_tokens) * a.Hq + 7) / 8);
    if (a.D == 128)
        prefix_merge_kernel<128><<<grid, 256, 0, s>>>(a);
    else
        prefix_merge_kernel<64><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
}

}  // namespace weaver
