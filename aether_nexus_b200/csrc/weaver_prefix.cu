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
// get nothing from elsewhere is written directly.  Lists of more than 8 or 16
// rows per kv head run on tcgen05 (weaver_prefix_tc.cu), the others here:
//
// prefix_rows16_kernel: tiles of 16 rows on mma.sync, as the multi-query
// attention of the flat caches: four warps take every fourth 16-token page of
// the item, each through its own two-stage cp.async ring; rows past a length
// are written as zeros in shared memory, so what the pool holds there never
// enters a product.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <functional>
#include <queue>
#include <stdexcept>

#include "weaver_device.cuh"
#include "weaver_fa.cuh"
#include "weaver_internal.hpp"
#include "weaver_prefix.cuh"

namespace weaver {
namespace {

constexpr uint32_t kPxThreads = 128;
// log2 of the factor on the probabilities: the largest is 2^15, inside f16, and
// what f16 cannot hold any more is 2^-40 of it (at 1 a long tail 2^-25 below one
// dominant token vanished from the output while the sum counted it)
constexpr int kPxShift = 15;

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
__device__ __forceinline__ void px_issue(uint8_t* st, const PrefixArgs& a, uint64_t block, uint32_t pos0, uint32_t len,
                                         uint32_t g, uint32_t lane) {
    constexpr uint32_t kChunks = D / 8;
#pragma unroll
    for (uint32_t i = lane; i < 16 * kChunks; i += 32) {
        const uint32_t row = i / kChunks, ch = i % kChunks;
        const bool valid = pos0 + row < len;
        const uint64_t off = valid ? ((block * kBlock + row) * a.Hkv + g) * D + ch * 8 : 0ull;
        const uint32_t so = (ch >> 3) * FaTile<D>::kBox + swz128(row, ch & 7);
        cp_async16_zfill(st + so, a.k + off, valid);
        cp_async16_zfill(st + PxLayout<D>::kTile + so, a.v + off, valid);
    }
}

template <int D>
__global__ void __launch_bounds__(kPxThreads) prefix_rows16_kernel(const __grid_constant__ PrefixArgs a) {
    using L = PxLayout<D>;
    constexpr int KS = D / 16, NT = D / 8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __half* qs = reinterpret_cast<__half*>(smem + (L::kRing > L::kRed ? L::kRing : L::kRed));
    float* red = reinterpret_cast<float*>(smem);
    launch_dependents();

    // Three latencies before the pages are under way: the item, then the lengths,
    // page references and tokens that it names, then query rows and pages.
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2;
    const uint32_t word = lane < sizeof(PrefixItem) / 4 ? reinterpret_cast<const uint32_t*>(a.items + blockIdx.x)[lane] : 0u;
    auto field = [&](uint32_t w) { return __shfl_sync(0xffffffffu, word, w); };
    const uint64_t part_row = static_cast<uint64_t>(field(1)) << 32 | field(0);
    const uint32_t tok0 = field(2), row0 = field(3), rows = field(4), g = field(5), ntok = field(6);
    const uint32_t pre_ref0 = field(7), pre_blocks = field(8), pre_i = field(9), suf_ref0 = field(11), suf_blocks = field(12),
                   suf_i = field(13), t0 = field(14), t1 = field(15), flags = field(16);
    const uint32_t pre_len = page_len(a.prefix_lens, pre_i, pre_blocks, a.status, tid == 0);
    const uint32_t suf_len = page_len(a.suffix_lens, suf_i, suf_blocks, a.status, tid == 0);
    // this warp's pages are t0 + warp, + 4, ...: lane i holds the reference of the i-th of 32
    auto reference = [&](uint32_t k0) {
        const uint32_t p = t0 + warp + 4 * (k0 + lane);
        return p >= t1 ? 0u : (p < pre_blocks ? a.prefix_refs[pre_ref0 + p] : a.suffix_refs[suf_ref0 + p - pre_blocks]) & kRefMask;
    };
    uint32_t ref = reference(0);
    uint32_t at = 0;  // lane r: row r of the tile in q and out
    if (lane < rows) {
        const uint32_t rr = row0 + lane, j = rr / a.G;
        at = a.row_tok[tok0 + j] * a.Hq + g * a.G + (rr - j * a.G);
    }
    for (uint32_t i = tid; i < 16 * (D / 8); i += kPxThreads) {
        const uint32_t r = i / (D / 8), ch = i % (D / 8);
        const uint64_t row = __shfl_sync(0xffffffffu, at, r);
        cp_async16_zfill(qs + r * D + ch * 8, a.q + row * D + ch * 8, r < rows);
    }
    cp_async_commit();
    const bool causal = flags & kPxCausal;
    int32_t lim_pre[2], lim_suf[2];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
        const uint32_t r = gid + 8 * hh;
        lim_pre[hh] = r < rows ? static_cast<int32_t>(pre_len) : 0;
        lim_suf[hh] = r < rows ? static_cast<int32_t>(suffix_limit(causal, suf_len, ntok, (row0 + r) / a.G)) : 0;
    }
    const uint32_t top = suffix_limit(causal, suf_len, ntok, (row0 + rows - 1) / a.G);  // the largest of the tile

    uint8_t* ring = smem + warp * L::kWarpRing;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;

    uint32_t qf[KS][4];
    bool have_q = false;
    for (uint32_t k0 = 0; t0 + warp + 4 * k0 < t1; k0 += 32) {
        if (k0) ref = reference(k0);
        // the pages with tokens that some row sees
        const uint32_t p = t0 + warp + 4 * (k0 + lane);
        const bool own = p >= pre_blocks;
        const uint32_t pos = (own ? p - pre_blocks : p) * kBlock;
        const bool in = p < t1 && pos < (own ? top : pre_len);
        const bool ok = ref < a.pool_blocks;
        if (in && !ok) atomicOr(a.status, DEVERR_REF_RANGE);
        uint32_t todo = __ballot_sync(0xffffffffu, in && ok), next = todo;  // pages to compute, to fetch
        uint32_t stage = 0, fetched = 0;
        auto issue = [&] {
            const uint32_t i = __ffs(next) - 1;
            next &= next - 1;
            px_issue<D>(ring + (fetched++ & 1) * L::kStage, a, __shfl_sync(0xffffffffu, ref, i), __shfl_sync(0xffffffffu, pos, i),
                        __shfl_sync(0xffffffffu, own, i) ? suf_len : pre_len, g, lane);
        };
        if (next) issue();
        cp_async_commit();
        while (todo) {
            const uint32_t i = __ffs(todo) - 1;
            todo &= todo - 1;
            if (next) issue();
            cp_async_commit();
            cp_async_wait1();  // the page (and the query rows) have landed, this lane's copies
            if (!have_q) {
                named_bar(1, kPxThreads);  // ... and every thread's
                fa_load_q<D>(qs, qf, lane);
                have_q = true;
            }
            __syncwarp();
            const uint8_t* Ks = ring + (stage++ & 1) * L::kStage;
            const bool o_own = __shfl_sync(0xffffffffu, own, i);
            fa_block<D, kPxShift>(Ks, Ks + L::kTile, qf, o_own ? lim_suf : lim_pre,
                        static_cast<int32_t>(__shfl_sync(0xffffffffu, pos, i)), a.scale, true, m_run, l_run, o, lane);
            __syncwarp();  // every lane done with the stage before it is refilled
        }
    }
    if (!have_q) {  // a warp without pages keeps the others' appointment
        cp_async_wait_all();
        named_bar(1, kPxThreads);
    }
    cp_async_wait_all();
    __syncthreads();  // the rings are dead: reuse the space for the warps' partials
    fa_store_partial<D>(red + warp * 16 * (D + 2), m_run, l_run, o, lane);
    __syncthreads();
    // each row's maximum and sum over the four warps, and the warps' factors
    if (tid < 16) {
        float M = -INFINITY, Lsum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, red[(w * 16 + tid) * (D + 2)]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float* pw = red + (w * 16 + tid) * (D + 2);
            const float f = exp_shift(pw[0], M) * (1.0f / (1 << kPxShift));
            Lsum += pw[1] * f;
            pw[0] = f;
        }
        red[tid * (D + 2) + 1] = inverse_sum(Lsum);
        if (!(flags & kPxDirect) && tid < rows) a.part_ml[part_row + tid] = make_float2(M, Lsum);
    }
    __syncthreads();
    // four dimensions of a row per thread, the next row to the next thread
    for (uint32_t x = tid; x < rows * (D / 4); x += kPxThreads) {
        const uint32_t r = x % rows, c = x / rows;
        float O[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float* pw = red + (w * 16 + r) * (D + 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) O[e] += pw[2 + c * 4 + e] * pw[0];
        }
        if (flags & kPxDirect) {
            const float inv = red[r * (D + 2) + 1];
            const uint32_t rr = row0 + r, j = rr / a.G;
            const uint64_t row = static_cast<uint64_t>(a.row_tok[tok0 + j]) * a.Hq + g * a.G + (rr - j * a.G);
            __half2 h[2] = {__floats2half2_rn(O[0] * inv, O[1] * inv), __floats2half2_rn(O[2] * inv, O[3] * inv)};
            *reinterpret_cast<uint2*>(a.out + row * D + c * 4) = *reinterpret_cast<const uint2*>(h);
        } else {
            *reinterpret_cast<float4*>(a.part_o + part_row * D + x * 4ull) = make_float4(O[0], O[1], O[2], O[3]);
        }
    }
}

// A thread per (merged row, four dimensions, share of the row's runs), rows
// fastest: one pass over the runs with the running maximum, then the kShares
// threads of a row and dimensions join theirs in shared memory.  Few rows
// behind a long prefix have a run per CTA that attended to it, and one thread
// would walk through them a latency at a time.
template <int D, uint32_t kShares>
__global__ void __launch_bounds__(8 * D / 4) prefix_merge_kernel(const __grid_constant__ PrefixArgs a) {
    constexpr uint32_t kRows = 8 / kShares;  // neighbouring rows per CTA of 8 * D / 4 threads
    __shared__ float sm[kShares > 1 ? kShares : 1][kRows][D / 4][6];
    const uint32_t tid = threadIdx.x;
    const uint32_t r = tid % kRows, c = tid / kRows % (D / 4), share = tid / (kRows * D / 4);
    const uint64_t i = static_cast<uint64_t>(blockIdx.x) * kRows + r;
    const bool in = i < a.n_merge;
    const PrefixMergeRow mr = a.merge_rows[in ? i : 0];
    wait_prerequisites();
    float M = -INFINITY, L = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto join = [&](float m, float l, float4 y) {
        const float Mn = fmaxf(M, m);
        const float f0 = exp_shift(M, Mn), f1 = exp_shift(m, Mn);
        M = Mn;
        L = L * f0 + l * f1;
        O = make_float4(O.x * f0 + y.x * f1, O.y * f0 + y.y * f1, O.z * f0 + y.z * f1, O.w * f0 + y.w * f1);
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        // row `row` of runs that start at rows run0, run0 + step, ...
        const uint64_t step = mr.step[s], run0 = mr.run0[s];
        const uint32_t row = mr.row[s];
        const uint32_t n = in ? mr.n[s] : 0u;
#pragma unroll 4
        for (uint32_t k = share; k < n; k += kShares) {
            const float2 x = a.part_ml[run0 + k * step + row];
            const float4 y = reinterpret_cast<const float4*>(a.part_o + (run0 + k * step) * D)[c * step + row];
            join(x.x, x.y, y);
        }
    }
    if (kShares > 1) {
        float* mine = sm[share][r][c];
        mine[0] = M, mine[1] = L, mine[2] = O.x, mine[3] = O.y, mine[4] = O.z, mine[5] = O.w;
        __syncthreads();
        if (share) return;
        M = -INFINITY, L = 0.0f;
        O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t k = 0; k < kShares; ++k) {
            const float* x = sm[k][r][c];
            join(x[0], x[1], make_float4(x[2], x[3], x[4], x[5]));
        }
    }
    if (!in) return;
    const uint64_t row = mr.out_row;
    if (a.out_m) {
        if (c == 0) {
            a.out_m[row] = M;
            a.out_l[row] = L;
        }
        *reinterpret_cast<float4*>(a.out_o + row * D + c * 4) = O;
        return;
    }
    const float inv = inverse_sum(L);
    __half2 h[2] = {__floats2half2_rn(O.x * inv, O.y * inv), __floats2half2_rn(O.z * inv, O.w * inv)};
    *reinterpret_cast<uint2*>(a.out + row * D + c * 4) = *reinterpret_cast<const uint2*>(h);
}

}  // namespace

// A sequence whose own queries fill this many rows of a kv head gets tiles of
// its own over prefix and own pages: its padding to 128 rows is at most a
// quarter then, and it saves writing and reading two partials a row.
constexpr uint32_t kOwnRows = 512;
// Starting an item (query rows in, results out, the pipeline filling) in the
// units of a token tile's cost.  8 sequences x 4 drafts run 22.6 to 23.6 us with
// 32, 24.3 to 24.9 with 24, 26.2 to 26.9 with 16, 23.0 to 25.0 with 40 to 56; 16 x
// 8 drafts 35.2 to 35.9, 33.2 to 33.9, 38.1 to 38.5 and 35.4 to 36.4 (two series
// of a graph of 20 calls).
constexpr uint32_t kItemCost = 32;
// Lists of up to 16 rows go to the 16-row tiles, whose many small CTAs start
// and end faster than items of the tensor-memory kernel; lists of 9 to 16 rows
// only where they are many (more than two tiles an SM), since a few more items
// there cost less than another kernel (8 sequences x 4 queries of 4 heads: 22.6
// us on tensor memory, 30.5 with both; 200 sequences x 3: 120.5 and 92.7).
constexpr uint32_t kRows16 = 16, kRowsFew = 8;

// The longest run of an item.  The tensor cores cut the bits below the
// accumulator's last off where they add a step of 16 tokens to it, so O comes out
// low by up to 2^-22 of itself a step, half of that over a run that grows evenly:
// 1.4e-3 after 2^14 steps, more than the rounding of the result.  2048 steps leave
// it below 2^-12; the runs are joined in fp32.  512 token tiles of four steps;
// 8192 pages of one step, dealt to four warps.
constexpr uint32_t kMostTiles = 512, kMostPages = 8192;

// The length of a 16-row item, in pages: that of least makespan on `slots`
// resident CTAs, where an item costs kStart16 rounds beside a round for every
// four of its pages (a page per warp).  64 sequences behind one prefix, 38 MB of
// own pages: 62.1 us a run so and with 3 or 12, 66.9 with a start of one round; 40
// sequences, 123 MB: 73.7, 74.1 and 82.3.
constexpr uint64_t kStart16 = 6;
static uint64_t rows16_item(const std::vector<uint64_t>& tiles, uint64_t slots) {
    uint64_t longest = 1, total = 0;
    for (uint64_t n : tiles) longest = std::max(longest, n), total += n;
    // no shorter than four waves of equal items, then in steps of a quarter; with
    // many tiles that shortest length already spreads them evenly (and the search
    // would take the host long)
    const uint64_t shortest = std::max<uint64_t>(4, total / (4 * slots) / 4 * 4);
    if (tiles.size() > 8 * slots) return shortest;
    uint64_t best = shortest, least = ~0ull;
    for (uint64_t per = shortest;; per += std::max<uint64_t>(4, per / 4 / 4 * 4)) {
        std::vector<uint64_t> cost;
        for (uint64_t n : tiles) {
            const uint64_t k = (n + per - 1) / per;
            for (uint64_t s = 0; s < k; ++s) cost.push_back(kStart16 + (n * (s + 1) / k - n * s / k + 3) / 4);
        }
        std::sort(cost.begin(), cost.end(), std::greater<uint64_t>());
        std::priority_queue<uint64_t, std::vector<uint64_t>, std::greater<uint64_t>> ends;
        uint64_t span = 0;
        for (uint64_t c : cost) {
            uint64_t from = 0;
            if (ends.size() == slots) from = ends.top(), ends.pop();
            ends.push(from + c);
            span = std::max(span, from + c);
        }
        if (span < least) least = span, best = per;
        if (per >= longest) break;
    }
    return best;
}

void plan_prefix(const PrefixGeometry& geo, uint32_t n_sm, PrefixTables* t) {
    const uint32_t G = geo.Hq / geo.Hkv, NG = geo.n_groups, B = geo.n_seqs, none = ~0u;
    // (list, token of it) of every token's pooled part and of its own part
    std::vector<uint4> at(geo.q_indptr[B], uint4{none, 0, none, 0});
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
                        at[q].x = static_cast<uint32_t>(t->lists.size());
                        at[q].y = L.ntok++;
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
                at[q].z = static_cast<uint32_t>(t->lists.size());
                at[q].w = L.ntok++;
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
    for (const uint4& x : at)
        if (x.x != none && pages(x.x) && x.z != none && pages(x.z)) joined[x.x] = joined[x.z] = 1;

    // tiles, and the work of either kind
    uint64_t mid = 0;
    for (uint32_t l = 0; l < n_lists; ++l)
        if (pages(l) && rows_of(l) > kRowsFew && rows_of(l) <= kRows16) mid += geo.Hkv;
    const uint64_t most_rows16 = mid > 2ull * n_sm ? kRows16 : kRowsFew;
    struct TcTile { uint32_t tile, n, cost; };
    std::vector<TcTile> tc;
    uint64_t cost_tc = 0, n_tc = 0;
    for (uint32_t l = 0; l < n_lists; ++l) {
        PrefixList& L = t->lists[l];
        const bool small = rows_of(l) <= most_rows16;
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
                T.rows = static_cast<uint32_t>(std::min<uint64_t>(L.tile_rows, rows_of(l) - T.row0));
                if (!small) {
                    // token tiles below the causal limit of the tile's last
                    // row, the pages taken as full
                    uint64_t own = static_cast<uint64_t>(L.suf_blocks) * kBlock;
                    if (L.causal) {
                        const int64_t lim = static_cast<int64_t>(own) - L.ntok + 1 + (T.row0 + T.rows - 1) / G;
                        own = lim > 0 ? std::min<uint64_t>(own, lim) : 0;
                    }
                    const uint32_t n = static_cast<uint32_t>((L.pre_blocks + kTcPages - 1) / kTcPages +
                                                             (own + kTcPages * kBlock - 1) / (kTcPages * kBlock));
                    // a token tile of 256 rows keeps the exponentials busy for two
                    // tiles of 128, one of fewer rows waits for HBM
                    const uint32_t cost = T.rows > 128 ? 8 : 5;
                    tc.push_back(TcTile{static_cast<uint32_t>(t->tiles.size()), std::max(n, 1u), cost});
                    cost_tc += static_cast<uint64_t>(tc.back().n) * cost + kItemCost;
                    n_tc += tc.back().n;
                }
                t->tiles.push_back(T);
            }
    }
    uint64_t part_rows = 0;

    auto item_of = [&](const PrefixTile& T, uint32_t unit) {
        const PrefixList& L = t->lists[T.list];
        PrefixItem it{};
        it.tok0 = L.tok0, it.row0 = T.row0, it.rows = T.rows, it.kvh = T.kvh, it.ntok = L.ntok;
        it.pre_ref0 = L.pre_ref0, it.pre_blocks = L.pre_blocks, it.pre_len = L.pre_len;
        it.pre_units = (L.pre_blocks + unit - 1) / unit;
        it.suf_ref0 = L.suf_ref0, it.suf_blocks = L.suf_blocks, it.suf_len = L.suf_len;
        it.flags = L.causal ? kPxCausal : 0;
        return it;
    };

    // 16-row tiles: a tile is cut into equal items, at any page.  Of the possible
    // item lengths the one whose items end first when dealt out longest first, as
    // the grid is, three CTAs to an SM at a time (what fits with heads of 128; with
    // heads of 64 four fit, and the lengths are those of three all the same).
    std::vector<uint64_t> sizes;
    for (const PrefixTile& T : t->tiles)
        if (t->lists[T.list].tile_rows == 16) sizes.push_back(pages(T.list));
    const uint64_t per = std::min<uint64_t>(rows16_item(sizes, 3 * n_sm), kMostPages);
    for (uint32_t ti = 0; ti < t->tiles.size(); ++ti) {
        PrefixTile& T = t->tiles[ti];
        if (t->lists[T.list].tile_rows != 16) continue;
        const uint64_t n = pages(T.list), rows = T.rows;
        T.n_slots = static_cast<uint32_t>((n + per - 1) / per);
        T.direct = T.n_slots == 1 && !joined[T.list];
        T.part_row0 = part_rows;
        for (uint32_t s = 0; s < T.n_slots; ++s) {
            PrefixItem it = item_of(T, 1);
            it.part_row = part_rows + s * rows;
            it.t0 = static_cast<uint32_t>(n * s / T.n_slots);
            it.t1 = static_cast<uint32_t>(n * (s + 1) / T.n_slots);
            it.flags |= T.direct ? kPxDirect : 0;
            t->items16.push_back(it);
        }
        if (!T.direct) part_rows += T.n_slots * rows;
    }
    std::stable_sort(t->items16.begin(), t->items16.end(),
                     [](const PrefixItem& x, const PrefixItem& y) { return x.t1 - x.t0 > y.t1 - y.t0; });

    // tensor-memory tiles: one CTA per SM, each with an equal share of the
    // cost along the list of tiles, so a tile is cut only where a share ends
    const uint32_t n_ctas = static_cast<uint32_t>(std::min<uint64_t>(n_sm, n_tc));
    t->tc_ptr.assign(1, 0);
    uint64_t spent = 0;
    uint32_t cta = 0;
    for (const TcTile& x : tc) {
        PrefixTile& T = t->tiles[x.tile];
        const size_t first = t->items_tc.size();
        T.part_row0 = part_rows;
        spent += kItemCost;
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
            take = std::min<uint64_t>({take, x.n - b, kMostTiles});
            PrefixItem it = item_of(T, kTcPages);
            it.part_row = part_rows + static_cast<uint64_t>(T.n_slots) * T.rows;
            it.t0 = b;
            it.t1 = static_cast<uint32_t>(b + take);
            const bool two = T.rows <= 128 && take > 1;
            it.flags |= two ? kPxTwo : 0;
            T.n_slots += two ? 2 : 1;
            t->items_tc.push_back(it);
            b += static_cast<uint32_t>(take);
            spent += take * x.cost;
        }
        T.direct = T.n_slots == 1 && !joined[T.list];
        if (T.direct)
            t->items_tc[first].flags |= kPxDirect;
        else
            part_rows += static_cast<uint64_t>(T.n_slots) * T.rows;
    }
    if (!tc.empty()) t->tc_ptr.push_back(static_cast<uint32_t>(t->items_tc.size()));
    t->part_rows = part_rows;

    // the rows that no single item writes, those with nothing to attend to
    // (their zeros) included
    for (uint32_t q = 0; q < geo.q_indptr[B]; ++q)
        for (uint32_t h = 0; h < geo.Hq; ++h) {
            PrefixMergeRow m{};
            m.out_row = q * geo.Hq + h;
            const uint32_t list[2] = {at[q].x, at[q].z}, tok[2] = {at[q].y, at[q].w};
            bool direct = false;
            for (int s = 0; s < 2; ++s) {
                if (list[s] == none || !pages(list[s])) continue;
                const PrefixList& L = t->lists[list[s]];
                const uint32_t r = tok[s] * G + h % G;
                const PrefixTile& T = t->tiles[L.tile0 + h / G * L.n_tiles + r / L.tile_rows];
                m.run0[s] = T.part_row0;
                m.step[s] = T.rows;
                m.n[s] = T.n_slots;
                m.row[s] = r % L.tile_rows;
                direct |= T.direct != 0;
            }
            if (!direct) t->max_slots = std::max(t->max_slots, m.n[0] + m.n[1]);
            if (!direct) t->merge_rows.push_back(m);
        }
}

namespace {

template <int D>
constexpr size_t rows16_smem() {
    return 1024 + PxLayout<D>::kBytes;
}

template <int D>
cudaError_t rows16(const PrefixArgs& a, uint32_t n_items, cudaStream_t s) {
    prefix_rows16_kernel<D><<<n_items, kPxThreads, rows16_smem<D>(), s>>>(a);
    return cudaGetLastError();
}

template <int D, uint32_t kShares>
cudaError_t merge(const PrefixArgs& a, cudaStream_t s) {
    constexpr uint32_t kRows = 8 / kShares;
    return launch_pdl(prefix_merge_kernel<D, kShares>, dim3((a.n_merge + kRows - 1) / kRows), dim3(8 * D / 4), 0, true, s, a);
}

}  // namespace

cudaError_t prepare_prefix(uint32_t D) {
    const cudaError_t e = D == 128 ? cudaFuncSetAttribute(prefix_rows16_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                          static_cast<int>(rows16_smem<128>()))
                                   : cudaFuncSetAttribute(prefix_rows16_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                          static_cast<int>(rows16_smem<64>()));
    return e == cudaSuccess ? prepare_prefix_tc(D) : e;
}

cudaError_t launch_prefix_rows16(const PrefixArgs& a, uint32_t n_items, cudaStream_t s) {
    return a.D == 128 ? rows16<128>(a, n_items, s) : rows16<64>(a, n_items, s);
}

cudaError_t launch_prefix_merge(const PrefixArgs& a, uint32_t max_slots, cudaStream_t s) {
    // two shares of the runs where a row has more than eight (64 sequences of 19
    // runs: 67.2 us a run of the plan with one share, 62.1 with two, 65.1 with
    // four, whose warps read two rows' neighbouring 16 bytes at a time and not four)
    if (max_slots > 8) return a.D == 128 ? merge<128, 2>(a, s) : merge<64, 2>(a, s);
    return a.D == 128 ? merge<128, 1>(a, s) : merge<64, 1>(a, s);
}

}  // namespace weaver
