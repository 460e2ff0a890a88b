// weaver_prefix_tc.cu — the shared-prefix attention of many query rows on the
// 5th-generation tensor cores.
//
// One persistent CTA per SM works through its items; an item is a tile of up
// to 256 query rows of one kv head against a run of 128-token tiles of its
// page list (the group's prefix pages, then the sequence's own).  Two halves
// of the CTA run the online softmax, one thread per row:
//   S = Q K^T (tcgen05.mma, Q and K in shared memory, S in tensor memory)
//   p = 2^(S * scale * log2 e - m), packed to f16 over S in tensor memory
//   O += P V (P from tensor memory, V in shared memory)
// A tile of more than 128 rows gives each half 128 rows of it and both take
// every token tile; a smaller one gives both halves the same rows and every
// other token tile, so the exponentials of one half overlap the products of the
// other either way.  m is the row's maximum up to 2^8: the accumulator is
// rescaled only when the maximum has grown by more than that, since p <= 2^8
// and its f16 rounding is relative.
//
// Tensor memory (512 columns): S of either half (128 each; P lies in its first
// 64), O of either half (D each).  Pages arrive by one TMA box per page and
// tensor, [2 groups of 8 rows][D/64 halves][8 rows][128 B]: K is a K-major
// operand with 8-row groups D * 16 bytes apart, V an MN-major one whose 16
// tokens per step are one page.
//
// Warps 0-3 and 4-7: the halves; warp 8: MMA; warp 9: TMA; warps 10 and 11
// only complete the third warpgroup, whose registers the first two take over
// (launched with 168 a thread: 384 * 168 = 64512 >= 256 * 216 + 128 * 64).
//
// Bound: up to about 250 rows per kv head by HBM (D * 4 bytes a token and kv
// head); above that by the exponential unit and the tensor cores, which need
// the same 2048 clocks per 256 x 128 tile at D = 128.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "weaver_device.cuh"
#include "weaver_internal.hpp"
#include "weaver_prefix.cuh"

namespace weaver {
namespace {

constexpr uint32_t kTcThreads = 384;  // three warpgroups
constexpr uint32_t kTileTokens = 128;
constexpr uint32_t kTilePages = kTileTokens / kBlock;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.0f;  // log2 of the growth of the maximum that forces a rescale

template <int D>
struct TcLayout {
    static constexpr uint32_t kPage = kBlock * D * 2;
    static constexpr uint32_t kBuf = kTileTokens * D * 2;  // 128 tokens of K (or V)
    static constexpr uint32_t kBufs = D == 128 ? 5 : 10;   // ring of buffers, K and V in turn
    static constexpr uint32_t kQ = 128 * D * 2;
    static constexpr uint32_t kBytes = 2 * kQ + kBufs * kBuf;
    static constexpr uint32_t kO = 256;                    // tensor-memory column of the first accumulator
};

struct TcBars {
    uint64_t full[10], empty[10];
    uint64_t q_full[2], s_full[2], p_ready[2], o_done[2];
    uint64_t drain;
    uint32_t tmem;
};

// The bounded wait, by every lane of a warp (same answer in all).  For the MMA
// and TMA warps the slow path is one function (inlined at every wait it cost
// their registers); the softmax warps, with a row of S in registers, inline it.
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
    return mbar_wait(bar, parity, status, site);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
    const bool ok = mbar_try_wait(bar, parity) || wait_slow(bar, parity, status, site);
    return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ bool row_wait(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, site));
}

// Shared-memory matrix descriptor, 128-byte swizzle (atoms of 8 x 128 bytes).
// K-major: sbo = bytes between 8-row groups (lbo unused).  MN-major: lbo =
// bytes between 64-element column groups, sbo = between 8-row groups.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lbo >> 4) << 16) |
           (static_cast<uint64_t>(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16, f16 operands, fp32 accumulators; b_mn: B is MN-major.
constexpr uint32_t f16_idesc(uint32_t M, uint32_t N, uint32_t b_mn) {
    return (1u << 4) | (b_mn << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 lanes x 32 columns, this lane's row.
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t r[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t r[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One page of one head (16 rows x D f16); x = 0, so the copy starts 128-byte
// aligned in every row; row groups past the pool read zeros.
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, uint64_t* bar, uint32_t half0,
                                              uint32_t group) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(0), "r"(half0), "r"(group)
        : "memory");
}

// What an item comes to, the same for every role.
struct Work {
    PrefixItem it;
    PrefixTile tile;
    PrefixList list;
    uint32_t R, rows;            // rows of the kv head, of this tile
    uint32_t pre_len, suf_len;
    uint32_t pre0, n_pre, suf0;  // token tiles: n_pre of the prefix from pre0, then own ones from suf0
    uint32_t n;                  // token tiles in all
    bool pair;                   // each half has rows of its own

    __device__ __forceinline__ Work(const PrefixArgs& a, uint32_t item, bool report) {
        it = a.tc_items[item];
        tile = a.tiles[it.tile];
        list = a.lists[tile.list];
        R = list.ntok * a.G;
        rows = min(256u, R - tile.row0);
        pair = rows > 128;
        pre_len = prefix_len(a, list, report);
        suf_len = suffix_len(a, list, report);
        // own tokens below the largest limit of the tile's rows
        const uint32_t top = suffix_limit(list, suf_len, (tile.row0 + rows - 1) / a.G);
        const uint32_t cap = (list.pre_blocks + kTilePages - 1) / kTilePages;  // prefix tiles counted by the plan
        const uint32_t p1 = min(it.blk1, (pre_len + kTileTokens - 1) / kTileTokens);
        pre0 = it.blk0;
        n_pre = p1 > pre0 ? p1 - pre0 : 0;
        suf0 = it.blk0 > cap ? it.blk0 - cap : 0;
        const uint32_t s1 = min(it.blk1 > cap ? it.blk1 - cap : 0, (top + kTileTokens - 1) / kTileTokens);
        n = n_pre + (s1 > suf0 ? s1 - suf0 : 0);
    }
    // token tiles of half h
    __device__ __forceinline__ uint32_t count(uint32_t h) const { return pair ? n : (n + 1 - h) / 2; }
    __device__ __forceinline__ uint32_t tile_of(uint32_t j, uint32_t h) const { return pair ? j : 2 * j + h; }
    // token tile t: whether of the own pages, its first token there, tokens of the list from it on
    __device__ __forceinline__ bool own(uint32_t t) const { return t >= n_pre; }
    __device__ __forceinline__ uint32_t first(uint32_t t) const {
        return (own(t) ? suf0 + (t - n_pre) : pre0 + t) * kTileTokens;
    }
    __device__ __forceinline__ uint32_t length(uint32_t t) const { return own(t) ? suf_len : pre_len; }
};

template <int D>
__global__ void __launch_bounds__(kTcThreads, 1) prefix_tc_kernel(const __grid_constant__ CUtensorMap tm_k,
                                                                  const __grid_constant__ CUtensorMap tm_v,
                                                                  const __grid_constant__ PrefixArgs a) {
    using L = TcLayout<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* qs = smem;                 // [half of the CTA][D/64][128 rows][128 B]
    uint8_t* bufs = smem + 2 * L::kQ;   // ring
    __shared__ __align__(8) TcBars bars;

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t i0 = a.tc_ptr[blockIdx.x], i1 = a.tc_ptr[blockIdx.x + 1];

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (uint32_t i = 0; i < L::kBufs; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 1);
        }
        for (uint32_t h = 0; h < 2; ++h) {
            mbar_init(&bars.q_full[h], 128);
            mbar_init(&bars.s_full[h], 1);
            mbar_init(&bars.p_ready[h], 4);
            mbar_init(&bars.o_done[h], 1);
        }
        mbar_init(&bars.drain, 1);
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars.tmem;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 9) {
            // ---- TMA: K and V of every token tile, in turn, into the ring
            bool ok = true;
            uint32_t c_full = 0;  // buffers filled so far
            for (uint32_t i = i0; i < i1 && ok; ++i) {
                const Work w(a, i, lane == 0);
                const uint32_t half0 = w.tile.kvh * (D / 64);
                for (uint32_t t = 0; t < w.n && ok; ++t) {
                    const uint32_t first = w.first(t), len = w.length(t);
                    const uint32_t pages = min(kTilePages, (len - first + kBlock - 1) / kBlock);
                    const uint32_t* refs = (w.own(t) ? a.suffix_refs + w.list.suf_ref0 : a.prefix_refs + w.list.pre_ref0) +
                                           first / kBlock;
                    uint32_t group = 0;
                    if (lane < pages) {
                        const uint32_t ref = refs[lane] & kRefMask;
                        if (ref >= a.pool_blocks) atomicOr(a.status, DEVERR_REF_RANGE);
                        group = 2 * static_cast<uint32_t>(min(static_cast<uint64_t>(ref), a.pool_blocks));  // past the pool: zeros
                    }
#pragma unroll
                    for (uint32_t kv = 0; kv < 2; ++kv) {
                        const uint32_t b = c_full % L::kBufs, round = c_full / L::kBufs;
                        if (round > 0) ok = warp_wait(&bars.empty[b], (round - 1) & 1, a.status, 50);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&bars.full[b], pages * L::kPage);
                        __syncwarp();
                        if (lane < pages)
                            tma_load_page(smem_u32(bufs + b * L::kBuf + lane * L::kPage), kv ? &tm_v : &tm_k, &bars.full[b],
                                          half0, group);
                        ++c_full;
                    }
                }
            }
            // every copy has landed before the CTA's shared memory goes (an
            // abandoned wait of the MMA warp may have left some unread)
            for (uint32_t b = 0; b < L::kBufs && lane == 0; ++b) {
                if (c_full <= b) break;
                const uint32_t last = (c_full - 1 - b) / L::kBufs;
                mbar_drain(&bars.full[b], last & 1);
            }
        } else if (warp == 8) {
            // ---- MMA
            bool ok = true;
            constexpr uint32_t kQK = f16_idesc(128, 128, 0), kPV = f16_idesc(128, D, 1);
            constexpr uint32_t kGroup = D * 16;  // bytes between 8-row groups of a K or V buffer
            uint32_t n_p[2] = {0, 0};            // tiles of each half so far (phase of p_ready, o_done)
            uint32_t n_q[2] = {0, 0};            // items with tiles for the half so far (phase of q_full)
            uint32_t base = 0;                   // buffers consumed by earlier items
            for (uint32_t i = i0; i < i1 && ok; ++i) {
                const Work w(a, i, false);
                if (w.n == 0) continue;
                const uint32_t steps = w.pair ? 2 * w.n : w.n;
                // Wait for buffer idx; own or prefix tile t's V is cleared from its length on.
                auto wait_full = [&](uint32_t idx) {
                    return warp_wait(&bars.full[idx % L::kBufs], (idx / L::kBufs) & 1, a.status, 51);
                };
                auto qk = [&](uint32_t h, uint32_t t) {  // S of half h = Q K(t)^T
                    const uint32_t idx = base + 2 * t;
                    if (!wait_full(idx)) return false;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t q = smem_u32(qs + h * L::kQ), k = smem_u32(bufs + (idx % L::kBufs) * L::kBuf);
#pragma unroll
                        for (uint32_t ks = 0; ks < D / 16; ++ks)
                            mma_ss(tmem + h * 128, sw128_desc(q + (ks / 4) * 16384 + (ks % 4) * 32, 16, 1024),
                                   sw128_desc(k + (ks / 4) * 1024 + (ks % 4) * 32, 16, kGroup), kQK, ks > 0);
                        tc_commit(&bars.s_full[h]);
                        if (!w.pair || h == 1) tc_commit(&bars.empty[idx % L::kBufs]);
                    }
                    __syncwarp();
                    return true;
                };
                const uint32_t halves = w.count(1) ? 2 : 1;
                for (uint32_t h = 0; h < halves && ok; ++h) {
                    ok = warp_wait(&bars.q_full[h], n_q[h]++ & 1, a.status, 52);
                    if (ok) ok = qk(h, w.tile_of(0, h));
                }
                for (uint32_t st = 0; st < steps && ok; ++st) {
                    const uint32_t h = st & 1, t = w.pair ? st / 2 : st;
                    const uint32_t idx = base + 2 * t + 1;
                    const bool last_use = !w.pair || h == 1;
                    if (!(ok = wait_full(idx))) break;
                    if (!w.pair || h == 0) {
                        // rows past the length hold whatever the pool or an earlier
                        // tile left: clear them, or 0 * NaN would reach the sums
                        const uint32_t have = w.length(t) - w.first(t);
                        if (have < kTileTokens) {
                            uint8_t* v = bufs + (idx % L::kBufs) * L::kBuf;
                            for (uint32_t x = lane; x < (kTileTokens - have) * (D / 8); x += 32) {
                                const uint32_t row = have + x / (D / 8), ch = x % (D / 8);
                                *reinterpret_cast<uint4*>(v + (row / 8) * kGroup + (ch >> 3) * 1024 + (row & 7) * 128 +
                                                          (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
                            }
                            fence_proxy_async_shared();
                            __syncwarp();
                        }
                    }
                    if (!(ok = warp_wait(&bars.p_ready[h], n_p[h] & 1, a.status, 53))) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t v = smem_u32(bufs + (idx % L::kBufs) * L::kBuf);
                        const bool more = t >= (w.pair ? 1u : 2u);  // not the half's first tile of the item
#pragma unroll
                        for (uint32_t ks = 0; ks < kTilePages; ++ks)
                            mma_ts(tmem + L::kO + h * D, tmem + h * 128 + ks * 8, sw128_desc(v + ks * L::kPage, 1024, kGroup), kPV,
                                   more || ks > 0);
                        tc_commit(&bars.o_done[h]);
                        if (last_use) tc_commit(&bars.empty[idx % L::kBufs]);
                    }
                    __syncwarp();
                    const uint32_t t_next = w.pair ? t + 1 : t + 2;
                    if (t_next < w.n) {  // P is read before its columns become the next S
                        ok = warp_wait(&bars.o_done[h], n_p[h] & 1, a.status, 54);
                        if (ok) ok = qk(h, t_next);
                    }
                    ++n_p[h];
                }
                // the last products are done before the next item's S and Q
                for (uint32_t h = 0; h < halves && ok; ++h)
                    ok = warp_wait(&bars.o_done[h], (n_p[h] - 1) & 1, a.status, 55);
                base += 2 * w.n;
            }
            // nothing in flight when the tensor memory goes (bounded)
            if (lane == 0) {
                tc_commit(&bars.drain);
                mbar_drain(&bars.drain, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- softmax: half h, one thread per row
        const uint32_t h = warp >> 2, r = tid & 127;
        const uint32_t lanes = (warp & 3) * 32;  // this warp's tensor-memory lanes
        const uint32_t ts = tmem + (lanes << 16) + h * 128, to = tmem + (lanes << 16) + L::kO + h * D;
        const float scale2 = fabsf(a.scale) * kLog2e;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale goes into Q
        uint32_t n_s = 0;                                         // tiles so far (phase of s_full, o_done)
        bool ok = true;
        for (uint32_t i = i0; i < i1 && ok; ++i) {
            const Work w(a, i, false);
            const uint32_t rbase = w.pair ? h * 128 : 0;
            const uint32_t mine = w.rows > rbase ? min(128u, w.rows - rbase) : 0;  // rows of this half
            const uint32_t g = w.tile.kvh, cnt = w.count(h);
            if (cnt) {
                for (uint32_t x = r; x < 128 * (D / 8); x += 128) {
                    const uint32_t row = x / (D / 8), ch = x % (D / 8);
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (row < mine) {
                        const uint32_t rr = w.tile.row0 + rbase + row, j = rr / a.G;
                        const uint64_t at = static_cast<uint64_t>(a.row_tok[w.list.tok0 + j]) * a.Hq + g * a.G + (rr - j * a.G);
                        v = *reinterpret_cast<const uint4*>(a.q + at * D + ch * 8);
                        v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
                    }
                    *reinterpret_cast<uint4*>(qs + h * L::kQ + (ch >> 3) * 16384 + swz128(row, ch & 7)) = v;
                }
                fence_proxy_async_shared();
                mbar_arrive(&bars.q_full[h]);
            }
            const bool has = r < mine;
            const uint32_t rr = w.tile.row0 + rbase + (has ? r : 0), tok = rr / a.G;
            const int32_t lim_pre = has ? static_cast<int32_t>(w.pre_len) : 0;
            const int32_t lim_suf = has ? static_cast<int32_t>(suffix_limit(w.list, w.suf_len, tok)) : 0;
            const bool idle = (warp & 3) * 32 >= mine;  // no row of this warp
            float m = -INFINITY, l = 0.0f;
            for (uint32_t j = 0; j < cnt; ++j) {
                const uint32_t t = w.tile_of(j, h);
                const uint32_t first = w.first(t);
                const int32_t lim = (w.own(t) ? lim_suf : lim_pre) - static_cast<int32_t>(first);
                // pages of this tile whose reference lies beyond the pool
                uint32_t bad = 0;
                {
                    const uint32_t* refs = (w.own(t) ? a.suffix_refs + w.list.suf_ref0 : a.prefix_refs + w.list.pre_ref0) +
                                           first / kBlock;
                    const bool in = lane < kTilePages && first + lane * kBlock < w.length(t);
                    bad = __ballot_sync(0xffffffffu, in && (refs[in ? lane : 0] & kRefMask) >= a.pool_blocks);
                }
                if (!(ok = row_wait(&bars.s_full[h], n_s & 1, a.status, 56))) break;
                tc_fence_after();
                if (!idle) {
                    uint32_t raw[128];
                    tc_ld32(ts, raw);
                    tc_ld32(ts + 32, raw + 32);
                    tc_ld32(ts + 64, raw + 64);
                    tc_ld32(ts + 96, raw + 96);
                    tc_wait_ld();
                    if (__any_sync(0xffffffffu, lim < static_cast<int32_t>(kTileTokens)) || bad) {
#pragma unroll
                        for (int c = 0; c < 128; ++c)
                            if (c >= lim || ((bad >> (c / 16)) & 1u)) raw[c] = 0xFF800000u;  // -inf
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 128; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(raw[c]));
                    const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                    const bool grow = m_new > m + kRescale;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float to_m = grow ? m_new : m;
                        if (j > 0) {
                            const float f = grow ? ex2(m - to_m) : 1.0f;
                            l *= f;
                            // the previous product has been added before O is rescaled
                            if (!(ok = row_wait(&bars.o_done[h], (n_s - 1) & 1, a.status, 57))) break;
                            tc_fence_after();
#pragma unroll
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                tc_ld32(to + c, o);
                                tc_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tc_st32(to + c, o);
                            }
                        }
                        m = to_m;
                    }
                    const float ms = m == -INFINITY ? 0.0f : m;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t pk[32];
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            const float p0 = ex2(__uint_as_float(raw[half * 64 + c]) * scale2 - ms);
                            const float p1 = ex2(__uint_as_float(raw[half * 64 + c + 1]) * scale2 - ms);
                            sum[c & 2] += p0;
                            sum[(c & 2) + 1] += p1;
                            const __half2 hp = __floats2half2_rn(p0, p1);
                            pk[c / 2] = *reinterpret_cast<const uint32_t*>(&hp);
                        }
                        tc_st32(ts + half * 32, pk);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tc_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.p_ready[h]);
                ++n_s;
            }
            if (!ok) break;
            // ---- this half's result
            if (cnt) {
                if (!(ok = row_wait(&bars.o_done[h], (n_s - 1) & 1, a.status, 58))) break;
                tc_fence_after();
            }
            const bool writes = mine && (w.pair || h == 0 || w.it.two);
            if (writes && !idle) {
                float4* po = nullptr;
                __half* out = nullptr;
                float inv = 0.0f;
                if (w.tile.direct) {
                    inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
                    out = a.out + (static_cast<uint64_t>(a.row_tok[w.list.tok0 + tok]) * a.Hq + g * a.G + (rr - tok * a.G)) * D;
                } else {
                    const uint64_t row = w.it.part_row + (w.pair ? rbase : (h ? w.rows : 0u)) + r;
                    po = reinterpret_cast<float4*>(a.part_o + row * D);
                    if (has) a.part_ml[row] = make_float2(m * kLn2, l);
                }
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    if (cnt) {
                        tc_ld32(to + c, o);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0;
                    }
                    if (!has) continue;
                    if (out) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint4 pack;
                            __half2* hp = reinterpret_cast<__half2*>(&pack);
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                hp[y] = __floats2half2_rn(__uint_as_float(o[e + 2 * y]) * inv,
                                                          __uint_as_float(o[e + 2 * y + 1]) * inv);
                            *reinterpret_cast<uint4*>(out + c + e) = pack;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            po[(c + e) / 4] = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]),
                                                          __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                    }
                }
            }
            tc_fence_before();  // O and S have been read before the next item's products
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D>
cudaError_t launch_tc(const PrefixArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, uint32_t n_ctas, cudaStream_t s) {
    const size_t smem = 1024 + TcLayout<D>::kBytes;
    cudaError_t e = cudaFuncSetAttribute(prefix_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    prefix_tc_kernel<D><<<n_ctas, kTcThreads, smem, s>>>(tm_k, tm_v, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_prefix_tc(const PrefixArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, uint32_t n_ctas,
                             cudaStream_t s) {
    return a.D == 128 ? launch_tc<128>(a, tm_k, tm_v, n_ctas, s) : launch_tc<64>(a, tm_k, tm_v, n_ctas, s);
}

}  // namespace weaver
