// weaver_prefix_tc.cu — the shared-prefix attention of many query rows on the
// 5th-generation tensor cores.
//
// One persistent CTA per SM works through its items; an item is a tile of up
// to 256 query rows of one kv head against a run of 64-token tiles of its
// page list (the group's prefix pages, then the sequence's own).  Two halves
// of the CTA run the online softmax, one thread per row:
//   S = Q K^T (tcgen05.mma, Q and K in shared memory, S in tensor memory)
//   p = 2^(S * scale * log2 e - m), packed to f16 over S in tensor memory
//   O += P V (P from tensor memory, V in shared memory)
// A tile of more than 128 rows gives each half 128 rows of it and both take
// every token tile; a smaller one gives both halves the same rows and every
// other token tile.  m follows the row's maximum at a distance: a rescale of
// the accumulator sets it 2^7 below, the next comes when p would pass 2^15.  So
// the largest p lies in 2^7 .. 2^15, inside f16, whose rounding is relative to
// 2^-14 and whose least step, 2^-24, is then 2^-31 of it or less: n tokens far
// below one dominant one lose at most n 2^-32 of max|v| (with the largest p from
// 1 to 2^15, 2^15 tokens 17 nats below an attention sink vanished).
//
// Tensor memory (512 columns): two S of either half (64 columns each; P lies
// in the first 32), O of either half (D each).  With two S the product for the
// tile after next is issued when P of this one has been used, so the softmax
// finds its next S ready: with one S of 128 tokens each half waited out P V
// and Q K of its own before its next tile (5400 clocks for a 256 x 128 tile,
// against 2048 of the exponential unit).  Pages arrive by one TMA box per page
// and tensor, [2 groups of 8 rows][D/64 halves][8 rows][128 B]: K is a K-major
// operand with 8-row groups D * 16 bytes apart, V an MN-major one whose 16
// tokens per step are one page.
//
// Warps 0-3 and 4-7: the halves; warp 8: Q K^T; warp 10: P V; warps 9 and 11:
// TMA of K and of V.  The first two warpgroups take over registers of the third
// (launched with 168 a thread: 384 * 168 = 64512 >= 256 * 216 + 128 * 64).
// Code that runs once per item is kept in rolled loops: the first pass over
// straight-line code is bound by instruction fetch (10 us for an unrolled copy
// of the query tile).
//
// Bound: up to about 250 rows per kv head by HBM (D * 4 bytes a token and kv
// head); above that by the exponential unit and the tensor cores.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "weaver_device.cuh"
#include "weaver_internal.hpp"
#include "weaver_prefix.cuh"

namespace weaver {
namespace {

constexpr uint32_t kTcThreads = 384;  // three warpgroups
constexpr uint32_t kTilePages = kTcPages;
constexpr uint32_t kTileTokens = kTilePages * kBlock;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// p = 2^(s - m) with m = maximum - kBias at a rescale, the next one where the
// maximum is more than kTop above m.  A larger bias keeps more of a long tail
// and rescales more often, a stop of 900 clocks for a half: 4 x 1024 queries
// behind 4096 tokens take 283.5 us a call with 0, 291.5 with 4, 294.5 with 7 and
// 308 with 10, 64 single tokens behind 32768 67.9, 68.5, 69.5 and 71.5.
constexpr float kBias = 7.0f, kTop = 15.0f;

template <int D>
struct TcLayout {
    static constexpr uint32_t kPage = kBlock * D * 2;
    static constexpr uint32_t kBuf = kTileTokens * D * 2;  // one token tile of K (or V)
    static constexpr uint32_t kBufs = D == 128 ? 10 : 20;  // ring of buffers, K and V in turn
    static constexpr uint32_t kQ = 128 * D * 2;
    static constexpr uint32_t kBytes = 2 * kQ + kBufs * kBuf;
    static constexpr uint32_t kO = 256;                    // tensor-memory column of the first accumulator
};

struct TcBars {
    uint64_t full[20], empty[20];
    // [half][tile of the half & 1]: the products of two tiles of a half may be
    // outstanding, and a parity tells only neighbouring phases apart
    uint64_t q_full[2], s_full[2][2], p_ready[2][2], o_done[2][2];
    uint64_t tail, drain[2];
    uint32_t tmem;
};

// Bounded waits as in mbar_wait, but the clock is first read after a while:
// reading %globaltimer takes longer than most of these waits.  For the MMA and
// TMA warps the slow path is one function (inlined at every wait it cost their
// registers); the softmax warps, with a row of S in registers, inline it.
__device__ __forceinline__ bool spin(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
    for (uint32_t i = 0; i < 256; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait(bar, parity, status, site);
}
__device__ __noinline__ bool wait_slow(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
    return spin(bar, parity, status, site);
}
// Whether the phase is over, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// By every lane of a warp, the same answer in all.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
    const bool ok = mbar_try_wait(bar, parity) || wait_slow(bar, parity, status, site);
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ bool row_wait(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t site) {
    return __all_sync(0xffffffffu, spin(bar, parity, status, site));
}

// Shared-memory matrix descriptors, 128-byte swizzle (atoms of 8 x 128 bytes).
// K-major: sbo = bytes between 8-row groups (lbo unused).  MN-major: lbo =
// bytes between 64-element column groups, sbo = between 8-row groups.  The low
// word holds address and lbo, the high word is a constant of the layout.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | (lbo >> 4 << 16); }
constexpr uint32_t desc_hi(uint32_t sbo) { return (sbo >> 4) | (1u << 14) | (2u << 29); }
// kind::f16, f16 operands, fp32 accumulators; b_mn: B is MN-major.
constexpr uint32_t f16_idesc(uint32_t M, uint32_t N, uint32_t b_mn) {
    return (1u << 4) | (b_mn << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
template <uint32_t kHiA, uint32_t kHiB>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %6};\n\t"
        "setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "n"(kHiA), "n"(kHiB)
        : "memory");
}
template <uint32_t kHiB>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b_lo), "r"(idesc), "r"(acc), "n"(kHiB)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 lanes x 32 (64) columns, this lane's row.  The wait is part of the
// statement: nothing that uses the values can be moved before it.
__device__ __forceinline__ void tc_ld32(uint32_t taddr, float r[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_ld64(uint32_t taddr, float r[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]),
          "=f"(r[32]), "=f"(r[33]), "=f"(r[34]), "=f"(r[35]), "=f"(r[36]), "=f"(r[37]), "=f"(r[38]), "=f"(r[39]),
          "=f"(r[40]), "=f"(r[41]), "=f"(r[42]), "=f"(r[43]), "=f"(r[44]), "=f"(r[45]), "=f"(r[46]), "=f"(r[47]),
          "=f"(r[48]), "=f"(r[49]), "=f"(r[50]), "=f"(r[51]), "=f"(r[52]), "=f"(r[53]), "=f"(r[54]), "=f"(r[55]),
          "=f"(r[56]), "=f"(r[57]), "=f"(r[58]), "=f"(r[59]), "=f"(r[60]), "=f"(r[61]), "=f"(r[62]), "=f"(r[63])
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

__device__ __forceinline__ void tc_st32(uint32_t taddr, const float r[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
        "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]),
        "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]),
        "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31])
        : "memory");
}

// Two fp32 lanes per instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
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

__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// What an item comes to, the same for every role; every value is the same in
// all lanes of the warp, by shuffle, so that the MMA operands stay in uniform
// registers (a thread that feeds them from its own registers issues an MMA at
// half the rate at which the tensor cores take it).
struct Work {
    uint64_t part_row;
    uint32_t tok0, row0, rows, kvh, ntok, flags;
    uint32_t pre_ref, suf_ref;   // first page of the lists
    uint32_t pre_len, suf_len;
    uint32_t pre0, n_pre, suf0;  // token tiles: n_pre of the prefix from pre0, then own ones from suf0
    uint32_t n;                  // token tiles in all
    bool pair;                   // more than 128 rows: each half of the CTA has rows of its own

    // This lane's word of item i's record.
    static __device__ __forceinline__ uint32_t fetch(const PrefixArgs& a, uint32_t i, uint32_t end, uint32_t lane) {
        return i < end && lane < sizeof(PrefixItem) / 4 ? reinterpret_cast<const uint32_t*>(a.tc_items + i)[lane] : 0u;
    }
    // Tokens of the prefix and own pages that a record names: a load each, apart
    // from the rest so that a role may have the next item's on their way.
    struct Lens {
        uint32_t pre, suf;
    };
    static __device__ __forceinline__ Lens lens(const PrefixArgs& a, uint32_t word, bool report) {
        auto at = [&](uint32_t w) { return __shfl_sync(0xffffffffu, word, w); };
        const uint32_t pre_blocks = at(8), pre_i = at(9), suf_blocks = at(12), suf_i = at(13);
        return Lens{page_len(a.prefix_lens, pre_i, pre_blocks, a.status, report),
                    page_len(a.suffix_lens, suf_i, suf_blocks, a.status, report)};
    }
    __device__ __forceinline__ Work(const PrefixArgs& a, uint32_t word, bool report) : Work(a, word, lens(a, word, report)) {}
    __device__ __forceinline__ Work(const PrefixArgs& a, uint32_t word, const Lens& len) {
        auto at = [&](uint32_t w) { return __shfl_sync(0xffffffffu, word, w); };
        part_row = static_cast<uint64_t>(at(1)) << 32 | at(0);
        tok0 = at(2), row0 = at(3), rows = at(4), kvh = at(5), ntok = at(6);
        pre_ref = at(7);
        const uint32_t cap = at(10);
        suf_ref = at(11);
        const uint32_t t0 = at(14), t1 = at(15);
        flags = at(16);
        pair = rows > 128;
        pre_len = __shfl_sync(0xffffffffu, len.pre, 0);
        suf_len = __shfl_sync(0xffffffffu, len.suf, 0);
        // own tokens below the largest limit of the tile's rows
        const uint32_t top = limit((row0 + rows - 1) / a.G);
        const uint32_t p1 = min(t1, (pre_len + kTileTokens - 1) / kTileTokens);
        pre0 = t0;
        n_pre = p1 > pre0 ? p1 - pre0 : 0;
        suf0 = t0 > cap ? t0 - cap : 0;
        const uint32_t s1 = min(t1 > cap ? t1 - cap : 0, (top + kTileTokens - 1) / kTileTokens);
        n = n_pre + (s1 > suf0 ? s1 - suf0 : 0);
    }
    __device__ __forceinline__ uint32_t limit(uint32_t j) const { return suffix_limit(flags & kPxCausal, suf_len, ntok, j); }
    // token tiles of half h
    __device__ __forceinline__ uint32_t count(uint32_t h) const { return pair ? n : (n + 1 - h) / 2; }
    // token tile t: whether of the own pages, its first token there, tokens of the list, its first page reference
    __device__ __forceinline__ bool own(uint32_t t) const { return t >= n_pre; }
    __device__ __forceinline__ uint32_t first(uint32_t t) const {
        return (own(t) ? suf0 + (t - n_pre) : pre0 + t) * kTileTokens;
    }
    __device__ __forceinline__ uint32_t length(uint32_t t) const { return own(t) ? suf_len : pre_len; }
    __device__ __forceinline__ const uint32_t* refs(const PrefixArgs& a, uint32_t t) const {
        return (own(t) ? a.suffix_refs + suf_ref : a.prefix_refs + pre_ref) + first(t) / kBlock;
    }
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
    launch_dependents();
    uint32_t word = Work::fetch(a, i0, i1, lane);  // the next item's record

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
            for (uint32_t b = 0; b < 2; ++b) {
                mbar_init(&bars.s_full[h][b], 1);
                mbar_init(&bars.p_ready[h][b], 4);
                mbar_init(&bars.o_done[h][b], 1);
            }
        }
        mbar_init(&bars.tail, 1);
        mbar_init(&bars.drain[0], 1);
        mbar_init(&bars.drain[1], 1);
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bars.tmem, 0);

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 9 || warp == 11) {
            // ---- TMA: warp 9 brings K, warp 11 V of every token tile into their half
            // of the ring (buffers 0, 2, ... and 1, 3, ...).  The page references of
            // the next tile are loaded ahead and the copies issued by one thread with
            // uniform operands: one warp that did both, loading as it went, took 1400
            // clocks a tile and bounded the kernel.
            const uint32_t kv = warp == 11;
            const CUtensorMap* map = kv ? &tm_v : &tm_k;
            constexpr uint32_t kPairs = L::kBufs / 2;
            bool ok = true;
            uint32_t b = 0, fill = 0;  // next buffer pair; how often the ring has been filled
            uint32_t n_tail = 0;
            for (uint32_t i = i0; i < i1 && ok; ++i) {
                const Work w(a, word, lane == 0 && !kv);
                word = Work::fetch(a, i + 1, i1, lane);
                const uint32_t half0 = w.kvh * (D / 64);
                auto reference = [&](uint32_t t) {
                    return t < w.n && lane < kTilePages && w.first(t) + lane * kBlock < w.length(t) ? w.refs(a, t)[lane] & kRefMask : 0u;
                };
                uint32_t next = reference(0);
                for (uint32_t t = 0; t < w.n && ok; ++t) {
                    const uint32_t ref = next;
                    next = reference(t + 1);
                    const uint32_t have = min(kTileTokens, w.length(t) - w.first(t));  // tokens of this tile
                    const uint32_t pages = (have + kBlock - 1) / kBlock;
                    if (ref >= a.pool_blocks && !kv) atomicOr(a.status, DEVERR_REF_RANGE);
                    const uint32_t group = 2 * static_cast<uint32_t>(min(static_cast<uint64_t>(ref), a.pool_blocks));  // past the pool: zeros
                    if (fill > 0 && !(ok = warp_wait(&bars.empty[2 * b + kv], (fill - 1) & 1, a.status, 50))) break;
                    // V of a partial tile: its rows past the length hold whatever the
                    // pool or an earlier tile left, and 0 * NaN would reach the sums.
                    // It lands on a barrier of its own, is cleared there and only then
                    // handed over.
                    const bool tail = kv && have < kTileTokens;
                    uint64_t* bar = tail ? &bars.tail : &bars.full[2 * b + kv];
                    uint8_t* buf = bufs + (2 * b + kv) * L::kBuf;
                    uint32_t at[kTilePages];
#pragma unroll
                    for (uint32_t p = 0; p < kTilePages; ++p) at[p] = __shfl_sync(0xffffffffu, group, p);
                    if (elect_one()) {
                        mbar_arrive_expect_tx(bar, pages * L::kPage);
#pragma unroll
                        for (uint32_t p = 0; p < kTilePages; ++p)
                            if (p < pages) tma_load_page(smem_u32(buf + p * L::kPage), map, bar, half0, at[p]);
                    }
                    __syncwarp();
                    if (tail) {
                        if (!(ok = warp_wait(&bars.tail, n_tail++ & 1, a.status, 51))) break;
#pragma unroll 1
                        for (uint32_t y = lane; y < (kTileTokens - have) * (D / 8); y += 32) {
                            const uint32_t row = have + y / (D / 8), ch = y % (D / 8);
                            *reinterpret_cast<uint4*>(buf + (row / 8) * (D * 16) + (ch >> 3) * 1024 + (row & 7) * 128 +
                                                      (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_proxy_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bars.full[2 * b + kv]);
                    }
                    if (++b == kPairs) {
                        b = 0;
                        ++fill;
                    }
                }
            }
            // every copy has landed before the CTA's shared memory goes (an
            // abandoned wait of the MMA warps may have left some unread)
            if (lane == 0) {
                for (uint32_t x = 0; x < kPairs; ++x) {
                    const uint32_t times = fill + (x < b ? 1 : 0);
                    if (times) mbar_drain(&bars.full[2 * x + kv], (times - 1) & 1);
                }
                if (!ok && n_tail) mbar_drain(&bars.tail, (n_tail - 1) & 1);
            }
        } else if (warp == 8 || warp == 10) {
            // ---- the products: warp 8 issues S = Q K^T, warp 10 O += P V, one
            // thread each.  A step of one thread that did both took 1200 clocks,
            // 80 to 100 for every barrier polled or committed to, against 670 of
            // the products themselves.
            constexpr uint32_t kQK = f16_idesc(128, kTileTokens, 0), kPV = f16_idesc(128, D, 1);
            constexpr uint32_t kGroup = D * 16;        // bytes between 8-row groups of a K or V buffer
            constexpr uint32_t kPairs = L::kBufs / 2;  // K in buffers 0, 2, ..., V in 1, 3, ...
            constexpr uint32_t kBufStep = L::kBuf >> 4, kQStep = L::kQ >> 4;
            const bool is_qk = warp == 8;
            const uint32_t q_lo = desc_lo(smem_u32(qs), 16), k_lo = desc_lo(smem_u32(bufs), 16),
                           v_lo = desc_lo(smem_u32(bufs) + L::kBuf, 1024);
            uint32_t b = 0, ph = 0;         // ring position of the next K (V) tile, its phase
            uint32_t n0 = 0, n1 = 0;        // tiles of either half so far
            uint32_t ph_q = 0;              // phases of q_full, a bit per half
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
                return mbar_try_wait(bar, parity) || wait_slow(bar, parity, a.status, site);
            };
            for (uint32_t i = i0; i < i1; ++i) {
                const Work w(a, word, false);
                word = Work::fetch(a, i + 1, i1, lane);
                // In the order h = 0, 1, 0, 1, ...: step s is token tile s / 2 of either
                // half's own rows, or tile s of the shared ones.
                const uint32_t steps = w.pair ? 2 * w.n : w.n;
                if (elect_one()) {
                    if (is_qk) {
#pragma unroll 1
                        for (uint32_t s = 0; s < steps; ++s) {
                            const uint32_t h = s & 1, k = h ? n1++ : n0++;
                            if (s < 2) {
                                if (!(ok = wait(&bars.q_full[h], (ph_q >> h) & 1, 52))) break;
                                ph_q ^= 1u << h;
                            }
                            if (!w.pair || h == 0)
                                if (!(ok = wait(&bars.full[2 * b], ph, 51))) break;
                            // the S whose P the half's step before last has used
                            if (k >= 2 && !(ok = wait(&bars.o_done[h][k & 1], ((k - 2) >> 1) & 1, 54))) break;
                            tc_fence_after();
                            const uint32_t q = q_lo + h * kQStep, kd = k_lo + 2 * b * kBufStep, sd = tmem + h * 128 + (k & 1) * 64;
#pragma unroll
                            for (uint32_t ks = 0; ks < D / 16; ++ks)
                                mma_ss<desc_hi(1024), desc_hi(kGroup)>(sd, q + (ks / 4) * 1024 + (ks % 4) * 2,
                                                                       kd + (ks / 4) * 64 + (ks % 4) * 2, kQK, ks > 0);
                            tc_commit(&bars.s_full[h][k & 1]);
                            if ((!w.pair || h == 1) && ++b == kPairs) b = 0, ph ^= 1;
                        }
                    } else {
#pragma unroll 1
                        for (uint32_t s = 0; s < steps; ++s) {
                            const uint32_t h = s & 1, k = h ? n1++ : n0++;
                            if (!w.pair || h == 0)
                                if (!(ok = wait(&bars.full[2 * b + 1], ph, 51))) break;
                            if (!(ok = wait(&bars.p_ready[h][k & 1], (k >> 1) & 1, 53))) break;
                            tc_fence_after();
                            // P of the tile's last half: its Q K^T is done, and K with it (an
                            // arrive takes a fifth of a commit's time)
                            if (!w.pair || h == 1) mbar_arrive(&bars.empty[2 * b]);
                            const uint32_t v = v_lo + 2 * b * kBufStep, p = tmem + h * 128 + (k & 1) * 64, o = tmem + L::kO + h * D;
                            mma_ts<desc_hi(kGroup)>(o, p, v, kPV, s >= 2);  // the half's first tile of the item starts O
#pragma unroll
                            for (uint32_t ks = 1; ks < kTilePages; ++ks)
                                mma_ts<desc_hi(kGroup)>(o, p + ks * 8, v + ks * (L::kPage >> 4), kPV, 1);
                            tc_commit(&bars.o_done[h][k & 1]);
                            if (!w.pair || h == 1) {
                                tc_commit(&bars.empty[2 * b + 1]);
                                if (++b == kPairs) b = 0, ph ^= 1;
                            }
                        }
                    }
                }
                if (!__all_sync(0xffffffffu, ok)) break;
            }
            // nothing in flight when the tensor memory goes (bounded)
            __syncwarp();
            if (elect_one()) {
                tc_commit(&bars.drain[is_qk]);
                mbar_drain(&bars.drain[is_qk], 0);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- softmax: half h, one thread per row
        const uint32_t h = warp >> 2, r = tid & 127;
        const uint32_t lanes = (warp & 3) * 32;  // this warp's rows: tensor-memory lanes
        const uint32_t ts = tmem + (lanes << 16) + h * 128, to = tmem + (lanes << 16) + L::kO + h * D;
        uint8_t* const qh = qs + h * L::kQ;
        // a scale of 0 is a query of zeros (0 times the -inf of a masked score is NaN)
        const float scale2 = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
        constexpr uint32_t kChunks = D / 8, kStep = 32 / kChunks;  // 16-byte chunks of a row; rows per warp-wide copy
        const uint32_t ch = lane % kChunks, sub = lane / kChunks;
        uint32_t k = 0;  // tiles so far
        bool ok = true;
        // The lengths and this thread's query token of the next item are loaded
        // while the one before ends (its start took 900 clocks for the lengths and
        // 2900 to the query rows in shared memory).
        Work::Lens len;
        uint32_t tok, row_j, row_h;  // token, query of the list, head of the group
        auto ahead = [&] {
            auto at = [&](uint32_t x) { return __shfl_sync(0xffffffffu, word, x); };
            len = Work::lens(a, word, false);
            const uint32_t tok0 = at(2), rows = at(4), rr = at(3) + (rows > 128 ? h * 128 : 0) + r;
            row_j = rr / a.G;
            row_h = rr - row_j * a.G;
            tok = rr - at(3) < rows ? a.row_tok[tok0 + row_j] : 0u;
        };
        ahead();
        for (uint32_t i = i0; i < i1 && ok; ++i) {
            const Work w(a, word, len);
            word = Work::fetch(a, i + 1, i1, lane);
            const uint32_t rbase = w.pair ? h * 128 : 0;
            const uint32_t mine = w.rows > rbase ? min(128u, w.rows - rbase) : 0;  // rows of this half
            const uint32_t cnt = w.count(h);
            const bool has = r < mine;
            const bool idle = lanes >= mine;  // no row of this warp
            // this thread's row of q and out
            const uint32_t at = has ? tok * a.Hq + w.kvh * a.G + row_h : 0u;
            const int32_t lim_pre = has ? static_cast<int32_t>(w.pre_len) : 0;
            const int32_t lim_suf = has ? static_cast<int32_t>(w.limit(row_j)) : 0;
            if (cnt) {
#pragma unroll 1
                for (uint32_t y = sub; y < 32; y += kStep) {
                    const uint64_t row = __shfl_sync(0xffffffffu, at, y);
                    cp_async16_zfill(qh + (ch >> 3) * 16384 + swz128(lanes + y, ch & 7), a.q + row * D + ch * 8,
                                     lanes + y < mine && a.scale != 0.0f);
                }
            }
            // Pages beyond the pool: looked for once per item, while the query rows
            // are on their way (a look at every tile took 130 clocks of it; one that
            // waited for each 8 tiles 4700 of an item of 28), and tile by tile only
            // where there are any.
            bool beyond = false;
#pragma unroll 4
            for (uint32_t t = 0; t < w.n; t += 32 / kTilePages) {
                const uint32_t tl = t + lane / kTilePages, pg = lane % kTilePages;
                const bool in = tl < w.n && w.first(tl) + pg * kBlock < w.length(tl);
                const uint32_t ref = in ? w.refs(a, tl)[pg] & kRefMask : 0u;
                beyond |= in & (ref >= a.pool_blocks);
            }
            if (cnt) {
                cp_async_wait_all();
                if (a.scale < 0.0f) {  // a negative scale goes into Q: each lane flips what it copied
#pragma unroll 1
                    for (uint32_t y = sub; y < 32; y += kStep) {
                        uint4* q = reinterpret_cast<uint4*>(qh + (ch >> 3) * 16384 + swz128(lanes + y, ch & 7));
                        *q = make_uint4(q->x ^ 0x80008000u, q->y ^ 0x80008000u, q->z ^ 0x80008000u, q->w ^ 0x80008000u);
                    }
                }
                fence_proxy_async_shared();
                mbar_arrive(&bars.q_full[h]);
            }
            const bool any_bad = __any_sync(0xffffffffu, beyond);
            float m = -INFINITY, l = 0.0f;
            // Tokens of the tile that this row sees, and that the warp's first row sees:
            // the rows' limits rise with the row, so the first one says whether any row
            // needs the mask.  They fall by a tile's tokens from tile to tile.
            const uint32_t step = w.pair ? 1 : 2;
            uint32_t t = w.pair ? 0 : h;
            int32_t lim = 0, low = 0;
            auto enter = [&] {  // tile t is the half's first of a list
                const int32_t first = static_cast<int32_t>(w.first(t));
                lim = (w.own(t) ? lim_suf : lim_pre) - first;
                low = __shfl_sync(0xffffffffu, lim, 0);
            };
            enter();
            bool ready = false;
#pragma unroll 1
            for (uint32_t j = 0; j < cnt; ++j, ++k) {
                const uint32_t tb = ts + (k & 1) * 64;
                if (!ready && !(ok = row_wait(&bars.s_full[h][k & 1], (k >> 1) & 1, a.status, 56))) break;
                tc_fence_after();
                uint32_t bad = 0;
                if (any_bad) {
                    const bool in = lane < kTilePages && w.first(t) + lane * kBlock < w.length(t);
                    bad = __ballot_sync(0xffffffffu, in && (w.refs(a, t)[in ? lane : 0] & kRefMask) >= a.pool_blocks);
                }
                if (!idle) {
                    float v[64];
                    tc_ld64(tb, v);
                    if (low < static_cast<int32_t>(kTileTokens) || bad) {
#pragma unroll
                        for (int c = 0; c < 64; ++c)
                            if (c >= lim || ((bad >> (c / 16)) & 1u)) v[c] = -INFINITY;
                    }
                    float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int c = 4; c < 60; c += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], v[c + e], v[c + 4 + e]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], v[60 + e]);
                    const float m_new = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * scale2;
                    const bool grow = m_new > m + kTop;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float to_m = grow ? m_new - kBias : m;
                        if (j > 0) {
                            const float f = grow ? ex2(m - to_m) : 1.0f;
                            l *= f;
                            // the previous product has been added before O is rescaled
                            if (!(ok = row_wait(&bars.o_done[h][(k - 1) & 1], ((k - 1) >> 1) & 1, a.status, 57))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                float o[32];
                                tc_ld32(to + c, o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] *= f;
                                tc_st32(to + c, o);
                            }
                        }
                        m = to_m;
                    }
                    const float ms = m == -INFINITY ? 0.0f : m;
                    const float2 sc = make_float2(scale2, scale2), mm = make_float2(-ms, -ms);
                    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                    uint32_t pk[32];
#pragma unroll
                    for (int c = 0; c < 64; c += 2) {
                        float2 x = fma2(make_float2(v[c], v[c + 1]), sc, mm);
                        x = make_float2(ex2(x.x), ex2(x.y));
                        sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], x);
                        const __half2 hp = __floats2half2_rn(x.x, x.y);
                        pk[c / 2] = *reinterpret_cast<const uint32_t*>(&hp);
                    }
                    tc_st32(tb, pk);
                    // the next S is usually there by now; a poll takes 170 clocks, here beside
                    // the store (before the store, which then waits for it, it cost a tenth)
                    const bool next = mbar_test(&bars.s_full[h][(k + 1) & 1], ((k + 1) >> 1) & 1);
                    sum[0] = add2(sum[0], sum[1]);
                    l += sum[0].x + sum[0].y;
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.p_ready[h][k & 1]);
                    ready = __all_sync(0xffffffffu, next);
                } else if (lane == 0) {
                    mbar_arrive(&bars.p_ready[h][k & 1]);
                }
                t += step;
                lim -= static_cast<int32_t>(step * kTileTokens);
                low -= static_cast<int32_t>(step * kTileTokens);
                if (t >= w.n_pre && t < w.n_pre + step) enter();
            }
            if (!ok) break;
            ahead();
            // ---- this half's result
            if (cnt) {
                if (!(ok = row_wait(&bars.o_done[h][(k - 1) & 1], ((k - 1) >> 1) & 1, a.status, 58))) break;
                tc_fence_after();
            }
            if (mine && (w.pair || h == 0 || (w.flags & kPxTwo))) {
                const bool direct = w.flags & kPxDirect;
                const float inv = inverse_sum(l);
                const uint64_t run = w.part_row + (!w.pair && h ? w.rows : 0u);
                if (!direct && has) a.part_ml[run + rbase + r] = make_float2(m * kLn2, l);
                if (!idle) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        if (cnt) {
                            tc_ld32(to + c, o);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = 0.0f;
                        }
                        if (direct) {
                            // f16 rows into this half's Q (its products are done), copied out row by row below
#pragma unroll
                            for (int e = 0; e < 32; e += 8) {
                                uint4 pack;
                                __half2* hp = reinterpret_cast<__half2*>(&pack);
#pragma unroll
                                for (int y = 0; y < 4; ++y)
                                    hp[y] = __floats2half2_rn(o[e + 2 * y] * inv, o[e + 2 * y + 1] * inv);
                                const uint32_t x = (c + e) / 8;
                                *reinterpret_cast<uint4*>(qh + (x >> 3) * 16384 + swz128(r, x & 7)) = pack;
                            }
                        } else if (has) {
                            float4* po = reinterpret_cast<float4*>(a.part_o + run * D) + rbase + r;
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                po[static_cast<uint64_t>((c + e) / 4) * w.rows] =
                                    make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                        }
                    }
                }
                if (direct) {
                    // each warp its own 32 rows: D / 8 lanes write a row's 16-byte chunks
                    __syncwarp();
#pragma unroll 2
                    for (uint32_t y = sub; y < 32; y += kStep) {
                        const uint64_t row = __shfl_sync(0xffffffffu, at, y);
                        if (lanes + y < mine)
                            *reinterpret_cast<uint4*>(a.out + row * D + ch * 8) =
                                *reinterpret_cast<const uint4*>(qh + (ch >> 3) * 16384 + swz128(lanes + y, ch & 7));
                    }
                    __syncwarp();  // the next item's Q goes where the rows were
                }
            }
            tc_fence_before();  // O and S have been read before the next item's products
        }
    }
    // the 16-row tiles' kernel has completed when this one has, for the merge
    if (tid == 0) wait_prerequisites();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D>
constexpr size_t tc_smem() {
    return 1024 + TcLayout<D>::kBytes;
}

template <int D>
cudaError_t launch_tc(const PrefixArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, uint32_t n_ctas, bool after,
                      cudaStream_t s) {
    return launch_pdl(prefix_tc_kernel<D>, dim3(n_ctas), dim3(kTcThreads), tc_smem<D>(), after, s, tm_k, tm_v, a);
}

}  // namespace

cudaError_t prepare_prefix_tc(uint32_t D) {
    return D == 128 ? cudaFuncSetAttribute(prefix_tc_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(tc_smem<128>()))
                    : cudaFuncSetAttribute(prefix_tc_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(tc_smem<64>()));
}

cudaError_t launch_prefix_tc(const PrefixArgs& a, const CUtensorMap& tm_k, const CUtensorMap& tm_v, uint32_t n_ctas, bool after,
                             cudaStream_t s) {
    return a.D == 128 ? launch_tc<128>(a, tm_k, tm_v, n_ctas, after, s) : launch_tc<64>(a, tm_k, tm_v, n_ctas, after, s);
}

}  // namespace weaver
