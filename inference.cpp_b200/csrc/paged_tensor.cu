// ib_attention_paged on tcgen05: head_dim up to 128, tiles of 256 query rows (128 for FP32 pages
// with head_dim over 64) -- the chunks of prompts.
//
// Two query tiles of 128 rows share each key tile.  As on mma.sync, FP32 operands are pairs hi + lo
// and 2^-21 of every product is kept (of a weight on FP16 pages 2^-35 of the row's largest, where that is
// more: it is where FP16 ends):
//   FP16 pages  q and p as FP16 pairs (q scaled to a largest element in [256, 512), p by 2^10),
//               K and V as they are: two MMAs; key tiles of 128 positions
//     S = q_lo K' + q_hi K'      A: q in shared memory, B: K            M 128, N 128
//     O = p_lo V  + p_hi V       A: p in tensor memory, B: V            M 128, N head_dim
//   FP32 pages  both operands as TF32 pairs: three MMAs (lo hi + hi lo + hi hi); key tiles of 64
//               positions, 32 for head_dim over 64
// The tensor core adds to its accumulator by cutting, which over a long sequence would drift; so
// O starts from zero in every key tile and the running sum is kept in registers, one row per
// thread, where acc = acc c + O takes the softmax's rescaling with it.
//
// Tensor memory, 512 columns: S of both query tiles (128 each), O of both (128 each).  p lies
// over its S: FP16, of a chunk of 16 scores a thread writes hi into the first 8 columns and lo into
// the other 8, and an MMA's 16 positions are one chunk; FP32, hi over the scores and lo behind.
// Shared memory: q of both tiles as hi and lo (128 KB) and a ring of slots for K and V tiles in
// turn (three FP16 tiles, or two of FP32 parts and the FP32 tiles as they come).  Rows are 128
// bytes under the 128-byte swizzle; K is read with head_dim along the MMA's K (K-major).  FP16 V is
// read with positions along it (MN-major) and so stored as it lies in the pages; TF32 operands are
// K-major only, so FP32 V is turned round on the way.
// Warps: 0-3 and 4-7 the softmax of a query tile each (thread = row), 8 issues the MMAs, the others
// bring K and V in, with TMA in boxes of as many rows as divide both a page and the tile (a box of
// a page that is not there lies outside the tensor and reads as zeros).  FP16: 9-11, row by row
// where boxes would have fewer than 8 rows.  FP32: 9 by TMA, 10-15 split the parts.  In tiles where some row
// does not see a position, they make V finite before it is used (0 x inf).  The order of MMAs is
//     O0(j) S0(j+1) O1(j) S1(j+1) O0(j+1) ...
// so that a tile's softmax has the other tile's MMAs to hide behind, and FP16 O begins with the
// second half of the positions while p of the first is computed (435 us without, 415 with).
// Work per CTA is a piece of the batch (paged_plan.cuh); the copies run on into the next
// segment.
//
// Trees of drafted tokens mostly fill less than one query tile, so for them there is a second shape
// (SPLIT): one query tile, whose key tiles the two softmax groups take in turn, each with a maximum, a
// sum and an accumulator of its own.  A group's softmax has the other group's MMAs to hide behind, as
// above.  At a segment's end the second group hands its maximum and sum over and the first one, which has
// a thread for the same rows and so the same lanes of tensor memory, writes the results, while the second
// one brings in the next segment's q.  The half of q that the other query tile would take goes to the
// ring (five slots of FP16, four of FP32), and the copies bring K a tile ahead of V.  In tiles behind the
// context a position counts where the node's bit is set.
//
// Measured, trees: 32 of 12 to 24 nodes over 200 .. 4096 positions (32 heads on 8, head_dim 128, FP16) 127
// to 132 us with the join, 332 MB at 2.6 TB/s (232 with the kernel for chunks); tensor pipe 0.35, issue
// 0.35; 100 of 8 to 24 over 50 .. 900 163 us (180 while each role looked its segments up like the first).  A key tile takes 3.9k cycles to its 2.05k of MMAs: its scores, softmax (3.5k) and weighted
// sum are a chain, and two groups hide half of it; a segment's beginning and end take 20k more, 1.7 of
// them to a CTA.  Two documents of 33 to 63 nodes over 20001 .. 32000 (32 heads on 4, head_dim 64, FP32)
// 182 us with two query tiles, 203 with one; tensor pipe 0.40.
//
// Measured, chunks: 2048 tokens behind 6144 (32 heads on 8, head_dim 128, FP16) 471 us, 1020 TFLOP/s of
// MMAs, 0.63 of the measured rate of library FP16 products (421 to 427 us in runs of a few
// milliseconds, before the power limit lowers the clock), and 299 us at head_dim 64; the tensor pipe
// is busy 0.60 of the cycles.  A step of both query tiles takes 6.3k cycles to the MMAs' 4.1k: the bound is the softmax
// between a tile's S and its p, 3.8k cycles of dependent instructions with two warps to a scheduler
// (a row's running sums in one thread leave registers for no more), which only half overlaps.  FP32
// pages at head_dim 64: a step of 6.3k cycles to 4.6k; 8.4k while the warp that starts the copies
// split them too.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "lookup.h"
#include "mma_tile.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "paged_ring.h"
#include "pdl.cuh"
#include "pipeline.cuh"

namespace ib {

int paged_tensor_fault_take(int* code) { return paged_fault_take_here(code); }

// A bad table entry and then a wait for an arrival that nobody makes.
__global__ void wait_selftest_kernel() {
    __shared__ uint64_t bar;
    mbar_init(&bar, 1);
    fence_mbar_init();
    paged_fault(PAGED_BAD_PAGE);
    mbar_wait(&bar, 0, &g_paged_faults.wait, PAGED_BAD_WAIT, 256);
}

// SPLIT (trees): one query tile, whose key tiles the two groups of softmax warps take in turn.
template <typename KV, int HDP, bool SPLIT>
struct TensorCfg {
    static constexpr bool F32 = sizeof(KV) == 4;
    static constexpr int QT = SPLIT || (F32 && HDP == 128) ? 1 : 2;  // query tiles of 128 rows
    static constexpr int R = 128 * QT;
    static constexpr int KT = !F32 ? 128 : HDP == 64 ? 64 : 32;  // positions of a key tile
    static constexpr int EB = F32 ? 4 : 2;                       // bytes of an operand element
    static constexpr int ROW = 128 / EB;                         // elements of a swizzled row
    static constexpr int Q_PLANE = 128 * HDP * EB;               // hi or lo of a query tile
    static constexpr int PLANE = KT * HDP * EB;                  // a K or V tile, or its hi or lo
    static constexpr int TILE = F32 ? 2 * PLANE : PLANE;         // a ring slot
    static constexpr int SLOTS = !SPLIT ? (F32 ? 2 : 3) : F32 ? (HDP == 64 ? 4 : 2) : HDP == 64 ? 6 : 5;
    static constexpr int RECENT = SPLIT ? 8 : 4;                 // key tiles whose masks are kept
    // tensor memory's columns for two more values of the second group's rows: behind its O, or its p
    static constexpr int ML = HDP == 64 ? 256 + 128 + 64 : F32 ? 128 + 2 * KT : -1;
    static constexpr int RAW = F32 ? 2 * PLANE : 0;              // FP32 K and V as they come
    static constexpr int Q_BLOCK = 128 * 128;                    // ROW columns of a query tile
    static constexpr int K_BLOCK = KT * 128;                     // and of a K tile
    // V: FP16 as it lies (K_BLOCK: 64 dimensions of all positions), FP32 turned round (32
    // positions of all dimensions)
    static constexpr int V_BLOCK = F32 ? HDP * 128 : K_BLOCK;
    // warps that fill ring slots: copies (FP16), or splitting what warp 9 brings in (FP32)
    static constexpr int SPLIT_WARPS = 6, FILL_WARPS = F32 ? SPLIT_WARPS : 3;
    static constexpr int WARPS = F32 ? 10 + FILL_WARPS : 9 + FILL_WARPS, THREADS = 32 * WARPS;
    // registers of the softmax warps and of the others, within what the launch has
    static constexpr int MANY = F32 ? 184 : 224, FEW = F32 ? 72 : 56;
    static_assert(256 * MANY + (THREADS - 256) * FEW <= THREADS * (65536 / THREADS / 8 * 8), "");
    static constexpr size_t SMEM = QT * 2 * Q_PLANE + SLOTS * TILE + RAW;
};

// ---- tcgen05 ---------------------------------------------------------------------------
__device__ __forceinline__ void pt_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void pt_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void pt_fence_async() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// 128-byte swizzle (layout type 2), 8-row groups 1024 bytes apart, sm_100 descriptor (version
// 1).  K-major: a row's 128 bytes lie along K.  MN-major (FP16): they lie along the MN dimension,
// its next 64 elements `lead` bytes on, and the groups of eight rows run along K.
__device__ __forceinline__ uint64_t pt_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// D FP32, A and B FP16 (kind::f16) or TF32 (kind::tf32); b_mn: B is MN-major.
constexpr uint32_t pt_idesc(int M, int N, bool b_mn, bool tf32 = false) {
    return (1u << 4) | (tf32 ? 2u << 7 | 2u << 10 : 0u) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

// The whole warp comes here with the same operands and `leader` lets one thread issue.  (The loops
// around it are kept short: unrolled, 64 MMAs missed the instruction cache and took 134 cycles each
// instead of 64.)
template <bool TF32>
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t add, uint32_t leader) {
    if constexpr (TF32)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "setp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "setp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
            : "memory");
}
template <bool TF32>
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                          uint32_t add, uint32_t leader) {
    if constexpr (TF32)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "setp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "setp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
            : "memory");
}

__device__ __forceinline__ void pt_commit(uint64_t* bar, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(
            smem_u32(bar)),
        "r"(leader)
        : "memory");
}

// One thread of the (converged) warp.
__device__ __forceinline__ uint32_t pt_elect() {
    uint32_t x;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(x));
    return x;
}

// 32 columns of this warp's 32 lanes; the wait is part of the statement, so that nothing uses the
// registers before it.
__device__ __forceinline__ void pt_read32(uint32_t at, float (&a)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
        "%28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(a[0]), "=f"(a[1]), "=f"(a[2]), "=f"(a[3]), "=f"(a[4]), "=f"(a[5]), "=f"(a[6]),
          "=f"(a[7]), "=f"(a[8]), "=f"(a[9]), "=f"(a[10]), "=f"(a[11]), "=f"(a[12]), "=f"(a[13]),
          "=f"(a[14]), "=f"(a[15]), "=f"(a[16]), "=f"(a[17]), "=f"(a[18]), "=f"(a[19]),
          "=f"(a[20]), "=f"(a[21]), "=f"(a[22]), "=f"(a[23]), "=f"(a[24]), "=f"(a[25]),
          "=f"(a[26]), "=f"(a[27]), "=f"(a[28]), "=f"(a[29]), "=f"(a[30]), "=f"(a[31])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ float2 pt_read2(uint32_t at) {
    float2 x;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0, %1}, [%2];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(x.x), "=f"(x.y)
        : "r"(at)
        : "memory");
    return x;
}
__device__ __forceinline__ void pt_st2(uint32_t at, float x, float y) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(at), "f"(x), "f"(y)
                 : "memory");
}
__device__ __forceinline__ void pt_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// Two FP32 operations in one instruction: x = a b + c and x + a, element by element.
__device__ __forceinline__ void fma2(float& x0, float& x1, float a0, float a1, float b0, float b1,
                                     float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 c, a, b, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t}"
        : "=f"(x0), "=f"(x1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void add2(float& x0, float& x1, float a0, float a1) {
    asm("{\n\t.reg .b64 a, c;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 c, {%0, %1};\n\t"
        "add.rn.f32x2 c, a, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t}"
        : "+f"(x0), "+f"(x1)
        : "f"(a0), "f"(a1));
}
// x - h, exact where h is x rounded
__device__ __forceinline__ float less_half(float x, __half h) {
    const uint16_t u = __half_as_ushort(h);
    float y;
    asm("{\n\t.reg .b16 m;\n\t"
        "mov.b16 m, 0xbc00;\n\t"  // -1
        "fma.rn.f32.f16 %0, %1, m, %2;\n\t}"
        : "=f"(y)
        : "h"(u), "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float x;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(x) : "f"(a), "f"(b), "f"(c));
    return x;
}

// Byte offset of 16-byte chunk c (0-7) of row r in a swizzled block.
__device__ __forceinline__ uint32_t pt_off(int r, int c) {
    return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}

// 2-D tiled TMA load (no multicast) of the box at (x = column, y = row), completing on bar.  x is
// a multiple of 64 FP16 (128 bytes).
__device__ __forceinline__ void pt_tma(uint32_t dst, const CUtensorMap* map, int x, int y,
                                       uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

struct TensorArgs {
    RowsArgs rows;
    CUtensorMap k, v;  // the layer's rows [page, kv head, position in page][head_dim]
    int box;           // log2 of a box's rows; FP16: 0 for no TMA
};

template <int SLOTS>
struct TensorBars {
    uint64_t kv_full[SLOTS], kv_empty[SLOTS], raw_full[2], raw_empty[2];
    uint64_t q_full[2], s_full[2], p_half[2], p_full[2], o_full[2], seg_done[2], v_there[SLOTS], done;
    uint64_t x_there, x_done;  // the second group's sums are in tensor memory; have been read
};

template <typename KV, int HDP, bool TREE, bool SPLIT>
__global__ void __launch_bounds__(TensorCfg<KV, HDP, SPLIT>::THREADS, 1)
    attn_tensor_kernel(const __grid_constant__ TensorArgs TA) {
    const RowsArgs& A = TA.rows;
    using C = TensorCfg<KV, HDP, SPLIT>;
    constexpr bool F32 = C::F32;
    constexpr int KT = C::KT;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) TensorBars<C::SLOTS> bar;
    __shared__ uint32_t tmem_base;
    // the same one for each warp, out of its registers
    __shared__ std::conditional_t<TREE, Following, Piece> sh_piece[C::WARPS];
    Piece* piece;
    if constexpr (TREE) {
        __shared__ Piece one;
        piece = &one;
    } else {
        piece = sh_piece;
    }
    __shared__ int found;
    // of the last key tiles: positions without a page; positions whose V is not finite
    constexpr int RECENT = C::RECENT;
    __shared__ __align__(16) uint16_t sh_gone[RECENT][8];
    __shared__ __align__(16) uint16_t sh_bad[F32 ? 1 : RECENT][8];
    __shared__ uint32_t sh_bad32[F32 ? RECENT : 1][C::SPLIT_WARPS][2];  // the same for FP32, of each splitting warp
    __shared__ uint8_t sh_scale[2][SPLIT && !F32 ? 128 : 1];  // of the segment's rows (exponents), see ScaleTurn
    // the second group's maximum and sum, where tensor memory has no columns left for them
    __shared__ float2 sh_ml[SPLIT && C::ML < 0 ? 128 : 1];
    const PagedView& w = A.w;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (!A.beside) pdl_wait();
    pdl_launch_dependents();
    find_piece<C::THREADS>(w, A.rule, blockIdx.x, piece, &found);
    __syncthreads();
    if (!found) {
        if (A.beside) pdl_wait();
        return;
    }
    if constexpr (!TREE) {
        if (tid > 0 && tid < C::WARPS) sh_piece[tid] = sh_piece[0];
    }
    const uint32_t base = smem_u32(smem_raw);  // on a boundary of 1024 bytes, for the swizzle
    uint8_t* const base_ptr = smem_raw;
    if (tid == 0) {
        if (F32 || TA.box) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&TA.k)) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&TA.v)) : "memory");
        }
        // SPLIT with TMA: one arrival, of the warp that sees to the tile
        const int fill = SPLIT && !F32 && TA.box ? 1 : 33 * C::FILL_WARPS;
        for (int i = 0; i < C::SLOTS; ++i) {
            mbar_init(&bar.kv_full[i], fill);
            mbar_init(&bar.kv_empty[i], 1);
            mbar_init(&bar.v_there[Looks::bar(i)], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.raw_full[i], 1);
            mbar_init(&bar.raw_empty[i], C::FILL_WARPS);
            mbar_init(&bar.q_full[i], 128);
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], 128);
            mbar_init(&bar.p_half[i], 128);
            mbar_init(&bar.o_full[i], 1);
            mbar_init(&bar.seg_done[i], 128);
        }
        mbar_init(&bar.x_there, 128);
        mbar_init(&bar.x_done, 128);
        mbar_init(&bar.done, 1);
        fence_mbar_init();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&tmem_base)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pt_fence_before();
    __syncthreads();
    pt_fence_after();
    const uint32_t tmem = tmem_base;
    const uint32_t ring = base + C::QT * 2 * C::Q_PLANE;
    const int G = w.H / w.Hkv, HD = w.HD;
    Segment it;
    auto next = [&]() -> bool {
        auto p = sh_piece[warp];
        bool more;
        if constexpr (TREE) more = following_segment(w, A.rule, p, it);
        else more = next_segment<false>(w, A.rule, p, it);
        __syncwarp();
        if (lane == 0) sh_piece[warp] = p;
        __syncwarp();
        return more;
    };
    // For the n-th completion, from 0; the same answer in a whole warp.  Every wait is bounded: a
    // role whose wait expired leaves its loop, and so do, one wait later, those that wait for it.
    auto wait = [&](uint64_t* b, int n) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(b, (uint32_t)(n & 1), &g_paged_faults.wait, PAGED_BAD_WAIT));
    };

    // The first segment here, for all roles: its code is brought in once.
    bool first = false;
    if constexpr (TREE) {
        Piece p = *piece;
        first = next_segment<true>(w, A.rule, p, it);
        if (lane == 0 && first) sh_piece[warp] = following(w, A.rule, p, it);
        __syncwarp();
    }
    auto go_on = [&](bool& begun) -> bool {  // `begun`: false at a role's beginning
        if (!TREE || begun) return next();
        begun = true;
        return first;
    };
    if (warp < 8) {
        // ---- softmax of query tile t: thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::MANY));
        const int t = warp >> 2, wr = (warp & 3) * 32;  // this warp's rows of the tile, its lanes
        // SPLIT: both groups have the tile's rows.  The second one has key tiles 0, 2 .., the first one
        // 1, 3 ..; the second one's sums go to the first through tensor memory, where both reach the same
        // lanes, and the first one writes the results while the second brings in the next segment's q and
        // begins with it.
        const int qt = SPLIT ? 0 : t, j0 = SPLIT ? 1 - t : 0;
        constexpr int DJ = SPLIT ? 2 : 1;
        uint8_t* const q_ptr = base_ptr + 2 * qt * C::Q_PLANE;
        const uint32_t s_at = tmem + ((uint32_t)wr << 16) + (uint32_t)(128 * t);
        const uint32_t o_at = tmem + ((uint32_t)wr << 16) + (uint32_t)(256 + 128 * t);
        [[maybe_unused]] const uint32_t ml_at = tmem + ((uint32_t)wr << 16) + (uint32_t)C::ML;
        int tiles = 0;      // key tiles so far, of all segments
        if constexpr (!TREE) first = next();
        uint32_t seen = 0;  // and counted as the copies do (both groups')
        // SPLIT: the first group's key tiles so far, the one that used q last
        [[maybe_unused]] int firsts = 0, q_used = -1, exchanges = 0;
        [[maybe_unused]] ScaleTurn segs;
        bool ok = true;
        const float sign = A.scale_log2 < 0.f ? -1.f : 1.f;
        // The segment's q into this warp's 32 rows of the tile, HDP / 8 lanes to a row; returns the
        // factor of row `lane`.  The last segment's scores are done (this warp has read some), so
        // nothing reads the rows any more.  All of q is on its way at once, into the places of the
        // parts that are made of it.
        auto stage_q = [&](const Segment& sg) -> float {
            constexpr int LPR = HDP / 8, RPI = 32 / LPR;
            const int rows = sg.rows - 128 * qt, d = (lane % LPR) * 8;
            float mine = F32 ? 1.f : 0.f;
            if (rows <= 0 || sg.kt0 == sg.kt1) return mine;
            // 16 bytes of the values d .. of row r: FP16 hi, lo; FP32 the first four's hi, the others'
            // (their lo parts Q_PLANE behind)
            auto place = [&](int r, int d, int half) -> uint32_t {
                if constexpr (F32)
                    return (uint32_t)((d >> 5) * C::Q_BLOCK) + pt_off(r, ((d & 31) >> 2) + half);
                else
                    return (uint32_t)((d >> 6) * C::Q_BLOCK + half * C::Q_PLANE) + pt_off(r, (d & 63) >> 3);
            };
            const uint32_t q_a = base + (uint32_t)(2 * qt * C::Q_PLANE);
            constexpr int CPR = HDP / 4, RPC = 32 / CPR;  // 16-byte chunks of a row, rows at a time
            const int dc = (lane % CPR) * 4;
            const int64_t per_token = A.q_stride - (int64_t)G * HD;  // rows of a token are consecutive
            const float* const q0 = A.q + (int64_t)sg.s.q0 * A.q_stride + (int64_t)sg.hk * G * HD + dc;
            const int first_row = sg.row0 + 128 * qt;
            const FastDiv group = w.group;
#pragma unroll 4
            for (int i = 0; i < 32; i += RPC) {
                const int r = wr + i + lane / CPR, row = first_row + r;
                const bool there = r < rows && dc < HD;
                const int64_t at = (int64_t)row * HD + (int64_t)group.div((uint32_t)row) * per_token;
                cp16(q_a + place(r, dc & ~7, (dc >> 2) & 1), q0 + (there ? at : 0), there);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
#pragma unroll 2
            for (int i = 0; i < 32; i += RPI) {
                const int r = wr + i + lane / LPR;
                uint4* const at0 = reinterpret_cast<uint4*>(q_ptr + place(r, d, 0));
                uint4* const at1 = reinterpret_cast<uint4*>(q_ptr + place(r, d, 1));
                const float4 x0 = *reinterpret_cast<const float4*>(at0);
                const float4 x1 = *reinterpret_cast<const float4*>(at1);
                uint4 h, l;
                if constexpr (F32) {
                    split_tf32(x0.x * sign, h.x, l.x), split_tf32(x0.y * sign, h.y, l.y);
                    split_tf32(x0.z * sign, h.z, l.z), split_tf32(x0.w * sign, h.w, l.w);
                    *at0 = h, at0[C::Q_PLANE / 16] = l;
                    split_tf32(x1.x * sign, h.x, l.x), split_tf32(x1.y * sign, h.y, l.y);
                    split_tf32(x1.z * sign, h.z, l.z), split_tf32(x1.w * sign, h.w, l.w);
                    *at1 = h, at1[C::Q_PLANE / 16] = l;
                } else {
                    float top = fmaxf(fmaxf(fmaxf(fabsf(x0.x), fabsf(x0.y)), fmaxf(fabsf(x0.z), fabsf(x0.w))),
                                      fmaxf(fmaxf(fabsf(x1.x), fabsf(x1.y)), fmaxf(fabsf(x1.z), fabsf(x1.w))));
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    float down;
                    const float up = pow2_scale(top, down) * sign;
                    split2(x0.x * up, x0.y * up, h.x, l.x), split2(x0.z * up, x0.w * up, h.y, l.y);
                    split2(x1.x * up, x1.y * up, h.z, l.z), split2(x1.z * up, x1.w * up, h.w, l.w);
                    *at0 = h, *at1 = l;
                    const float f = __shfl_sync(0xffffffffu, down, ((lane - i) & (RPI - 1)) * LPR);
                    if (lane >= i && lane < i + RPI) mine = f;
                }
            }
            pt_fence_async();
            mbar_arrive(&bar.q_full[qt]);
            return mine;
        };
        // SPLIT: by the second group, whose registers are free then, the rows that there are spread over
        // its warps (the others' scores are not used).  The rows' factors, powers of two, go to sh_scale.
        [[maybe_unused]] auto stage_split = [&](const Segment& sg, int buffer) {
            // (small loops: it is met once a segment, and its instructions come from far then)
            constexpr int LPR = HDP / 8, RPI = 32 / LPR, CPR = HDP / 4, RPC = 32 / CPR;
            if (sg.kt0 == sg.kt1) return;
            const int d = (lane % LPR) * 8, dc = (lane % CPR) * 4, w4 = warp & 3;
            // 16 bytes of the values d .. of row r: FP16 hi, lo; FP32 the first four's hi, the others'
            // (their lo parts Q_PLANE behind)
            auto place = [&](int r, int d, int half) -> uint32_t {
                if constexpr (F32)
                    return (uint32_t)((d >> 5) * C::Q_BLOCK) + pt_off(r, ((d & 31) >> 2) + half);
                else
                    return (uint32_t)((d >> 6) * C::Q_BLOCK + half * C::Q_PLANE) + pt_off(r, (d & 63) >> 3);
            };
            const int64_t per_token = A.q_stride - (int64_t)G * HD;  // rows of a token are consecutive
            const float* const q0 = A.q + (int64_t)sg.s.q0 * A.q_stride + (int64_t)sg.hk * G * HD + dc;
            const FastDiv group = w.group;
            // warp w4 has rows RPI (w4 + 4 i) .. + RPI
#pragma unroll 1
            for (int r0 = w4 * RPI; r0 < sg.rows; r0 += 4 * RPI)
#pragma unroll
                for (int i = 0; i < RPI; i += RPC) {
                    const int r = r0 + i + lane / CPR, row = sg.row0 + r;
                    const bool there = r < sg.rows && dc < HD;
                    const int64_t at = (int64_t)row * HD + (int64_t)group.div((uint32_t)row) * per_token;
                    cp16(base + place(r, dc & ~7, (dc >> 2) & 1), q0 + (there ? at : 0), there);
                }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
#pragma unroll 1
            for (int r0 = w4 * RPI; r0 < sg.rows; r0 += 4 * RPI) {
                const int r = r0 + lane / LPR;
                uint4* const at0 = reinterpret_cast<uint4*>(q_ptr + place(r, d, 0));
                uint4* const at1 = reinterpret_cast<uint4*>(q_ptr + place(r, d, 1));
                const float4 x0 = *reinterpret_cast<const float4*>(at0);
                const float4 x1 = *reinterpret_cast<const float4*>(at1);
                uint4 h, l;
                if constexpr (F32) {
                    split_tf32(x0.x * sign, h.x, l.x), split_tf32(x0.y * sign, h.y, l.y);
                    split_tf32(x0.z * sign, h.z, l.z), split_tf32(x0.w * sign, h.w, l.w);
                    *at0 = h, at0[C::Q_PLANE / 16] = l;
                    split_tf32(x1.x * sign, h.x, l.x), split_tf32(x1.y * sign, h.y, l.y);
                    split_tf32(x1.z * sign, h.z, l.z), split_tf32(x1.w * sign, h.w, l.w);
                    *at1 = h, at1[C::Q_PLANE / 16] = l;
                } else {
                    float top = fmaxf(fmaxf(fmaxf(fabsf(x0.x), fabsf(x0.y)), fmaxf(fabsf(x0.z), fabsf(x0.w))),
                                      fmaxf(fmaxf(fabsf(x1.x), fabsf(x1.y)), fmaxf(fabsf(x1.z), fabsf(x1.w))));
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    float down;
                    const float up = pow2_scale(top, down) * sign;
                    split2(x0.x * up, x0.y * up, h.x, l.x), split2(x0.z * up, x0.w * up, h.y, l.y);
                    split2(x1.x * up, x1.y * up, h.z, l.z), split2(x1.z * up, x1.w * up, h.w, l.w);
                    *at0 = h, *at1 = l;
                    if (d == 0) sh_scale[buffer][r] = (uint8_t)(__float_as_uint(down) >> 23);
                }
            }
            pt_fence_async();
            mbar_arrive(&bar.q_full[0]);
        };
        bool more = first;
        float next_scale = 1.f;
        if (!SPLIT && more) next_scale = stage_q(it);
        while (ok && more) {
            const Segment cur = it;
            const int n_kt = cur.kt1 - cur.kt0;
            const int rows = cur.rows - 128 * qt;  // of this query tile
            const uint32_t first = seen;
            seen += (uint32_t)n_kt;
            if constexpr (SPLIT) {
                if (t == 1) {
                    // q's place is free once the last segment's scores are done, where the first group's came
                    // last: this group has waited for its own
                    if (q_used >= 0) ok = wait(&bar.s_full[0], q_used);
                    q_used = -1;
                    if (ok) stage_split(cur, segs.buffer());
                }
                firsts += n_kt / 2;
                if (n_kt > 0 && !(n_kt & 1)) q_used = firsts - 1;
            }
            // scores are multiplied by this; kept off zero, where -inf would turn into NaN
            float sc = fmaxf(fabsf(A.scale_log2) * next_scale, 1e-37f);
            if (!SPLIT && rows <= 0) {
                more = next();
                if (more) next_scale = stage_q(it);
                continue;
            }
            const int r = wr + lane;
            const int row = cur.row0 + 128 * qt + r;  // of the sequence
            const int lim = r < rows ? cur.start + (int)w.group.div((uint32_t)row) : -1;
            const int first_lim = all_see<TREE>(cur.start, cur.row0 + 128 * qt, G);
            [[maybe_unused]] const uint32_t* nodes = nullptr;
            if constexpr (TREE) nodes = mask_row(A, cur.s.q0, row, r < rows);
            float acc[HDP];
#pragma unroll
            for (int d = 0; d < HDP; ++d) acc[d] = 0.f;
            float m = -INFINITY, l = 0.f, c_last = 1.f;
            // SPLIT: sc, from what the second group has left
            [[maybe_unused]] auto row_scale = [&]() -> float {
                if constexpr (!SPLIT || F32) return sc;
                else
                    return fmaxf(fabsf(A.scale_log2) * __uint_as_float((uint32_t)sh_scale[segs.buffer()][r] << 23),
                                 1e-37f);
            };
            // trees: the masks' bits of the key tile, read ahead of its scores; they serve until its O
            [[maybe_unused]] uint32_t tree_see[TREE ? KT / 32 : 1];
            // positions of key tile j (of the segment) that this row sees and that have a page
            auto visible = [&](int j, int word) -> uint32_t {
                const int n = lim + 1 - ((cur.kt0 + j) * KT + 32 * word);
                uint32_t below = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
                if constexpr (TREE) {
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i)
                        if (i == word) below &= tree_see[i];
                }
                const uint16_t* gone = sh_gone[(first + j) & (RECENT - 1)];
                return below & ~((uint32_t)gone[2 * word] | ((uint32_t)gone[2 * word + 1] << 16));
            };
            // O of key tile j into the running sum
            auto add_o = [&](int j) {
                ok = wait(&bar.o_full[t], tiles - 1) && ok;
                pt_fence_after();
#pragma unroll
                for (int d0 = 0; d0 < HDP; d0 += 32) {
                    float o[32];
                    pt_read32(o_at + d0, o);
#pragma unroll
                    for (int d = 0; d < 32; d += 2) {
                        float* a = acc + d0 + d;
                        fma2(a[0], a[1], a[0], a[1], c_last, c_last, o[d], o[d + 1]);
                    }
                }
                if ((cur.kt0 + j) * KT + KT - 1 > all_see<TREE>(cur.start, cur.row0, G)) {
                    // where some row does not see all of the tile, V was made finite: rows that
                    // see such a position are not
                    const uint16_t* bad16 = sh_bad[(first + j) & (RECENT - 1)];
                    const auto& bad32 = sh_bad32[(first + j) & (RECENT - 1)];
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i) {
                        uint32_t bad;
                        if constexpr (F32) {
                            bad = 0;
#pragma unroll
                            for (int k = 0; k < C::SPLIT_WARPS; ++k) bad |= bad32[k][i];
                        }
                        else bad = (uint32_t)bad16[2 * i] | ((uint32_t)bad16[2 * i + 1] << 16);
                        if (visible(j, i) & bad) l = NAN;
                    }
                }
            };
            // (each step of the code has one place: a CTA meets it for the first time a few times only, and
            // its instructions come from far then)
            for (int j = j0;; j += DJ) {
                const bool end = j >= n_kt || !ok;
                if (end) {
                    more = next();
                    // the next segment's q goes in while the last O is computed; its first scores follow
                    if (!SPLIT && more) next_scale = stage_q(it);
                }
                if (j > j0 && ok) add_o(j - DJ);
                if (end) break;
                if constexpr (TREE) {
                    const int p0 = (cur.kt0 + j) * KT;
#pragma unroll
                    for (int i = 0; i < KT / 32; ++i)
                        tree_see[i] = p0 + KT > cur.start ? tree_bits(nodes, A.words, p0 + 32 * i - cur.start)
                                                          : 0xffffffffu;
                }
                ok = wait(&bar.s_full[t], tiles) && ok;
                ++tiles;
                pt_fence_after();
                if (SPLIT && j == j0) sc = row_scale();
                bool all = (cur.kt0 + j) * KT + KT - 1 <= first_lim && r < rows;
                {
                    const uint4 gone = *reinterpret_cast<const uint4*>(sh_gone[(first + j) & (RECENT - 1)]);
                    all = all && (gone.x | (KT > 32 ? gone.y : 0) | (KT > 64 ? gone.z | gone.w : 0)) == 0;
                }
                all = __all_sync(0xffffffffu, all);
                auto mask = [&](float (&s)[32], int i) {
                    const uint32_t see = visible(j, i);
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (!((see >> k) & 1)) s[k] = -INFINITY;
                };
                // The row's maximum, 32 columns at a time; the last ones stay for below.  (Small loops:
                // the softmax shares the instruction cache with the MMAs' thread.)
                float top = -INFINITY;
                float sv[32];
#pragma unroll 1
                for (int i = 0; i < KT / 32; ++i) {
                    pt_read32(s_at + 32 * i, sv);
                    if (!all) mask(sv, i);
                    float top1 = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        top = max3(top, sv[k], sv[k + 1]);
                        top1 = max3(top1, sv[k + 2], sv[k + 3]);
                    }
                    top = fmaxf(top, top1);
                }
                top = fmaxf(m, top);  // of the scores before scaling
                const bool none = top == -INFINITY;
                const float c = none ? 1.f : ex2((m - top) * sc);
                // (FP32: rounded down, so that no p is above 1, which the largest V values need)
                const float off = none ? 0.f : F32 ? __fmul_rd(-top, sc) : fmaf(-top, sc, 10.f);
                m = top;
                float sum0 = 0.f, sum1 = 0.f;
#pragma unroll 1
                for (int i = KT / 32 - 1; i >= 0; --i) {
                    if (i < KT / 32 - 1) {
                        pt_read32(s_at + 32 * i, sv);
                        if (!all) mask(sv, i);
                    }
#pragma unroll
                    for (int c16 = 0; c16 < 2; ++c16) {
                        const float* const s = sv + 16 * c16;
                        if constexpr (F32) {  // hi over the scores, lo KT columns on
                            uint32_t hi[16], lo[16];
#pragma unroll
                            for (int k = 0; k < 16; k += 2) {
                                float x, y;
                                fma2(x, y, s[k], s[k + 1], sc, sc, off, off);
                                x = ex2(x), y = ex2(y);
                                add2(sum0, sum1, x, y);
                                split_tf32_weight(x, hi[k], lo[k]);
                                split_tf32_weight(y, hi[k + 1], lo[k + 1]);
                            }
                            pt_st16(s_at + 32 * i + 16 * c16, hi);
                            pt_st16(s_at + KT + 32 * i + 16 * c16, lo);
                        } else {
                            uint32_t hl[16];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                float x, y;
                                fma2(x, y, s[2 * k], s[2 * k + 1], sc, sc, off, off);
                                x = ex2(x), y = ex2(y);
                                add2(sum0, sum1, x, y);
                                const __half2 h = __floats2half2_rn(x, y);
                                x = less_half(x, __low2half(h)), y = less_half(y, __high2half(h));
                                const __half2 r = __floats2half2_rn(x, y);
                                hl[k] = *reinterpret_cast<const uint32_t*>(&h);
                                hl[8 + k] = *reinterpret_cast<const uint32_t*>(&r);
                            }
                            pt_st16(s_at + 32 * i + 16 * c16, hl);
                        }
                    }
                    if (!F32 && i == KT / 64) {  // half of p: O can begin
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        pt_fence_before();
                        mbar_arrive(&bar.p_half[t]);
                    }
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                l = fmaf(l, c, sum0 + sum1);
                c_last = c;
                pt_fence_before();
                mbar_arrive(&bar.p_full[t]);
            }
            if (n_kt > j0 && ok) mbar_arrive(&bar.seg_done[t]);
            if constexpr (SPLIT) {
                if (n_kt > 0 && ok) {
                    if (t == 1) {
#pragma unroll
                        for (int d0 = 0; d0 < HDP; d0 += 16) {
                            uint32_t y[16];
#pragma unroll
                            for (int d = 0; d < 16; ++d) y[d] = __float_as_uint(acc[d0 + d]);
                            pt_st16(o_at + d0, y);
                        }
                        if constexpr (C::ML < 0) sh_ml[r] = make_float2(m, l);
                        else pt_st2(ml_at, m, l);
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        pt_fence_before();
                        mbar_arrive(&bar.x_there);
                    } else {
                        ok = wait(&bar.x_there, exchanges++);
                        pt_fence_after();
                        sc = row_scale();  // (it may have had no key tile)
                        float2 y;
                        if constexpr (C::ML < 0) y = sh_ml[r];
                        else y = pt_read2(ml_at);
                        const float top = fmaxf(m, y.x);
                        const float f = top == -INFINITY ? 1.f : ex2((m - top) * sc);
                        const float g = top == -INFINITY ? 1.f : ex2((y.x - top) * sc);
                        m = top;
                        l = l * f + y.y * g;
#pragma unroll
                        for (int d0 = 0; d0 < HDP; d0 += 32) {
                            float o[32];
                            pt_read32(o_at + 128 + d0, o);
#pragma unroll
                            for (int d = 0; d < 32; ++d) acc[d0 + d] = fmaf(acc[d0 + d], f, o[d] * g);
                        }
                        pt_fence_before();
                        mbar_arrive(&bar.x_done);
                    }
                }
                segs.next(n_kt);
                if (t == 1) continue;
            }
            if (r < rows && ok) {  // a row per thread
                const bool whole = cur.part < 0;
                const int64_t at = (int64_t)cur.part * C::R + 128 * qt + r;
                const float f = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
                float* p = whole ? out_row(A, cur, G, row) : part_at(A, cur.part, 128 * qt + r, 0);
                const int step = whole ? 4 : 4 * C::R;
                if (SPLIT && whole && A.sectors) {  // whole sectors of 32 bytes
#pragma unroll
                    for (int d = 0; d < HDP; d += 8, p += 8)
                        if (d < HD)
                            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p),
                                         "f"(acc[d] * f), "f"(acc[d + 1] * f), "f"(acc[d + 2] * f),
                                         "f"(acc[d + 3] * f), "f"(acc[d + 4] * f), "f"(acc[d + 5] * f),
                                         "f"(acc[d + 6] * f), "f"(acc[d + 7] * f)
                                         : "memory");
                } else {
#pragma unroll
                    for (int d = 0; d < HDP; d += 4, p += step)
                        if (d < HD)
                            *reinterpret_cast<float4*>(p) =
                                make_float4(acc[d] * f, acc[d + 1] * f, acc[d + 2] * f, acc[d + 3] * f);
                }
                if (!whole) A.part_ml[at] = make_float2(m * sc, l);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::FEW));
        if (warp == 8) {
            // ---- MMAs ----
            constexpr uint32_t id_s = pt_idesc(128, KT, false, F32), id_o = pt_idesc(128, HDP, !F32, F32);
            int half = 0;               // K and V tiles so far: the ring's order
            // q tiles (segments) and key tiles so far; SPLIT: q tiles, then segments of the two groups
            int n_q[3] = {0, 0, 0}, n_s[2] = {0, 0};
            // A segment's last sh_gone and sh_bad are read after its last MMA: the next segment's
            // second key tile waits for that, before the copies come round to them.
            uint32_t owed = 0;  // of which query tiles
            bool ok = true;
            const uint32_t leader = pt_elect();
            // loops of a few MMAs: the code stays in the instruction cache, 64 cycles an MMA are time.
            // FP16: lo k, hi k.  FP32: lo hi, hi lo, hi hi (pass 0, 1, 2).
            constexpr int PASSES = F32 ? 3 : 2;
            auto scores = [&](int t, uint32_t k_at) {
                const uint32_t q_at = base + (uint32_t)(SPLIT ? 0 : 2 * t * C::Q_PLANE);
                uint32_t add = 0;
#pragma unroll 1
                for (int pass = 0; pass < PASSES; ++pass) {
                    uint64_t qa = pt_desc(q_at + (pass == 0 ? C::Q_PLANE : 0), 16);
                    uint64_t kb = pt_desc(k_at + (F32 && pass == 1 ? C::PLANE : 0), 16);
#pragma unroll 1
                    for (int b = 0; b < HDP / C::ROW; ++b, qa += C::Q_BLOCK >> 4, kb += C::K_BLOCK >> 4)
#pragma unroll
                        for (int k = 0; k < 4; ++k, add = 1)  // 32 bytes a step
                            pt_mma_ss<F32>(tmem + 128 * t, qa + 2 * k, kb + 2 * k, id_s, add, leader);
                }
            };
            // FP16: half h of the positions, the second one first
            auto outputs = [&](int t, uint32_t v_at, int h) {
                uint32_t add = !F32 && h == 0;
#pragma unroll 1
                for (int pass = 0; pass < PASSES; ++pass) {
                    if constexpr (F32) {
                        uint64_t vb = pt_desc(v_at + (pass == 1 ? C::PLANE : 0), 16);
                        uint32_t pa = tmem + 128 * t + (pass == 0 ? KT : 0);
#pragma unroll 1
                        for (int b = 0; b < KT / 32; ++b, vb += C::V_BLOCK >> 4, pa += 32)
#pragma unroll
                            for (int k = 0; k < 4; ++k, add = 1)  // 8 positions, 32 bytes, a step
                                pt_mma_ts<true>(tmem + 256 + 128 * t, pa + 8 * k, vb + 2 * k, id_o, add,
                                                leader);
                    } else {
                        uint64_t vb = pt_desc(v_at, C::V_BLOCK) + h * 4 * 128;
                        uint32_t pa = tmem + 128 * t + (pass == 0 ? 8 : 0) + h * 64;
#pragma unroll
                            for (int k = 0; k < 4; ++k, add = 1)  // 16 rows, 2048 bytes, a step
                                pt_mma_ts<false>(tmem + 256 + 128 * t, pa + 16 * k, vb + 128 * k, id_o,
                                                 add, leader);
                    }
                }
            };
            [[maybe_unused]] int exchanges = 0;
            [[maybe_unused]] bool x_owed = false;
            // SPLIT: the next slot, how often it has been used, its place
            [[maybe_unused]] int slot = 0, uses = 0;
            [[maybe_unused]] uint32_t slot_a = ring;
            [[maybe_unused]] auto advance = [&]() {
                ++slot, slot_a += C::TILE;
                if (slot == C::SLOTS) slot = 0, slot_a = ring, ++uses;
            };
            bool begun = false;
            while (ok && go_on(begun)) {
                const int n_kt = it.kt1 - it.kt0, n_t = it.rows > 128 ? 2 : 1;
                if (n_kt == 0) continue;
                auto slot_at = [&](int h) { return ring + (uint32_t)((h % C::SLOTS) * C::TILE); };
                auto arrived = [&](int h) {
                    ok = ok && wait(&bar.kv_full[h % C::SLOTS], h / C::SLOTS);
                    // written by cp.async, read by the tensor core (stores are followed by a fence of their
                    // own, TMA needs none)
                    pt_fence_async();
                };
                if constexpr (SPLIT) {
                    // Every K and V tile once, in the ring's order: O of key tile j, then the scores of key tile
                    // j + 2 in the same columns.  Both tiles are waited for before O, so that between the two
                    // the tensor core has the next MMA in time (4.0k cycles a key tile without that).
#pragma unroll 1
                    for (int j = -2; j < n_kt && ok; ++j) {
                        const bool s = j + 2 < n_kt;
                        const int t = ~j & 1;
                        uint64_t* empty_v = nullptr;
                        uint32_t v_at = 0;
                        if (j >= 0) {
                            ok = wait(&bar.kv_full[slot], uses);
                            empty_v = &bar.kv_empty[slot], v_at = slot_a;
                            advance();
                        }
                        if (s) ok = ok && wait(&bar.kv_full[slot], uses);
                        if (!F32 && !TA.box) pt_fence_async();  // written by cp.async
                        if (j >= 0) {
                            if (j == 0) {  // the last segment's masks and its second group's sums have been read
#pragma unroll 1
                                for (int g = 0; g < 2; ++g, owed >>= 1)
                                    if (owed & 1) ok = ok && wait(&bar.seg_done[g], n_q[1 + g]++);
                                if (x_owed) ok = ok && wait(&bar.x_done, exchanges++);
                            }
                            const int n = t ? n_s[1]++ : n_s[0]++;
                            ok = ok && wait(F32 ? &bar.p_full[t] : &bar.p_half[t], n);
                            pt_fence_after();
                            if (ok) {
                                if constexpr (!F32) {
                                    outputs(t, v_at, 1);
                                    ok = wait(&bar.p_full[t], n);
                                    pt_fence_after();
                                }
                                if (ok) outputs(t, v_at, 0);
                                pt_commit(&bar.o_full[t], leader);
                                pt_commit(empty_v, leader);
                            }
                        }
                        if (s) {
                            if (j == -2) ok = ok && wait(&bar.q_full[0], n_q[0]++);
                            pt_fence_after();
                            if (ok) {
                                scores(t, slot_a);
                                pt_commit(&bar.s_full[t], leader);
                                pt_commit(&bar.kv_empty[slot], leader);
                            }
                            advance();
                        }
                        __syncwarp();
                    }
                    owed = n_kt > 1 ? 3 : 2;
                    x_owed = true;
                    continue;
                }
                arrived(half);
                for (int t = 0; t < n_t && ok; ++t) {
                    ok = wait(&bar.q_full[t], n_q[t]++);
                    pt_fence_after();
                    if (ok) {
                        scores(t, slot_at(half));
                        pt_commit(&bar.s_full[t], leader);
                        if (t == n_t - 1) pt_commit(&bar.kv_empty[half % C::SLOTS], leader);
                    }
                }
#pragma unroll 1
                for (int t = 0; t < 2; ++t, owed >>= 1)  // phase: of the segment before
                    if (owed & 1) ok = ok && wait(&bar.seg_done[t], n_q[t] - (t < n_t ? 2 : 1));
                owed = (1u << n_t) - 1;
                for (int j = 0; j < n_kt && ok; ++j) {
                    const int hv = half + 2 * j + 1, hk = hv + 1;
                    for (int t = 0; t < n_t && ok; ++t) {
                        if (t == 0) arrived(hv);
                        // p of this key tile (half of it) is there, and O of the one before has been
                        // read
                        ok = ok && wait(F32 ? &bar.p_full[t] : &bar.p_half[t], n_s[t]++);
                        pt_fence_after();
                        if (ok) {
                            if constexpr (!F32) {
                                outputs(t, slot_at(hv), 1);
                                ok = wait(&bar.p_full[t], n_s[t] - 1);
                                pt_fence_after();
                                if (ok) outputs(t, slot_at(hv), 0);
                            } else {
                                outputs(t, slot_at(hv), 0);
                            }
                            pt_commit(&bar.o_full[t], leader);
                            if (t == n_t - 1) pt_commit(&bar.kv_empty[hv % C::SLOTS], leader);
                        }
                        if (j + 1 < n_kt) {
                            if (t == 0) arrived(hk);
                            if (ok) {
                                scores(t, slot_at(hk));
                                pt_commit(&bar.s_full[t], leader);
                                if (t == n_t - 1) pt_commit(&bar.kv_empty[hk % C::SLOTS], leader);
                            }
                        }
                        __syncwarp();
                    }
                }
                half += 2 * n_kt;
            }
            // the MMAs issued are done before tensor memory is given back
            pt_commit(&bar.done, leader);
            wait(&bar.done, 0);
        } else if constexpr (!F32) {
            // ---- copies.  Row by row: 16 rows at a time, lane j (and j + 16) sees to row j; with
            // TMA: lane i of warp 9 sees to box i. ----
            const int lw = warp - 9;
            constexpr int CH = HDP / 8, RL = 32 / CH;  // chunks of a row, rows at a time
            constexpr int BLOCKS = HDP / 64;
            const int row_bytes = HD * 2, x = lane % CH, r0 = lane / CH;
            const bool in_row = x * 16 < row_bytes;
            const uint8_t* const src_x[2] = {(const uint8_t*)A.k + x * 16, (const uint8_t*)A.v + x * 16};
            const int box = TA.box, box_row = (lane / BLOCKS) << box, box_col = lane % BLOCKS;
            const bool has_box = box && box_row < KT && (SPLIT || lw == 0);
            int half = 0;
            uint32_t seg_tile = 0;
            Looks looks;  // at V tiles, each on a barrier of its slot
            bool looking = false;  // such a wait ran out
            bool ok = true;
            bool begun = false;
            while (ok && go_on(begun)) {
                const int last_lim = it.start + (it.row0 + it.rows - 1) / G;
                const int first_lim = all_see<TREE>(it.start, it.row0, G);
                if (lw == 1) {  // the softmax warps ask for the segment's q soon
                    const int bytes = HD * 4;
                    for (int r = lane; r < it.rows; r += 32) {
                        const uint8_t* p = (const uint8_t*)q_row(A, it, G, it.row0 + r);
                        for (int b = 0; b < bytes; b += 128)
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(p + b));
                    }
                }
                auto row_of = [&](int pos) -> int {  // in the layer; -1: no page, or not seen
                    if (pos > last_lim) return -1;
                    const int col = (int)w.ps.div((uint32_t)pos);
                    const int page = page_at(w, it.s.row[col]);
                    return page < 0 ? -1 : (page * w.Hkv + it.hk) * w.page_size + (pos - col * w.page_size);
                };
                const int n_kt = it.kt1 - it.kt0;
                int box_at = -1, rows3[3] = {-1, -1, -1};
                // SPLIT with TMA: the warps see to a tile in turn (starting the 16 copies of one takes a
                // warp 2.8k cycles, as long as the MMAs and the softmax need for it), each with the table
                // entries of its next one on their way
                auto entry = [&](int e) -> int {
                    const int pos = (it.kt0 + (tile_order<SPLIT>(e, n_kt) >> 1)) * KT + box_row;
                    return has_box && e < 2 * n_kt && pos <= last_lim ? it.s.row[w.ps.div((uint32_t)pos)] : -1;
                };
                int turn = (lw - tile_owner(half) + 3) % 3;  // this warp's next
                [[maybe_unused]] int soon = SPLIT && box ? entry(turn) : -1;
#pragma unroll 1
                for (int e = 0; e < 2 * n_kt && ok; ++e, ++half) {
                    const int of = tile_order<SPLIT>(e, n_kt), j = of >> 1, kt = it.kt0 + j, kv = of & 1;
                    const uint32_t tile_no = seg_tile + (uint32_t)j;
                    const bool careful = kt * KT + KT - 1 > first_lim;
                    const bool mine = !SPLIT || !box || e == turn;
                    if (SPLIT && box) {
                        if (!mine) {
                            if (kv == 1 && careful) looks.take(half % C::SLOTS);  // the phases of all looks count
                            continue;
                        }
                        const int page = page_at(w, soon), pos = kt * KT + box_row;
                        box_at = page < 0 ? -1
                                          : (page * w.Hkv + it.hk) * w.page_size +
                                                (pos - (int)w.ps.div((uint32_t)pos) * w.page_size);
                        turn += 3;
                        soon = entry(turn);
                    } else if (SPLIT || kv == 0) {  // (else V: those of K)
                        if (has_box) box_at = row_of(kt * KT + box_row);
                        if (!box) {
#pragma unroll
                            for (int i = 0; i < 3; ++i)
                                if (lw + 3 * i < 8)
                                    rows3[i] = row_of(kt * KT + (lw + 3 * i) * 16 + (lane & 15));
                        }
                    }
                    {
                        const int slot = half % C::SLOTS, use = half / C::SLOTS;
                        if (use > 0 && !wait(&bar.kv_empty[slot], use - 1)) {
                            ok = false;
                            break;  // (half is not counted)
                        }
                        const bool look = kv == 1 && careful;  // V to be looked through
                        const uint32_t tile_at = ring + (uint32_t)(slot * C::TILE);
                        if (box) {
                            uint64_t* const there =
                                look ? &bar.v_there[Looks::bar(slot)] : &bar.kv_full[slot];
                            if (SPLIT || lw == 0) {
                                // (before the arrival, which is the tile's only one with SPLIT)
                                if (has_box && kv == 0 && box_col == 0)
                                    for (int b = 0; b < 1 << (box - 3); ++b)
                                        reinterpret_cast<uint8_t*>(sh_gone[tile_no & (RECENT - 1)])[box_row / 8 + b] =
                                            box_at < 0 ? 0xff : 0;
                                __syncwarp();
                                if (lane == 0) mbar_arrive_expect_tx(there, C::TILE);
                                __syncwarp();
                                if (has_box)
                                    pt_tma(tile_at + (uint32_t)(box_col * C::K_BLOCK + box_row * 128),
                                           kv ? &TA.v : &TA.k, box_col * 64, box_at < 0 ? -KT : box_at,
                                           there);
                            }
                            if (look && !wait(&bar.v_there[Looks::bar(slot)], looks.take(slot))) {
                                ok = false, looking = true;
                                break;
                            }
                        } else {
                            const uint8_t* src = src_x[kv];
                            // small loops: this code shares the instruction cache with the softmax
#pragma unroll 1
                            for (int i = 0; i < 3; ++i) {
                                const int g16 = lw + 3 * i;
                                if (g16 >= 8) break;
                                const int row = i == 0 ? rows3[0] : i == 1 ? rows3[1] : rows3[2];
#pragma unroll 4
                                for (int k = 0; k < 16 / RL; ++k) {
                                    const int from = k * RL + r0;
                                    const int n = __shfl_sync(0xffffffffu, row, from);
                                    const bool there = n >= 0 && in_row;
                                    cp16(tile_at + (uint32_t)((x >> 3) * C::K_BLOCK) +
                                             pt_off(g16 * 16 + from, x & 7),
                                         src + (there ? (int64_t)n * row_bytes : 0), there);
                                }
                                const uint32_t none = __ballot_sync(0xffffffffu, row < 0) & 0xffffu;
                                if (kv == 0 && lane == 0) sh_gone[tile_no & (RECENT - 1)][g16] = (uint16_t)none;
                            }
                            if (look) {
                                asm volatile("cp.async.wait_all;" ::: "memory");
                                __syncwarp();  // a warp looks through the rows it has copied
                            }
                        }
                        if (look) {
                            uint8_t* const tile = base_ptr + (tile_at - base);
                            if (SPLIT && box) {
                                // is there any such value at all?  0 x is 0 for every other one (two FP16 values an
                                // instruction; with the loop below alone one warp took 24k cycles for a tile)
                                const __half2 zero = __floats2half2_rn(0.f, 0.f);
                                __half2 any[4] = {zero, zero, zero, zero};
#pragma unroll 4
                                for (int i = lane; i < C::TILE / 16; i += 32) {
                                    const uint4 v = *reinterpret_cast<const uint4*>(tile + i * 16);
                                    const __half2* const x = reinterpret_cast<const __half2*>(&v);
#pragma unroll
                                    for (int k = 0; k < 4; ++k) any[k] = __hfma2(x[k], zero, any[k]);
                                }
                                uint32_t bits = 0;
#pragma unroll
                                for (int k = 0; k < 4; ++k) bits |= *reinterpret_cast<const uint32_t*>(&any[k]);
                                if (!__any_sync(0xffffffffu, (bits & 0x7fff7fffu) != 0)) {
                                    if (lane < 8) sh_bad[tile_no & (RECENT - 1)][lane] = 0;
                                    __syncwarp();
                                    if (lane == 0) mbar_arrive(&bar.kv_full[slot]);
                                    continue;
                                }
                            }
#pragma unroll 1
                            for (int g16 = SPLIT && box ? 0 : lw; g16 < 8; g16 += SPLIT && box ? 1 : 3) {
                                uint32_t bad = 0;
#pragma unroll 4
                                for (int k = 0; k < 4 * BLOCKS; ++k) {  // four rows of a block
                                    uint4* const at = reinterpret_cast<uint4*>(
                                        tile + (k >> 2) * C::K_BLOCK + (g16 * 16 + (k & 3) * 4) * 128 + lane * 16);
                                    uint4 v = *at;
                                    bool odd = false;
                                    v.x = finite16x2(v.x, odd), v.y = finite16x2(v.y, odd);
                                    v.z = finite16x2(v.z, odd), v.w = finite16x2(v.w, odd);
                                    if (odd) *at = v;
                                    const uint32_t any = __ballot_sync(0xffffffffu, odd);
                                    if (any)
                                        for (int r = 0; r < 4; ++r)
                                            if (any & (0xffu << (8 * r))) bad |= 1u << ((k & 3) * 4 + r);
                                }
                                if (lane == 0) sh_bad[tile_no & (RECENT - 1)][g16] = (uint16_t)bad;
                            }
                            pt_fence_async();
                        }
                        if (SPLIT && box) {
                            // (else the bytes' arrival is the one)
                            __syncwarp();
                            if (lane == 0 && look) mbar_arrive(&bar.kv_full[slot]);
                            continue;
                        }
                        // 33 arrivals a warp, whichever way: with TMA one of them is the bytes'
                        if (box || look) mbar_arrive(&bar.kv_full[slot]);
                        else
                            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                                             smem_u32(&bar.kv_full[slot]))
                                         : "memory");
                        // after sh_gone and sh_bad
                        __syncwarp();
                        if (lane == 0 && !(box && !look && lw == 0)) mbar_arrive(&bar.kv_full[slot]);
                    }
                }
                seg_tile += (uint32_t)n_kt;
            }
            // no copy may still be landing when the CTA ends
            asm volatile("cp.async.wait_all;" ::: "memory");
            drain_copies<C::SLOTS>(
                half, looking, looks, [&](int slot, int use) { wait(&bar.kv_full[slot], use); },
                [&](int slot, int parity) { wait(&bar.v_there[Looks::bar(slot)], parity); });
        } else if (warp == 9) {
            // ---- copies of FP32 pages: TMA brings K and V as they are ----
            const int box = TA.box, box_row = lane << box;
            const bool has_box = box_row < KT;
            const bool singles = KT > 32 && box == 0;  // odd page sizes: two rows for a lane
            const uint32_t raw_a = ring + C::SLOTS * C::TILE;
            int issued = 0;  // key tiles
            RawSent sent;
            bool ok = true;
            bool begun = false;
            while (ok && go_on(begun)) {
                const int last_lim = it.start + (it.row0 + it.rows - 1) / G;
                auto row_of = [&](int kt, int row) -> int {  // in the layer; -1: no page, or not seen
                    const int pos = kt * KT + row;
                    if (row >= KT || kt >= it.kt1 || pos > last_lim) return -1;
                    const int col = (int)w.ps.div((uint32_t)pos);
                    const int page = page_at(w, it.s.row[col]);
                    return page < 0 ? -1 : (page * w.Hkv + it.hk) * w.page_size + (pos - col * w.page_size);
                };
                const int n_kt = it.kt1 - it.kt0;
                int at = SPLIT ? -1 : row_of(it.kt0, box_row);
                // the softmax warps ask for the segment's q soon
                for (int r = lane; r < it.rows; r += 32) {
                    const uint8_t* p = (const uint8_t*)q_row(A, it, G, it.row0 + r);
                    for (int b = 0; b < HD * 4; b += 128)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(p + b));
                }
                if constexpr (SPLIT) {
                    // table entries of the next two key tiles, on their way, and the rows of the last two
                    auto entry = [&](int j, int row) -> int {
                        const int pos = (it.kt0 + j) * KT + row;
                        return row < KT && j < n_kt && pos <= last_lim ? it.s.row[w.ps.div((uint32_t)pos)] : -1;
                    };
                    auto layer_row = [&](int e, int j, int row) -> int {
                        const int pos = (it.kt0 + j) * KT + row, page = page_at(w, e);
                        return page < 0 ? -1
                                        : (page * w.Hkv + it.hk) * w.page_size +
                                              (pos - (int)w.ps.div((uint32_t)pos) * w.page_size);
                    };
                    int soon[2] = {entry(0, box_row), entry(1, box_row)}, rows[2] = {-1, -1};
                    int soon2[2] = {-1, -1}, rows2[2] = {-1, -1};
                    if (singles) soon2[0] = entry(0, lane + 32), soon2[1] = entry(1, lane + 32);
#pragma unroll 1
                    for (int e = 0; e < 2 * n_kt && ok; ++e) {
                        const int of = tile_order<true>(e, n_kt), j = of >> 1, kv = of & 1;
                        if (kv == 0) {
                            rows[0] = rows[1], rows[1] = layer_row(soon[0], j, box_row);
                            soon[0] = soon[1], soon[1] = entry(j + 2, box_row);
                            if (singles) {
                                rows2[0] = rows2[1], rows2[1] = layer_row(soon2[0], j, lane + 32);
                                soon2[0] = soon2[1], soon2[1] = entry(j + 2, lane + 32);
                            }
                        }
                        const bool newest = kv == 0 || j == n_kt - 1;
                        at = newest ? rows[1] : rows[0];
                        const int at2 = newest ? rows2[1] : rows2[0];
                        uint64_t none = __ballot_sync(0xffffffffu, has_box && at < 0);
                        if (singles) none |= (uint64_t)__ballot_sync(0xffffffffu, at2 < 0) << 32;
                        uint32_t gone = 0;  // of positions 16 lane ..
                        if (none)
                            for (int r = 0; r < 16; ++r)
                                gone |= (uint32_t)((none >> (((lane * 16 + r) >> box) & 63)) & 1) << r;
                        const int n = issued + j;  // of its kind
                        if (n > 0) ok = wait(&bar.raw_empty[kv], n - 1);
                        if (!ok) break;
                        if (kv == 0 && lane < KT / 16) sh_gone[n & (RECENT - 1)][lane] = (uint16_t)gone;
                        __syncwarp();
                        if (lane == 0) mbar_arrive_expect_tx(&bar.raw_full[kv], C::PLANE);
                        sent.add(kv);
                        __syncwarp();
                        const uint32_t to = raw_a + (uint32_t)(kv * C::PLANE + box_row * HDP * 4);
                        const CUtensorMap* const map = kv ? &TA.v : &TA.k;
                        if (has_box) pt_tma(to, map, 0, at < 0 ? -KT : at, &bar.raw_full[kv]);
                        if (singles)
                            pt_tma(to + 32 * HDP * 4, map, 0, at2 < 0 ? -KT : at2, &bar.raw_full[kv]);
                    }
                    issued += n_kt;
                }
                for (int kt = SPLIT ? it.kt1 : it.kt0; kt < it.kt1 && ok; ++kt, ++issued) {
                    const int at_next = row_of(kt + 1, box_row);
                    uint64_t none = __ballot_sync(0xffffffffu, has_box && at < 0);
                    int at2 = -1;
                    if (singles) {
                        at2 = row_of(kt, lane + 32);
                        none |= (uint64_t)__ballot_sync(0xffffffffu, at2 < 0) << 32;
                    }
                    uint32_t gone = 0;  // of positions 16 lane ..
                    if (none)
                        for (int r = 0; r < 16; ++r)
                            gone |= (uint32_t)((none >> (((lane * 16 + r) >> box) & 63)) & 1) << r;
#pragma unroll 1
                    for (int kv = 0; kv < 2 && ok; ++kv) {
                        if (issued > 0) ok = wait(&bar.raw_empty[kv], issued - 1);
                        if (!ok) break;
                        if (kv == 0 && lane < KT / 16) sh_gone[issued & (RECENT - 1)][lane] = (uint16_t)gone;
                        __syncwarp();
                        if (lane == 0) mbar_arrive_expect_tx(&bar.raw_full[kv], C::PLANE);
                        sent.add(kv);
                        __syncwarp();
                        const uint32_t to = raw_a + (uint32_t)(kv * C::PLANE + box_row * HDP * 4);
                        const CUtensorMap* const map = kv ? &TA.v : &TA.k;
                        if (has_box) pt_tma(to, map, 0, at < 0 ? -KT : at, &bar.raw_full[kv]);
                        if (singles)
                            pt_tma(to + 32 * HDP * 4, map, 0, at2 < 0 ? -KT : at2, &bar.raw_full[kv]);
                    }
                    at = at_next;
                }
            }
            // no copy may still be landing when the CTA ends
            sent.drain([&](int kv, int phase) { wait(&bar.raw_full[kv], phase); });
        } else {
            // ---- and these warps split them into TF32 parts, hi in a slot's first half, lo in the
            // second.  K: rows are positions, 128 bytes 32 dimensions.  V is turned round, since TF32
            // operands have to lie along K: rows are dimensions, 128 bytes 32 positions. ----
            const int sw = warp - 10;
            const uint8_t* const raw_ptr = base_ptr + (ring - base) + C::SLOTS * C::TILE;
            int half = 0;
            uint32_t seg_tile = 0;
            bool ok = true;
            bool begun = false;
            while (ok && go_on(begun)) {
                const int first_lim = all_see<TREE>(it.start, it.row0, G);
                const int n_kt = it.kt1 - it.kt0;
#pragma unroll 1
                for (int e = 0; e < 2 * n_kt && ok; ++e, ++half) {
                    const int of = tile_order<SPLIT>(e, n_kt), kt = it.kt0 + (of >> 1), kv = of & 1;
                    const uint32_t tile_no = seg_tile + (uint32_t)(of >> 1);
                    const bool careful = kt * KT + KT - 1 > first_lim;
                    {
                        const int slot = half % C::SLOTS, use = half / C::SLOTS;
                        ok = wait(&bar.raw_full[kv], (int)tile_no);
                        if (use > 0) ok = ok && wait(&bar.kv_empty[slot], use - 1);
                        if (!ok) break;
                        uint8_t* const tile = base_ptr + (ring - base) + slot * C::TILE;
                        const uint8_t* const raw = raw_ptr + kv * C::PLANE;
                        if (kv == 0) {
                            // (small loops: unrolled four and two times they missed the instruction
                            // cache, 91 us against 84.5 for prompts on pages of 24)
#pragma unroll 1
                            for (int i = sw * 32 + lane; i < C::PLANE / 16; i += 32 * C::SPLIT_WARPS) {
                                const int r = i / (HDP / 4), d = (i % (HDP / 4)) * 4;
                                const float4 x = *reinterpret_cast<const float4*>(raw + i * 16);
                                uint4 h, l;
                                split_tf32(x.x, h.x, l.x), split_tf32(x.y, h.y, l.y);
                                split_tf32(x.z, h.z, l.z), split_tf32(x.w, h.w, l.w);
                                uint8_t* const at = tile + (d >> 5) * C::K_BLOCK + pt_off(r, (d & 31) >> 2);
                                *reinterpret_cast<uint4*>(at) = h;
                                *reinterpret_cast<uint4*>(at + C::PLANE) = l;
                            }
                        } else {
                            uint32_t bad0 = 0, bad1 = 0;
                            // four positions of 32 dimensions at a time, a dimension to a lane
#pragma unroll 1
                            for (int u = sw; u < KT / 4 * (HDP / 32); u += C::SPLIT_WARPS) {
                                const int p4 = u / (HDP / 32), d = (u % (HDP / 32)) * 32 + lane;
                                float y[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    y[j] = *reinterpret_cast<const float*>(raw + ((p4 * 4 + j) * HDP + d) * 4);
                                if (careful) {
                                    uint32_t odd4 = 0;
#pragma unroll
                                    for (int j = 0; j < 4; ++j) {
                                        const bool odd = !(fabsf(y[j]) < INFINITY);
                                        if (odd) y[j] = 0.f;
                                        if (__any_sync(0xffffffffu, odd)) odd4 |= 1u << j;
                                    }
                                    if (p4 < 8) bad0 |= odd4 << (4 * p4);
                                    else bad1 |= odd4 << (4 * p4 - 32);
                                }
                                uint4 h, l;
                                split_tf32(y[0], h.x, l.x), split_tf32(y[1], h.y, l.y);
                                split_tf32(y[2], h.z, l.z), split_tf32(y[3], h.w, l.w);
                                uint8_t* const at = tile + (p4 >> 3) * C::V_BLOCK + pt_off(d, p4 & 7);
                                *reinterpret_cast<uint4*>(at) = h;
                                *reinterpret_cast<uint4*>(at + C::PLANE) = l;
                            }
                            if (lane == 0) {
                                sh_bad32[tile_no & (RECENT - 1)][sw][0] = bad0;
                                sh_bad32[tile_no & (RECENT - 1)][sw][1] = bad1;
                            }
                        }
                        pt_fence_async();
                        mbar_arrive(&bar.kv_full[slot]);
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(&bar.kv_full[slot]);
                            mbar_arrive(&bar.raw_empty[kv]);
                        }
                    }
                }
                seg_tile += (uint32_t)n_kt;
            }
        }
    }
    // every use of tensor memory is over before it is given back
    pt_fence_before();
    __syncthreads();
    if (warp == 8) {
        pt_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                     : "memory");
    }
    if (A.beside) pdl_wait();
}

// The layer's rows as a tensor [rows][head_dim]: FP16 in swizzled boxes of 64 columns, FP32 in
// plain boxes of all (padded) columns.
template <typename KV, int HDP>
static int tensor_map(CUtensorMap* map, const void* base, int64_t rows, int head_dim, int box_rows) {
    constexpr bool F32 = sizeof(KV) == 4;
    static Lookup<PFN_cuTensorMapEncodeTiled> lookup;
    const PFN_cuTensorMapEncodeTiled encode = lookup.get([] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool there = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault,
                                                   &q) == cudaSuccess &&
                           q == cudaDriverEntryPointSuccess;
        return there ? (PFN_cuTensorMapEncodeTiled)fn : nullptr;
    });
    if (!encode) {
        set_error("ib_attention_paged: cuTensorMapEncodeTiled is not available");
        return IB_ERR_CUDA;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)head_dim * sizeof(KV)};
    const cuuint32_t box[2] = {F32 ? HDP : 64, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode(
        map, F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
        const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
        F32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("ib_attention_paged: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
        return IB_ERR_CUDA;
    }
    return IB_OK;
}

template <typename KV, bool SPLIT>
static CutRule rule_of(int head_dim, int min_rows, int max_rows) {
    // one CTA to an SM, a piece for each
    using S = TensorCfg<KV, 64, SPLIT>;
    using L = TensorCfg<KV, 128, SPLIT>;
    return head_dim <= 64 ? CutRule{S::R, S::KT, min_rows, max_rows, kSMs, 128}
                          : CutRule{L::R, L::KT, min_rows, max_rows, kSMs, 128};
}
template <typename KV, bool TREE>
CutRule tensor_rule(int head_dim, int min_rows, int max_rows, bool split) {
    CutRule r = split ? rule_of<KV, true>(head_dim, min_rows, max_rows)
                      : rule_of<KV, false>(head_dim, min_rows, max_rows);
    if (TREE) {
        // Beginning a tile takes some 20k cycles, as long as 800 positions on FP16 pages and 200 on FP32
        // ones.  Eight batches of 32 trees of 12 to 24 nodes over 200 .. 4096 positions (FP16) take
        // 160 us with 100, 151 with 200, 141 with 300, 132 with 500, 126 with 800; two documents of
        // 20000 .. 32000 (FP32) 171.5, 171.5, 173, 174 and 176.
        r.fixed = sizeof(KV) == 4 ? 200 : 800;
        // Tiles of under 768 positions (FP32: 512) stay whole, and no side of a cut has less than two FP16 key
        // tiles: a join takes as long as a few of them.  Four trees of 41 nodes over 104 .. 194 positions take
        // 31 us so, 42 cut; 56 of 15 over 204 .. 472 (8 rows to a token) 78 and 88; 59 of 1 to 10 over
        // 4 .. 1184 take 45 us, and 50 if tiles of under 1024 stay whole too.  FP32: four of 16 to 24 over
        // 400 .. 750 (32 heads on 8 of 128) 43 us, 73 whole; 16 over 150 .. 350 46 us, 53 cut.
        r.flat = true;
        r.uncut = sizeof(KV) == 4 ? 512 : 768;
        r.least = sizeof(KV) == 4 ? 128 : 256;
        r.split = split;
    }
    return r;
}
template CutRule tensor_rule<float, false>(int, int, int, bool);
template CutRule tensor_rule<__half, false>(int, int, int, bool);
template CutRule tensor_rule<float, true>(int, int, int, bool);
template CutRule tensor_rule<__half, true>(int, int, int, bool);

template <typename KV, int HDP, bool TREE, bool SPLIT>
static int launch(const RowsArgs& a, int64_t grid, cudaStream_t st) {
    using C = TensorCfg<KV, HDP, SPLIT>;
    auto kern = attn_tensor_kernel<KV, HDP, TREE, SPLIT>;
    TensorArgs t{};
    t.rows = a;
    const PagedView& w = a.w;
    // a box: the largest power of two that divides the page, up to the tile
    int box = 0;
    while (2 << box <= C::KT && w.page_size % (2 << box) == 0) ++box;
    if (C::F32 || box >= 3) {
        const int64_t rows = (int64_t)w.n_pages * w.Hkv * w.page_size;
        int r = tensor_map<KV, HDP>(&t.k, a.k, rows, w.HD, 1 << box);
        if (r == IB_OK) r = tensor_map<KV, HDP>(&t.v, a.v, rows, w.HD, 1 << box);
        if (r != IB_OK) return r;
        t.box = box;
    }
    static DeviceOnce once;
    IB_CUDA_CHECK(once.run([&] {
        return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    }));
    IB_CUDA_CHECK(launch_pdl(kern, dim3((unsigned)grid), dim3(C::THREADS), C::SMEM, st, true, t));
    return IB_OK;
}

template <typename KV, bool TREE>
int attn_tensor_launch(const RowsArgs& a, int64_t tiles, int64_t max_pos, cudaStream_t st) {
    const int64_t most = tiles * (max_pos / a.rule.least + 1 + a.rule.R);
    const int64_t grid = std::min<int64_t>(a.rule.n_pieces, most);
    if constexpr (TREE) {
        if (a.rule.split)
            return a.w.HD <= 64 ? launch<KV, 64, true, true>(a, grid, st) : launch<KV, 128, true, true>(a, grid, st);
    }
    return a.w.HD <= 64 ? launch<KV, 64, TREE, false>(a, grid, st) : launch<KV, 128, TREE, false>(a, grid, st);
}
template int attn_tensor_launch<float, false>(const RowsArgs&, int64_t, int64_t, cudaStream_t);
template int attn_tensor_launch<__half, false>(const RowsArgs&, int64_t, int64_t, cudaStream_t);
template int attn_tensor_launch<float, true>(const RowsArgs&, int64_t, int64_t, cudaStream_t);
template int attn_tensor_launch<__half, true>(const RowsArgs&, int64_t, int64_t, cudaStream_t);

}  // namespace ib

extern "C" int ib_kv_wait_selftest(void* stream) {
    ib::wait_selftest_kernel<<<1, 1, 0, ib::as_stream(stream)>>>();
    IB_LAUNCH_CHECK("wait_selftest_kernel");
    return IB_OK;
}
