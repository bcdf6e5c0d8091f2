// ib_attention_paged on tcgen05: FP16 pages, head_dim up to 128, tiles of 256 query rows -- the
// chunks of prompts.
//
// Two query tiles of 128 rows share each key tile of 128 positions.  As on mma.sync, q and p are
// FP16 pairs hi + lo (q scaled to a largest element in [256, 512), p by 2^10), K and V are taken
// as they are, so every product is two MMAs and 2^-21 of it is kept:
//     S = q_lo K' + q_hi K'      A: q in shared memory, B: K            M 128, N 128
//     O = p_lo V  + p_hi V       A: p in tensor memory, B: V            M 128, N head_dim
// The tensor core adds to its accumulator by cutting, which over a long sequence would drift; so
// O starts from zero in every key tile and the running sum is kept in registers, one row per
// thread, where acc = acc c + O takes the softmax's rescaling with it.
//
// Tensor memory, 512 columns: S of both query tiles (128 each), O of both (128 each).  p lies
// over its S: of a chunk of 16 scores a thread writes hi into the first 8 columns and lo into the
// other 8, and an MMA's 16 positions are one chunk.
// Shared memory: q of both tiles as hi and lo (128 KB at head_dim 128) and a ring of three slots
// for K and V tiles in turn.  Rows are 128 bytes (64 elements) under the 128-byte swizzle; K is
// read with head_dim along the MMA's K (K-major), V with positions along it (MN-major), so both
// are stored as they lie in the pages.
// Warps: 0-3 and 4-7 the softmax of a query tile each (thread = row), 8 issues the MMAs, 9-11
// copy K and V row by row with cp.async, since pages end anywhere.  The order of MMAs is
//     O0(j) S0(j+1) O1(j) S1(j+1) O0(j+1) ...
// so that a tile's softmax has the other tile's MMAs to hide behind.
// Work per CTA is a piece of the batch (paged_plan.cuh); the copies run on into the next
// segment.
#include <cuda_fp16.h>

#include <algorithm>
#include <string>

#include "common.cuh"
#include "mma_tile.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "pdl.cuh"
#include "pipeline.cuh"

namespace ib {

int paged_tensor_fault_take(int* code) { return paged_fault_take_here(code); }

constexpr int PT_R = 256, PT_KT = 128, PT_SLOTS = 3, PT_THREADS = 384;
constexpr int PT_LOADERS = 96;

template <int HDP>
struct TensorCfg {
    static constexpr int BLOCKS = HDP / 64;           // of 64 columns
    static constexpr int BLOCK = 128 * 128;           // bytes: 128 rows of 64 elements
    static constexpr int TILE = BLOCKS * BLOCK;       // a K or V tile, or a part of a q tile
    static constexpr size_t SMEM = 4 * TILE + PT_SLOTS * TILE + 1024;
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
// 1).  K-major: 64 columns to a row.  MN-major: the 64 columns are the MN dimension, the next
// 64 lie TILE rows on (the leading offset), the groups of eight rows run along K.
__device__ __forceinline__ uint64_t pt_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) |
           ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// kind::f16: D FP32, A and B FP16; b_mn: B is MN-major.
constexpr uint32_t pt_idesc(int M, int N, bool b_mn) {
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

// The whole warp comes here with the same operands and `leader` lets one thread issue: the
// operands then are uniform registers, as the instruction takes them.  Issued inside a branch of
// one thread, every operand is moved there first, and an MMA took 134 cycles instead of 64.
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t add, uint32_t leader) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                          uint32_t add, uint32_t leader) {
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

// 16 columns of this warp's 32 lanes, to be waited for
__device__ __forceinline__ void pt_ld16(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
        "%12, %13, %14, %15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
          "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
          "=f"(v[14]), "=f"(v[15])
        : "r"(taddr));
}
// The loads' registers pass through the wait, so that nothing uses them before it.
__device__ __forceinline__ void pt_wait_ld(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                   "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                   "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void pt_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
        : "memory");
}

// Byte offset of 16-byte chunk c (0-7) of row r in a swizzled block.
__device__ __forceinline__ uint32_t pt_off(int r, int c) {
    return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}

struct TensorBars {
    uint64_t kv_full[PT_SLOTS], kv_empty[PT_SLOTS];
    uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2], done;
};

template <int HDP>
__global__ void __launch_bounds__(PT_THREADS, 1)
    attn_tensor_kernel(const __grid_constant__ RowsArgs A) {
    using C = TensorCfg<HDP>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) TensorBars bar;
    __shared__ uint32_t tmem_base;
    __shared__ Piece sh_piece[PT_THREADS / 32];  // the same one for each warp, out of its registers
    __shared__ int found;
    // of the last four key tiles: positions without a page; positions whose V is not finite
    __shared__ __align__(16) uint16_t sh_gone[4][8], sh_bad[4][8];
    const PagedView& w = A.w;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_launch_dependents();
    find_pieces<PT_THREADS, 1, false>(w, A.rule, blockIdx.x, sh_piece, &found, nullptr);
    __syncthreads();
    if (!found) return;
    if (tid > 0 && tid < PT_THREADS / 32) sh_piece[tid] = sh_piece[0];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const base_ptr = smem_raw + (base - smem_u32(smem_raw));
    if (tid == 0) {
        for (int i = 0; i < PT_SLOTS; ++i) {
            mbar_init(&bar.kv_full[i], PT_LOADERS + PT_LOADERS / 32);
            mbar_init(&bar.kv_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.q_full[i], 128);
            mbar_init(&bar.q_empty[i], 128);
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], 128);
            mbar_init(&bar.o_full[i], 1);
            mbar_init(&bar.o_empty[i], 128);
        }
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
    const uint32_t ring = base + 4 * C::TILE;
    const int G = w.H / w.Hkv, HD = w.HD;
    Segment it;
    auto next = [&]() -> bool {
        Piece p = sh_piece[warp];
        const bool more = next_segment(w, A.rule, p, it);
        __syncwarp();
        if (lane == 0) sh_piece[warp] = p;
        __syncwarp();
        return more;
    };
    // For the n-th completion, from 0; the same answer in a whole warp.  Every wait is bounded: a
    // role whose wait expired leaves its loop, and so do, one wait later, those that wait for it.
    auto wait = [&](uint64_t* b, int n) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(b, (uint32_t)(n & 1), &g_paged_fault, PAGED_BAD_WAIT));
    };

    if (warp < 8) {
        // ---- softmax of query tile t: thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int t = warp >> 2, wr = (warp & 3) * 32;  // this warp's rows of the tile, its lanes
        uint8_t* const q_ptr = base_ptr + 2 * t * C::TILE;
        const uint32_t s_at = tmem + ((uint32_t)wr << 16) + (uint32_t)(128 * t);
        const uint32_t o_at = tmem + ((uint32_t)wr << 16) + (uint32_t)(256 + 128 * t);
        int tiles = 0, segs = 0;  // key tiles so far, of all segments; segments so far
        uint32_t seen = 0;  // and counted as the copies do (both query tiles)
        bool ok = true;
        while (ok && next()) {
            const int n_kt = it.kt1 - it.kt0;
            const int rows = it.rows - 128 * t;  // of this query tile
            const uint32_t first = seen;
            seen += (uint32_t)n_kt;
            if (rows <= 0) continue;
            // q: this warp's 32 rows, HDP / 4 lanes to a row
            constexpr int LPR = HDP / 4, RPI = 32 / LPR;  // lanes per row, rows at a time
            float my_scale = 0.f;
            const float sign = A.scale_log2 < 0.f ? -1.f : 1.f;
            // every warp of the tile has stored the last segment's rows from here
            if (segs > 0) ok = wait(&bar.q_empty[t], segs - 1);
            ++segs;
            if (!ok) break;
            if (n_kt > 0) {
#pragma unroll 4
                for (int i = 0; i < 32; i += RPI) {
                    const int r = wr + i + lane / LPR, d = (lane % LPR) * 4;
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (r < rows && d < HD)
                        x = __ldg(reinterpret_cast<const float4*>(
                            q_row(A, it, G, it.row0 + 128 * t + r) + d));
                    float top = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    float down;
                    const float up = pow2_scale(top, down) * sign;
                    uint32_t h[2], l[2];
                    split2(x.x * up, x.y * up, h[0], l[0]);
                    split2(x.z * up, x.w * up, h[1], l[1]);
                    const uint32_t at = (uint32_t)((d >> 6) * C::BLOCK) + pt_off(r, (d & 63) >> 3) +
                                        (uint32_t)((d & 4) << 1);
                    *reinterpret_cast<uint2*>(q_ptr + at) = make_uint2(h[0], h[1]);
                    *reinterpret_cast<uint2*>(q_ptr + C::TILE + at) = make_uint2(l[0], l[1]);
#pragma unroll
                    for (int k = 0; k < RPI; ++k) {
                        const float f = __shfl_sync(0xffffffffu, down, k * LPR);
                        if (lane == i + k) my_scale = f;
                    }
                }
                pt_fence_async();
                mbar_arrive(&bar.q_full[t]);
            }
            // scores are multiplied by this; kept off zero, where -inf would turn into NaN
            const float sc = fmaxf(fabsf(A.scale_log2) * my_scale, 1e-37f);
            const int r = wr + lane;
            const int lim = r < rows ? it.start + (it.row0 + 128 * t + r) / G : -1;
            const int first_lim = it.start + (it.row0 + 128 * t) / G;  // of the tile's first row
            float acc[HDP];
#pragma unroll
            for (int d = 0; d < HDP; ++d) acc[d] = 0.f;
            float m = -INFINITY, l = 0.f, c_last = 1.f;
            // positions of key tile j (of the segment) that this row sees and that have a page
            auto visible = [&](int j, int word) -> uint32_t {
                const int n = lim + 1 - ((it.kt0 + j) * PT_KT + 32 * word);
                const uint32_t below = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
                const uint16_t* gone = sh_gone[(first + j) & 3];
                return below & ~((uint32_t)gone[2 * word] | ((uint32_t)gone[2 * word + 1] << 16));
            };
            // O of key tile j into the running sum
            auto add_o = [&](int j) {
                ok = wait(&bar.o_full[t], tiles - 1) && ok;
                pt_fence_after();
#pragma unroll
                for (int d0 = 0; d0 < HDP; d0 += 32) {
                    float o[16], o2[16];
                    pt_ld16(o_at + d0, o);
                    pt_ld16(o_at + d0 + 16, o2);
                    pt_wait_ld(o);
                    pt_wait_ld(o2);
#pragma unroll
                    for (int d = 0; d < 16; ++d) {
                        acc[d0 + d] = fmaf(acc[d0 + d], c_last, o[d]);
                        acc[d0 + 16 + d] = fmaf(acc[d0 + 16 + d], c_last, o2[d]);
                    }
                }
                pt_fence_before();
                mbar_arrive(&bar.o_empty[t]);
                if ((it.kt0 + j) * PT_KT + PT_KT - 1 > it.start + it.row0 / G) {
                    // where some row does not see all of the tile, V was made finite: rows that
                    // see such a position are not
                    const uint16_t* bad = sh_bad[(first + j) & 3];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (visible(j, i) & ((uint32_t)bad[2 * i] | ((uint32_t)bad[2 * i + 1] << 16)))
                            l = NAN;
                }
            };
            for (int j = 0; j < n_kt && ok; ++j) {
                if (j > 0) add_o(j - 1);
                ok = wait(&bar.s_full[t], tiles) && ok;
                ++tiles;
                pt_fence_after();
                bool all = (it.kt0 + j) * PT_KT + PT_KT - 1 <= first_lim && r < rows;
                {
                    const uint4 gone = *reinterpret_cast<const uint4*>(sh_gone[(first + j) & 3]);
                    all = all && (gone.x | gone.y | gone.z | gone.w) == 0;
                }
                all = __all_sync(0xffffffffu, all);
                // the next 16 scores are on their way while these are worked on
                auto mask = [&](float (&s)[16], int i) {
                    const uint32_t see = visible(j, i >> 1) >> (16 * (i & 1));
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (!((see >> k) & 1)) s[k] = -INFINITY;
                };
                float top = -INFINITY;
                auto maximum = [&](float (&s)[16], int i) {
                    if (!all) mask(s, i);
#pragma unroll
                    for (int k = 0; k < 16; ++k) top = fmaxf(top, s[k]);
                };
                float s0[16], s1[16];
                pt_ld16(s_at, s0);
#pragma unroll 1
                for (int i = 0; i < 8; i += 2) {
                    pt_wait_ld(s0);
                    pt_ld16(s_at + 16 * i + 16, s1);
                    maximum(s0, i);
                    pt_wait_ld(s1);
                    pt_ld16(s_at + ((16 * i + 32) & 127), s0);  // the last: the first, for below
                    maximum(s1, i + 1);
                }
                top = fmaxf(m, top);  // of the scores before scaling
                const bool none = top == -INFINITY;
                const float c = none ? 1.f : ex2((m - top) * sc);
                const float off = none ? 0.f : 10.f - top * sc;
                m = top;
                float sum = 0.f;
                auto weights = [&](float (&s)[16], int i) {
                    if (!all) mask(s, i);
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float x = ex2(fmaf(s[2 * k], sc, off));
                        const float y = ex2(fmaf(s[2 * k + 1], sc, off));
                        sum += x + y;
                        split2(x, y, hi[k], lo[k]);
                    }
                    pt_st8(s_at + 16 * i, hi);
                    pt_st8(s_at + 16 * i + 8, lo);
                };
#pragma unroll 1
                for (int i = 0; i < 8; i += 2) {
                    pt_wait_ld(s0);
                    pt_ld16(s_at + 16 * i + 16, s1);
                    weights(s0, i);
                    pt_wait_ld(s1);
                    if (i < 6) pt_ld16(s_at + 16 * i + 32, s0);
                    weights(s1, i + 1);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                l = fmaf(l, c, sum);
                c_last = c;
                pt_fence_before();
                mbar_arrive(&bar.p_full[t]);
            }
            if (n_kt > 0 && ok) add_o(n_kt - 1);

            // ---- the segment's rows, through this warp's quarter of the q tile (every MMA on
            // it is done), so that they go out row by row ----
            const bool whole = it.part < 0;
            const float f = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
            constexpr int RB = HDP * 4;  // bytes of a row
            uint8_t* const mine = q_ptr + (warp & 3) * 32 * RB;
#pragma unroll
            for (int c4 = 0; c4 < HDP / 4; ++c4)
                *reinterpret_cast<float4*>(mine + lane * RB + ((c4 ^ (lane & 7)) << 4)) =
                    make_float4(acc[4 * c4] * f, acc[4 * c4 + 1] * f, acc[4 * c4 + 2] * f,
                                acc[4 * c4 + 3] * f);
            __syncwarp();
            for (int i = 0; i < 32; i += RPI) {
                const int rr = i + lane / LPR, c4 = lane % LPR, row = wr + rr;
                if (row >= rows || c4 * 4 >= HD) continue;
                const float4 x = *reinterpret_cast<const float4*>(mine + rr * RB + ((c4 ^ (rr & 7)) << 4));
                float* p = whole ? out_row(A, it, G, it.row0 + 128 * t + row)
                                 : A.part_acc + ((int64_t)it.part * PT_R + 128 * t + row) * HD;
                *reinterpret_cast<float4*>(p + 4 * c4) = x;
            }
            mbar_arrive(&bar.q_empty[t]);
            if (!whole && r < rows)
                A.part_ml[(int64_t)it.part * PT_R + 128 * t + r] = make_float2(m * sc, l);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            // ---- MMAs ----
            constexpr uint32_t id_s = pt_idesc(128, 128, false), id_o = pt_idesc(128, HDP, true);
            int half = 0;               // K and V tiles so far: the ring's order
            int n_q[2] = {0, 0}, n_s[2] = {0, 0};  // q tiles and key tiles so far
            bool ok = true;
            const uint32_t leader = pt_elect();
            auto scores = [&](int t, uint32_t k_at) {
                const uint64_t qa = pt_desc(base + (uint32_t)(2 * t * C::TILE), 16);
                const uint64_t kb = pt_desc(k_at, 16);
#pragma unroll
                for (int part = 1; part >= 0; --part)  // lo, then hi
#pragma unroll
                    for (int k = 0; k < HDP / 16; ++k) {
                        const uint32_t off = (uint32_t)((k >> 2) * (C::BLOCK >> 4) + (k & 3) * 2);
                        pt_mma_ss(tmem + 128 * t, qa + (uint32_t)(part * (C::TILE >> 4)) + off, kb + off,
                                  id_s, part == 0 || k > 0, leader);
                    }
            };
            auto outputs = [&](int t, uint32_t v_at) {
                const uint64_t vb = pt_desc(v_at, C::BLOCK);
#pragma unroll
                for (int part = 1; part >= 0; --part)
#pragma unroll
                    for (int k = 0; k < PT_KT / 16; ++k)  // 16 rows, 2048 bytes, a step
                        pt_mma_ts(tmem + 256 + 128 * t, tmem + 128 * t + 16 * k + 8 * part,
                                  vb + (uint32_t)(k * 128), id_o, part == 0 || k > 0, leader);
            };
            while (ok && next()) {
                const int n_kt = it.kt1 - it.kt0, n_t = it.rows > 128 ? 2 : 1;
                if (n_kt == 0) continue;
                auto slot_at = [&](int h) { return ring + (uint32_t)((h % PT_SLOTS) * C::TILE); };
                auto arrived = [&](int h) {
                    ok = ok && wait(&bar.kv_full[h % PT_SLOTS], h / PT_SLOTS);
                    pt_fence_async();  // written by cp.async and stores, read by the tensor core
                };
                arrived(half);
                for (int t = 0; t < n_t && ok; ++t) {
                    ok = wait(&bar.q_full[t], n_q[t]++);
                    pt_fence_after();
                    if (ok) {
                        scores(t, slot_at(half));
                        pt_commit(&bar.s_full[t], leader);
                        if (t == n_t - 1) pt_commit(&bar.kv_empty[half % PT_SLOTS], leader);
                    }
                }
                for (int j = 0; j < n_kt && ok; ++j) {
                    const int hv = half + 2 * j + 1, hk = hv + 1;
                    for (int t = 0; t < n_t && ok; ++t) {
                        if (t == 0) arrived(hv);
                        ok = ok && wait(&bar.p_full[t], n_s[t]);
                        if (n_s[t] > 0) ok = ok && wait(&bar.o_empty[t], n_s[t] - 1);
                        ++n_s[t];
                        pt_fence_after();
                        if (ok) {
                            outputs(t, slot_at(hv));
                            pt_commit(&bar.o_full[t], leader);
                            if (t == n_t - 1) pt_commit(&bar.kv_empty[hv % PT_SLOTS], leader);
                        }
                        if (j + 1 < n_kt) {
                            if (t == 0) arrived(hk);
                            if (ok) {
                                scores(t, slot_at(hk));
                                pt_commit(&bar.s_full[t], leader);
                                if (t == n_t - 1) pt_commit(&bar.kv_empty[hk % PT_SLOTS], leader);
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
        } else {
            // ---- copies: 16 rows at a time, lane j (and j + 16) sees to row j ----
            const int lw = warp - 9;
            constexpr int CH = HDP / 8, RL = 32 / CH;  // chunks of a row, rows at a time
            const int row_bytes = HD * 2, x = lane % CH, r0 = lane / CH;
            const bool in_row = x * 16 < row_bytes;
            const uint8_t* const src_x[2] = {(const uint8_t*)A.k + x * 16, (const uint8_t*)A.v + x * 16};
            int half = 0;
            uint32_t tile_no = 0;
            bool ok = true;
            while (ok && next()) {
                const int last_lim = it.start + (it.row0 + it.rows - 1) / G;
                const int first_lim = it.start + it.row0 / G;
                for (int kt = it.kt0; kt < it.kt1 && ok; ++kt, ++tile_no) {
                    // the tile's table entries, for K and V; -1: no page, or not seen
                    int rows3[3];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        const int pos = kt * PT_KT + (lw + 3 * i) * 16 + (lane & 15);
                        rows3[i] = -1;
                        if (lw + 3 * i < 8 && pos <= last_lim) {
                            const int col = (int)w.ps.div((uint32_t)pos);
                            const int page = page_at(w, it.s.row[col]);
                            if (page >= 0)
                                rows3[i] = (page * w.Hkv + it.hk) * w.page_size + (pos - col * w.page_size);
                        }
                    }
                    const bool careful = kt * PT_KT + PT_KT - 1 > first_lim;
#pragma unroll 1
                    for (int kv = 0; kv < 2 && ok; ++kv, ++half) {
                        const int slot = half % PT_SLOTS, use = half / PT_SLOTS;
                        if (use > 0 && !wait(&bar.kv_empty[slot], use - 1)) {
                            ok = false;
                            break;
                        }
                        const uint32_t dst = ring + (uint32_t)(slot * C::TILE + (x >> 3) * C::BLOCK);
                        const uint8_t* src = src_x[kv];
                        // small loops: this code shares the instruction cache with the softmax
#pragma unroll 1
                        for (int i = 0; i < 3; ++i) {
                            const int g16 = lw + 3 * i;
                            if (g16 >= 8) break;
                            const int row = i == 0 ? rows3[0] : i == 1 ? rows3[1] : rows3[2];
                            uint32_t bad = 0;
                            if (kv == 0 || !careful) {
#pragma unroll 4
                                for (int k = 0; k < 16 / RL; ++k) {
                                    const int from = k * RL + r0;
                                    const int n = __shfl_sync(0xffffffffu, row, from);
                                    const bool there = n >= 0 && in_row;
                                    cp16(dst + pt_off(g16 * 16 + from, x & 7),
                                         src + (there ? (int64_t)n * row_bytes : 0), there);
                                }
                            } else {
#pragma unroll 1
                                for (int k = 0; k < 16 / RL; ++k) {
                                    const int from = k * RL + r0;
                                    const int n = __shfl_sync(0xffffffffu, row, from);
                                    uint4 v = make_uint4(0, 0, 0, 0);
                                    if (n >= 0 && in_row)
                                        v = __ldg(reinterpret_cast<const uint4*>(src + (int64_t)n * row_bytes));
                                    bool odd = false;
                                    v.x = finite16x2(v.x, odd), v.y = finite16x2(v.y, odd);
                                    v.z = finite16x2(v.z, odd), v.w = finite16x2(v.w, odd);
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                                     dst + pt_off(g16 * 16 + from, x & 7)),
                                                 "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                                                 : "memory");
                                    const uint32_t any = __ballot_sync(0xffffffffu, odd);
#pragma unroll
                                    for (int b = 0; b < RL; ++b)
                                        if (any & (((1u << CH) - 1u) << (b * CH))) bad |= 1u << (k * RL + b);
                                }
                            }
                            const uint32_t none = __ballot_sync(0xffffffffu, row < 0) & 0xffffu;
                            if (lane == 0) {
                                if (kv == 0) sh_gone[tile_no & 3][g16] = (uint16_t)none;
                                else sh_bad[tile_no & 3][g16] = (uint16_t)bad;
                            }
                        }
                        if (kv == 1 && careful) {
                            pt_fence_async();
                            mbar_arrive(&bar.kv_full[slot]);
                        } else {
                            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                                             smem_u32(&bar.kv_full[slot]))
                                         : "memory");
                        }
                        if (lane == 0) mbar_arrive(&bar.kv_full[slot]);  // sh_gone, sh_bad
                    }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
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
}

CutRule tensor_rule(int min_rows, int max_rows) {
    // one CTA to an SM (148 of a B200), a piece for each
    return CutRule{PT_R, PT_KT, min_rows, max_rows, 148, 128};
}

template <int HDP>
static int launch(const RowsArgs& a, int64_t grid, cudaStream_t st) {
    auto kern = attn_tensor_kernel<HDP>;
    IB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)TensorCfg<HDP>::SMEM));
    IB_CUDA_CHECK(launch_pdl(kern, dim3((unsigned)grid), dim3(PT_THREADS), TensorCfg<HDP>::SMEM, st,
                             true, a));
    return IB_OK;
}

int attn_tensor_launch(const RowsArgs& a, int64_t tiles, int64_t max_pos, cudaStream_t st) {
    const int64_t most = tiles * (max_pos / a.rule.least + 1 + a.rule.R);
    const int64_t grid = std::min<int64_t>(a.rule.n_pieces, most);
    return a.w.HD <= 64 ? launch<64>(a, grid, st) : launch<128>(a, grid, st);
}

}  // namespace ib
