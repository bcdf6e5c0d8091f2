// ib_attention_paged: causal GQA attention of a batch of new tokens over the paged cache.
//
// The query rows of a sequence that share a kv head -- (token, head of the group), token by
// token -- are consecutive: row r is token r / G, head r % G.  A tile is R such rows against the
// positions they see.  Tiles are cut so that a batch of any mix of lengths keeps every SM busy to
// the end (paged_plan.cuh); a tile that is cut leaves partial results (running maximum m,
// exponential sum l, unnormalised sum of p v), and a second kernel joins them:
//     out = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s.
// Lengths are device data: every CTA works the cuts out for itself from cu_q and len (one pass
// over the batch; no planning launch).
//
// Products of FP32 operands keep 2^-20 or better on the tensor cores:
//   FP16 pages  q = hi + lo and p = hi + lo in FP16, K and V as they are: two products.  q rows
//               are scaled to a largest element in [256, 512) and p by 2^10, powers of two that
//               keep the lo parts out of FP16's subnormals (a p below 2^-13 of the row's largest,
//               whose lo part gets there, is off by at most 2^-35 of that largest).
//   FP32 pages  both operands as TF32 hi + lo, hi hi + hi lo + lo hi: three products, with the
//               range of FP32.
// The MMA adds to its FP32 accumulator by cutting, half a unit of the accumulator per step on
// average and always towards zero: a running sum over a long sequence would drift (2.6e-6 of
// the result over 131072 positions, 4e-7 this way).  So lo parts have accumulators of their own
// or go first, and p v of each tile starts from zero and is added to the running sum by FFMA,
// which rounds and takes the rescaling with it.
// Positions that a row does not see get a score of -inf; pages that are not there are filled
// with zeros, and in tiles where some row does not see a position that has a page (`careful`),
// V is checked for values that are not finite (0 x inf).
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "common.cuh"
#include "mma_tile.cuh"
#include "paged.cuh"
#include "paged_plan.cuh"
#include "pdl.cuh"
#include "pipeline.cuh"

namespace ib {

int paged_attention_fault_take(int* code) {
    int r = paged_fault_take_here(code), c = 0;
    if (r == IB_OK) r = paged_tensor_fault_take(&c);
    *code = paged_fault_worse(*code, c);
    return r;
}

// ---- a warp's 16 rows on mma.sync, for the wide kernel ---------------------------------------
// One query row into shared memory as hi and lo parts, by one warp.  Returns the factor that
// turns its scores into base-2 exponents.
template <bool F32, int HDP>
__device__ __forceinline__ float stage_q_row(const float* row, int HD, uint8_t* hi, uint8_t* lo,
                                             float scale_log2) {
    const int lane = threadIdx.x & 31;
    float x[HDP / 32], top = 0.f;
#pragma unroll
    for (int i = 0; i < HDP / 32; ++i) {
        const int d = lane + 32 * i;
        x[i] = row && d < HD ? row[d] : 0.f;
        top = fmaxf(top, fabsf(x[i]));
    }
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i)
            split_tf32(x[i], reinterpret_cast<uint32_t*>(hi)[lane + 32 * i],
                       reinterpret_cast<uint32_t*>(lo)[lane + 32 * i]);
        return scale_log2;
    } else {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float down;
        const float up = pow2_scale(top, down);
#pragma unroll
        for (int i = 0; i < HDP / 32; ++i) {
            const float y = x[i] * up;
            const __half h = __float2half_rn(y);
            reinterpret_cast<__half*>(hi)[lane + 32 * i] = h;
            reinterpret_cast<__half*>(lo)[lane + 32 * i] = __float2half_rn(y - __half2float(h));
        }
        return scale_log2 * down;
    }
}

// LD: bytes between K or V rows in shared memory (16 more than a row: the 8 rows of an ldmatrix,
// and the TF32 V columns, hit distinct banks); QLD: the same for q.
template <typename KV, int HDP, int KW, bool TREE>
struct WarpRows {
    static constexpr bool F32 = sizeof(KV) == 4;
    static constexpr int LD = HDP * (int)sizeof(KV) + 16, QLD = HDP * (F32 ? 4 : 2) + 16;
    static constexpr int NB = KW / 8, DB = HDP / 8, KS = F32 ? HDP / 8 : HDP / 16;
    // p is carried times 2^10 (FP16 pages)
    static constexpr float P_BIAS = F32 ? 0.f : 10.f;

    float acc[DB][4];
    float m[2], l[2];
    int lim[2];     // last positions that rows g and g + 8 see
    float sc[2];
    uint32_t q_hi, q_lo;  // this lane's fragment addresses
    [[maybe_unused]] const uint32_t* nodes[2];  // trees: the rows' masks
    [[maybe_unused]] int first_node, words;     // position of bit 0

    // whether row h sees position p
    __device__ __forceinline__ bool sees(int h, int p) const {
        if (p > lim[h]) return false;
        if constexpr (TREE) {
            const int c = p - first_node;
            return c < 0 || (c < 32 * words && ((__ldg(nodes[h] + (c >> 5)) >> (c & 31)) & 1));
        }
        return true;
    }

    __device__ __forceinline__ void start(uint32_t hi, uint32_t lo) {
        const int lane = threadIdx.x & 31;
        q_hi = hi + (uint32_t)((lane & 15) * QLD + (lane >> 4) * 16);
        q_lo = lo + (uint32_t)((lane & 15) * QLD + (lane >> 4) * 16);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[d][i] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    __device__ __forceinline__ void load_q(int k, uint32_t (&h)[4], uint32_t (&e)[4]) const {
        ldsm_x4(q_hi + k * 32, h[0], h[1], h[2], h[3]);
        ldsm_x4(q_lo + k * 32, e[0], e[1], e[2], e[3]);
    }

    // kd, vd: the tile's K and V in shared memory (v_ptr: vd as a pointer); pos_of(j): the
    // position of tile row j, j = 8 n + 2 t4 + (0 or 1) of this lane or, for a j that is the
    // same in the whole warp, any.
    template <typename Pos>
    __device__ __forceinline__ void step(uint32_t kd, uint32_t vd, const uint8_t* v_ptr, bool careful,
                                         Pos pos_of) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
        float s[NB][4], e[NB][4];
        zero(s), zero(e);
        if constexpr (!F32) {
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t ah[4], al[4];
                load_q(k, ah, al);
#pragma unroll
                for (int n = 0; n < NB; n += 2) {  // 16 positions x 16 dimensions
                    uint32_t b[4];
                    ldsm_x4(kd + (uint32_t)((n * 8 + (lane & 7) + ((lane >> 4) << 3)) * LD + k * 32 +
                                            ((lane >> 3) & 1) * 16),
                            b[0], b[1], b[2], b[3]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_f16(s[n + j], ah, b[2 * j], b[2 * j + 1], s[n + j]);
                        mma_f16(e[n + j], al, b[2 * j], b[2 * j + 1], e[n + j]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                uint32_t ah[2][4], al[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) load_q(k + j, ah[j], al[j]);
                float t[NB][4];  // two k-steps at a time
                zero(t);
#pragma unroll
                for (int n = 0; n < NB; ++n) {  // 8 positions x 16 dimensions
                    uint32_t b[4], h[4], r[4];
                    ldsm_x4(kd + (uint32_t)((n * 8 + (lane & 7)) * LD + k * 32 + (lane >> 3) * 16),
                            b[0], b[1], b[2], b[3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) split_tf32_cut(__uint_as_float(b[j]), h[j], r[j]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_tf32(t[n], ah[j], h[2 * j], h[2 * j + 1], t[n]);
                        mma_tf32(e[n], ah[j], r[2 * j], r[2 * j + 1], e[n]);
                        mma_tf32(e[n], al[j], h[2 * j], h[2 * j + 1], e[n]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[n][j] += t[n][j];
                }
            }
        }
        // what the rows do not see, and the running maximum
        float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int p0 = pos_of(n * 8 + 2 * t4), p1 = pos_of(n * 8 + 2 * t4 + 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float &a = s[n][2 * h], &b = s[n][2 * h + 1];
                a = sees(h, p0) ? (a + e[n][2 * h]) * sc[h] : -INFINITY;
                b = sees(h, p1) ? (b + e[n][2 * h + 1]) * sc[h] : -INFINITY;
                x[h] = fmaxf(x[h], fmaxf(a, b));
            }
        }
        float c[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) x[h] = fmaxf(x[h], __shfl_xor_sync(0xffffffffu, x[h], o));
            x[h] = fmaxf(m[h], x[h]);
            c[h] = x[h] == -INFINITY ? 1.f : ex2(m[h] - x[h]);
            m[h] = x[h];
            l[h] *= c[h];
            const float base = m[h] == -INFINITY ? 0.f : m[h] - P_BIAS;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float &a = s[n][2 * h], &b = s[n][2 * h + 1];
                a = ex2(a - base), b = ex2(b - base);
                l[h] += a + b;
            }
        }
        bool odd = false;  // a V value that is not finite, among this thread's
        if constexpr (!F32) {
            uint32_t ph[KW / 16][4], pl[KW / 16][4];
#pragma unroll
            for (int k = 0; k < KW / 16; ++k) {
                split2(s[2 * k][0], s[2 * k][1], ph[k][0], pl[k][0]);
                split2(s[2 * k][2], s[2 * k][3], ph[k][1], pl[k][1]);
                split2(s[2 * k + 1][0], s[2 * k + 1][1], ph[k][2], pl[k][2]);
                split2(s[2 * k + 1][2], s[2 * k + 1][3], ph[k][3], pl[k][3]);
            }
#pragma unroll
            for (int d = 0; d < DB; d += 2) {
                float t[2][4];
                zero(t);
#pragma unroll
                for (int k = 0; k < KW / 16; ++k) {
                    uint32_t b[4];
                    ldsm_x4_t(vd + (uint32_t)((k * 16 + (lane & 15)) * LD + d * 16 + (lane >> 4) * 16),
                              b[0], b[1], b[2], b[3]);
                    if (careful) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) b[j] = finite16x2(b[j], odd);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma_f16(t[j], pl[k], b[2 * j], b[2 * j + 1], t[j]);
                        mma_f16(t[j], ph[k], b[2 * j], b[2 * j + 1], t[j]);
                    }
                }
                add(d, t[0], c), add(d + 1, t[1], c);
            }
        } else {
            // the MMA's k index t holds position 2 t, t + 4 position 2 t + 1, in both operands:
            // then the scores' accumulator is the A operand as it lies
            uint32_t ph[NB][4], pl[NB][4];
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                split_tf32_weight(s[k][0], ph[k][0], pl[k][0]);
                split_tf32_weight(s[k][2], ph[k][1], pl[k][1]);
                split_tf32_weight(s[k][1], ph[k][2], pl[k][2]);
                split_tf32_weight(s[k][3], ph[k][3], pl[k][3]);
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                float t[1][4], r[1][4];
                zero(t), zero(r);
#pragma unroll
                for (int k = 0; k < NB; ++k) {
                    const uint8_t* v0 = v_ptr + (k * 8 + 2 * t4) * LD + d * 32 + g * 4;
                    float y0 = *reinterpret_cast<const float*>(v0);
                    float y1 = *reinterpret_cast<const float*>(v0 + LD);
                    if (careful) {
                        if (!(fabsf(y0) < INFINITY)) odd = true, y0 = 0.f;
                        if (!(fabsf(y1) < INFINITY)) odd = true, y1 = 0.f;
                    }
                    uint32_t h0, r0, h1, r1;
                    split_tf32_cut(y0, h0, r0);
                    split_tf32_cut(y1, h1, r1);
                    mma_tf32(t[0], ph[k], h0, h1, t[0]);
                    mma_tf32(r[0], ph[k], r0, r1, r[0]);
                    mma_tf32(r[0], pl[k], h0, h1, r[0]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)  // towards zero: split_tf32_cut
                    t[0][j] = __fadd_rz(t[0][j], r[0][j]);
                add(d, t[0], c);
            }
        }
        if (__any_sync(0xffffffffu, odd)) {
            // rows that see such a value are not finite there
#pragma unroll 1
            for (int j = 0; j < KW; ++j) {
                const int pos = pos_of(j);
                const uint8_t* vr = v_ptr + j * LD;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int at = d * 8 + 2 * t4 + i;
                        float y;
                        if constexpr (F32) y = reinterpret_cast<const float*>(vr)[at];
                        else y = __half2float(reinterpret_cast<const __half*>(vr)[at]);
                        if (fabsf(y) < INFINITY) continue;
                        if (sees(0, pos)) acc[d][i] = NAN;
                        if (sees(1, pos)) acc[d][2 + i] = NAN;
                    }
            }
        }
    }

    // the sums of a row are spread over its four lanes
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int o = 1; o <= 2; o <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
    }

    template <int N>
    static __device__ __forceinline__ void zero(float (&x)[N][4]) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[n][j] = 0.f;
    }
    __device__ __forceinline__ void add(int d, const float (&t)[4], const float (&c)[2]) {
        acc[d][0] = fmaf(acc[d][0], c[0], t[0]), acc[d][1] = fmaf(acc[d][1], c[0], t[1]);
        acc[d][2] = fmaf(acc[d][2], c[1], t[2]), acc[d][3] = fmaf(acc[d][3], c[1], t[3]);
    }
};

// ---- up to 32 rows: single tokens and short drafts ---------------------------------------
// The bound is reading K and V once, and next to it a warp's own chain of loads, scores, maximum
// and products.  So the products are turned round -- 16 positions are the MMA's M, eight query
// rows its N: scores K q', outputs V' p -- which halves the instructions and registers of eight
// rows against 16-row tiles (four query heads on a kv head fill half of N, not a quarter of M);
// and each of a CTA's warps runs through every NW-th tile of 16 positions by itself, with its
// own ring in shared memory filled by its own cp.async and no barrier in the loop; they join at
// the end.  A ring slot is one half of a tile, K or V.  64 single tokens over 200..4096 positions
// (32 heads on 8, head_dim 128): 113 us with FP16 pages, 5.1 TB/s or 0.78 of the measured rate (join
// included), 5.2 to 5.3 TB/s with FP32 pages (1.23 GB in 233 us); two tokens over 100001..131072
// positions (64 heads on 8, FP16) 168 to 178 us, 5.2 to 5.5 TB/s.  At head_dim 256, with fewer and
// longer ring slots to an SM, 3.7 TB/s (FP16) and 3.4 TB/s (FP32).  (Warps with pieces of their own, their
// copies running on from tile to tile, took 135 us against 119 us for 64 single tokens over
// 200..4096 positions: warps far apart in the code miss the instruction cache.)
template <typename KV, int HDP>
struct NarrowCfg {
    static constexpr bool F32 = sizeof(KV) == 4;
    static constexpr int R = 8, KW = 16;
    static constexpr int LD = HDP * (int)sizeof(KV) + 16, QLD = HDP * 4 + 16;
    static constexpr int HALF = KW * LD;
    // 64 single tokens at head_dim 128 in FP16: 117 us with three CTAs of four warps to an SM,
    // 126 us with two, 130 us with four of three half tiles a warp
    static constexpr int ROWB = HDP * (int)sizeof(KV);
    static constexpr int D = ROWB <= 256 ? 4 : ROWB <= 512 ? 3 : 2;  // ring slots of a warp
    static constexpr int CTAS = ROWB <= 256 ? 3 : ROWB <= 512 ? 2 : 1;  // to an SM
    static constexpr int NW = 4, NT = NW * 32;
    static constexpr bool QREG = HDP * (F32 ? 2 : 1) <= 256;  // q fragments stay in registers
    static constexpr int Q_BYTES = QREG ? 0 : 2 * R * QLD;  // or lie in shared memory (FP32)
    static constexpr size_t RING = (size_t)NW * (Q_BYTES + D * HALF);
    static constexpr size_t MERGE = (size_t)NW * R * (HDP + 4) * 4;  // of the warps' results
    static constexpr size_t SMEM = RING > MERGE ? RING : MERGE;
    static_assert(QREG || F32, "");
};

template <typename KV, int HDP, bool TREE>
__global__ void __launch_bounds__(NarrowCfg<KV, HDP>::NT, NarrowCfg<KV, HDP>::CTAS)
    attn_narrow_kernel(const __grid_constant__ RowsArgs A) {
    using C = NarrowCfg<KV, HDP>;
    constexpr bool F32 = C::F32;
    constexpr int R = C::R, KW = C::KW, LD = C::LD, QLD = C::QLD, D = C::D, NW = C::NW;
    constexpr int KS = F32 ? HDP / 8 : HDP / 16, DB = HDP / 16;
    constexpr float P_BIAS = F32 ? 0.f : 10.f;  // p is carried times 2^10 (FP16 pages)
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float sh_m[NW][R], sh_l[NW][R];
    const PagedView& w = A.w;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    pdl_wait();
    pdl_launch_dependents();
    Item item;
    if (!find_item<C::NT, false>(w, A.rule, blockIdx.x, item)) return;
    const int G = w.H / w.Hkv, HD = w.HD;
    Segment it;
    it.s = item.s;
    it.hk = item.hk;
    it.row0 = item.tile * R;
    it.rows = min(R, it.s.n * G - it.row0);
    it.start = it.s.L - it.s.n;
    it.part = item.n_parts == 1 ? -1 : item.part_base + item.part;
    const int first_lim = all_see<TREE>(it.start, it.row0, G);
    const int last_lim = it.start + (it.row0 + it.rows - 1) / G;
    // this warp's tiles: kt0, kt0 + NW ..
    const int kt0 = item.kt0 + warp, kt1 = min(item.kt1, last_lim < 0 ? 0 : last_lim / KW + 1);
    uint8_t* ring = smem + warp * (C::Q_BYTES + D * C::HALF);
    const uint32_t ring_a = smem_u32(ring);
    uint8_t* q_smem = ring + D * C::HALF;

    // ---- copies ----
    // Lane j (and j + 16) sees to position j of a tile: its table entry is read a tile ahead of
    // the copies, its row number in the layer is shuffled to the lanes that copy the row.
    auto entry_of = [&](int kt) -> int {
        const int pos = kt * KW + (lane & (KW - 1));
        if (kt >= kt1 || pos > last_lim) return -1;
        return page_at(w, it.s.row[w.ps.div((uint32_t)pos)]);
    };
    const int row_bytes = HD * (int)sizeof(KV);
    constexpr int CH = HDP * (int)sizeof(KV) / 16, CHL = CH < 32 ? CH : 32, RL = 32 / CHL;
    const int x0 = (lane % CHL) * 16, r0 = lane / CHL;
    const uint8_t* k_src = (const uint8_t*)A.k + x0;
    const uint8_t* v_src = (const uint8_t*)A.v + x0;
    const uint32_t dst0 = ring_a + (uint32_t)(r0 * LD + x0);
    int in_kt = kt0, page = entry_of(kt0), row = -1, slot_in = 0;
    uint32_t gone[3] = {0, 0, 0};  // positions without a page: of the tile at work and those after
    auto copy_half = [&](const uint8_t* src) {
        if (in_kt < kt1) {
            const uint32_t d0 = dst0 + (uint32_t)(slot_in * C::HALF);
#pragma unroll
            for (int i = 0; i < KW / RL; ++i) {
                const int r = __shfl_sync(0xffffffffu, row, i * RL + r0);
                const int64_t at = (int64_t)max(r, 0) * row_bytes;
#pragma unroll
                for (int x = 0; x < CH / CHL; ++x) {
                    const bool ok = r >= 0 && x0 + x * 512 < row_bytes;
                    // nothing is read through the address of a chunk that is not there
                    cp16(d0 + (uint32_t)(i * RL * LD + x * 512), src + (ok ? at + x * 512 : 0), ok);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        slot_in = slot_in == D - 1 ? 0 : slot_in + 1;
    };
    auto copy_k = [&](int place) {  // place: of this tile in gone[]
        const int pos = in_kt * KW + (lane & (KW - 1));
        const int in_page = pos - (int)w.ps.div((uint32_t)pos) * w.page_size;
        row = page < 0 ? -1 : (page * w.Hkv + it.hk) * w.page_size + in_page;
        gone[place] = __ballot_sync(0xffffffffu, page < 0);
        page = entry_of(in_kt + NW);
        copy_half(k_src);
    };
    auto copy_v = [&]() {
        copy_half(v_src);
        in_kt += NW;
    };
#pragma unroll
    for (int h = 0; h < D - 1; ++h) {
        if (h & 1) copy_v();
        else copy_k(h / 2);
    }

    int slot = 0;
    const uint32_t k_frag = (uint32_t)((lane & 15) * LD + (lane >> 4) * 16);
    const uint32_t v_frag = (uint32_t)(((lane & 7) + ((lane >> 4) << 3)) * LD + ((lane >> 3) & 1) * 16);
    // this lane's rows are 2 t4 and 2 t4 + 1
    int lim[2];
    [[maybe_unused]] const uint32_t* nodes[2];
    float sc[2], m[2], l[2], acc[DB][4];
    uint32_t qh[C::QREG ? KS : 1][2], ql[C::QREG ? KS : 1][2];
    // q as B: row g; FP16 k-steps of dimensions 2 t4, + 1, + 8, + 9, TF32 t4, + 4
    const float* src = g < it.rows ? q_row(A, it, G, it.row0 + g) : nullptr;
    float f = A.scale_log2;
    if constexpr (F32) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
            const int d = k * 8 + t4 + 4 * j;
            const float x = src && d < HD ? __ldg(src + d) : 0.f;
            uint32_t hi, lo;
            split_tf32(x, hi, lo);
            if constexpr (C::QREG) {
                qh[k][j] = hi, ql[k][j] = lo;
            } else {
                *reinterpret_cast<uint32_t*>(q_smem + g * QLD + d * 4) = hi;
                *reinterpret_cast<uint32_t*>(q_smem + (R + g) * QLD + d * 4) = lo;
            }
        }
        if constexpr (!C::QREG) __syncwarp();
    } else {
        float2 x[KS][2];
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
            const int d = k * 16 + 2 * t4 + 8 * j;
            x[k][j] = src && d < HD ? __ldg(reinterpret_cast<const float2*>(src + d))
                                    : make_float2(0.f, 0.f);
            top = fmaxf(top, fmaxf(fabsf(x[k][j].x), fabsf(x[k][j].y)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float down;
        const float up = pow2_scale(top, down);
        f *= down;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                split2(x[k][j].x * up, x[k][j].y * up, qh[k][j], ql[k][j]);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int mine = 2 * t4 + j;
        lim[j] = mine < it.rows ? it.start + (it.row0 + mine) / G : -1;
        if constexpr (TREE) nodes[j] = mask_row(A, it.s.q0, it.row0 + mine, mine < it.rows);
        sc[j] = __shfl_sync(0xffffffffu, f, (2 * t4 + j) * 4);
        m[j] = -INFINITY;
        l[j] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[d][j] = 0.f;
    for (int kt = kt0; kt < kt1; kt += NW) {
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
        __syncwarp();  // every lane's copies of K, and its reads of the half before
        if constexpr (D & 1) copy_k((D - 1) / 2);
        else copy_v();
        const uint32_t kd = ring_a + (uint32_t)(slot * C::HALF) + k_frag;
        slot = slot == D - 1 ? 0 : slot + 1;
        // scores: rows of a fragment are positions g and g + 8, columns the lane's two rows.
        // sa, sb: two chains; e: the lo parts.
        float s[4];
        {
            float sa[4], sb[4], e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) sa[j] = sb[j] = e[j] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t a[4];
                ldsm_x4(kd + k * 32, a[0], a[1], a[2], a[3]);
                uint32_t ah[4], al[4];
                if constexpr (F32) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) split_tf32_cut(__uint_as_float(a[j]), ah[j], al[j]);
                }
                uint32_t q0, q1, r0, r1;
                if constexpr (C::QREG) {
                    q0 = qh[k][0], q1 = qh[k][1], r0 = ql[k][0], r1 = ql[k][1];
                } else {
                    const uint8_t* p = q_smem + g * QLD + (k * 8 + t4) * 4;
                    q0 = *reinterpret_cast<const uint32_t*>(p);
                    q1 = *reinterpret_cast<const uint32_t*>(p + 16);
                    r0 = *reinterpret_cast<const uint32_t*>(p + R * QLD);
                    r1 = *reinterpret_cast<const uint32_t*>(p + R * QLD + 16);
                }
                float(&x)[4] = k & 1 ? sb : sa;
                if constexpr (F32) {
                    mma_tf32(x, ah, q0, q1, x);
                    mma_tf32(e, ah, r0, r1, e);
                    mma_tf32(e, al, q0, q1, e);
                } else {
                    mma_f16(x, a, q0, q1, x);
                    mma_f16(e, a, r0, r1, e);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = (sa[j] + sb[j]) + e[j];
        }
        // what the rows do not see, the running maximum, p
        const uint32_t missing = gone[0];
        const int p0 = (missing >> g) & 1 ? 0x7fffffff : kt * KW + g;
        const int p1 = (missing >> (g + 8)) & 1 ? 0x7fffffff : kt * KW + g + 8;
        const bool careful = kt * KW + KW - 1 > first_lim;
        [[maybe_unused]] uint32_t sees[2] = {0xffffffffu, 0xffffffffu};  // of the tile's positions
        if constexpr (TREE)
            if (careful)
#pragma unroll
                for (int j = 0; j < 2; ++j) sees[j] = tree_bits(nodes[j], A.words, kt * KW - it.start);
        float c[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float &x = s[j], &y = s[2 + j];
            x = p0 <= lim[j] && (!TREE || ((sees[j] >> g) & 1)) ? x * sc[j] : -INFINITY;
            y = p1 <= lim[j] && (!TREE || ((sees[j] >> (g + 8)) & 1)) ? y * sc[j] : -INFINITY;
            float top = fmaxf(x, y);
#pragma unroll
            for (int o = 4; o <= 16; o <<= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(top, m[j]);
            c[j] = top == -INFINITY ? 1.f : ex2(m[j] - top);
            m[j] = top;
            const float base = top == -INFINITY ? 0.f : top - P_BIAS;
            x = ex2(x - base), y = ex2(y - base);
            l[j] = fmaf(l[j], c[j], x + y);
        }
        // p as B: positions along k, the row along n
        uint32_t ph[F32 ? 4 : 2], pl[F32 ? 4 : 2];
        if constexpr (F32) {
            // the MMA's k index t holds position 2 t, t + 4 position 2 t + 1, as V below
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                const int from = 8 * t4 + 4 * j + (g >> 1);
                const float x = __shfl_sync(0xffffffffu, s[2 * i], from);
                const float y = __shfl_sync(0xffffffffu, s[2 * i + 1], from);
                split_tf32_weight(g & 1 ? y : x, ph[2 * i + j], pl[2 * i + j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                split2(s[2 * i], s[2 * i + 1], ph[i], pl[i]);
                ph[i] = movm(ph[i]), pl[i] = movm(pl[i]);
            }
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
        __syncwarp();
        gone[0] = gone[1], gone[1] = gone[2];
        if constexpr (D & 1) copy_v();
        else copy_k((D - 1) / 2);
        const uint32_t vd = ring_a + (uint32_t)(slot * C::HALF);
        const uint8_t* v_ptr = ring + slot * C::HALF;
        slot = slot == D - 1 ? 0 : slot + 1;
        bool odd = false;  // a V value that is not finite, among this lane's
        // outputs: rows of a fragment are dimensions g and g + 8 of a block of 16
        auto products = [&](auto check) {
            constexpr bool CHECK = decltype(check)::value;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                uint32_t a[F32 ? 2 : 1][4];
                [[maybe_unused]] uint32_t al[2][4];
                if constexpr (F32) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {  // position 2 t4 + (j >> 1), dimension g + 8 (j & 1)
                        float y = *reinterpret_cast<const float*>(
                            v_ptr + (i * 8 + 2 * t4 + (j >> 1)) * LD +
                            (d * 16 + g + 8 * (j & 1)) * 4);
                        if (CHECK && !(fabsf(y) < INFINITY)) odd = true, y = 0.f;
                        split_tf32_cut(y, a[i][j], al[i][j]);
                    }
                } else {
                    ldsm_x4_t(vd + v_frag + d * 32, a[0][0], a[0][1], a[0][2], a[0][3]);
                    if (CHECK) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) a[0][j] = finite16x2(a[0][j], odd);
                    }
                }
                const float none[4] = {0.f, 0.f, 0.f, 0.f};
                float t[4];
                if constexpr (F32) {
                    float r[4];
                    mma_tf32(t, a[0], ph[0], ph[1], none);
                    mma_tf32(t, a[1], ph[2], ph[3], t);
                    mma_tf32(r, a[0], pl[0], pl[1], none);
                    mma_tf32(r, al[0], ph[0], ph[1], r);
                    mma_tf32(r, a[1], pl[2], pl[3], r);
                    mma_tf32(r, al[1], ph[2], ph[3], r);
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // towards zero: split_tf32_cut
                        t[j] = __fadd_rz(t[j], r[j]);
                } else {
                    mma_f16(t, a[0], pl[0], pl[1], none);
                    mma_f16(t, a[0], ph[0], ph[1], t);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[d][j] = fmaf(acc[d][j], c[j & 1], t[j]);
            }
        };
        if (careful) products(std::true_type{});
        else products(std::false_type{});
        if (careful && __any_sync(0xffffffffu, odd)) {
            // rows that see such a value are not finite there
#pragma unroll 1
            for (int i = 0; i < KW; ++i) {
                if ((missing >> i) & 1) continue;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                    const int at = i * LD / (int)sizeof(KV) + d * 16 + g + 8 * (j >> 1);
                    float y;
                    if constexpr (F32) y = reinterpret_cast<const float*>(v_ptr)[at];
                    else y = __half2float(reinterpret_cast<const __half*>(v_ptr)[at]);
                    if (fabsf(y) < INFINITY) continue;
                    if (kt * KW + i <= lim[j & 1] && (!TREE || ((sees[j & 1] >> i) & 1)))
                        acc[d][j] = NAN;
                }
            }
        }
    }

    // ---- the warps' results together, in the rings ----
    constexpr int MLD = HDP + 4;
    float* ma = reinterpret_cast<float*>(smem);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            ma[(warp * R + 2 * t4 + (j & 1)) * MLD + d * 16 + g + 8 * (j >> 1)] =
                acc[d][j];
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // a row's sum is spread over eight lanes
        float x = l[j];
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        if (g == 0) {
            sh_m[warp][2 * t4 + j] = m[j];
            sh_l[warp][2 * t4 + j] = x;
        }
    }
    __syncthreads();
    const int v4 = HD / 4;
    for (int e = tid; e < it.rows * v4; e += C::NT) {
        const int r = e / v4, x = (e - r * v4) * 4;
        float M = sh_m[0][r], sum = 0.f;
#pragma unroll
        for (int i = 1; i < NW; ++i) M = fmaxf(M, sh_m[i][r]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const float f = M == -INFINITY ? 1.f : ex2(sh_m[i][r] - M);
            const float4 y = *reinterpret_cast<const float4*>(ma + (i * R + r) * MLD + x);
            sum += f * sh_l[i][r];
            o.x += f * y.x, o.y += f * y.y, o.z += f * y.z, o.w += f * y.w;
        }
        if (it.part < 0) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            *reinterpret_cast<float4*>(out_row(A, it, G, it.row0 + r) + x) =
                make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        } else {
            const int64_t at = (int64_t)it.part * R + r;
            *reinterpret_cast<float4*>(A.part_acc + at * HD + x) = o;
            if (x == 0) A.part_ml[at] = make_float2(M, sum);
        }
    }
}

// ---- more rows on mma.sync, for head_dim over 128 -----------------------------------------
// WR warps of 16 rows each over the same key tiles, which the CTA brings in together.  Bound by
// the legacy tensor path and the splitting of its operands: the last 1024 of 4096 positions (16
// heads on 8, head_dim 256) 624 to 650 us on FP16 pages, 93 to 96 TFLOP/s of the formula, where
// head_dim 128 on tcgen05 has 510 to 560; 1.95 ms on FP32 pages.
template <typename KV, int HDP>
struct WideCfg {
    static constexpr bool F32 = sizeof(KV) == 4;
    static constexpr int WR = 4, NT = WR * 32, R = 16 * WR;
    static constexpr int ROWB = HDP * (int)sizeof(KV);
    static constexpr int KT = F32 ? 16 : 32;
    template <bool TREE>
    using Tile = WarpRows<KV, HDP, KT, TREE>;
    static constexpr int STAGES = 2;
    static constexpr int Q_BYTES = 2 * R * Tile<false>::QLD;
    static constexpr int STAGE = 2 * KT * Tile<false>::LD;
    static constexpr int RING = STAGES + 1;  // of row offsets: a tile's outlive its copies
    static constexpr size_t SMEM = (size_t)Q_BYTES + STAGES * STAGE;
};

template <typename KV, int HDP, bool TREE>
__global__ void __launch_bounds__(WideCfg<KV, HDP>::NT)
    attn_wide_kernel(const __grid_constant__ RowsArgs A) {
    using C = WideCfg<KV, HDP>;
    using T = typename C::template Tile<TREE>;
    constexpr int NT = C::NT, R = C::R, KT = C::KT, LD = T::LD, S = C::STAGES;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ long long row_off[C::RING][KT];  // where a position's row starts, -1: nowhere
    __shared__ int key_pos[C::RING][KT];        // its position, INT_MAX: none
    __shared__ float row_scale[R];
    const PagedView& w = A.w;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2;
    if (!A.beside) pdl_wait();
    pdl_launch_dependents();
    __shared__ Piece sh_piece;
    __shared__ int found;
    find_piece<NT>(w, A.rule, blockIdx.x, &sh_piece, &found);
    __syncthreads();
    if (!found) {
        if (A.beside) pdl_wait();
        return;
    }
    Piece piece = sh_piece;
    Segment it;
    const int G = w.H / w.Hkv, HD = w.HD;
    while (next_segment<false>(w, A.rule, piece, it)) {
    const int row0 = it.row0, rows = it.rows, start = it.start;
    const int first_lim = all_see<TREE>(start, row0, G), last_lim = start + (row0 + rows - 1) / G;
    const int kt0 = it.kt0, kt1 = it.kt1;
    const int n_kt = max(0, kt1 - kt0);
    const uint32_t q_base = smem_u32(smem), kv_base = q_base + C::Q_BYTES;

    auto entry_of = [&](int kt) -> int {  // read a tile ahead of the copies that need it
        const int pos = kt * KT + tid;
        if (tid >= KT || kt >= kt1 || pos > last_lim) return -1;
        return page_at(w, it.s.row[w.ps.div((uint32_t)pos)]);
    };
    auto put_offsets = [&](int i, int page) {  // tile i of the range
        if (tid >= KT) return;
        const int pos = (kt0 + i) * KT + tid;
        const int in_page = pos - (int)w.ps.div((uint32_t)pos) * w.page_size;
        row_off[i % C::RING][tid] =
            page < 0 ? -1 : (((long long)page * w.Hkv + it.hk) * w.page_size + in_page) * HD;
        key_pos[i % C::RING][tid] = page < 0 ? 0x7fffffff : pos;
    };
    const int cpr = HD * (int)sizeof(KV) / 16;
    auto issue = [&](int i) {
        if (i < n_kt) {
            const uint32_t kd = kv_base + (uint32_t)((i % S) * C::STAGE);
            constexpr int CH = C::ROWB / 16, N = KT * CH;
#pragma unroll 4
            for (int c = tid; c < N; c += NT) {
                const int r = c / CH, x = c % CH;
                const long long off = row_off[i % C::RING][r];
                const bool ok = off >= 0 && x < cpr;
                const size_t byte = ok ? (size_t)off * sizeof(KV) + (size_t)x * 16 : 0;
                const uint32_t d = kd + (uint32_t)(r * LD + x * 16);
                cp16(d, (const uint8_t*)A.k + byte, ok);
                cp16(d + KT * LD, (const uint8_t*)A.v + byte, ok);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) put_offsets(i, entry_of(kt0 + i));
    __syncthreads();
    for (int i = 0; i < S - 1; ++i) issue(i);
    int next_page = entry_of(kt0 + S - 1);

    for (int r = warp; r < R; r += C::WR) {
        const float* src = r < rows ? q_row(A, it, G, row0 + r) : nullptr;
        uint8_t* hi = smem + r * T::QLD;
        const float f = stage_q_row<C::F32, HDP>(src, HD, hi, hi + R * T::QLD, A.scale_log2);
        if (lane == 0) row_scale[r] = f;
    }
    __syncthreads();
    T t;
    t.start(q_base + warp * 16 * T::QLD, q_base + (R + warp * 16) * T::QLD);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = warp * 16 + g + 8 * h;
        t.lim[h] = r < rows ? start + (row0 + r) / G : -1;
        t.sc[h] = row_scale[r];
        if constexpr (TREE) {
            t.nodes[h] = mask_row(A, it.s.q0, row0 + r, r < rows);
            t.first_node = start, t.words = A.words;
        }
    }
    for (int i = 0; i < n_kt; ++i) {
        if (i + S - 1 < n_kt) put_offsets(i + S - 1, next_page);
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncthreads();
        issue(i + S - 1);
        next_page = entry_of(kt0 + i + S);
        const uint32_t kd = kv_base + (uint32_t)((i % S) * C::STAGE);
        const int* kp = key_pos[i % C::RING];
        t.step(kd, kd + KT * LD, smem + (kd - q_base) + KT * LD, (kt0 + i) * KT + KT - 1 > first_lim,
               [&](int j) { return kp[j]; });
    }
    t.finish();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = warp * 16 + g + 8 * h;
        if (r >= rows) continue;
        const bool whole = it.part < 0;
        const int64_t at = (int64_t)it.part * R + r;
        const float inv = !whole ? 1.f : t.l[h] == 0.f ? 0.f : 1.f / t.l[h];
        float* p = whole ? out_row(A, it, G, row0 + r) : nullptr;
#pragma unroll
        for (int d = 0; d < T::DB; ++d)
            if (d * 8 < HD) {
                const int x = d * 8 + 2 * (lane & 3);
                *reinterpret_cast<float2*>(whole ? p + x : part_at(A, it.part, r, x)) =
                    make_float2(t.acc[d][2 * h] * inv, t.acc[d][2 * h + 1] * inv);
            }
        if (!whole && (lane & 3) == 0) A.part_ml[at] = make_float2(t.m[h], t.l[h]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // the ring and q are free for the next segment
    }
    if (A.beside) pdl_wait();
}

// ---- joining the parts of a tile ---------------------------------------------------------
struct JoinArgs {
    PagedView w;
    CutRule rule;
    float* out;
    int64_t out_stride;
    const float* part_acc;
    const float2* part_ml;
};

__device__ __forceinline__ void join_store(const JoinArgs& A, const SeqInfo& s, int hk, int gr, int x4,
                                           const float4& o, float l) {
    const int G = A.w.H / A.w.Hkv, tok = (int)A.w.group.div((uint32_t)gr);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float* out = A.out + (int64_t)(s.q0 + tok) * A.out_stride + (int64_t)(hk * G + gr - tok * G) * A.w.HD;
    reinterpret_cast<float4*>(out)[x4] = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// Tiles of 8 rows that find_item cut, into many parts where they are long: a CTA to a tile, WPR
// warps to a row.  (A CTA to a row took 16 us against 6 on 64 single tokens: each of them plans.)
// Two warps keep two CTAs on an SM for many tiles; four get through the parts of a few long
// ones sooner.
template <int WPR>
__device__ __forceinline__ void join_parts(const JoinArgs& A, int item) {
    constexpr int NT = 8 * WPR * 32, MAXV = 2;  // float4 per lane: head_dim 256
    __shared__ float4 sh_acc[8 * WPR][32 * MAXV];
    __shared__ float sh_l[8 * WPR];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = warp / WPR;
    const int G = A.w.H / A.w.Hkv, HD = A.w.HD;
    Item it;
    // cu_q and len were complete before the attention kernel started; its partials follow
    const bool any = find_item<NT, true>(A.w, A.rule, item, it);
    pdl_wait();
    if (!any || it.n_parts == 1) return;
    const bool some = r < it.s.n * G - it.tile * 8;  // the other warps come along to the barrier
    auto at = [&](int i) { return (int64_t)(it.part_base + i) * 8 + r; };
    float M = -INFINITY, l = 0.f;
    float4 o[MAXV];
#pragma unroll
    for (int i = 0; i < MAXV; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = lane; some && i < it.n_parts; i += 32) M = fmaxf(M, A.part_ml[at(i)].x);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
#pragma unroll 8
    for (int i = warp % WPR; i < (some ? it.n_parts : 0); i += WPR) {
        const float2 y = A.part_ml[at(i)];
        const float c = M == -INFINITY ? 1.f : ex2(y.x - M);
        l += c * y.y;
        const float4* acc = reinterpret_cast<const float4*>(A.part_acc + at(i) * HD);
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
            if (lane + 32 * k < HD / 4) {
                const float4 x = acc[lane + 32 * k];
                o[k].x += c * x.x, o[k].y += c * x.y, o[k].z += c * x.z, o[k].w += c * x.w;
            }
    }
#pragma unroll
    for (int k = 0; k < MAXV; ++k) sh_acc[warp][lane + 32 * k] = o[k];
    if (lane == 0) sh_l[warp] = l;
    __syncthreads();
    if (warp % WPR || !some) return;
#pragma unroll
    for (int i = 1; i < WPR; ++i) {
        l += sh_l[warp + i];
#pragma unroll
        for (int k = 0; k < MAXV; ++k) {
            const float4 z = sh_acc[warp + i][lane + 32 * k];
            o[k].x += z.x, o[k].y += z.y, o[k].z += z.z, o[k].w += z.w;
        }
    }
#pragma unroll
    for (int k = 0; k < MAXV; ++k)
        if (lane + 32 * k < HD / 4) join_store(A, it.s, it.hk, it.tile * 8 + r, lane + 32 * k, o[k], l);
}

// Tiles of many rows that find_piece cut, mostly in two: CTA (no, y) looks whether piece `no`
// begins inside a tile, and sees to its share of that tile's rows JOIN_ROWS y ..: as many CTAs as the
// tile has cuts share it (one CTA took 44 us for trees of 230 rows over 12000 positions in eight parts).
// All CTAs are on the SMs at once, since each has to plan first: with 32 rows to a CTA, four times
// as many of them, the join of a mixed step took 36 us against 22 (cold caches).  The parts lie in L2; what bounds
// it is the plan and a few dependent reads: 12.5 us with cold caches for 148 cut tiles of 32 trees, of which
// some 6 are behind the attention kernel's end.
constexpr int JOIN_ROWS = 128, JOIN_THREADS = 512;
__device__ __forceinline__ void join_pieces(const JoinArgs& A, int no, int y) {
    __shared__ Piece sh_piece;
    __shared__ int found;
    const PagedView& w = A.w;
    const CutRule& rule = A.rule;
    const int tid = threadIdx.x;
    const int G = w.H / w.Hkv, HD = w.HD, R = rule.R;
    find_piece<JOIN_THREADS>(w, rule, no, &sh_piece, &found);
    __syncthreads();
    if (!found) return pdl_wait();
    // the tile that the piece begins in
    Piece p = sh_piece;
    const SeqInfo s = p.x.s;
    const long long start_g = start_work(rule, s, G);
    const TileAt t = tile_at<false>(w, rule, p, start_g);
    // its work is [a, b), and pieces c0 .. c1 hold shares of it: the first one's is its last
    // segment (unless the tile begins with the piece), the others' is their first
    const long long a = p.at - t.x0, b = a + t.all;
    int c0 = (int)(a / p.len), c1 = (int)((b - 1) / p.len);
    if (c0 == no || c1 >= rule.n_pieces) return pdl_wait();
    const int share = no - c0 - 1, shares = c1 - c0;
    const int first = 2 * c0 + (a == c0 * p.len ? 0 : 1), first_piece = c0;
    const int row0 = t.tile * R, rows = min(R, s.n * G - row0);
    if (rule.flat) {  // shares at its ends may be empty
        const int nkt = seen_tiles(rule, s.L - s.n, row0, rows, G);
        while (c0 < c1 && flat_cut(rule, (c0 + 1) * p.len - a, G, nkt) == 0) ++c0;
        while (c0 < c1 && flat_cut(rule, c1 * p.len - a, G, nkt) == nkt) --c1;
        if (c0 == c1) return pdl_wait();
    }
    // A thread to 32 bytes of a row, four to 128, eight rows to a warp: the parts lie that way.
    const int lg = R < JOIN_ROWS ? 6 : 7, y0 = y * JOIN_ROWS, D4 = HD / 4;
    const int n = (HD + 31) / 32 * 4 << lg, begin = n * share / shares, end = n * (share + 1) / shares;
    auto join = [&](auto units) {  // U of them at a time, so that enough is on its way
        constexpr int U = decltype(units)::value;
#pragma unroll 1
        for (int e = begin + tid; e < end; e += U * JOIN_THREADS) {
            int r[U], d[U];
            bool ok[U];
            float M[U], l[U];
            float4 o[U][2];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = e + u * JOIN_THREADS;
                r[u] = y0 + ((at >> 2) & ((1 << lg) - 1)), d[u] = ((at >> (lg + 2)) * 4 + (at & 3)) * 2;
                ok[u] = at < end && r[u] < rows && d[u] < D4;
                if (!ok[u]) r[u] = d[u] = 0;
                M[u] = -INFINITY, l[u] = 0.f;
                o[u][0] = o[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll(U == 1 ? 4 : 2)
            for (int c = c0; c <= c1; ++c) {
                const int64_t part = c == first_piece ? first : 2 * c;
                float2 ml[U];
                float4 v[U][2];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    ml[u] = A.part_ml[part * R + r[u]];
                    const float4* const p =
                        reinterpret_cast<const float4*>(A.part_acc) + (part * D4 + d[u]) * R + r[u];
                    v[u][0] = p[0], v[u][1] = p[R];
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float top = fmaxf(M[u], ml[u].x);
                    const float f = top == -INFINITY ? 1.f : ex2(M[u] - top);
                    const float g = top == -INFINITY ? 1.f : ex2(ml[u].x - top);
                    M[u] = top;
                    l[u] = fmaf(l[u], f, g * ml[u].y);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float4& x = o[u][k];
                        const float4& z = v[u][k];
                        x.x = fmaf(x.x, f, g * z.x), x.y = fmaf(x.y, f, g * z.y);
                        x.z = fmaf(x.z, f, g * z.z), x.w = fmaf(x.w, f, g * z.w);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (ok[u]) join_store(A, s, t.hk, row0 + r[u], d[u] + k, o[u][k], l[u]);
        }
    };
    pdl_wait();
    if (end - begin > JOIN_THREADS) join(std::integral_constant<int, 2>{});
    else join(std::integral_constant<int, 1>{});
}

template <int WPR>
__global__ void __launch_bounds__(8 * WPR * 32) join_parts_kernel(const __grid_constant__ JoinArgs A) {
    join_parts<WPR>(A, blockIdx.x);
}
__global__ void __launch_bounds__(JOIN_THREADS, 2)
    join_pieces_kernel(const __grid_constant__ JoinArgs A) {
    join_pieces(A, blockIdx.x, blockIdx.y);
}
// Both in one launch, the pieces first.
__global__ void __launch_bounds__(JOIN_THREADS, 2)
    join_both_kernel(const __grid_constant__ JoinArgs parts, const __grid_constant__ JoinArgs pieces) {
    constexpr int WPR = JOIN_THREADS / 256;
    const int n = pieces.rule.n_pieces, y = blockIdx.x / n;
    if (y * JOIN_ROWS < pieces.rule.R) join_pieces(pieces, blockIdx.x - y * n, y);
    else join_parts<WPR>(parts, blockIdx.x - (pieces.rule.R + JOIN_ROWS - 1) / JOIN_ROWS * n);
}

// ---- launches ----------------------------------------------------------------------------
// One kernel's share of a call.
struct Share {
    CutRule rule;
    int64_t tiles;  // most row tiles, over all kv heads
    size_t acc_off, ml_off;
};

struct Plan {
    int n = 0;
    Share share[2];
    size_t bytes = 0;
};

// Parts for two rounds of the CTAs that the GPU holds at once, or one piece for each of them,
// of at least 128 positions: below that joining costs more.
template <typename KV, int HDP>
static CutRule narrow_rule(int min_rows, int max_rows) {
    using C = NarrowCfg<KV, HDP>;
    return CutRule{C::R, C::KW, min_rows, max_rows, kSMs * C::CTAS * 2, 128};
}
// Trees, whose rows fill a tile: where every SM has a part, parts are 1024 positions (us, with 128 and with
// 1024; two to four nodes, 32 heads on 8 of 128: 8 trees over 480, 900 and 200 .. 4096 positions, FP16, 21:17
// 31:23 44:35; 48 over 240, 480, 100 .. 900 and 200 .. 4096 34:29 46:37 47:39 99:99; 24 on FP32 pages over 240,
// 900 and 200 .. 4096 30:24 51:57 108:102; one over 60000 73:76).  Over tables of no more than 192 positions
// nothing is cut, which takes a launch less (us over tables of 144 to 192 positions, cut at 128 and whole; one and
// four nodes): FP32, 6 heads of 48, 1 tree 9.8:9.1 10.1:9.0, 64 trees 21:15 22:16; 32 heads on 8 of 128, FP16, 1 tree
// 10.5:9.3 11.1:9.9, 4 trees 10.8:10.7 14.6:10.6, 64 trees 30:22 53:36; FP32, 1 tree 12.5:12.4 13.2:13.0, 64 trees
// 42:33 77:60; 4 of 64, FP16, 64 trees 17.5:11.3 25.2:25.1.
template <typename KV, int HDP>
static CutRule narrow_tree_rule(int min_rows, int max_rows, int64_t max_pos) {
    CutRule r = narrow_rule<KV, HDP>(min_rows, max_rows);
    r.filled = 1024;
    if (max_pos <= 192) r.least = 192;
    return r;
}
template <typename KV, int HDP>
static CutRule wide_rule(int min_rows, int max_rows) {
    using C = WideCfg<KV, HDP>;
    return CutRule{C::R, C::KT, min_rows, max_rows, kSMs, 128};
}

// KERN: the kernel
template <auto KERN>
static int rows_launch(int threads, size_t smem, bool pieces, const RowsArgs& a,
                       int64_t tiles, int64_t max_pos, cudaStream_t st) {
    static DeviceOnce once;  // of each kernel
    IB_CUDA_CHECK(once.run([&] {
        return cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    }));
    // pieces: no more than `least` allows; parts: at most one more per tile
    const int64_t most = tiles * (max_pos / a.rule.least + 1 + a.rule.R);
    const int64_t grid = std::min<int64_t>(a.rule.n_pieces + (pieces ? 0 : tiles), most);
    IB_CUDA_CHECK(launch_pdl(KERN, dim3((unsigned)grid), dim3(threads), smem, st, true, a));
    return IB_OK;
}

// The kernels of a call, by the rows (new tokens x group) that a sequence may have: up to
// narrow_rows in tiles of eight on the narrow kernel, more on the wide one, by the caller's bound
// one of them alone.  Narrow against tcgen05 in us, at 16, 32 and 64 rows, 32 heads:
//   sequences over        FP16, 8 kv heads of 128         FP16, 4 kv heads of 64
//   2 x 30000..32000      90:140  152:139  274:140        37:68   51:68   82:66
//   8 x 200..4096         42:69   59:67    95:65          23:36   25:36   34:36
//   32 x 200..4096        101:180 167:185  317:196        37:77   58:76   103:78
//   96 x 200..2000        162:310 292:317  534:337        62:121  102:128 181:130
//                         FP32, 8 kv heads of 128         FP32, 4 kv heads of 64
//   2 x 30000..32000      209:305 393:305  769:310        59:112  103:112 177:112
//   8 x 200..4096         76:113  120:115  202:120        33:49   44:48   64:49
//   32 x 200..4096        215:362 426:370  750:385        72:119  115:119 199:121
//   96 x 200..2000        352:588 633:609  1214:630       104:186 184:192 336:193
// The number of sequences and their lengths move the crossing little: the kernel not taken is ahead
// only for two long sequences of 32 rows (FP16, head_dim 128), by 8 %, and for 64 rows of a few short
// ones (FP16, head_dim 64), by 6 %.
template <typename KV, int HDP>
constexpr int narrow_rows = sizeof(KV) == 4 && HDP == 128 ? 16 : 32;

// The same for trees, whose wide kernel takes one query tile and its key tiles in turn (us, 16, 24, 32
// and 48 rows, 32 heads):
//   sequences over   FP16, 8 kv heads of 128                  FP16, 4 kv heads of 64
//   2 x 30000        92:87    123:87   155:85   217:86        42:50   46:50   62:49   82:49
//   8 x 2000         36:49    37:50    62:49    70:50         20:30   24:30   23:29   26:29
//   32 x 2000        102:112  137:113  170:112  228:112       44:53   50:53   69:53   92:53
//   64 x 400         69:74    92:75    117:75   166:77        30:35   38:35   48:35   66:36
//                    FP32, 8 kv heads of 128                  FP32, 4 kv heads of 64
//   2 x 30000        218:296  317:296  409:296  571:296       67:90   80:90   103:89  141:89
//   8 x 2000         57:112   104:112  109:112  161:112       27:41   35:41   41:41   41:41
//   32 x 2000        213:347  296:347  390:347  581:347       70:99   83:99   110:99  149:100
//   64 x 400         120:174  174:175  214:176  319:178       43:55   51:55   68:55   93:55
// (head_dim over 128, whose wide kernel is the causal one: as there)
template <typename KV, int HDP>
constexpr int narrow_tree_rows = HDP > 128 ? 32 : sizeof(KV) == 2 && HDP == 128 ? 16 : 24;

// Few trees over tables of short rows are the narrow kernel's whatever their rows: the wide one's start alone
// takes 10 us and more, two tiles of eight rows to an SM less.  Narrow against wide (us in a graph, 32 heads; FP16
// pages, 8 kv heads of 128 and 4 of 64; FP32 pages likewise), by the tables' positions:
//   trees x rows  tiles        224                           480                           720
//   1 x 256       264, 132     16:28  16:20  22:34  17:29    21:36  17:25  32:54  20:28    27:35  18:25  41:38  22:28
//   4 x 64        272, 136     16:17  16:14  23:32  17:20    21:22  17:17  33:52  20:22    27:26  18:20  43:42  23:23
//   8 x 64        544, 272     29:17  15:14  40:32  17:20    40:22  16:18  62:54  23:28    50:33  19:22  83:67  30:30
//   4 x 256       1040, 520    49:28  22:20  72:34  28:29    65:36  28:25  117:55 41:32    80:48  34:29  158:66 52:32
// and fewer tiles, by tiles x positions:
//                 tiles        64000                         100000                        140000
//   1 x 64        72, 36       18:23  16:20  24:36  20:24    21:23  18:21  33:37  23:26    23:24  21:22  39:38  28:34
//   2 x 128       264, 132     17:21  17:18  24:33  20:22    19:23  18:20  29:43  23:23    22:25  20:20  34:38  27:23
// so: two tiles to an SM, and 128000 positions in all of them.
static bool few_short_trees(int64_t tiles, int64_t max_pos) {
    return tiles <= 2 * kSMs && tiles * max_pos <= 128000;
}

// Wide tiles run on tcgen05 for head_dim up to 128.  Above, S and O of two query tiles do not fit
// into tensor memory, nor FP32 sums of a row into a thread's registers; one query tile whose sums are
// shared by both softmax groups would fit on FP16 pages and is not built, on FP32 pages the TF32 parts
// of 128 query rows alone take 256 KB of shared memory.
template <int HDP>
constexpr bool on_tcgen05 = HDP <= 128;

template <typename KV, int HDP, bool TREE>
static Plan make_plan(const ib_kv_pages* p, const ib_kv_batch* b, int n_heads, int64_t max_pos) {
    constexpr int ALL = 0x7fffffff;
    const int64_t G = n_heads / p->n_kv_heads;
    const int64_t most_q = b->max_q > 0 ? std::min(b->max_q, b->n_tokens) : b->n_tokens;
    const int64_t seqs = std::min(b->n_seqs, b->n_tokens);
    Plan plan;
    auto add = [&](const CutRule& r, int64_t tiles_per_head) {
        Share& s = plan.share[plan.n++];
        s.rule = r;
        s.tiles = tiles_per_head * p->n_kv_heads;
        auto take = [&](size_t n) {
            const size_t at = plan.bytes;
            plan.bytes += (n + 255) / 256 * 256;
            return at;
        };
        // a piece cuts at most the tile it begins in and the one it ends in; a tile of k > len key
        // tiles has ceil(k / len) <= 2 k / len parts
        s.acc_off = take((size_t)2 * r.n_pieces * r.R * p->head_dim * sizeof(float));
        s.ml_off = take((size_t)2 * r.n_pieces * r.R * sizeof(float2));
    };
    const int64_t rows = b->n_tokens * G;
    constexpr int NARROW = TREE ? narrow_tree_rows<KV, HDP> : narrow_rows<KV, HDP>;
    const bool short_ones =
        TREE && on_tcgen05<HDP> && few_short_trees((rows / 8 + (seqs + 1) / 2) * p->n_kv_heads, max_pos);
    const bool few_rows = rows <= (int64_t)NARROW * b->n_seqs;  // to a sequence on average
    if (most_q * G <= NARROW || short_ones || (TREE && few_rows && most_q * G <= 2 * NARROW)) {
        add(TREE ? narrow_tree_rule<KV, HDP>(1, ALL, max_pos) : narrow_rule<KV, HDP>(1, ALL), seqs + rows / 8);
    } else {
        // trees: where a sequence has more rows on average, short ones are left to the wide kernel too (an
        // empty launch of the narrow one and its share of the join take 10 us), and where it has no more and
        // none has twice as many, all are the narrow one's.  On both kernels and on the narrow one (us): 24 of 4
        // to 28 rows over 500 .. 2000 positions (FP16, 8 kv heads of 128) 79 and 64, 60 of them over 100 .. 400
        // 75 and 56; 60 of 4 to 44 (FP16, 8 of 64) 68 and 53; FP32 178 and 151, 92 and 69; at head_dim 256
        // (24 of 4 to 56, 4 kv heads) 136 and 98, but 274 and 302 on FP32 pages.
        const bool few = b->n_seqs == 1 || G > NARROW || (TREE && !few_rows);
        const int narrow = few ? 0 : NARROW;
        if (narrow)
            add(TREE ? narrow_tree_rule<KV, HDP>(1, narrow, max_pos) : narrow_rule<KV, HDP>(1, narrow), std::min(seqs * (narrow / 8), seqs + rows / 8));
        CutRule r;
        // trees: two query tiles that share their key tiles where the sequences fill them on average, one
        // elsewhere (two long documents of 33 to 63 nodes, FP32 pages: 181 us with two tiles, 203 with one; 32
        // trees of 12 to 24 nodes, FP16: 213 and 133, both before cuts were moved to where they gain).  FP32 pages at head_dim above 64 have one anyway.
        const bool split = TREE && ((sizeof(KV) == 4 && HDP == 128) || rows <= 128 * seqs);
        if constexpr (on_tcgen05<HDP>) r = tensor_rule<KV, TREE>(p->head_dim, narrow + 1, ALL, split);
        else r = wide_rule<KV, HDP>(narrow + 1, ALL);
        add(r, seqs + rows / r.R);
    }
    return plan;
}

template <typename KV, int HDP, bool TREE>
static int run_plan(const ib_kv_pages* p, const ib_kv_batch* b, const Plan& plan, RowsArgs a,
                    uint8_t* ws, int64_t max_pos, cudaStream_t st) {
    using N = NarrowCfg<KV, HDP>;
    for (int i = 0; i < plan.n; ++i) {
        const Share& s = plan.share[i];
        a.rule = s.rule;
        const bool wide = s.rule.R > 8;
        a.beside = i > 0;
        a.part_acc = reinterpret_cast<float*>(ws + s.acc_off);
        a.part_ml = reinterpret_cast<float2*>(ws + s.ml_off);
        int r = IB_OK;
        if (!wide) {
            r = rows_launch<attn_narrow_kernel<KV, HDP, TREE>>(N::NT, N::SMEM, false, a, s.tiles, max_pos, st);
        } else if constexpr (on_tcgen05<HDP>) {
            r = attn_tensor_launch<KV, TREE>(a, s.tiles, max_pos, st);
        } else {
            using W = WideCfg<KV, HDP>;
            r = rows_launch<attn_wide_kernel<KV, HDP, TREE>>(W::NT, W::SMEM, true, a, s.tiles, max_pos, st);
        }
        if (r != IB_OK) return r;
    }
    JoinArgs parts{}, pieces{};
    int64_t n_parts = 0, n_pieces = 0;  // CTAs
    for (int i = 0; i < plan.n; ++i) {
        const Share& s = plan.share[i];
        const JoinArgs j{a.w, s.rule, a.out, a.out_stride, reinterpret_cast<float*>(ws + s.acc_off),
                         reinterpret_cast<float2*>(ws + s.ml_off)};
        if (s.rule.flat && max_pos <= s.rule.uncut - s.rule.KT) {
            // (no tile is cut: flat_cut)
        } else if (s.rule.R > 8) {
            pieces = j;
            n_pieces = (int64_t)s.rule.n_pieces * ((s.rule.R + JOIN_ROWS - 1) / JOIN_ROWS);
        } else if (max_pos > s.rule.least) {
            // (no tile is cut into parts where the tables' rows are no longer than the least part)
            parts = j;
            n_parts = s.tiles;
        }
    }
    const unsigned rounds = n_pieces ? (unsigned)(n_pieces / pieces.rule.n_pieces) : 0;
    if (n_parts && n_pieces)
        IB_CUDA_CHECK(launch_pdl(join_both_kernel, dim3((unsigned)(n_pieces + n_parts)),
                                 dim3(JOIN_THREADS), 0, st, true, parts, pieces));
    else if (n_pieces)
        IB_CUDA_CHECK(launch_pdl(join_pieces_kernel, dim3((unsigned)pieces.rule.n_pieces, rounds),
                                 dim3(JOIN_THREADS), 0, st, true, pieces));
    else if (n_parts && n_parts <= kSMs)
        IB_CUDA_CHECK(launch_pdl(join_parts_kernel<4>, dim3((unsigned)n_parts), dim3(8 * 4 * 32), 0, st,
                                 true, parts));
    else if (n_parts)
        IB_CUDA_CHECK(launch_pdl(join_parts_kernel<2>, dim3((unsigned)n_parts), dim3(8 * 2 * 32), 0, st,
                                 true, parts));
    return IB_OK;
}

template <typename KV>
static int attention_paged(const ib_kv_pages* p, const ib_kv_batch* b, RowsArgs a, void* ws,
                           size_t* bytes, int64_t max_pos, cudaStream_t st) {
    auto go = [&](auto hdp) {
        constexpr int HDP = decltype(hdp)::value;
        const Plan plan = a.mask ? make_plan<KV, HDP, true>(p, b, a.w.H, max_pos)
                                 : make_plan<KV, HDP, false>(p, b, a.w.H, max_pos);
        if (bytes) {
            *bytes = plan.bytes;
            return (int)IB_OK;
        }
        return a.mask ? run_plan<KV, HDP, true>(p, b, plan, a, (uint8_t*)ws, max_pos, st)
                      : run_plan<KV, HDP, false>(p, b, plan, a, (uint8_t*)ws, max_pos, st);
    };
    if (p->head_dim <= 64) return go(std::integral_constant<int, 64>{});
    if (p->head_dim <= 128) return go(std::integral_constant<int, 128>{});
    return go(std::integral_constant<int, 256>{});
}

static int attention_paged_any(const ib_kv_pages* p, const ib_kv_batch* b, const RowsArgs& a,
                               void* ws, size_t* bytes, int64_t max_pos, cudaStream_t st) {
    return p->type == IB_TYPE_F32 ? attention_paged<float>(p, b, a, ws, bytes, max_pos, st)
                                  : attention_paged<__half>(p, b, a, ws, bytes, max_pos, st);
}

}  // namespace ib

using namespace ib;

static size_t attention_workspace(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                  const ib_kv_batch* batch, const ib_kv_tree* tree, int n_heads) {
    if (batch->n_tokens == 0 || batch->n_seqs == 0) return 256;
    RowsArgs a{};
    a.w = paged_view(pages, seqs, batch, n_heads, tree);
    if (tree) a.mask = tree->mask;
    size_t n = 0;
    attention_paged_any(pages, batch, a, nullptr, &n, (int64_t)seqs->max_pages * pages->page_size, nullptr);
    return n;
}

extern "C" size_t ib_attention_paged_workspace(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                               const ib_kv_batch* batch, int n_heads) {
    if (paged_check_batch(pages, seqs, batch, 0, n_heads, "ib_attention_paged_workspace") != IB_OK)
        return 0;
    return attention_workspace(pages, seqs, batch, nullptr, n_heads);
}

extern "C" size_t ib_attention_paged_tree_workspace(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                                    const ib_kv_batch* batch, const ib_kv_tree* tree,
                                                    int n_heads) {
    const char* who = "ib_attention_paged_tree_workspace";
    if (paged_check_batch(pages, seqs, batch, 0, n_heads, who) != IB_OK ||
        paged_check_tree(batch, tree, who) != IB_OK)
        return 0;
    return attention_workspace(pages, seqs, batch, tree, n_heads);
}

// The structs are checked.
static int attention_call(const ib_kv_pages* pages, const ib_kv_seqs* seqs, const ib_kv_batch* batch,
                          const ib_kv_tree* tree, int layer, int n_heads, const float* q, int64_t q_stride,
                          float* out, int64_t out_stride, float scale, void* workspace,
                          size_t workspace_bytes, void* stream, const char* who) {
    if (batch->n_tokens == 0 || batch->n_seqs == 0) return IB_OK;
    if (!(q && out)) return paged_refuse(who, "null pointer argument");
    if ((((uintptr_t)q | (uintptr_t)out) & 15) || ((q_stride | out_stride) & 3))
        return paged_refuse(who, "q and out must be 16-byte aligned, with row strides that are "
                                 "multiples of 4");
    if (!(q_stride >= 0 && out_stride >= (int64_t)n_heads * pages->head_dim))
        return paged_refuse(who, "bad row strides");
    const int64_t row = (int64_t)n_heads * pages->head_dim;
    if (!((out == q && out_stride == q_stride) ||
          !paged_rows_overlap(out, out_stride, row, q, q_stride, row, batch->n_tokens)))
        return paged_refuse(who, "out may be q, with its row stride, and must not overlap it otherwise");
    RowsArgs a{};
    a.w = paged_view(pages, seqs, batch, n_heads, tree);
    if (tree) {
        a.mask = tree->mask;
        a.words = (tree->max_nodes + 31) / 32;
    }
    size_t need = 0;
    const int64_t max_pos = (int64_t)seqs->max_pages * pages->page_size;
    attention_paged_any(pages, batch, a, nullptr, &need, max_pos, nullptr);
    if (!(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need))
        return paged_refuse(who, "workspace missing, too small or not 256-byte aligned");
    const int64_t layer_bytes = (int64_t)pages->n_pages * pages->n_kv_heads * pages->page_size *
                                pages->head_dim * (pages->type == IB_TYPE_F32 ? 4 : 2);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.k = (const uint8_t*)pages->k + layer * layer_bytes;
    a.v = (const uint8_t*)pages->v + layer * layer_bytes;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.sectors = (((uintptr_t)out | (uintptr_t)(out_stride * 4)) & 31) == 0;
    return attention_paged_any(pages, batch, a, workspace, nullptr, max_pos, as_stream(stream));
}

extern "C" int ib_attention_paged(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                  const ib_kv_batch* batch, int layer, int n_heads, const float* q,
                                  int64_t q_stride, float* out, int64_t out_stride, float scale,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "ib_attention_paged";
    const int r = paged_check_batch(pages, seqs, batch, layer, n_heads, who);
    if (r != IB_OK) return r;
    return attention_call(pages, seqs, batch, nullptr, layer, n_heads, q, q_stride, out, out_stride, scale,
                          workspace, workspace_bytes, stream, who);
}

extern "C" int ib_attention_paged_tree(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                       const ib_kv_batch* batch, const ib_kv_tree* tree, int layer,
                                       int n_heads, const float* q, int64_t q_stride, float* out,
                                       int64_t out_stride, float scale, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    const char* who = "ib_attention_paged_tree";
    int r = paged_check_batch(pages, seqs, batch, layer, n_heads, who);
    if (r == IB_OK) r = paged_check_tree(batch, tree, who);
    if (r != IB_OK) return r;
    return attention_call(pages, seqs, batch, tree, layer, n_heads, q, q_stride, out, out_stride, scale,
                          workspace, workspace_bytes, stream, who);
}
