// ib_attention_paged: causal GQA attention of a batch of new tokens over the paged cache.
//
// The query rows of a sequence that share a kv head -- (token, head of the group), token by
// token -- are consecutive: row r is token r / G, head r % G.  A work item is a tile of such
// rows against a range of the sequence's positions; items whose range is not the whole leave
// a partial result (running maximum m, exponential sum l, unnormalised sum of p v), and a
// second kernel joins them:
//     out = sum_s 2^(m_s - M) acc_s / sum_s 2^(m_s - M) l_s.
// Lengths are device data, so every CTA works the split out for itself from cu_q and len (one
// pass over the batch; no planning launch), and grids are sized by the host's bounds.
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "common.cuh"
#include "mma_tile.cuh"
#include "paged.cuh"
#include "pdl.cuh"
#include "pipeline.cuh"

namespace ib {

int paged_attention_fault_take(int* code) { return paged_fault_take_here(code); }

// ---- the split of a batch into items -----------------------------------------------------
// Sequences with rows in [min_rows, max_rows] take part.  A sequence has ceil(rows / R) row
// tiles per kv head, each over ceil(L / KT) key tiles; the ranges are as long as it takes to
// have about `target` items, but at least `least` key tiles.
struct SplitRule {
    int R, KT, min_rows, max_rows, target, least;
};

// Item `item` of the batch.  n_parts: ranges of its row tile; part_base: index of the first
// of their partials (unused when n_parts == 1).
struct Item {
    int b, hk, tile, part, n_parts, part_base;
    int kt0, kt1;  // key tiles of the range
    SeqInfo s;
};

struct SeqSplit {
    int tiles, nkt, parts;  // row tiles per kv head, key tiles, ranges
};

__device__ __forceinline__ void seq_shape(const PagedView& w, const SplitRule& rule,
                                          const SeqInfo& s, int& tiles, int& nkt) {
    const int rows = s.n * (w.H / w.Hkv);
    const bool in = rows >= rule.min_rows && rows <= rule.max_rows;
    tiles = in ? (rows + rule.R - 1) / rule.R : 0;
    nkt = max(1, (s.L + rule.KT - 1) / rule.KT);  // a sequence without positions: zeros
}

// Every thread of the CTA (NT threads) calls it; false when there are fewer items.  BY_TILE
// counts row tiles instead of items (the joining kernel).
template <int NT, bool BY_TILE>
__device__ __forceinline__ bool find_item(const PagedView& w, const SplitRule& rule, int item,
                                          Item& out) {
    __shared__ long long sh_units[NT / 32];
    __shared__ int sh_scan[NT / 32][2];
    __shared__ Item sh_item;
    __shared__ int sh_found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    SeqInfo s0{};
    int tiles0 = 0, nkt0 = 1;
    long long units = 0;
    for (int b = tid; b < w.n_seqs; b += NT) {
        const SeqInfo s = seq_info(w, b);
        int tiles, nkt;
        seq_shape(w, rule, s, tiles, nkt);
        units += min((long long)tiles * nkt, 1ll << 40);
        if (b == tid) s0 = s, tiles0 = tiles, nkt0 = nkt;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
    if (lane == 0) sh_units[warp] = units;
    if (tid == 0) sh_found = 0;
    __syncthreads();
    units = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) units += sh_units[i];
    units = min(units, 1ll << 45) * w.Hkv;
    const int len = (int)min(max((long long)rule.least, (units + rule.target - 1) / rule.target),
                             0x3fffffffll);
    // cu_q can hold anything: counts are clamped to what cannot be, so that sums stay in range
    // (valid batches have at most 2^22 + n_seqs row tiles, see paged_check_batch)
    constexpr long long MOST = 1 << 23;
    const int room = 2 * rule.target;  // partials in the workspace
    long long items_before = 0;
    int parts_before = 0;
    for (int b0 = 0; b0 < w.n_seqs; b0 += NT) {
        const int b = b0 + tid;
        SeqInfo s = s0;
        int tiles = tiles0, nkt = nkt0;
        if (b0 > 0) {
            tiles = 0;
            if (b < w.n_seqs) {
                s = seq_info(w, b);
                seq_shape(w, rule, s, tiles, nkt);
            }
        }
        const int parts = (nkt + len - 1) / len;
        const long long n_tiles = b < w.n_seqs ? (long long)tiles * w.Hkv : 0;
        const int n_items = (int)min(BY_TILE ? n_tiles : n_tiles * parts, MOST);
        const int n_parts = parts > 1 ? (int)min(n_tiles * parts, (long long)room + 1) : 0;
        int a = n_items, p = n_parts;  // inclusive scans
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int xa = __shfl_up_sync(0xffffffffu, a, o), xp = __shfl_up_sync(0xffffffffu, p, o);
            if (lane >= o) a += xa, p += xp;
        }
        if (lane == 31) sh_scan[warp][0] = a, sh_scan[warp][1] = p;
        __syncthreads();
        int ta = 0, tp = 0;
#pragma unroll
        for (int i = 0; i < NT / 32; ++i) {
            if (i == warp) a += ta, p += tp;
            ta += sh_scan[i][0], tp += sh_scan[i][1];
        }
        const long long at = item - items_before - (a - n_items);
        if (at >= 0 && at < n_items) {
            const int local = (int)at;
            Item it;
            it.b = b;
            it.s = s;
            it.n_parts = parts;
            const int t = BY_TILE ? local : local / parts;
            it.part = BY_TILE ? 0 : local - t * parts;
            it.tile = t / w.Hkv;
            it.hk = t - it.tile * w.Hkv;
            it.part_base = parts_before + (p - n_parts) + t * parts;
            // ranges of equal length, to one key tile
            it.kt0 = (int)((long long)nkt * it.part / parts);
            it.kt1 = (int)((long long)nkt * (it.part + 1) / parts);
            sh_item = it;
            sh_found = parts == 1 || it.part_base + parts <= room ? 1 : 2;
        }
        __syncthreads();
        if (sh_found) break;
        items_before += ta;
        parts_before += tp;
    }
    __syncthreads();
    out = sh_item;
    if (sh_found == 2) paged_fault(PAGED_BAD_LEN);  // more partials than a valid batch has
    return sh_found == 1;
}

// ---- 16 rows on mma.sync -----------------------------------------------------------------
// A warp's 16 query rows against KW positions at a time.  Products of FP32 operands keep about
// 2^-21:
//   FP16 pages  q = hi + lo and p = hi + lo in FP16, K and V as they are: two m16n8k16 per
//               product.  q rows are scaled to a largest element in [256, 512) and p by 2^10,
//               powers of two that keep the lo parts out of FP16's subnormals.
//   FP32 pages  both operands as TF32 hi + lo, hi hi + hi lo + lo hi: three m16n8k8, with the
//               range of FP32.
// The MMA adds to its FP32 accumulator by cutting, half a unit of the accumulator per step on
// average and always towards zero: a running sum over a long sequence would drift (2.6e-6 of
// the result over 131072 positions).  So lo parts have accumulators of their own, and p v of
// each tile starts from zero and is added to the running sum by FFMA, which rounds and takes
// the rescaling with it.
// Positions that a row does not see get a score of -inf; pages that are not there are filled
// with zeros, and in tiles where some row does not see a position that has a page (`careful`),
// V is checked for values that are not finite (0 x inf).
struct RowsArgs {
    PagedView w;
    SplitRule rule;
    const float* q;
    float* out;
    int64_t q_stride, out_stride;
    const void *k, *v;  // the layer
    float* part_acc;    // [partial][R][HD]
    float2* part_ml;    // [partial][R]
    float scale_log2;   // scale * log2(e)
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(valid ? 16 : 0)
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two FP16 values with those that are not finite as zero; odd is set when there were any.
__device__ __forceinline__ uint32_t finite16x2(uint32_t x, bool& odd) {
    if ((x & 0x7c00u) == 0x7c00u) odd = true, x &= 0xffff0000u;
    if ((x & 0x7c000000u) == 0x7c000000u) odd = true, x &= 0x0000ffffu;
    return x;
}

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
        // 2^(8 - e) with e the exponent of the largest element, and its inverse
        const int e = max(-100, (int)((__float_as_uint(top) >> 23) & 255u) - 127);
        const bool plain = top == 0.f || e > 127;
        const float up = plain ? 1.f : __uint_as_float((uint32_t)(8 - e + 127) << 23);
        const float down = plain ? 1.f : __uint_as_float((uint32_t)(e - 8 + 127) << 23);
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

// QREG: the q fragments stay in registers.  LD: bytes between K or V rows in shared memory
// (16 more than a row: the 8 rows of an ldmatrix, and the TF32 V columns, hit distinct banks);
// QLD: the same for q.
template <typename KV, int HDP, int KW, bool QREG>
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
    uint32_t qh[QREG ? KS : 1][4], ql[QREG ? KS : 1][4];
    uint32_t q_hi, q_lo;  // this lane's fragment addresses

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
        if constexpr (QREG) {
#pragma unroll
            for (int k = 0; k < KS; ++k) load_q(k, qh[k], ql[k]);
        }
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
            float s2[NB <= 2 ? NB : 1][4];  // a second chain for the upper half of head_dim
            zero(s2);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t ah[4], al[4];
                if constexpr (QREG) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) ah[j] = qh[k][j], al[j] = ql[k][j];
                } else {
                    load_q(k, ah, al);
                }
#pragma unroll
                for (int n = 0; n < NB; n += 2) {  // 16 positions x 16 dimensions
                    uint32_t b[4];
                    ldsm_x4(kd + (uint32_t)((n * 8 + (lane & 7) + ((lane >> 4) << 3)) * LD + k * 32 +
                                            ((lane >> 3) & 1) * 16),
                            b[0], b[1], b[2], b[3]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if constexpr (NB <= 2) mma16816(k < KS / 2 ? s[n + j] : s2[n + j], ah, b[2 * j], b[2 * j + 1]);
                        else mma16816(s[n + j], ah, b[2 * j], b[2 * j + 1]);
                        mma16816(e[n + j], al, b[2 * j], b[2 * j + 1]);
                    }
                }
            }
            if constexpr (NB <= 2) {
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[n][j] += s2[n][j];
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
                    for (int j = 0; j < 4; ++j) split_tf32(__uint_as_float(b[j]), h[j], r[j]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mma1688_tf32(t[n], ah[j], h[2 * j], h[2 * j + 1]);
                        mma1688_tf32(e[n], ah[j], r[2 * j], r[2 * j + 1]);
                        mma1688_tf32(e[n], al[j], h[2 * j], h[2 * j + 1]);
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
                a = p0 <= lim[h] ? (a + e[n][2 * h]) * sc[h] : -INFINITY;
                b = p1 <= lim[h] ? (b + e[n][2 * h + 1]) * sc[h] : -INFINITY;
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
                        mma16816(t[j], pl[k], b[2 * j], b[2 * j + 1]);
                        mma16816(t[j], ph[k], b[2 * j], b[2 * j + 1]);
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
                split_tf32(s[k][0], ph[k][0], pl[k][0]);
                split_tf32(s[k][2], ph[k][1], pl[k][1]);
                split_tf32(s[k][1], ph[k][2], pl[k][2]);
                split_tf32(s[k][3], ph[k][3], pl[k][3]);
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
                    split_tf32(y0, h0, r0);
                    split_tf32(y1, h1, r1);
                    mma1688_tf32(t[0], ph[k], h0, h1);
                    mma1688_tf32(r[0], ph[k], r0, r1);
                    mma1688_tf32(r[0], pl[k], h0, h1);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) t[0][j] += r[0][j];
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
                        if (pos <= lim[0]) acc[d][i] = NAN;
                        if (pos <= lim[1]) acc[d][2 + i] = NAN;
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

__device__ __forceinline__ float* out_row(const RowsArgs& A, const Item& it, int G, int gr) {
    const int tok = gr / G;
    return A.out + (int64_t)(it.s.q0 + tok) * A.out_stride +
           (int64_t)(it.hk * G + gr - tok * G) * A.w.HD;
}

// ---- up to 16 rows: single tokens and short drafts ---------------------------------------
// The bound is reading K and V once.  A CTA holds the 16 rows; each of its warps runs through
// every NW-th group of KW positions by itself -- its own ring in shared memory, filled by its
// own cp.async, no barrier in the loop -- so that one warp's chain of loads, scores, maximum and
// products hides behind the others'; they join at the end.
template <typename KV, int HDP>
struct NarrowCfg {
    static constexpr bool F32 = sizeof(KV) == 4;
    static constexpr int KW = F32 ? 8 : 16;
    static constexpr bool QREG = !F32 && HDP <= 128;
    using Tile = WarpRows<KV, HDP, KW, QREG>;
    static constexpr int NW = HDP == 256 ? 4 : 8, NT = NW * 32;
    static constexpr int STAGES = F32 && HDP == 256 ? 2 : 3;
    static constexpr int STAGE = 2 * KW * Tile::LD;
    static constexpr int Q_BYTES = 2 * 16 * Tile::QLD;
    static constexpr int RING = NW * STAGES * STAGE;
    static constexpr int MERGE = NW * 16 * (HDP + 4) * 4;  // of the warps' results, in the ring
    static constexpr size_t SMEM = Q_BYTES + (RING > MERGE ? RING : MERGE);
    // CTAs that an SM holds
    static constexpr int CTAS = HDP == 64 ? 2 : 1;
};

template <typename KV, int HDP>
__global__ void __launch_bounds__(NarrowCfg<KV, HDP>::NT, NarrowCfg<KV, HDP>::CTAS)
    attn_narrow_kernel(const __grid_constant__ RowsArgs A) {
    using C = NarrowCfg<KV, HDP>;
    using T = typename C::Tile;
    constexpr int KW = C::KW, LD = T::LD, S = C::STAGES, NW = C::NW;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float row_scale[16], sh_m[NW][16], sh_l[NW][16];
    const PagedView& w = A.w;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2;
    pdl_wait();
    pdl_launch_dependents();
    Item it;
    if (!find_item<C::NT, false>(w, A.rule, blockIdx.x, it)) return;
    const int G = w.H / w.Hkv, HD = w.HD, row0 = it.tile * 16;
    const int rows = min(16, it.s.n * G - row0);
    const int start = it.s.L - it.s.n;  // position of the first new token
    const int first_lim = start + row0 / G, last_lim = start + (row0 + rows - 1) / G;
    const int kt0 = it.kt0 + warp, kt1 = min(it.kt1, last_lim < 0 ? 0 : last_lim / KW + 1);
    uint8_t* ring = smem + C::Q_BYTES + warp * S * C::STAGE;
    const uint32_t ring_a = smem_u32(ring);

    // Lane j holds position j of a tile (j < KW, twice or four times over): where its row starts
    // in the layer (-1: nowhere) and the position itself (INT_MAX: none).
    auto entry_of = [&](int kt) -> int {  // read a tile ahead of the copies that need it
        const int pos = kt * KW + (lane & (KW - 1));
        if (kt >= kt1 || pos > last_lim) return -1;
        return page_at(w, it.s.row[w.ps.div((uint32_t)pos)]);
    };
    const int cpr = HD * (int)sizeof(KV) / 16;  // 16-byte chunks of a row that exist
    constexpr int CH = HDP * (int)sizeof(KV) / 16;  // and with padding
    auto issue = [&](int kt, int slot, int page) -> int {
        const int pos = kt * KW + (lane & (KW - 1));
        if (kt < kt1) {
            const int in_page = pos - (int)w.ps.div((uint32_t)pos) * w.page_size;
            const long long off =
                page < 0 ? -1 : (((long long)page * w.Hkv + it.hk) * w.page_size + in_page) * HD;
            const uint32_t d0 = ring_a + (uint32_t)(slot * C::STAGE);
#pragma unroll
            for (int c = lane; c < KW * CH; c += 32) {
                const int r = c / CH, x = c % CH;  // CH: 8 or more, so r is within the lanes
                const long long o = __shfl_sync(0xffffffffu, off, r);
                const bool ok = o >= 0 && x < cpr;
                const size_t byte = ok ? (size_t)o * sizeof(KV) + (size_t)x * 16 : 0;
                const uint32_t d = d0 + (uint32_t)(r * LD + x * 16);
                cp16(d, (const uint8_t*)A.k + byte, ok);
                cp16(d + KW * LD, (const uint8_t*)A.v + byte, ok);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return page < 0 ? 0x7fffffff : pos;
    };
    int pos[S];  // of the tiles in flight, the oldest first
    {
        int page[S - 1];
#pragma unroll
        for (int i = 0; i < S - 1; ++i) page[i] = entry_of(kt0 + i * NW);
#pragma unroll
        for (int i = 0; i < S - 1; ++i) pos[i] = issue(kt0 + i * NW, i, page[i]);
    }
    int next_page = entry_of(kt0 + (S - 1) * NW);

    for (int r = warp; r < 16; r += NW) {
        const int gr = row0 + r, tok = gr / G;
        const float* src = r < rows ? A.q + (int64_t)(it.s.q0 + tok) * A.q_stride +
                                          (int64_t)(it.hk * G + gr - tok * G) * HD
                                    : nullptr;
        uint8_t* hi = smem + r * T::QLD;
        const float f = stage_q_row<C::F32, HDP>(src, HD, hi, hi + 16 * T::QLD, A.scale_log2);
        if (lane == 0) row_scale[r] = f;
    }
    __syncthreads();
    T t;
    t.start(smem_u32(smem), smem_u32(smem) + 16 * T::QLD);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        t.lim[h] = r < rows ? start + (row0 + r) / G : -1;
        t.sc[h] = row_scale[r];
    }
    int slot = 0;
    for (int kt = kt0; kt < kt1; kt += NW) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        __syncwarp();  // every lane's copies of this tile, and its reads of the one before
        const int fill = slot == 0 ? S - 1 : slot - 1;  // the slot before: the tile of last time
        pos[S - 1] = issue(kt + (S - 1) * NW, fill, next_page);
        next_page = entry_of(kt + S * NW);
        const uint32_t kd = ring_a + (uint32_t)(slot * C::STAGE);
        const int mine = pos[0];
        t.step(kd, kd + KW * LD, ring + slot * C::STAGE + KW * LD, kt * KW + KW - 1 > first_lim,
               [&](int j) { return __shfl_sync(0xffffffffu, mine, j); });
#pragma unroll
        for (int i = 0; i < S - 1; ++i) pos[i] = pos[i + 1];
        slot = slot == S - 1 ? 0 : slot + 1;
    }
    t.finish();

    // ---- the warps' results together, in the ring ----
    constexpr int MLD = HDP + 4;
    float* ma = reinterpret_cast<float*>(smem + C::Q_BYTES);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int d = 0; d < T::DB; ++d) {
        float* p = ma + (warp * 16 + g) * MLD + d * 8 + 2 * (lane & 3);
        *reinterpret_cast<float2*>(p) = make_float2(t.acc[d][0], t.acc[d][1]);
        *reinterpret_cast<float2*>(p + 8 * MLD) = make_float2(t.acc[d][2], t.acc[d][3]);
    }
    if ((lane & 3) == 0) {
        sh_m[warp][g] = t.m[0], sh_m[warp][g + 8] = t.m[1];
        sh_l[warp][g] = t.l[0], sh_l[warp][g + 8] = t.l[1];
    }
    __syncthreads();
    const int64_t pidx = (int64_t)it.part_base + it.part;
    const int v4 = HD / 4;
    for (int e = tid; e < rows * v4; e += C::NT) {
        const int r = e / v4, x = (e - r * v4) * 4;
        float M = sh_m[0][r], l = 0.f;
#pragma unroll
        for (int i = 1; i < NW; ++i) M = fmaxf(M, sh_m[i][r]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const float c = M == -INFINITY ? 1.f : ex2(sh_m[i][r] - M);
            const float4 y = *reinterpret_cast<const float4*>(ma + (i * 16 + r) * MLD + x);
            l += c * sh_l[i][r];
            o.x += c * y.x, o.y += c * y.y, o.z += c * y.z, o.w += c * y.w;
        }
        if (it.n_parts == 1) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            *reinterpret_cast<float4*>(out_row(A, it, G, row0 + r) + x) =
                make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        } else {
            *reinterpret_cast<float4*>(A.part_acc + (pidx * 16 + r) * HD + x) = o;
            if (x == 0) A.part_ml[pidx * 16 + r] = make_float2(M, l);
        }
    }
}

// ---- more rows on mma.sync ---------------------------------------------------------------
// WR warps of 16 rows each over the same key tiles, which the CTA brings in together.
template <typename KV, int HDP>
struct WideCfg {
    static constexpr bool F32 = sizeof(KV) == 4;
    static constexpr int WR = HDP == 256 ? 4 : 8, NT = WR * 32, R = 16 * WR;
    static constexpr int ROWB = HDP * (int)sizeof(KV);
    static constexpr int KT = ROWB <= 128 ? 64 : ROWB <= 512 ? 32 : 16;
    static constexpr bool QREG = !F32 && HDP <= 128;
    using Tile = WarpRows<KV, HDP, KT, QREG>;
    static constexpr int STAGES = ROWB > 256 ? 2 : 4;
    static constexpr int Q_BYTES = 2 * R * Tile::QLD;
    static constexpr int STAGE = 2 * KT * Tile::LD;
    static constexpr int RING = STAGES + 1;  // of row offsets: a tile's outlive its copies
    static constexpr size_t SMEM = (size_t)Q_BYTES + STAGES * STAGE;
};

template <typename KV, int HDP>
__global__ void __launch_bounds__(WideCfg<KV, HDP>::NT)
    attn_wide_kernel(const __grid_constant__ RowsArgs A) {
    using C = WideCfg<KV, HDP>;
    using T = typename C::Tile;
    constexpr int NT = C::NT, R = C::R, KT = C::KT, LD = T::LD, S = C::STAGES;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ long long row_off[C::RING][KT];  // where a position's row starts, -1: nowhere
    __shared__ int key_pos[C::RING][KT];        // its position, INT_MAX: none
    __shared__ float row_scale[R];
    const PagedView& w = A.w;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2;
    pdl_wait();
    pdl_launch_dependents();
    Item it;
    if (!find_item<NT, false>(w, A.rule, blockIdx.x, it)) return;
    const int G = w.H / w.Hkv, HD = w.HD, row0 = it.tile * R;
    const int rows = min(R, it.s.n * G - row0);
    const int start = it.s.L - it.s.n;
    const int first_lim = start + row0 / G, last_lim = start + (row0 + rows - 1) / G;
    const int kt0 = it.kt0, kt1 = min(it.kt1, last_lim < 0 ? 0 : last_lim / KT + 1);
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
        const int gr = row0 + r, tok = gr / G;
        const float* src = r < rows ? A.q + (int64_t)(it.s.q0 + tok) * A.q_stride +
                                          (int64_t)(it.hk * G + gr - tok * G) * HD
                                    : nullptr;
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
    const int64_t pidx = (int64_t)it.part_base + it.part;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = warp * 16 + g + 8 * h;
        if (r >= rows) continue;
        const bool whole = it.n_parts == 1;
        const float inv = !whole ? 1.f : t.l[h] == 0.f ? 0.f : 1.f / t.l[h];
        float* p = whole ? out_row(A, it, G, row0 + r) : A.part_acc + (pidx * R + r) * HD;
#pragma unroll
        for (int d = 0; d < T::DB; ++d)
            if (d * 8 < HD)
                *reinterpret_cast<float2*>(p + d * 8 + 2 * (lane & 3)) =
                    make_float2(t.acc[d][2 * h] * inv, t.acc[d][2 * h + 1] * inv);
        if (!whole && (lane & 3) == 0) A.part_ml[pidx * R + r] = make_float2(t.m[h], t.l[h]);
    }
}

// ---- joining the ranges of a row tile ----------------------------------------------------
// One CTA per (row tile, row): its four warps take every fourth range each.
struct JoinArgs {
    PagedView w;
    SplitRule rule;
    float* out;
    int64_t out_stride;
    const float* part_acc;
    const float2* part_ml;
};

__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ JoinArgs A) {
    constexpr int NT = 128, MAXV = 2;  // float4 per lane: head_dim 256
    __shared__ float4 sh_acc[4][32 * MAXV];
    __shared__ float sh_l[4];
    const PagedView& w = A.w;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Item it;
    // cu_q and len were complete before the attention kernel started; its partials follow
    const bool any = find_item<NT, true>(w, A.rule, blockIdx.x, it);
    pdl_wait();
    if (!any || it.n_parts == 1) return;
    const int G = w.H / w.Hkv, HD = w.HD, R = A.rule.R, r = blockIdx.y;
    if (r >= it.s.n * G - it.tile * R) return;
    float M = -INFINITY, l = 0.f;
    float4 o[MAXV];
#pragma unroll
    for (int i = 0; i < MAXV; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float2* ml = A.part_ml + (int64_t)it.part_base * R + r;
    for (int p = lane; p < it.n_parts; p += 32) M = fmaxf(M, ml[(int64_t)p * R].x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
#pragma unroll 4
    for (int p = warp; p < it.n_parts; p += 4) {
        const float2 y = ml[(int64_t)p * R];
        const float c = M == -INFINITY ? 1.f : ex2(y.x - M);
        l += c * y.y;
        const float4* a =
            reinterpret_cast<const float4*>(A.part_acc + ((int64_t)(it.part_base + p) * R + r) * HD);
#pragma unroll
        for (int i = 0; i < MAXV; ++i)
            if (lane + 32 * i < HD / 4) {
                const float4 x = a[lane + 32 * i];
                o[i].x += c * x.x, o[i].y += c * x.y, o[i].z += c * x.z, o[i].w += c * x.w;
            }
    }
#pragma unroll
    for (int i = 0; i < MAXV; ++i) sh_acc[warp][lane + 32 * i] = o[i];
    if (lane == 0) sh_l[warp] = l;
    __syncthreads();
    l = sh_l[0] + sh_l[1] + sh_l[2] + sh_l[3];
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int gr = it.tile * R + r, tok = gr / G;
    float* out = A.out + (int64_t)(it.s.q0 + tok) * A.out_stride +
                 (int64_t)(it.hk * G + gr - tok * G) * HD;
    for (int x = threadIdx.x; x < HD / 4; x += NT) {
        float4 y = sh_acc[0][x];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            const float4 z = sh_acc[i][x];
            y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
        }
        reinterpret_cast<float4*>(out)[x] = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
    }
}

// ---- launches ----------------------------------------------------------------------------
constexpr int kSMs = 148;  // of a B200: the items aimed at, and so the workspace, follow it

// One kernel's share of a call.
struct Share {
    SplitRule rule;
    int64_t tiles;  // most row tiles, over all kv heads
    size_t acc_off, ml_off;
};

struct Plan {
    int n = 0;
    Share share[2];
    size_t bytes = 0;
};

// Rules of the two: about two rounds of CTAs, so that uneven ranges even out, and at least 128
// positions a range, below which joining costs more.
template <typename KV, int HDP>
static SplitRule narrow_rule(int min_rows, int max_rows) {
    using C = NarrowCfg<KV, HDP>;
    return SplitRule{16, C::KW, min_rows, max_rows, kSMs * C::CTAS * 2, 128 / C::KW};
}
template <typename KV, int HDP>
static SplitRule wide_rule(int min_rows, int max_rows) {
    using C = WideCfg<KV, HDP>;
    return SplitRule{C::R, C::KT, min_rows, max_rows, kSMs * 2, 128 / C::KT};
}

template <typename Kern>
static int rows_launch(Kern kern, int threads, size_t smem, const RowsArgs& a, int64_t tiles,
                       cudaStream_t st) {
    IB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    const int64_t grid = tiles + a.rule.target;
    IB_CUDA_CHECK(launch_pdl(kern, dim3((unsigned)grid), dim3(threads), smem, st, true, a));
    return IB_OK;
}

// The kernels of a call, by the rows (new tokens x group) that a sequence may have: up to 16
// on the narrow kernel, more on the wide one.  With one sequence, or a bound that rules the
// wide one out, a single kernel takes everything.
template <typename KV, int HDP>
static Plan make_plan(const ib_kv_pages* p, const ib_kv_batch* b, int n_heads) {
    constexpr int ALL = 0x7fffffff;
    constexpr int WIDE = WideCfg<KV, HDP>::R;
    const int64_t G = n_heads / p->n_kv_heads;
    const int64_t most_q = b->max_q > 0 ? std::min(b->max_q, b->n_tokens) : b->n_tokens;
    const int64_t seqs = std::min(b->n_seqs, b->n_tokens);
    Plan plan;
    auto add = [&](const SplitRule& r, int64_t tiles_per_head) {
        Share& s = plan.share[plan.n++];
        s.rule = r;
        s.tiles = tiles_per_head * p->n_kv_heads;
        auto take = [&](size_t n) {
            const size_t at = plan.bytes;
            plan.bytes += (n + 255) / 256 * 256;
            return at;
        };
        // at most 2 x target partials: a tile of k > len key tiles has ceil(k / len) <= 2 k / len
        s.acc_off = take((size_t)2 * r.target * r.R * p->head_dim * sizeof(float));
        s.ml_off = take((size_t)2 * r.target * r.R * sizeof(float2));
    };
    const int64_t rows = b->n_tokens * G;
    if (most_q * G <= 16) {
        add(narrow_rule<KV, HDP>(1, ALL), seqs + rows / 16);
    } else {
        if (b->n_seqs > 1) add(narrow_rule<KV, HDP>(1, 16), seqs);
        add(wide_rule<KV, HDP>(b->n_seqs > 1 ? 17 : 1, ALL), seqs + rows / WIDE);
    }
    return plan;
}

template <typename KV, int HDP>
static int run_plan(const ib_kv_pages* p, const ib_kv_batch* b, const Plan& plan, RowsArgs a,
                    uint8_t* ws, int64_t max_pos, cudaStream_t st) {
    using N = NarrowCfg<KV, HDP>;
    using W = WideCfg<KV, HDP>;
    for (int i = 0; i < plan.n; ++i) {
        const Share& s = plan.share[i];
        a.rule = s.rule;
        a.part_acc = reinterpret_cast<float*>(ws + s.acc_off);
        a.part_ml = reinterpret_cast<float2*>(ws + s.ml_off);
        const int r =
            s.rule.R == 16
                ? rows_launch(attn_narrow_kernel<KV, HDP>, N::NT, N::SMEM, a, s.tiles, st)
                : rows_launch(attn_wide_kernel<KV, HDP>, W::NT, W::SMEM, a, s.tiles, st);
        if (r != IB_OK) return r;
        // no range is cut where the longest row of a table is no longer than the least
        if (max_pos > (int64_t)s.rule.least * s.rule.KT) {
            const JoinArgs j{a.w, s.rule, a.out, a.out_stride, a.part_acc, a.part_ml};
            const int64_t G = a.w.H / a.w.Hkv;
            const int64_t most_rows = std::min<int64_t>(s.rule.R, b->n_tokens * G);
            IB_CUDA_CHECK(launch_pdl(attn_join_kernel, dim3((unsigned)s.tiles, (unsigned)most_rows),
                                     dim3(128), 0, st, true, j));
        }
    }
    return IB_OK;
}

template <typename KV>
static int attention_paged(const ib_kv_pages* p, const ib_kv_batch* b, RowsArgs a, void* ws,
                           size_t* bytes, int64_t max_pos, cudaStream_t st) {
    auto go = [&](auto hdp) {
        constexpr int HDP = decltype(hdp)::value;
        const Plan plan = make_plan<KV, HDP>(p, b, a.w.H);
        if (bytes) {
            *bytes = plan.bytes;
            return (int)IB_OK;
        }
        return run_plan<KV, HDP>(p, b, plan, a, (uint8_t*)ws, max_pos, st);
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

extern "C" size_t ib_attention_paged_workspace(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                               const ib_kv_batch* batch, int n_heads) {
    if (paged_check_batch(pages, seqs, batch, 0, n_heads, "ib_attention_paged_workspace") != IB_OK)
        return 0;
    if (batch->n_tokens == 0 || batch->n_seqs == 0) return 256;
    RowsArgs a{};
    a.w = paged_view(pages, seqs, batch, n_heads);
    size_t n = 0;
    attention_paged_any(pages, batch, a, nullptr, &n, 0, nullptr);
    return n;
}

extern "C" int ib_attention_paged(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                  const ib_kv_batch* batch, int layer, int n_heads, const float* q,
                                  int64_t q_stride, float* out, int64_t out_stride, float scale,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    int r = paged_check_batch(pages, seqs, batch, layer, n_heads, "ib_attention_paged");
    if (r != IB_OK || batch->n_tokens == 0 || batch->n_seqs == 0) return r;
    IB_REQUIRE(q && out, "ib_attention_paged: null pointer argument");
    IB_REQUIRE((((uintptr_t)q | (uintptr_t)out) & 15) == 0 && ((q_stride | out_stride) & 3) == 0,
               "ib_attention_paged: q and out must be 16-byte aligned, with row strides that are "
               "multiples of 4");
    IB_REQUIRE(q_stride >= 0 && out_stride >= (int64_t)n_heads * pages->head_dim,
               "ib_attention_paged: bad row strides");
    RowsArgs a{};
    a.w = paged_view(pages, seqs, batch, n_heads);
    size_t need = 0;
    attention_paged_any(pages, batch, a, nullptr, &need, 0, nullptr);
    IB_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0 && workspace_bytes >= need,
               "ib_attention_paged: workspace missing, too small or not 256-byte aligned");
    const int64_t layer_bytes = (int64_t)pages->n_pages * pages->n_kv_heads * pages->page_size *
                                pages->head_dim * (pages->type == IB_TYPE_F32 ? 4 : 2);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.k = (const uint8_t*)pages->k + layer * layer_bytes;
    a.v = (const uint8_t*)pages->v + layer * layer_bytes;
    a.scale_log2 = scale * 1.4426950408889634f;
    return attention_paged_any(pages, batch, a, workspace, nullptr,
                               (int64_t)seqs->max_pages * pages->page_size, as_stream(stream));
}
