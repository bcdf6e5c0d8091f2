// ib_beam_select: the k best continuations of each group of beams.
//
// Row r (a beam) offers every token t with v(r, t) = score(r) + x(r, t) - log sum_t' e^x(r, t'); the
// k largest of a group's rows win, equal ones in the order of (row, token).  The reference takes the
// first maximum of one row (src/ops/ops.cpp:424-438, ib_argmax).
//
// One pass over the logits: a CTA takes a slice of a row, keeps a running maximum and sum of
// exponentials, and the slice's k best, found through a threshold: once k values are known to lie at or
// above it, all others need is one comparison.  Inside a row the order of v is that of x, so a slice's
// candidates are chosen by x alone.  A second kernel, a CTA per group, makes the rows' log sums of the
// slices' and picks the group's k best in 64 bits: candidates of different beams may be closer than FP32
// tells apart.
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <string>

#include "common.cuh"
#include "paged.cuh"
#include "pdl.cuh"

namespace ib {

constexpr int BS_THREADS = 256, BS_WARPS = BS_THREADS / 32;
constexpr int BS_TILE = 16 * BS_THREADS;  // values of a CTA's step
constexpr int BS_CAP = 2048;              // candidates of a slice in shared memory

// A value and its place as one number: larger values first, then lower places.  0: none (-inf, NaN).
// -0 and 0 are equal.
__device__ __forceinline__ uint64_t beam_key(float x, uint32_t at) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.f);
    const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
    return ((uint64_t)o << 32) | (0xffffffffu - at);
}
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint32_t key_place(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

__device__ __forceinline__ uint64_t shfl_max(uint64_t x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t y = __shfl_xor_sync(0xffffffffu, x, o);
        x = y > x ? y : x;
    }
    return x;
}

// Sum over the CTA; `turn` alternates, so that one barrier does.
__device__ __forceinline__ int block_sum(int c, int (&sh)[2][BS_WARPS], int turn) {
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0) sh[turn & 1][threadIdx.x >> 5] = c;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int i = 0; i < BS_WARPS; ++i) s += sh[turn & 1][i];
    return s;
}

// The largest key, or one less, such that at least k of the CTA's keys (N a thread, zeros are none) are at
// or above it, and at most `most` where that can be had by halving; 1 where there are fewer than k.
template <int N>
__device__ __forceinline__ uint64_t threshold(const uint64_t (&key)[N], int k, int most, int (&sh)[2][BS_WARPS],
                                              int& turn) {
    uint64_t lo = 1, hi = ~0ull;  // at least k at lo, fewer at hi
    auto count = [&](uint64_t t) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += key[i] >= t;
        return block_sum(c, sh, turn++);
    };
    int at_lo = count(1);
    if (at_lo < k) return 1;
    while (at_lo > most && hi - lo > 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        const int c = count(mid);
        if (c >= k) lo = mid, at_lo = c;
        else hi = mid;
    }
    return lo;
}

struct SliceMeta {
    float m;
    float pad;
    double sum;  // of e^(x - m)
};

struct SelectArgs {
    const void* logits;
    int64_t stride;
    const float* scores;     // null: zeros
    const int32_t* ended;    // null: none
    int rows, beams, vocab, k, slices, end_token;
    int64_t per_slice;       // values, a multiple of BS_TILE
    uint64_t* list;          // [row][slice][k] keys, largest first, zeros behind
    SliceMeta* meta;         // [row][slice]
    float* out_score;        // [group][k]
    int32_t *out_token, *out_row;
};

template <typename T>
__device__ __forceinline__ float logit(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return __half2float(x);
}

// The n <= BS_CAP keys in buf: the k largest, in order, to the front (zeros behind the last).
__device__ __forceinline__ void keep_best(uint64_t* buf, int n, int k, int (&sh)[2][BS_WARPS], int& turn,
                                          int* count) {
    constexpr int N = BS_CAP / BS_THREADS;
    const int tid = threadIdx.x;
    __syncthreads();
    uint64_t key[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = i * BS_THREADS + tid;
        key[i] = at < n ? buf[at] : 0;
    }
    // keys are all different, so exactly k can be had
    const uint64_t t = threshold(key, k, k, sh, turn);
    if (tid == 0) *count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (key[i] >= t) buf[atomicAdd(count, 1)] = key[i];
    __syncthreads();
    const int c = min(*count, k);
    uint64_t mine = 0;
    int rank = 0;
    if (tid < c) {
        mine = buf[tid];
        for (int j = 0; j < c; ++j) rank += buf[j] > mine;
    }
    __syncthreads();
    if (tid < c) buf[rank] = mine;
    for (int j = c + tid; j < k; j += BS_THREADS) buf[j] = 0;
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(BS_THREADS) beam_slice_kernel(const __grid_constant__ SelectArgs A) {
    __shared__ uint64_t buf[BS_CAP];
    __shared__ int sh[2][BS_WARPS];
    __shared__ int n_buf, n_kept;
    __shared__ double sh_sum[BS_WARPS];
    __shared__ float sh_m[BS_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / A.slices, slice = blockIdx.x - row * A.slices;
    pdl_wait();
    pdl_launch_dependents();
    if (A.ended && A.ended[row]) return;
    const T* const x = static_cast<const T*>(A.logits) + (int64_t)row * A.stride;
    const int64_t begin = slice * A.per_slice, end = min((int64_t)A.vocab, begin + A.per_slice);
    int turn = 0;
    if (tid == 0) n_buf = 0;
    float m = -INFINITY, sum = 0.f;
    uint64_t floor_key = 1;  // nothing below it is looked at
    const int k = A.k;
    for (int64_t at = begin; at < end; at += BS_TILE) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int64_t p = at + i * BS_THREADS + tid;
            v[i] = p < end ? logit(x[p]) : -INFINITY;
        }
        float top = v[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, v[i]);
        if (top > m) {
            sum *= expf(m - top);
            m = top;
        }
        if (m > -INFINITY || top != top) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += expf(v[i] - m);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += v[i] != v[i] ? NAN : 0.f;
        }
        uint64_t key[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) key[i] = beam_key(v[i], (uint32_t)(at + i * BS_THREADS + tid));
        // a value for each thread that may take part, the same way in every step
        int c = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) c += key[i] >= floor_key;
        int more = block_sum(c, sh, turn++);
        if (n_buf + more > BS_CAP) {
            // raise the floor: of what is here first, then of everything
            const uint64_t t = threshold(key, k, k, sh, turn);
            floor_key = t > floor_key ? t : floor_key;
            keep_best(buf, n_buf, k, sh, turn, &n_kept);
            if (tid == 0) n_buf = n_kept < k ? n_kept : k;
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (key[i] >= floor_key) buf[atomicAdd(&n_buf, 1)] = key[i];
        __syncthreads();
        if (at == begin && at + BS_TILE < end) {
            keep_best(buf, n_buf, k, sh, turn, &n_kept);
            if (tid == 0) n_buf = n_kept < k ? n_kept : k;
            __syncthreads();
            if (n_buf == k) floor_key = buf[k - 1];
        }
    }
    keep_best(buf, n_buf, k, sh, turn, &n_kept);
    const int64_t out = (int64_t)row * A.slices + slice;
    for (int j = tid; j < k; j += BS_THREADS) A.list[out * k + j] = buf[j];
    // the slice's maximum and sum
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0) sh_m[warp] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BS_WARPS; ++i) M = fmaxf(M, sh_m[i]);
    double d = m > -INFINITY ? (double)sum * exp((double)m - (double)M) : (double)sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) sh_sum[warp] = d;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < BS_WARPS; ++i) d += sh_sum[i];
        A.meta[out] = SliceMeta{M, 0.f, d};
    }
}

struct Best {
    double v;
    uint64_t place;  // row in the group, token
};
__device__ __forceinline__ bool better(const Best& a, const Best& b) {
    return a.v > b.v || (a.v == b.v && a.place < b.place);
}

// One CTA per group.  Each thread has some of the group's lists (a row's slice each) and offers the best
// of their heads; k rounds of a maximum over the CTA.
__global__ void __launch_bounds__(BS_THREADS) beam_group_kernel(const __grid_constant__ SelectArgs A) {
    extern __shared__ double base[];  // [beams] score - log sum of e^(x - M)
    double* const row_m = base + A.beams;                      // [beams] M
    int* const head = reinterpret_cast<int*>(row_m + A.beams);  // [beams * slices]
    __shared__ Best sh_best[2][BS_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = blockIdx.x, row0 = g * A.beams, lists = A.beams * A.slices, k = A.k;
    pdl_wait();
    for (int b = warp; b < A.beams; b += BS_WARPS) {
        const int row = row0 + b;
        const bool end = A.ended && A.ended[row];
        double log_sum = 0;
        float M = 0.f;
        if (!end) {
            const SliceMeta* const meta = A.meta + (int64_t)row * A.slices;
            double s = 0;
            M = -INFINITY;
            for (int i = lane; i < A.slices; i += 32) M = fmaxf(M, meta[i].m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
            for (int i = lane; i < A.slices; i += 32) {
                const SliceMeta y = meta[i];
                s += y.m > -INFINITY ? y.sum * exp((double)y.m - (double)M) : y.sum;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            log_sum = log(s);  // (a row of nothing but -inf has no candidates)
        }
        if (lane == 0) {
            base[b] = (A.scores ? (double)A.scores[row] : 0.0) - log_sum;
            row_m[b] = M;
        }
    }
    for (int l = tid; l < lists; l += BS_THREADS) head[l] = 0;
    __syncthreads();
    const Best none = {-INFINITY, ~0ull};
    for (int j = 0; j < k; ++j) {
        Best best = none;
        int from = -1;
        for (int l = tid; l < lists; l += BS_THREADS) {
            const int b = l / A.slices;
            Best y = none;
            if (A.ended && A.ended[row0 + b]) {
                if (head[l] == 0 && l == b * A.slices) y = Best{base[b], ((uint64_t)b << 32) | (uint32_t)A.end_token};
            } else if (head[l] < k) {
                const uint64_t key = A.list[((int64_t)row0 * A.slices + l) * k + head[l]];
                if (key) y = Best{base[b] + ((double)key_value(key) - row_m[b]), ((uint64_t)b << 32) | key_place(key)};
            }
            if (y.v > -INFINITY && better(y, best)) best = y, from = l;  // NaN: not a number is no candidate
        }
        Best top = best;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Best y;
            y.v = __shfl_xor_sync(0xffffffffu, top.v, o);
            y.place = __shfl_xor_sync(0xffffffffu, top.place, o);
            if (better(y, top)) top = y;
        }
        if (lane == 0) sh_best[j & 1][warp] = top;
        __syncthreads();
        top = sh_best[j & 1][0];
#pragma unroll
        for (int i = 1; i < BS_WARPS; ++i)
            if (better(sh_best[j & 1][i], top)) top = sh_best[j & 1][i];
        const bool any = top.v > -INFINITY;
        if (any && from >= 0 && best.place == top.place) ++head[from];
        if (tid == 0) {
            const int64_t at = (int64_t)g * k + j;
            A.out_score[at] = any ? (float)top.v : -INFINITY;
            A.out_token[at] = any ? (int32_t)(uint32_t)top.place : -1;
            A.out_row[at] = any ? row0 + (int32_t)(top.place >> 32) : -1;
        }
    }
}

// How a call is cut.
struct SelectPlan {
    int slices;
    int64_t per_slice;
    size_t list_off, meta_off, bytes;
};

static SelectPlan select_plan(int64_t rows, int64_t vocab, int k) {
    SelectPlan p;
    const int64_t tiles = (vocab + BS_TILE - 1) / BS_TILE;
    const int64_t want = std::max<int64_t>(1, 148 * 4 / rows);  // CTAs for each row
    const int64_t per = std::max<int64_t>(1, (tiles + want - 1) / want);
    p.per_slice = per * BS_TILE;
    p.slices = (int)((tiles + per - 1) / per);
    p.list_off = 0;
    p.meta_off = ((size_t)rows * p.slices * k * 8 + 255) / 256 * 256;
    p.bytes = p.meta_off + ((size_t)rows * p.slices * sizeof(SliceMeta) + 255) / 256 * 256;
    return p;
}

static int select_check(int type, int64_t n_groups, int beams, int vocab, int k, const char* who) {
    if (type != IB_TYPE_F32 && type != IB_TYPE_F16) {
        set_error(std::string(who) + ": the logits must be F32 or F16, not " + type_name(type));
        return IB_ERR_UNSUPPORTED;
    }
    if (n_groups < 0 || beams < 1 || beams > IB_BEAM_MAX_BEAMS || n_groups * beams > (1 << 20))
        return paged_refuse(who, "n_groups or beams out of range");
    if (vocab < 1 || vocab > (1 << 28)) return paged_refuse(who, "vocab out of range");
    if (k < 1 || k > IB_BEAM_MAX_K) return paged_refuse(who, "k must be in [1, 128]");
    return IB_OK;
}

}  // namespace ib

using namespace ib;

extern "C" size_t ib_beam_select_workspace(int n_groups, int beams, int vocab, int k) {
    if (select_check(IB_TYPE_F32, n_groups, beams, vocab, k, "ib_beam_select_workspace") != IB_OK) return 0;
    if (n_groups == 0) return 256;
    return select_plan((int64_t)n_groups * beams, vocab, k).bytes;
}

extern "C" int ib_beam_select(int type, const void* logits, int64_t stride, const float* scores,
                              const int32_t* ended, int end_token, int n_groups, int beams, int vocab,
                              int k, float* out_score, int32_t* out_token, int32_t* out_row,
                              void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "ib_beam_select";
    const int r = select_check(type, n_groups, beams, vocab, k, who);
    if (r != IB_OK || n_groups == 0) return r;
    if (!logits || !out_score || !out_token || !out_row) return paged_refuse(who, "null pointer argument");
    if (stride < vocab && (int64_t)n_groups * beams > 1) return paged_refuse(who, "bad row stride");
    if ((uintptr_t)logits & (type == IB_TYPE_F32 ? 3 : 1)) return paged_refuse(who, "logits not aligned");
    const int64_t rows = (int64_t)n_groups * beams;
    const SelectPlan p = select_plan(rows, vocab, k);
    if (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < p.bytes)
        return paged_refuse(who, "workspace missing, too small or not 256-byte aligned");
    SelectArgs a{};
    a.logits = logits;
    a.stride = stride;
    a.scores = scores;
    a.ended = ended;
    a.rows = (int)rows;
    a.beams = beams;
    a.vocab = vocab;
    a.k = k;
    a.slices = p.slices;
    a.end_token = end_token;
    a.per_slice = p.per_slice;
    a.list = reinterpret_cast<uint64_t*>((uint8_t*)workspace + p.list_off);
    a.meta = reinterpret_cast<SliceMeta*>((uint8_t*)workspace + p.meta_off);
    a.out_score = out_score;
    a.out_token = out_token;
    a.out_row = out_row;
    cudaStream_t st = as_stream(stream);
    const dim3 grid((unsigned)(rows * p.slices));
    IB_CUDA_CHECK(launch_pdl(type == IB_TYPE_F32 ? beam_slice_kernel<float> : beam_slice_kernel<__half>, grid,
                             dim3(BS_THREADS), 0, st, false, a));
    const size_t smem = (size_t)beams * 16 + (size_t)beams * p.slices * 4;
    IB_CUDA_CHECK(launch_pdl(beam_group_kernel, dim3(n_groups), dim3(BS_THREADS), smem, st, true, a));
    return IB_OK;
}
