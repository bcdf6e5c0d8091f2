// ib_beam_select: the k best continuations of each group of beams.
//
// Row r (a beam) offers every token t with v(r, t) = score(r) + x(r, t) - log sum_t' e^x(r, t'); the
// k largest of a group's rows win, equal ones in the order of (row, token).  The reference takes the
// first maximum of one row (src/ops/ops.cpp:424-438, ib_argmax).
//
// One pass over the logits: a CTA takes a slice of a row, keeps a running maximum and sum of
// exponentials, and the slice's k best.  Inside a row the order of v is that of x, so they are chosen by
// x alone, through a threshold that at least k values are known to reach: it comes from the first step's
// 256 threads' maxima, and from then on a value costs one comparison; the few that pass lie in shared
// memory and are ranked at the end.  A second kernel, a CTA per group, makes the rows' log sums of the
// slices' and picks the group's k best in 64 bits, through a threshold again: candidates of different
// beams may be closer than FP32 tells apart.
//
// What that holds.  Inside a row the choice and its order are exact.  A row's log sum has the error of its FP32
// parts: a thread adds 16 weights e^(x - m) in a step of 4096 values, the threads' and slices' sums are joined
// in 64 bits, so with S steps to a slice it is off by at most (S + 1) (A + 24) 2^-24, A = sum p (max x - x).
// Candidates of different rows that are closer than their rows' errors come in either order, and the
// errors, not the candidates, depend on how the rows are cut.
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <string>

#include "common.cuh"
#include "paged.cuh"  // FastDiv, kSMs, checks
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

// Numbers that sort as the values do (no NaN).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A number that at least k of the CTA's threads' `best` reach, where that many are above 0 (else 0).  First
// the least of the warps' n-th largest, n = k / BS_WARPS rounded up; then, where many more reach it,
// halving between it and the largest of all, a barrier a step, until no more than a quarter above k do or the
// interval is used up (at most 32 steps: it is one of 32-bit numbers).  n: how many reach it.
__device__ __forceinline__ uint32_t reached(uint32_t best, int k, uint32_t (&sh)[2][BS_WARPS], int& n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t top = 0, most = 0, x = best;
    for (int i = (k + BS_WARPS - 1) / BS_WARPS; i > 0; --i) {
        top = __reduce_max_sync(0xffffffffu, x);
        most = max(most, top);
        if (lane == __ffs(__ballot_sync(0xffffffffu, x == top)) - 1) x = 0;
    }
    if (lane == 0) sh[0][warp] = top, sh[1][warp] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BS_WARPS; ++i) top = min(top, sh[0][i]), most = max(most, sh[1][i]);
    top = max(top, 1u);  // (a warp may have none)
    n = __syncthreads_count(best >= top);
    if (n < k) return 0;
    for (int turn = 0; n > k + k / 4 && most - top > 1 && turn < 32; ++turn) {
        const uint32_t half = top + (most - top) / 2;
        const int c = __syncthreads_count(best >= half);
        if (c >= k) top = half, n = c;
        else most = half;
    }
    return top;
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
    int beams, vocab, k, slices, end_token;
    int64_t per_slice;       // values
    FastDiv of_k, of_slices;
    uint64_t* list;          // [row][slice][k] keys, largest first, zeros behind
    SliceMeta* meta;         // [row][slice]
    float* out_score;        // [group][k]
    int32_t *out_token, *out_row;
};

// Two FP32 values, an instruction for both.
struct Two {
    uint64_t x;
    __device__ __forceinline__ static Two of(float a, float b) {
        Two t;
        asm("mov.b64 %0, {%1, %2};" : "=l"(t.x) : "f"(a), "f"(b));
        return t;
    }
    __device__ __forceinline__ void get(float& a, float& b) const {
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
    }
};
__device__ __forceinline__ Two add(Two a, Two b) {
    Two t;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(t.x) : "l"(a.x), "l"(b.x));
    return t;
}
// e^t for t <= 0: 2^(t log2 e) with log2 e in two parts (one alone is 1e-8 short, for all values alike).  Off by
// at most (4 + 2 |t|) 2^-24 of itself: 2^-22 of ex2.approx, and two roundings of its argument.
__device__ __forceinline__ Two exp_of(Two t) {
    constexpr double LOG2E = 1.4426950408889634;
    constexpr float HI = (float)LOG2E, LO = (float)(LOG2E - (double)HI);
    const Two hi = Two::of(HI, HI), lo = Two::of(LO, LO);
    Two y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y.x) : "l"(t.x), "l"(hi.x));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(y.x) : "l"(t.x), "l"(lo.x));
    float a, b;
    y.get(a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    return Two::of(a, b);
}

template <typename T>
__device__ __forceinline__ float logit(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return __half2float(x);
}

struct SliceShared {
    uint64_t buf[BS_CAP];
    int n;
    uint32_t top[2][BS_WARPS];
    double sum[BS_WARPS];
    float m[BS_WARPS];
};

// The k largest of the first n <= BS_CAP keys in sh.buf, in order, to out (zeros behind the last).
// Every thread of the CTA calls it, after a barrier.
__device__ __forceinline__ void rank_best(SliceShared& sh, int n, int k, uint64_t* __restrict__ out) {
    const int tid = threadIdx.x;
    if (n > 3 * k && n > 64) {  // a threshold again, of what has passed the first
        constexpr int N = BS_CAP / BS_THREADS;
        uint64_t key[N], best = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = i * BS_THREADS + tid;
            key[i] = at < n ? sh.buf[at] : 0;
            best = key[i] > best ? key[i] : best;
        }
        int reach;
        const uint32_t least = reached((uint32_t)(best >> 32), k, sh.top, reach);
        if (tid == 0) sh.n = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if ((uint32_t)(key[i] >> 32) >= least && key[i]) sh.buf[atomicAdd(&sh.n, 1)] = key[i];
        __syncthreads();
        n = sh.n;
    }
    for (int i = tid; i < n; i += BS_THREADS) {
        const uint64_t mine = sh.buf[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += sh.buf[j] > mine;
        if (rank < k) out[rank] = mine;
    }
    for (int j = n + tid; j < k; j += BS_THREADS) out[j] = 0;
}

// The slice's k best where too many values reached the threshold (many equal ones, or values that
// rise): step by step and a value of each thread at a time, with a threshold that is raised whenever the
// room is used up.  sh.buf holds the k best so far, in no order, and what has come since.
template <typename T>
__device__ __noinline__ void slice_again(SliceShared& sh, const T* x, int64_t begin, int64_t end, int k,
                                         uint64_t* __restrict__ out) {
    constexpr int N = BS_CAP / BS_THREADS;
    const int tid = threadIdx.x;
    uint64_t floor_key = 1;
    __syncthreads();
    if (tid == 0) sh.n = 0;
    for (int64_t at = begin; at < end; at += BS_THREADS) {
        __syncthreads();
        const int have = sh.n;
        __syncthreads();  // everybody has read it
        if (have > BS_CAP - BS_THREADS) {
            // keys are all different: halving finds the k-th largest
            uint64_t key[N], lo = 1, hi = ~0ull;
#pragma unroll
            for (int i = 0; i < N; ++i) key[i] = i * BS_THREADS + tid < have ? sh.buf[i * BS_THREADS + tid] : 0;
            while (hi - lo > 1) {
                const uint64_t half = lo + (hi - lo) / 2;
                int c = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) c += __syncthreads_count(key[i] >= half);
                if (c >= k) lo = half;
                else hi = half;
                if (c == k) break;
            }
            floor_key = lo;
            __syncthreads();
            if (tid == 0) sh.n = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (key[i] >= lo) sh.buf[atomicAdd(&sh.n, 1)] = key[i];
            __syncthreads();
        }
        const int64_t p = at + tid;
        const uint64_t key = p < end ? beam_key(logit(x[p]), (uint32_t)p) : 0;
        if (key >= floor_key) sh.buf[atomicAdd(&sh.n, 1)] = key;
    }
    __syncthreads();
    rank_best(sh, sh.n, k, out);
}

// 16 groups of 8 beams over 128256 FP32 logits, 62 MB, take 21 us with cold caches, 3.0 TB/s; the call 23 us in
// a graph, 74 before loads of 16 bytes a step ahead and a threshold of the first step's.  Neither HBM (0.36) nor
// issue slots (0.53) are used up: a step's instructions, 17 to a value, wait for one another (10 cycles
// between two of a warp's), and four CTAs are on the busiest SM, 3.5 on the mean one; more and shorter
// slices cost what they gain (select_plan).
// VEC: values of one load (16 bytes where the rows allow it, else one).
template <typename T, int VEC>
__global__ void __launch_bounds__(BS_THREADS) beam_slice_kernel(const __grid_constant__ SelectArgs A) {
    __shared__ SliceShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / A.slices, slice = blockIdx.x - row * A.slices;
    pdl_launch_dependents();
    if (A.ended && A.ended[row]) return;
    const T* const x = static_cast<const T*>(A.logits) + (int64_t)row * A.stride;
    const int begin = (int)(slice * A.per_slice), end = (int)min((int64_t)A.vocab, begin + A.per_slice);
    if (tid == 0) sh.n = 0;
    float m = -INFINITY, sum = 0.f, least = 0.f;
    // value i of the thread's is token at + place(i)
    auto place = [&](int i) { return (i / VEC * BS_THREADS + tid) * VEC + i % VEC; };
    struct alignas(16) Values {
        T x[16];
    };
    auto load = [&](int at, Values& y) {
        const T* const p = x + at;
        if (VEC > 1 && at + BS_TILE <= end) {
#pragma unroll
            for (int i = 0; i < 16; i += VEC)
                *reinterpret_cast<uint4*>(y.x + i) = __ldg(reinterpret_cast<const uint4*>(p + place(i)));
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) y.x[i] = at + place(i) < end ? p[place(i)] : (T)-INFINITY;
        }
    };
    Values now;
    load(begin, now);
    for (int at = begin; at < end; at += BS_TILE) {
        Values next;  // on its way while this one is looked at
        if (at + BS_TILE < end) load(at + BS_TILE, next);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = logit(now.x[i]);
        float top = v[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, v[i]);  // (a NaN only where there is nothing else)
        if (at == begin) {
            int n;
            const uint32_t o = reached(top > -INFINITY ? ordered(top) : 0, A.k, sh.top, n);
            // the value itself; where not enough threads have one, all that are no -inf pass
            least = o > ordered(-FLT_MAX) ? __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o) : -FLT_MAX;
        }
        if (top > m) {
            sum *= expf(m - top);
            m = top;
        }
        const float base = m > -INFINITY ? m : 0.f;  // e^-inf is 0, and a NaN stays one
        const Two below = Two::of(-base, -base);
        Two more[2] = {Two::of(0.f, 0.f), Two::of(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < 16; i += 2)
            more[i / 2 & 1] = add(more[i / 2 & 1], exp_of(add(Two::of(v[i], v[i + 1]), below)));
        float part[4];
        more[0].get(part[0], part[1]), more[1].get(part[2], part[3]);
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        if (top >= least) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (v[i] >= least) {
                    const int to = atomicAdd(&sh.n, 1);
                    if (to < BS_CAP) sh.buf[to] = beam_key(v[i], (uint32_t)(at + place(i)));
                }
        }
        now = next;
    }
    const int64_t list = (int64_t)row * A.slices + slice;
    // the slice's maximum and sum
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (lane == 0) sh.m[warp] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BS_WARPS; ++i) M = fmaxf(M, sh.m[i]);
    double d = (double)(m > -INFINITY ? sum * expf(m - M) : sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) sh.sum[warp] = d;
    const int n = sh.n;
    if (n <= BS_CAP) rank_best(sh, n, A.k, A.list + list * A.k);
    else slice_again(sh, x, (int64_t)begin, (int64_t)end, A.k, A.list + list * A.k);
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < BS_WARPS; ++i) d += sh.sum[i];
        A.meta[list] = SliceMeta{M, 0.f, d};
    }
}

// Of two candidates of a row the one with the larger key is better, whatever their values round to in 64 bits.
struct Best {
    double v;
    uint64_t key;  // of the logit and its token
    int row;       // in the group
};
constexpr int BS_NO_ROW = 0x7fffffff;
__device__ __forceinline__ bool better(const Best& a, const Best& b) {
    return a.v > b.v || (a.v == b.v && (a.row < b.row || (a.row == b.row && a.key > b.key)));
}

constexpr int BS_GROUP_CAP = 1024;

__device__ __forceinline__ void put_choice(const SelectArgs& A, int g, int j, const Best& y) {
    const bool any = y.v > -INFINITY;
    const int64_t at = (int64_t)g * A.k + j;
    A.out_score[at] = any ? (float)y.v : -INFINITY;
    A.out_token[at] = any ? (int32_t)key_place(y.key) : -1;
    A.out_row[at] = any ? g * A.beams + y.row : -1;
}

// Candidate c of group g, whose key is `key`: entry c % k of list c / k, a row's slice; v is -inf where
// there is none.  base: score - log sum e^(x - M), and M; M is NaN for a row that has ended.
__device__ __forceinline__ Best candidate(const SelectArgs& A, int c, uint64_t key, const double2* base) {
    const int b = (int)A.of_slices.div(A.of_k.div((uint32_t)c));
    const double2 y0 = base[b];
    Best y = {-INFINITY, 0, BS_NO_ROW};
    if (y0.y != y0.y) {
        if (c == b * A.slices * A.k) y = Best{y0.x, beam_key(0.f, (uint32_t)A.end_token), b};
    } else if (key) {
        y = Best{y0.x + ((double)key_value(key) - y0.y), key, b};
    }
    if (!(y.v > -INFINITY)) y.v = -INFINITY;  // NaN is no candidate
    y.v += 0.0;                               // -0 and 0 are equal
    return y;
}

// The group's choice where too many candidates reached the threshold: k rounds of a maximum over the CTA,
// each behind the last one's.
__device__ __noinline__ void group_again(const SelectArgs& A, int g, int n, const uint64_t* list,
                                         const double2* base) {
    __shared__ Best sh_best[2][BS_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Best last = {INFINITY, 0, 0};
    bool first = true;
    for (int j = 0; j < A.k; ++j, first = false) {
        Best top = {-INFINITY, 0, BS_NO_ROW};
        for (int c = tid; c < n; c += BS_THREADS) {
            const Best y = candidate(A, c, list[c], base);
            if ((first || better(last, y)) && better(y, top)) top = y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            Best y;
            y.v = __shfl_xor_sync(0xffffffffu, top.v, o);
            y.key = __shfl_xor_sync(0xffffffffu, top.key, o);
            y.row = __shfl_xor_sync(0xffffffffu, top.row, o);
            if (better(y, top)) top = y;
        }
        if (lane == 0) sh_best[j & 1][warp] = top;
        __syncthreads();
        top = sh_best[j & 1][0];
#pragma unroll
        for (int i = 1; i < BS_WARPS; ++i)
            if (better(sh_best[j & 1][i], top)) top = sh_best[j & 1][i];
        if (tid == 0) put_choice(A, g, j, top);
        last = top;
    }
}

// A CTA per group, the slices' lists in its threads' registers where they fit.  A chain of reads, a
// threshold's barriers and FP64 values: 8 us with cold caches for 16 groups of 8 rows of 4 slices; three to
// four in a graph, where it is launched beside the slices.
__global__ void __launch_bounds__(BS_THREADS) beam_group_kernel(const __grid_constant__ SelectArgs A) {
    extern __shared__ __align__(16) double2 base[];  // [beams]
    __shared__ double buf_v[BS_GROUP_CAP];  // of those that are ranked; the rest is read where values are equal
    __shared__ uint64_t buf_key[BS_GROUP_CAP];
    __shared__ int buf_row[BS_GROUP_CAP];
    __shared__ uint32_t sh_top[2][BS_WARPS];
    __shared__ int sh_n;
    const int tid = threadIdx.x, g = blockIdx.x, row0 = g * A.beams, k = A.k;
    if (tid == 0) sh_n = 0;
    const int n = A.beams * A.slices * k;
    const uint64_t* const list = A.list + (int64_t)g * n;
    pdl_wait();
    constexpr int AHEAD = 4;  // a thread's first keys, on their way meanwhile
    uint64_t key[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) key[i] = tid + i * BS_THREADS < n ? list[tid + i * BS_THREADS] : 0;
    // as many lanes to a row as it has slices
    int lanes = 1;
    while (lanes < 32 && lanes < A.slices) lanes *= 2;
    const int sub = tid & (lanes - 1), per = BS_THREADS / lanes;
    for (int b0 = 0; b0 < A.beams; b0 += per) {
        const int b = b0 + tid / lanes, row = row0 + b;
        const bool there = b < A.beams, end = there && A.ended && A.ended[row];
        const SliceMeta* const meta = A.meta + (int64_t)row * A.slices;
        const int slices = there && !end ? A.slices : 0;
        float M = -INFINITY;
        double s = 0;
        for (int i = sub; i < slices; i += lanes) M = fmaxf(M, meta[i].m);
        for (int o = lanes / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        for (int i = sub; i < slices; i += lanes) {
            const SliceMeta y = meta[i];
            s += y.m > -INFINITY ? y.sum * exp((double)y.m - (double)M) : y.sum;
        }
        for (int o = lanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        // (a row of nothing but -inf has no candidates)
        if (there && sub == 0)
            base[b] = make_double2((A.scores ? (double)A.scores[row] : 0.0) - (end ? 0.0 : log(s)), end ? (double)NAN : (double)M);
    }
    __syncthreads();
    // rounding down keeps the order, so that k values at or above it are above all below it
    auto low = [](double v) { return v > -INFINITY ? ordered(__double2float_rd(v)) : 0u; };
    uint32_t best = 0;
    double mine[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const int c = tid + i * BS_THREADS;
        mine[i] = c < n ? candidate(A, c, key[i], base).v : -INFINITY;
        best = max(best, low(mine[i]));
    }
    for (int c = tid + AHEAD * BS_THREADS; c < n; c += BS_THREADS)
        best = max(best, low(candidate(A, c, list[c], base).v));
    int reach;
    const uint32_t least = max(reached(best, k, sh_top, reach), 1u);
    auto take = [&](const Best& y) {
        const int to = atomicAdd(&sh_n, 1);
        if (to < BS_GROUP_CAP) buf_v[to] = y.v, buf_key[to] = y.key, buf_row[to] = y.row;
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (low(mine[i]) >= least) take(candidate(A, tid + i * BS_THREADS, key[i], base));
    for (int c = tid + AHEAD * BS_THREADS; c < n; c += BS_THREADS) {
        const Best y = candidate(A, c, list[c], base);
        if (low(y.v) >= least) take(y);
    }
    __syncthreads();
    const int some = sh_n;
    if (some > BS_GROUP_CAP) {
        group_again(A, g, n, list, base);
        return;
    }
    for (int i = tid; i < some; i += BS_THREADS) {
        const Best own = {buf_v[i], buf_key[i], buf_row[i]};
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < some; ++j) {
            rank += buf_v[j] > own.v;
            if (buf_v[j] == own.v && j != i) rank += better(Best{own.v, buf_key[j], buf_row[j]}, own);
        }
        if (rank < k) put_choice(A, g, rank, own);
    }
    for (int j = some + tid; j < k; j += BS_THREADS) put_choice(A, g, j, Best{-INFINITY, 0, BS_NO_ROW});
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
    // The number of slices that keeps the SM with most of them busy for the shortest time: it has four at
    // once (fewer do not fill it), and a slice costs two tiles besides its own.  (us with one slice to a row
    // and with these: 360 rows over 38573 FP16 values 21.8 and 19.1, 304 over 15427 FP32 18.9 and 16.1, 192
    // over 32003 FP16 17.3 and 14.5; 128 over 128256 FP32 take 22.9 in 4 slices each, 25.8 in 5, 23.6 in 8.)
    int64_t best = INT64_MAX;
    p.slices = 1;
    for (int64_t s = 1; s <= std::min(tiles, std::max<int64_t>(1, kSMs * 8 / rows)); ++s) {
        const int64_t per = (tiles + s - 1) / s, n = (tiles + per - 1) / per;
        const int64_t cost = std::max<int64_t>(4, (rows * n + kSMs - 1) / kSMs) * (per + 2);
        if (cost < best) best = cost, p.slices = (int)n;
    }
    // of equal length
    p.per_slice = ((vocab + p.slices - 1) / p.slices + BS_THREADS - 1) / BS_THREADS * BS_THREADS;
    p.slices = (int)((vocab + p.per_slice - 1) / p.per_slice);
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
    {
        const int64_t size = type == IB_TYPE_F32 ? 4 : 2, out = (int64_t)n_groups * k * 4;
        const void* const to[4] = {out_score, out_token, out_row, workspace};
        const int64_t to_n[4] = {out, out, out, (int64_t)p.bytes};
        bool bad = false;
        for (int i = 0; i < 4; ++i) {
            bad = bad || bytes_meet(to[i], to_n[i], logits, ((rows - 1) * stride + vocab) * size);
            bad = bad || (scores && bytes_meet(to[i], to_n[i], scores, rows * 4));
            bad = bad || (ended && bytes_meet(to[i], to_n[i], ended, rows * 4));
            for (int j = 0; j < i; ++j) bad = bad || bytes_meet(to[i], to_n[i], to[j], to_n[j]);
        }
        if (bad) return paged_refuse(who, "results and workspace must not overlap the inputs or one another");
    }
    SelectArgs a{};
    a.logits = logits;
    a.stride = stride;
    a.scores = scores;
    a.ended = ended;
    a.beams = beams;
    a.vocab = vocab;
    a.k = k;
    a.slices = p.slices;
    a.end_token = end_token;
    a.per_slice = p.per_slice;
    a.of_k = FastDiv::make((uint32_t)k);
    a.of_slices = FastDiv::make((uint32_t)p.slices);
    a.list = reinterpret_cast<uint64_t*>((uint8_t*)workspace + p.list_off);
    a.meta = reinterpret_cast<SliceMeta*>((uint8_t*)workspace + p.meta_off);
    a.out_score = out_score;
    a.out_token = out_token;
    a.out_row = out_row;
    cudaStream_t st = as_stream(stream);
    const dim3 grid((unsigned)(rows * p.slices));
    const int64_t size = type == IB_TYPE_F32 ? 4 : 2;
    const bool wide = (((uintptr_t)logits | (uintptr_t)(rows > 1 ? stride * size : 0)) & 15) == 0;
    auto* const slice = type == IB_TYPE_F32 ? (wide ? beam_slice_kernel<float, 4> : beam_slice_kernel<float, 1>)
                                            : (wide ? beam_slice_kernel<__half, 8> : beam_slice_kernel<__half, 1>);
    IB_CUDA_CHECK(launch_pdl(slice, grid, dim3(BS_THREADS), 0, st, false, a));
    const size_t smem = (size_t)beams * sizeof(double2);
    IB_CUDA_CHECK(launch_pdl(beam_group_kernel, dim3(n_groups), dim3(BS_THREADS), smem, st, true, a));
    return IB_OK;
}
