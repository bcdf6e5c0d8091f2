// The paged KV cache: pages of page_size positions, handed to sequences through a table, so
// that many sequences of different lengths share one pool and forks share their prefix.  No
// counterpart in the reference, which keeps one contiguous cache per model
// (src/models/model_cuda.cpp:204-211).
//
// Pool: k and v each [layer][page][kv head][position in page][head_dim], FP32 or FP16.  The
// bookkeeping is on the device (refs[page] = sequences holding it, 0 = free), so a serving
// step -- release, fork, extend, append, attention -- runs without the host reading anything
// and can be captured in a graph.  Pages are given out lowest first and in list order, so a
// run's tables are reproducible.
//
// The planning kernels (extend, the first half of fork, the first half of compact) are one
// CTA of 1024 threads: their work is a scan over refs (4 bytes a page; 6000 pages are one
// 16-KB and one partial iteration) that needs one prefix order, and what bounds them is the
// latency of a few block-wide scans, not bandwidth.  The data moves in a second, wide kernel.
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "common.cuh"
#include "kv.cuh"
#include "paged.cuh"
#include "pdl.cuh"

namespace ib {

constexpr int KV_PLAN_THREADS = 1024;
constexpr int KV_SCAN = 8;  // refs per thread and iteration of a scan
constexpr int KV_COPY_THREADS = 256;

// ---- checks ----------------------------------------------------------------------------
static int paged_refuse(const char* who, const char* what) {
    set_error(std::string(who) + ": " + what);
    return IB_ERR_INVALID;
}

int paged_check(const ib_kv_pages* p, const ib_kv_seqs* s, const char* who) {
    if (!p || !s) return paged_refuse(who, "null pointer argument");
    if (p->type != IB_TYPE_F32 && p->type != IB_TYPE_F16) {
        set_error(std::string(who) + ": the pages must be F32 or F16, not " + type_name(p->type));
        return IB_ERR_UNSUPPORTED;
    }
    if (!p->k || !p->v || !s->table || !s->len || !s->refs)
        return paged_refuse(who, "null pointer argument");
    if (p->n_layers <= 0 || p->n_pages <= 0 || p->n_pages > IB_KV_MAX_PAGES || p->n_kv_heads <= 0)
        return paged_refuse(who, "n_layers, n_pages or n_kv_heads out of range");
    if (p->head_dim < 8 || p->head_dim > 256 || p->head_dim % 8)
        return paged_refuse(who, "head_dim must be a multiple of 8 in [8, 256]");
    if (p->page_size < 1 || p->page_size > IB_KV_MAX_PAGE_SIZE)
        return paged_refuse(who, "page_size out of range");
    // kernels number the rows of a layer with 31 bits
    if ((int64_t)p->n_pages * p->n_kv_heads * p->page_size >= (1ll << 31))
        return paged_refuse(who, "n_pages x n_kv_heads x page_size must be below 2^31");
    if (((uintptr_t)p->k & 15) || ((uintptr_t)p->v & 15))
        return paged_refuse(who, "the pages must be 16-byte aligned");
    if (s->n_slots < 1 || s->n_slots > IB_KV_MAX_SLOTS || s->max_pages < 1)
        return paged_refuse(who, "n_slots or max_pages out of range");
    if ((int64_t)s->max_pages * p->page_size > (1 << 28))
        return paged_refuse(who, "max_pages x page_size must be at most 2^28");
    return IB_OK;
}

int paged_check_batch(const ib_kv_pages* p, const ib_kv_seqs* s, const ib_kv_batch* b, int layer,
                      int n_heads, const char* who) {
    const int r = paged_check(p, s, who);
    if (r != IB_OK) return r;
    if (!b || !b->cu_q) return paged_refuse(who, "null pointer argument");
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_q < 0)
        return paged_refuse(who, "bad batch sizes");
    if (b->n_seqs > s->n_slots) return paged_refuse(who, "more sequences than slots");
    if (layer < 0 || layer >= p->n_layers) return paged_refuse(who, "layer out of range");
    if (n_heads <= 0 || n_heads % p->n_kv_heads)
        return paged_refuse(who, "n_heads must be a multiple of n_kv_heads");
    if (n_heads > 1024) return paged_refuse(who, "n_heads must be at most 1024");
    if ((int64_t)b->n_tokens * n_heads > (1 << 26))
        return paged_refuse(who, "n_tokens x n_heads must be at most 2^26");
    return IB_OK;
}

PagedView paged_view(const ib_kv_pages* p, const ib_kv_seqs* s, const ib_kv_batch* b, int n_heads) {
    PagedView w;
    w.table = s->table;
    w.len = s->len;
    w.refs = s->refs;
    w.cu_q = b->cu_q;
    w.slots = b->slots;
    w.n_slots = s->n_slots;
    w.max_pages = s->max_pages;
    w.n_pages = p->n_pages;
    w.n_seqs = b->n_seqs;
    w.n_tokens = b->n_tokens;
    w.H = n_heads;
    w.Hkv = p->n_kv_heads;
    w.HD = p->head_dim;
    w.page_size = p->page_size;
    w.ps = FastDiv::make((uint32_t)p->page_size);
    w.group = FastDiv::make((uint32_t)(n_heads / p->n_kv_heads));
    return w;
}

int paged_fault_take(int* code) { return paged_fault_take_here(code); }

bool paged_rows_overlap(const float* a, int64_t sa, int64_t wa, const float* b, int64_t sb, int64_t wb,
                        int64_t n) {
    const int64_t d = ((intptr_t)b - (intptr_t)a) / (int64_t)sizeof(float);
    if (sa != sb || sa <= 0)  // no common step: the whole ranges
        return d < (n - 1) * sa + wa && -d < (n - 1) * sb + wb;
    // row i of a and row i + k of b meet where -wb < d + k sa < wa, for k within n - 1 of 0: the
    // least such k is the first one above (-wb - d) / sa
    const int64_t x = -wb - d, floor = x >= 0 ? x / sa : -((-x + sa - 1) / sa);
    const int64_t k = std::max(floor + 1, 1 - n);
    return k <= n - 1 && d + k * sa < wa;
}

static int elem_bytes(const ib_kv_pages* p) { return p->type == IB_TYPE_F32 ? 4 : 2; }

static int sm_count(int* n) {
    int dev = 0;
    IB_CUDA_CHECK(cudaGetDevice(&dev));
    IB_CUDA_CHECK(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, dev));
    return IB_OK;
}

// ---- block-wide exclusive scan ---------------------------------------------------------
// Every thread of the CTA calls it; returns the sum of v over the threads before this one
// and the CTA's total.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += x;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    total = warp_sums[31];
    const int before = warp ? warp_sums[warp - 1] : 0;
    __syncthreads();  // warp_sums is free again
    return before + inc - v;
}

// KV_SCAN consecutive refs of this thread in the scan iteration that starts at `base`;
// pages behind the last read as held.
__device__ __forceinline__ void load_refs(const int32_t* refs, int base, int n_pages,
                                          int (&r)[KV_SCAN]) {
    const int64_t p0 = (int64_t)base + (int64_t)threadIdx.x * KV_SCAN;
#pragma unroll
    for (int i = 0; i < KV_SCAN; ++i) r[i] = p0 + i < n_pages ? refs[p0 + i] : 1;
}

// ---- extend and fork: who gets how many pages ------------------------------------------
struct KvSeqsDev {
    int32_t *table, *len, *refs;
    int n_slots, max_pages, n_pages, page_size;
};

// One CTA.  FORK: a = parents, b = children; entry i needs the one page that its partial
// last page is copied to.  Otherwise a = slots, b = tokens to make room for.  Pages go out
// lowest first in list order; once an entry finds too few, it and every later entry that
// needs pages get none.  status: 1 done, 0 no room, -1 refused.
// What the entries need stays in shared memory: the kernel is a chain of dependent accesses (list,
// length, table, refs, hand-out) and little else: 11 us for 96 children or slots with cold caches.
template <bool FORK>
__global__ void __launch_bounds__(KV_PLAN_THREADS)
    kv_assign_kernel(const KvSeqsDev s, int n, const int32_t* __restrict__ a,
                     const int32_t* __restrict__ b, int32_t* __restrict__ status) {
    extern __shared__ int sh[];
    __shared__ int warp_sums[32];
    const int n_first = max(s.n_slots, n);
    int* first = sh;                // [n_slots]: lowest list index naming the slot; then
    int* len = sh;                  // [n]: length of the entry's source
    int* off = sh + n_first;        // [n + 1]: pages needed by the entries before
    uint16_t* slot_of = reinterpret_cast<uint16_t*>(off + n + 1);  // [n]
    int8_t* state = reinterpret_cast<int8_t*>(slot_of + n);        // [n]
    const int tid = threadIdx.x, cap = s.max_pages * s.page_size;
    const int32_t* slots = FORK ? b : a;
    pdl_launch_dependents();
    int r[KV_SCAN];
    load_refs(s.refs, 0, s.n_pages, r);  // the first scan's, on their way
    for (int i = tid; i < n; i += KV_PLAN_THREADS) {
        const int slot = slots[i];
        const bool in = slot >= 0 && slot < s.n_slots;
        slot_of[i] = (uint16_t)(in ? slot : 0xffff);
        if (in) first[slot] = 0x7fffffff;
    }
    __syncthreads();
    for (int i = tid; i < n; i += KV_PLAN_THREADS)
        if (slot_of[i] != 0xffff) atomicMin(&first[slot_of[i]], i);
    __syncthreads();
    for (int i = tid; i < n; i += KV_PLAN_THREADS)
        state[i] = slot_of[i] != 0xffff && first[slot_of[i]] == i ? 1 : -1;
    __syncthreads();  // first is done with
    int total = 0;
    for (int i0 = 0; i0 < n; i0 += KV_PLAN_THREADS) {
        const int i = i0 + tid;
        int need = 0;
        if (i < n) {
            const int slot = slot_of[i], src = FORK ? a[i] : slot;
            int st = -1;
            if (state[i] == 1 && src >= 0 && src < s.n_slots &&
                (!FORK || (src != slot && s.len[slot] == 0))) {
                const int L = s.len[src], more = FORK ? 0 : b[i];
                len[i] = L;
                if (L < 0 || L > cap) {
                    paged_fault(PAGED_BAD_LEN);
                } else if (FORK) {
                    st = 1;
                    if (L % s.page_size) {  // a page that was given back (-1) has nothing to copy
                        const int t = s.table[(size_t)src * s.max_pages + L / s.page_size];
                        if (t < -1 || t >= s.n_pages) paged_fault(PAGED_BAD_PAGE);
                        need = t >= 0 && t < s.n_pages;
                    }
                } else if (more >= 0) {
                    st = more > cap - L ? 0 : 1;
                    if (st)
                        need = (L + more + s.page_size - 1) / s.page_size -
                               (L + s.page_size - 1) / s.page_size;
                }
            }
            state[i] = (int8_t)(st == 1 && need ? 2 : st);  // 2: if the pages are there
        }
        // more than the pool holds is as good as one page more: the sums stay in 31 bits
        // (1024 x (2^20 + 1)), and a saturated end is past any number of free pages
        const int most = s.n_pages + 1;
        int sum;
        const int before = block_scan(min(need, most), warp_sums, sum);
        if (i < n) off[i] = min(total + before, most);
        total = min(total + sum, most);
    }
    if (tid == 0) off[n] = total;
    // free pages, up to what is asked for; with one round of refs they are numbered with it
    constexpr int ROUND = KV_PLAN_THREADS * KV_SCAN;
    const bool one_round = s.n_pages <= ROUND;
    int avail = 0, number = 0;
    for (int base = 0; base < s.n_pages && avail < total; base += ROUND) {
        int c = 0, sum;
        if (base) load_refs(s.refs, base, s.n_pages, r);
#pragma unroll
        for (int k = 0; k < KV_SCAN; ++k) c += r[k] <= 0;
        number = block_scan(c, warp_sums, sum);
        avail += sum;
    }
    __syncthreads();  // off
    // entry i is served when the pages up to and with its own are there
    int served = 0;  // pages handed out
    for (int i = tid; i < n; i += KV_PLAN_THREADS) {
        int st = state[i];
        if (st == 2) {
            st = off[i + 1] <= avail;
            if (st) served = max(served, off[i + 1]);
            state[i] = (int8_t)st;
        }
        status[i] = st;
        if (st == 1) s.len[slot_of[i]] = FORK ? len[i] : len[i] + b[i];
    }
    for (int o = 16; o > 0; o >>= 1) served = max(served, __shfl_xor_sync(0xffffffffu, served, o));
    if ((tid & 31) == 0) warp_sums[tid >> 5] = served;
    __syncthreads();
    for (int k = 0; k < 32; ++k) served = max(served, warp_sums[k]);
    __syncthreads();
    // hand them out: the k-th free page belongs to the entry with off[i] <= k < off[i + 1]
    int given = 0;
    for (int base = 0; base < s.n_pages && given < served; base += ROUND) {
        int k = number;
        if (one_round) {
            given = avail;
        } else {
            int c = 0, sum;
            load_refs(s.refs, base, s.n_pages, r);
#pragma unroll
            for (int j = 0; j < KV_SCAN; ++j) c += r[j] <= 0;
            k = given + block_scan(c, warp_sums, sum);
            given += sum;
        }
#pragma unroll
        for (int j = 0; j < KV_SCAN; ++j) {
            if (r[j] > 0) continue;
            if (k < served) {
                int lo = 0, hi = n;  // last i with off[i] <= k
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (off[mid] <= k) lo = mid;
                    else hi = mid;
                }
                const int page = base + tid * KV_SCAN + j, L = len[lo];
                const int col = FORK ? L / s.page_size
                                     : (L + s.page_size - 1) / s.page_size + (k - off[lo]);
                s.table[(size_t)slot_of[lo] * s.max_pages + col] = page;
                s.refs[page] = 1;
            }
            ++k;
        }
    }
}

// Copies `bytes` (a multiple of 16, both sides 16-byte aligned) by one warp, eight 16-byte
// loads per lane in flight.
__device__ __forceinline__ void warp_copy(uint4* __restrict__ d, const uint4* __restrict__ s,
                                          int n16) {
    const int lane = threadIdx.x & 31;
    for (int i = lane; i < n16; i += 256) {
        uint4 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + 32 * k < n16) x[k] = s[i + 32 * k];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + 32 * k < n16) d[i + 32 * k] = x[k];
    }
}

// The pool as bytes: layer l, page p at l * layer_bytes + p * page_bytes.
struct PoolBytes {
    uint8_t *k, *v;
    int n_layers, n_kv_heads, row_bytes;  // row: head_dim elements
    int64_t page_bytes, layer_bytes;
};

// Second half of a fork: children's rows, reference counts and the filled rows of the
// partial pages, one warp per (child, layer, k or v, kv head) of those.  Bound by HBM once there are
// many: 96 children of 22 layers 18 us, most of 119 MB read and written.
__global__ void __launch_bounds__(KV_COPY_THREADS)
    kv_fork_kernel(const KvSeqsDev s, const PoolBytes pool, int n,
                   const int32_t* __restrict__ parents, const int32_t* __restrict__ children,
                   const int32_t* __restrict__ status) {
    const int n_warps = gridDim.x * (KV_COPY_THREADS / 32);
    const int w0 = blockIdx.x * (KV_COPY_THREADS / 32) + (threadIdx.x >> 5);
    pdl_wait();
    for (int i = blockIdx.x; i < n; i += gridDim.x) {  // rows: one CTA per child
        if (status[i] != 1) continue;
        const int full = s.len[children[i]] / s.page_size;
        const int32_t* from = s.table + (size_t)parents[i] * s.max_pages;
        int32_t* to = s.table + (size_t)children[i] * s.max_pages;
        for (int j = threadIdx.x; j < full; j += KV_COPY_THREADS) {
            const int t = from[j];
            to[j] = t;
            if (t >= 0 && t < s.n_pages) atomicAdd(&s.refs[t], 1);
            else if (t != -1) paged_fault(PAGED_BAD_PAGE);
        }
    }
    const int per = pool.n_layers * 2 * pool.n_kv_heads;
    const int64_t units = (int64_t)n * per;
    for (int64_t u = w0; u < units; u += n_warps) {
        const int i = (int)(u / per);
        int r = (int)(u - (int64_t)i * per);
        if (status[i] != 1) continue;
        const int L = s.len[children[i]], part = L % s.page_size;
        if (!part) continue;
        const int col = L / s.page_size;
        const int src = s.table[(size_t)parents[i] * s.max_pages + col];
        const int dst = s.table[(size_t)children[i] * s.max_pages + col];
        if (src < 0 || src >= s.n_pages || dst < 0) continue;
        const int head = r % pool.n_kv_heads;
        r /= pool.n_kv_heads;
        uint8_t* base = (r & 1) ? pool.v : pool.k;
        const int64_t head_off = (int64_t)head * s.page_size * pool.row_bytes +
                                 (int64_t)(r >> 1) * pool.layer_bytes;
        warp_copy((uint4*)(base + head_off + dst * pool.page_bytes),
                  (const uint4*)(base + head_off + src * pool.page_bytes),
                  part * pool.row_bytes / 16);
    }
}

__global__ void __launch_bounds__(KV_COPY_THREADS)
    kv_granted_kernel(int n, const int32_t* slots, const int32_t* __restrict__ status,
                      int32_t* granted) {  // may be slots
    const int i = blockIdx.x * KV_COPY_THREADS + threadIdx.x;
    if (i < n) granted[i] = status[i] == 1 ? slots[i] : -1;
}

// One CTA per list entry.  The length is taken with an exchange, so a slot named twice is
// released once.  A chain of four dependent accesses: 5 us for 96 slots with cold caches.
__global__ void __launch_bounds__(KV_COPY_THREADS)
    kv_release_kernel(const KvSeqsDev s, int n, const int32_t* __restrict__ slots) {
    __shared__ int len;
    const int slot = slots[blockIdx.x];
    if (slot < 0 || slot >= s.n_slots) {
        if (threadIdx.x == 0) paged_fault(PAGED_BAD_SLOT);
        return;
    }
    if (threadIdx.x == 0) len = atomicExch(&s.len[slot], 0);
    __syncthreads();
    int L = len;
    const int cap = s.max_pages * s.page_size;
    if (L < 0 || L > cap) {
        if (threadIdx.x == 0) paged_fault(PAGED_BAD_LEN);
        L = min(max(L, 0), cap);
    }
    int32_t* row = s.table + (size_t)slot * s.max_pages;
    const int used = (L + s.page_size - 1) / s.page_size;
    for (int j = threadIdx.x; j < used; j += KV_COPY_THREADS) {
        const int t = row[j];
        row[j] = -1;
        if (t >= 0 && t < s.n_pages) {
            if (atomicSub(&s.refs[t], 1) <= 0) {  // held by nobody: leave it free
                atomicAdd(&s.refs[t], 1);
                paged_fault(PAGED_BAD_REFS);
            }
        } else if (t != -1) {
            paged_fault(PAGED_BAD_PAGE);
        }
    }
}

// ---- compact ---------------------------------------------------------------------------
// One CTA: with n_live held pages, the i-th held page at an index >= n_live moves to the
// i-th free index below n_live, so the fewest pages move and no page is both read and
// written.  moves: (source, destination) pairs; info: n_live, number of moves.
__global__ void __launch_bounds__(KV_PLAN_THREADS)
    kv_compact_plan_kernel(const int32_t* refs, int32_t* refs_out, int n_pages,
                           int32_t* __restrict__ map, int32_t* __restrict__ moves,
                           int32_t* __restrict__ info) {
    __shared__ int warp_sums[32];
    constexpr int STEP = KV_PLAN_THREADS * KV_SCAN;
    const int tid = threadIdx.x;
    pdl_launch_dependents();
    int r[KV_SCAN];  // of the last round; with one round they are read once
    int n_live = 0;
    for (int base = 0; base < n_pages; base += STEP) {
        int c = 0, sum;
        load_refs(refs, base, n_pages, r);
#pragma unroll
        for (int k = 0; k < KV_SCAN; ++k)
            c += r[k] > 0 && base + tid * KV_SCAN + k < n_pages;
        block_scan(c, warp_sums, sum);
        n_live += sum;
    }
    int holes = 0, movers = 0;  // of the rounds before
    for (int base = 0; base < n_pages; base += STEP) {
        int h = 0, m = 0, sum;
        if (n_pages > STEP) load_refs(refs, base, n_pages, r);
        const int p0 = base + tid * KV_SCAN;
#pragma unroll
        for (int k = 0; k < KV_SCAN; ++k) {
            const int p = p0 + k;
            h += p < n_live && r[k] <= 0;
            m += p >= n_live && p < n_pages && r[k] > 0;
        }
        int hi = holes + block_scan(h, warp_sums, sum);
        holes += sum;
        int mi = movers + block_scan(m, warp_sums, sum);
        movers += sum;
#pragma unroll
        for (int k = 0; k < KV_SCAN; ++k) {
            const int p = p0 + k;
            if (p >= n_pages) break;
            if (r[k] > 0 && p >= n_live) {
                moves[2 * mi++] = p;  // map and refs_out follow below
            } else {
                if (r[k] <= 0 && p < n_live) moves[2 * hi++ + 1] = p;
                map[p] = r[k] > 0 ? p : -1;
                if (r[k] > 0) refs_out[p] = r[k];
                else if (p >= n_live) refs_out[p] = 0;  // a filled hole is set below
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < movers; i += KV_PLAN_THREADS) {
        const int src = moves[2 * i], dst = moves[2 * i + 1];
        map[src] = dst;
        refs_out[dst] = refs[src];
        refs_out[src] = 0;
    }
    if (tid == 0) {
        info[0] = n_live;
        info[1] = movers;
    }
}

// Renames the tables and copies the moved pages, one warp per 4 KB of a page of a layer.  Bound by
// HBM: 1.04 GB read and written in 169 us, 6.17 TB/s, 0.94 of the measured rate.
__global__ void __launch_bounds__(KV_COPY_THREADS)
    kv_compact_kernel(const int32_t* table, int32_t* table_out, int64_t n_entries, int n_pages,
                      const int32_t* __restrict__ map, const int32_t* __restrict__ moves,
                      const int32_t* __restrict__ info, const PoolBytes pool) {
    pdl_wait();
    for (int64_t e = (int64_t)blockIdx.x * KV_COPY_THREADS + threadIdx.x; e < n_entries;
         e += (int64_t)gridDim.x * KV_COPY_THREADS) {
        const int t = table[e];
        int to = -1;
        if (t >= 0 && t < n_pages) {
            to = map[t];
            if (to < 0) paged_fault(PAGED_BAD_REFS);  // a page that nobody is counted to hold
        } else if (t != -1) {
            paged_fault(PAGED_BAD_PAGE);
        }
        table_out[e] = to;
    }
    constexpr int CHUNK = 4096;
    const int chunks = (int)((pool.page_bytes + CHUNK - 1) / CHUNK);
    const int per = pool.n_layers * 2 * chunks;
    const int64_t units = (int64_t)info[1] * per;
    const int64_t n_warps = (int64_t)gridDim.x * (KV_COPY_THREADS / 32);
    for (int64_t u = (int64_t)blockIdx.x * (KV_COPY_THREADS / 32) + (threadIdx.x >> 5); u < units;
         u += n_warps) {
        const int i = (int)(u / per);
        int r = (int)(u - (int64_t)i * per);
        const int c = r % chunks;
        r /= chunks;
        const int src = moves[2 * i], dst = moves[2 * i + 1];
        uint8_t* base = ((r & 1) ? pool.v : pool.k) + (int64_t)(r >> 1) * pool.layer_bytes +
                        (int64_t)c * CHUNK;
        const int64_t left = pool.page_bytes - (int64_t)c * CHUNK;
        warp_copy((uint4*)(base + dst * pool.page_bytes),
                  (const uint4*)(base + src * pool.page_bytes),
                  (int)(left < CHUNK ? left : CHUNK) / 16);
    }
}

// ---- append ----------------------------------------------------------------------------
// Sequence of batch row t: the last b with cu_q[b] <= t, found by a warp that tests 32
// places per step (two dependent loads up to 1024 sequences).  -1 behind the last sequence.
__device__ __forceinline__ int seq_of_token(const PagedView& w, int t) {
    int lo = 0, n = w.n_seqs;  // the answer is in [lo, lo + n)
    if (t >= w.cu_q[n] || t < w.cu_q[0]) return -1;
    const int lane = threadIdx.x & 31;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lane * step;
        const unsigned below =
            __ballot_sync(0xffffffffu, at < n && w.cu_q[lo + min(at, n - 1)] <= t);
        // the places tested are in order, so the set bits are a prefix
        const int k = below ? 31 - __clz(below) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// RoPE on q and k (interleaved pairs, the reference's table, src/ops/cuda_kernels.cu:372-400)
// and the write of k and v into the pages: one CTA per token, one thread per eight elements
// of a head.  Bound by HBM (every element read once and written once).  The page and its reference
// count are looked up first: with a thread's first elements loaded before them 64 single tokens took
// 4.33 us in a graph, 4.23 this way, a launch and its dependent loads; 6798 prompt tokens (32 heads
// on 8, head_dim 128, FP32) 57.3 and 57.7 us, 5.8 TB/s, 0.89 of the measured rate.
template <typename KV>
__global__ void __launch_bounds__(256)
    kv_append_kernel(const PagedView w, const float* q, int64_t q_stride,
                     const float* __restrict__ k, int64_t k_stride, const float* __restrict__ v,
                     int64_t v_stride, float* q_out, int64_t qo_stride,  // may be q
                     const float* __restrict__ rope, int rope_len, KV* kpool, KV* vpool) {
    const int t = blockIdx.x;
    const int b = seq_of_token(w, t);
    if (b < 0) return;
    const SeqInfo s = seq_info(w, b);
    const int pos = s.L - s.n + (t - s.q0);
    if (t < s.q0 || t >= s.q0 + s.n || pos < 0) return;  // no position: nothing to do
    if (pos >= rope_len) {
        if (threadIdx.x == 0) paged_fault(PAGED_BAD_ROPE);
        return;
    }
    const int col = (int)w.ps.div((uint32_t)pos), slot = pos - col * w.page_size;
    const int page = page_at(w, s.row[col]);
    // a page that others hold too is not written: it would change what they have stored
    const bool own = page >= 0 && w.refs[page] <= 1;
    if (page >= 0 && !own && threadIdx.x == 0) paged_fault(PAGED_SHARED);
    const int per = w.HD / 8;
    const int total = (w.H + 2 * w.Hkv) * per;
    for (int e = threadIdx.x; e < total; e += blockDim.x) {
        int h = e / per;
        const int d = (e - h * per) * 8;
        const bool is_q = h < w.H, is_v = h >= w.H + w.Hkv;
        h -= is_q ? 0 : is_v ? w.H + w.Hkv : w.H;
        const float* src = is_q ? q + t * q_stride : is_v ? v + t * v_stride : k + t * k_stride;
        const float4* p = reinterpret_cast<const float4*>(src + (int64_t)h * w.HD + d);
        float4 x[2] = {p[0], p[1]};
        if (!is_v) {
            const float4* r = reinterpret_cast<const float4*>(rope + (int64_t)pos * w.HD + d);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 c = __ldg(r + i), y = x[i];
                x[i] = make_float4(y.x * c.x - y.y * c.y, y.x * c.y + y.y * c.x,
                                   y.z * c.z - y.w * c.w, y.z * c.w + y.w * c.z);
            }
        }
        if (is_q) {
            float4* o = reinterpret_cast<float4*>(q_out + t * qo_stride + (int64_t)h * w.HD + d);
            o[0] = x[0];
            o[1] = x[1];
        } else if (own) {
            KV* pool = is_v ? vpool : kpool;
            KV* o = pool + (((int64_t)page * w.Hkv + h) * w.page_size + slot) * w.HD + d;
            if constexpr (sizeof(KV) == 4) {
                reinterpret_cast<float4*>(o)[0] = x[0];
                reinterpret_cast<float4*>(o)[1] = x[1];
            } else {
                __half2 y[4] = {__floats2half2_rn(x[0].x, x[0].y), __floats2half2_rn(x[0].z, x[0].w),
                                __floats2half2_rn(x[1].x, x[1].y), __floats2half2_rn(x[1].z, x[1].w)};
                *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(y);
            }
        }
    }
}

// ---- launchers -------------------------------------------------------------------------
static KvSeqsDev seqs_dev(const ib_kv_pages* p, const ib_kv_seqs* s) {
    return KvSeqsDev{s->table, s->len, s->refs, s->n_slots, s->max_pages, p->n_pages, p->page_size};
}

static PoolBytes pool_bytes(const ib_kv_pages* p) {
    PoolBytes b;
    b.k = (uint8_t*)p->k;
    b.v = (uint8_t*)p->v;
    b.n_layers = p->n_layers;
    b.n_kv_heads = p->n_kv_heads;
    b.row_bytes = p->head_dim * elem_bytes(p);
    b.page_bytes = (int64_t)p->n_kv_heads * p->page_size * b.row_bytes;
    b.layer_bytes = b.page_bytes * p->n_pages;
    return b;
}

// kv_assign_kernel's arrays
constexpr size_t assign_smem(int n_slots, int n) {
    return ((size_t)(n_slots > n ? n_slots : n) + n + 1) * 4 + (size_t)n * 3;
}
constexpr int KV_ASSIGN_SMEM_MAX = (int)assign_smem(IB_KV_MAX_SLOTS, IB_KV_MAX_SLOTS);

template <bool FORK>
static int assign_launch(const KvSeqsDev& s, int n, const int32_t* a, const int32_t* b,
                         int32_t* status, cudaStream_t st) {
    const size_t sm = assign_smem(s.n_slots, n);
    static DeviceOnce once;
    IB_CUDA_CHECK(once.run([] {
        return cudaFuncSetAttribute(kv_assign_kernel<FORK>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    KV_ASSIGN_SMEM_MAX);
    }));
    kv_assign_kernel<FORK><<<1, KV_PLAN_THREADS, sm, st>>>(s, n, a, b, status);
    IB_LAUNCH_CHECK("kv_assign_kernel");
    return IB_OK;
}

}  // namespace ib

using namespace ib;

static int check_list(int n, const void* a, const char* who) {
    if (n < 0 || n > IB_KV_MAX_SLOTS) {
        set_error(std::string(who) + ": list length out of range");
        return IB_ERR_INVALID;
    }
    if (!a) {
        set_error(std::string(who) + ": null pointer argument");
        return IB_ERR_INVALID;
    }
    return IB_OK;
}

// the result (status, granted) is written while the lists are still being read
static int check_status(int n, const int32_t* a, const int32_t* b, const int32_t* status,
                        const char* who) {
    const int r = check_list(n, a && b ? status : nullptr, who);
    if (r != IB_OK) return r;
    for (const int32_t* list : {a, b})
        if ((uintptr_t)status < (uintptr_t)(list + n) && (uintptr_t)list < (uintptr_t)(status + n)) {
            set_error(std::string(who) + ": the result must not overlap the lists");
            return IB_ERR_INVALID;
        }
    return IB_OK;
}

extern "C" int ib_kv_extend(const ib_kv_pages* pages, const ib_kv_seqs* seqs, int n,
                            const int32_t* slots, const int32_t* n_new, int32_t* status,
                            void* stream) {
    int r = paged_check(pages, seqs, "ib_kv_extend");
    if (r != IB_OK || n == 0) return r;
    if ((r = check_status(n, slots, n_new, status, "ib_kv_extend")) != IB_OK) return r;
    return assign_launch<false>(seqs_dev(pages, seqs), n, slots, n_new, status, as_stream(stream));
}

extern "C" int ib_kv_fork(const ib_kv_pages* pages, const ib_kv_seqs* seqs, int n,
                          const int32_t* parents, const int32_t* children, int32_t* status,
                          void* stream) {
    int r = paged_check(pages, seqs, "ib_kv_fork");
    if (r != IB_OK || n == 0) return r;
    if ((r = check_status(n, parents, children, status, "ib_kv_fork")) != IB_OK) return r;
    const KvSeqsDev s = seqs_dev(pages, seqs);
    cudaStream_t st = as_stream(stream);
    if ((r = assign_launch<true>(s, n, parents, children, status, st)) != IB_OK) return r;
    int sms = 0;
    if ((r = sm_count(&sms)) != IB_OK) return r;
    const int64_t warps = (int64_t)n * pages->n_layers * 2 * pages->n_kv_heads;
    const int grid = (int)std::min<int64_t>(
        (int64_t)sms * 8, std::max<int64_t>(n, (warps + KV_COPY_THREADS / 32 - 1) / (KV_COPY_THREADS / 32)));
    IB_CUDA_CHECK(launch_pdl(kv_fork_kernel, dim3(grid), dim3(KV_COPY_THREADS), 0, st, true, s,
                             pool_bytes(pages), n, parents, children, (const int32_t*)status));
    return IB_OK;
}

extern "C" int ib_kv_granted(int n, const int32_t* slots, const int32_t* status, int32_t* granted,
                             void* stream) {
    if (n == 0) return IB_OK;
    const int r = check_status(n, granted == slots ? status : slots, status, granted, "ib_kv_granted");
    if (r != IB_OK) return r;
    kv_granted_kernel<<<(n + KV_COPY_THREADS - 1) / KV_COPY_THREADS, KV_COPY_THREADS, 0,
                        as_stream(stream)>>>(n, slots, status, granted);
    IB_LAUNCH_CHECK("kv_granted_kernel");
    return IB_OK;
}

extern "C" int ib_kv_release(const ib_kv_pages* pages, const ib_kv_seqs* seqs, int n,
                             const int32_t* slots, void* stream) {
    int r = paged_check(pages, seqs, "ib_kv_release");
    if (r != IB_OK || n == 0) return r;
    if ((r = check_list(n, slots, "ib_kv_release")) != IB_OK) return r;
    kv_release_kernel<<<n, KV_COPY_THREADS, 0, as_stream(stream)>>>(seqs_dev(pages, seqs), n, slots);
    IB_LAUNCH_CHECK("kv_release_kernel");
    return IB_OK;
}

extern "C" int ib_kv_compact(const ib_kv_pages* pages, const ib_kv_seqs* seqs, int32_t* table_out,
                             int32_t* refs_out, int32_t* map, int32_t* moves, int32_t* info,
                             void* stream) {
    int r = paged_check(pages, seqs, "ib_kv_compact");
    if (r != IB_OK) return r;
    IB_REQUIRE(table_out && refs_out && map && moves && info,
               "ib_kv_compact: null pointer argument");
    int sms = 0;
    if ((r = sm_count(&sms)) != IB_OK) return r;
    cudaStream_t st = as_stream(stream);
    kv_compact_plan_kernel<<<1, KV_PLAN_THREADS, 0, st>>>(seqs->refs, refs_out, pages->n_pages, map,
                                                          moves, info);
    IB_LAUNCH_CHECK("kv_compact_plan_kernel");
    IB_CUDA_CHECK(launch_pdl(kv_compact_kernel, dim3(sms * 8), dim3(KV_COPY_THREADS), 0, st, true,
                             (const int32_t*)seqs->table, table_out,
                             (int64_t)seqs->n_slots * seqs->max_pages, (int)pages->n_pages,
                             (const int32_t*)map, (const int32_t*)moves, (const int32_t*)info,
                             pool_bytes(pages)));
    return IB_OK;
}

extern "C" int ib_kv_append(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                            const ib_kv_batch* batch, int layer, int n_heads, const float* q,
                            int64_t q_stride, const float* k, int64_t k_stride, const float* v,
                            int64_t v_stride, float* q_out, int64_t q_out_stride,
                            const float* rope_table, int rope_len, void* stream) {
    int r = paged_check_batch(pages, seqs, batch, layer, n_heads, "ib_kv_append");
    if (r != IB_OK || batch->n_tokens == 0 || batch->n_seqs == 0) return r;
    IB_REQUIRE(q && k && v && q_out && rope_table && rope_len >= 0,
               "ib_kv_append: null pointer argument");
    IB_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out |
                 (uintptr_t)rope_table) & 15) == 0 &&
                   ((q_stride | k_stride | v_stride | q_out_stride) & 3) == 0,
               "ib_kv_append: q, k, v, q_out and the RoPE table must be 16-byte aligned, with row "
               "strides that are multiples of 4");
    const int64_t qw = (int64_t)n_heads * pages->head_dim;
    IB_REQUIRE(q_stride >= 0 && k_stride >= 0 && v_stride >= 0 && q_out_stride >= qw,
               "ib_kv_append: bad row strides");
    const int64_t kw = (int64_t)pages->n_kv_heads * pages->head_dim, n = batch->n_tokens;
    IB_REQUIRE(((q_out == q && q_out_stride == q_stride) ||
                !paged_rows_overlap(q_out, q_out_stride, qw, q, q_stride, qw, n)) &&
                   !paged_rows_overlap(q_out, q_out_stride, qw, k, k_stride, kw, n) &&
                   !paged_rows_overlap(q_out, q_out_stride, qw, v, v_stride, kw, n),
               "ib_kv_append: q_out may be q, with its row stride, and must not overlap it otherwise, "
               "nor k or v");
    const PagedView w = paged_view(pages, seqs, batch, n_heads);
    const int64_t layer_elems = pool_bytes(pages).layer_bytes / elem_bytes(pages);
    cudaStream_t st = as_stream(stream);
    if (pages->type == IB_TYPE_F32)
        kv_append_kernel<float><<<batch->n_tokens, 256, 0, st>>>(
            w, q, q_stride, k, k_stride, v, v_stride, q_out, q_out_stride, rope_table, rope_len,
            (float*)pages->k + layer * layer_elems, (float*)pages->v + layer * layer_elems);
    else
        kv_append_kernel<__half><<<batch->n_tokens, 256, 0, st>>>(
            w, q, q_stride, k, k_stride, v, v_stride, q_out, q_out_stride, rope_table, rope_len,
            (__half*)pages->k + layer * layer_elems, (__half*)pages->v + layer * layer_elems);
    IB_LAUNCH_CHECK("kv_append_kernel");
    return IB_OK;
}
