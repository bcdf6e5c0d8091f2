// Trees of drafted tokens over the paged cache: what the tree's shape means for attention and RoPE
// (ib_kv_tree_plan), which path through it the model confirms (ib_kv_tree_verify), and the cache with
// that path alone (ib_kv_tree_accept).  No counterpart in the reference, which decodes one token at a
// time (src/models/model_cuda.cpp:372-407).
//
// A sequence's n new tokens are nodes 0 .. n - 1; node i is stored at position L - n + i and stands
// at L - n + depth(i) of the text, behind its ancestors: depth(i) = number of ancestors in the tree.
#include <string>

#include "common.cuh"
#include "paged.cuh"
#include "pdl.cuh"

namespace ib {

int paged_tree_fault_take(int* code) { return paged_fault_take_here(code); }

constexpr int TREE_THREADS = 128;

// ---- plan --------------------------------------------------------------------------------
// One CTA per sequence, a thread per node that goes up to the root: parents come before their
// children, so a row's words are met from the last to the first.  A chain of reads of shared memory,
// as long as the tree is deep; what bounds a step's one call is its launch: 6 us with cold caches for 64
// trees of 16 to 64 nodes.  The append behind it starts beside it.
__global__ void __launch_bounds__(TREE_THREADS)
    tree_plan_kernel(const int32_t* __restrict__ cu_q, const int32_t* __restrict__ slots, int n_tokens,
                     const int32_t* __restrict__ parents, int max_nodes, int32_t* __restrict__ depth,
                     uint32_t* __restrict__ mask) {
    __shared__ int16_t up[IB_KV_MAX_NODES];
    pdl_launch_dependents();
    int q0;
    const int n = tree_nodes(cu_q, slots, n_tokens, blockIdx.x, max_nodes, q0);
    for (int i = threadIdx.x; i < n; i += TREE_THREADS) {
        int p = parents[q0 + i];
        if (p < -1 || p >= i) {
            paged_fault(PAGED_BAD_TREE);
            p = -1;
        }
        up[i] = (int16_t)p;
    }
    __syncthreads();
    const int words = (max_nodes + 31) / 32;
    for (int i = threadIdx.x; i < n; i += TREE_THREADS) {
        uint32_t* const row = mask + (size_t)(q0 + i) * words;
        int w = words - 1, d = 0;
        uint32_t bits = 0;
        for (int c = i; c >= 0; c = up[c], ++d) {
            for (; w > c >> 5; --w, bits = 0) row[w] = bits;
            bits |= 1u << (c & 31);
        }
        for (; w >= 0; --w, bits = 0) row[w] = bits;
        depth[q0 + i] = d - 1;
    }
}

// ---- verify ------------------------------------------------------------------------------
// Node 0 holds a token that is certain; from a confirmed node the path goes on to its first child
// whose token is what the model chose behind the node.  One warp per sequence over the nodes in order
// (a child comes after its parent, so the search only moves on): n / 32 steps and one for each node
// of the path.  Bound by its launch and those reads, 5 us with cold caches for 32 trees of 16 to 64 nodes.
__global__ void __launch_bounds__(32)
    tree_verify_kernel(const int32_t* __restrict__ cu_q, const int32_t* __restrict__ slots, int n_tokens,
                       int max_nodes, const int32_t* __restrict__ parents,
                       const int32_t* __restrict__ tokens, const int32_t* __restrict__ best,
                       int32_t* __restrict__ path, int32_t* __restrict__ n_path, int32_t* __restrict__ next) {
    const int lane = threadIdx.x;
    int q0;
    const int n = tree_nodes(cu_q, slots, n_tokens, blockIdx.x, max_nodes, q0);
    int at = n > 0 ? 0 : -1, m = 0, want = 0;
    pdl_launch_dependents();
    if (at == 0) {
        want = best[q0];
        if (lane == 0) path[q0] = 0;
        m = 1;
    }
    for (int c0 = 1; c0 < n; c0 += 32) {
        const int c = c0 + lane;
        const int p = c < n ? parents[q0 + c] : -2, t = c < n ? tokens[q0 + c] : 0;
        const int b = c < n ? best[q0 + c] : 0;
        for (;;) {
            const unsigned hit = __ballot_sync(0xffffffffu, c > at && p == at && t == want);
            if (!hit) break;
            const int j = __ffs(hit) - 1;
            at = c0 + j;
            want = __shfl_sync(0xffffffffu, b, j);
            if (lane == 0) path[q0 + m] = at;
            ++m;
        }
    }
    for (int i = m + lane; i < n; i += 32) path[q0 + i] = -1;
    if (lane == 0) {
        n_path[blockIdx.x] = m;
        next[blockIdx.x] = m ? want : -1;
    }
}

// ---- accept ------------------------------------------------------------------------------
// Two kernels: the moves, and what the sequences give back.  Whether others hold a page too is decided by
// the counts before the call, so no count changes before every sequence has its moves behind it (in
// one kernel a sequence that gave up a page could let another's move into it through for some layers
// and not for others).
//
// A path's nodes are in order, so entry j of it comes from a row at or behind its own place and rows can
// be moved in that order; a thread has 16 bytes of a row of one (layer, K or V, head) and takes them
// through all moves, a few loads in flight at a time, without waiting for others.  Bound by latency
// (length, path, table, reference count, row, one after the other): with the verification before it
// 11.2 us in a graph for 32 trees of 16 to 64 nodes through 32 layers (7.9 MB), 6.4 for one of 7 nodes, as
// in one kernel with a cluster's barrier (11.3, 6.5); the second launch is 2 us of the host.
constexpr int ACCEPT_THREADS = 512, ACCEPT_CTAS = 8, ACCEPT_BATCH = 4;

// What stays of sequence b: its first m new tokens' places; -1: it is left as it is.
struct Accepted {
    SeqInfo s;
    int slot, start, m;
};
__device__ __forceinline__ Accepted accepted(const PagedView& w, int max_nodes, const int32_t* n_path, int b,
                                             bool record) {
    Accepted a;
    a.s = seq_info(w, b);
    a.slot = w.slots ? w.slots[b] : b;
    a.start = a.s.L - a.s.n;
    a.m = n_path[b];
    // nothing to do: left out of the step, no new tokens, or a slot that is none
    const bool idle = a.s.n == 0 || a.slot < 0 || a.slot >= w.n_slots;
    const bool large = a.s.n > max_nodes;  // left out of the step: its K and V were never written
    if (idle || a.start < 0 || large || a.m < 0 || a.m > a.s.n) {
        if (!idle && record) paged_fault(a.start < 0 ? PAGED_BAD_LEN : PAGED_BAD_TREE);
        a.m = !idle && a.start >= 0 && large ? 0 : -1;
    }
    return a;
}
// Whether entry j of a path of n nodes is one behind the entry before.
__device__ __forceinline__ bool path_goes_on(const int32_t* path, int j, int n) {
    return path[j] > (j ? path[j - 1] : -1) && path[j] < n;
}

__global__ void __launch_bounds__(ACCEPT_THREADS)
    tree_move_kernel(const PagedView w, int max_nodes, const PoolBytes pool, const int32_t* __restrict__ path,
                     const int32_t* __restrict__ n_path) {
    __shared__ int from[IB_KV_MAX_NODES], to[IB_KV_MAX_NODES];  // rows of head 0 in a layer, -1: no move
    __shared__ int bad, first;
    const int b = blockIdx.x / ACCEPT_CTAS, part = blockIdx.x % ACCEPT_CTAS;
    const int tid = threadIdx.x;
    if (tid == 0) bad = first = IB_KV_MAX_NODES;
    pdl_wait();
    pdl_launch_dependents();
    const Accepted a = accepted(w, max_nodes, n_path, b, part == 0 && tid == 0);
    int m = a.m;
    __syncthreads();
    for (int j = tid; j < m; j += ACCEPT_THREADS) {
        if (!path_goes_on(path + a.s.q0, j, a.s.n)) {
            atomicMin(&bad, j);
            continue;
        }
        const int c = path[a.s.q0 + j];
        if (c != j) atomicMin(&first, j);
        auto row = [&](int pos, bool written) -> int {
            const int col = (int)w.ps.div((uint32_t)pos);
            const int page = page_at(w, a.s.row[col]);
            if (page >= 0 && written && w.refs[page] > 1) {
                paged_fault(PAGED_SHARED);  // others hold it too: not written
                return -1;
            }
            return page < 0 ? -1 : page * w.Hkv * w.page_size + (pos - col * w.page_size);
        };
        const int x = c == j ? -1 : row(a.start + c, false);
        const int z = c == j ? -1 : row(a.start + j, true);
        from[j] = z < 0 ? -1 : x;
        to[j] = z;
    }
    __syncthreads();
    if (m > bad) {  // the path ends before an entry that is none of it
        if (part == 0 && tid == 0) paged_fault(PAGED_BAD_TREE);
        m = bad;
    }
    const int per_row = pool.row_bytes / 16;
    const int per_layer = 2 * w.Hkv * per_row;
    const int64_t items = first < m ? (int64_t)pool.n_layers * per_layer : 0;
    for (int64_t i = (int64_t)part * ACCEPT_THREADS + tid; i < items; i += ACCEPT_CTAS * ACCEPT_THREADS) {
        const int layer = (int)(i / per_layer);
        int r = (int)(i - (int64_t)layer * per_layer);
        const int x = r % per_row;
        r /= per_row;
        const int head = r % w.Hkv;
        uint8_t* const base = (r >= w.Hkv ? pool.v : pool.k) + layer * pool.layer_bytes +
                              (int64_t)head * w.page_size * pool.row_bytes + x * 16;
        for (int j0 = first; j0 < m; j0 += ACCEPT_BATCH) {
            uint4 y[ACCEPT_BATCH];
#pragma unroll
            for (int k = 0; k < ACCEPT_BATCH; ++k)
                if (j0 + k < m && from[j0 + k] >= 0)
                    y[k] = *reinterpret_cast<const uint4*>(base + (int64_t)from[j0 + k] * pool.row_bytes);
#pragma unroll
            for (int k = 0; k < ACCEPT_BATCH; ++k)
                if (j0 + k < m && from[j0 + k] >= 0)
                    *reinterpret_cast<uint4*>(base + (int64_t)to[j0 + k] * pool.row_bytes) = y[k];
        }
    }
}

// Lengths, and the pages behind them given back: a CTA to a sequence.  It starts beside the moves, which
// change nothing that it reads, and waits for them before it changes what they read.
constexpr int GIVE_THREADS = 128;
__global__ void __launch_bounds__(GIVE_THREADS)
    tree_give_back_kernel(const PagedView w, int max_nodes, int32_t* table, int32_t* len, int32_t* refs,
                          const int32_t* __restrict__ path, const int32_t* __restrict__ n_path) {
    __shared__ int bad;
    const int b = blockIdx.x, tid = threadIdx.x;
    if (tid == 0) bad = IB_KV_MAX_NODES;
    const Accepted a = accepted(w, max_nodes, n_path, b, false);
    __syncthreads();
    for (int j = tid; j < a.m; j += GIVE_THREADS)
        if (!path_goes_on(path + a.s.q0, j, a.s.n)) atomicMin(&bad, j);
    __syncthreads();
    const int now = a.start + min(a.m, bad);
    const int keep = (now + w.page_size - 1) / w.page_size, used = (a.s.L + w.page_size - 1) / w.page_size;
    pdl_wait();
    if (a.m < 0) return;
    int32_t* const row = table + (size_t)a.slot * w.max_pages;
    for (int j = keep + tid; j < used; j += GIVE_THREADS) {
        const int t = row[j];
        row[j] = -1;
        if (t >= 0 && t < w.n_pages) {
            if (atomicSub(&refs[t], 1) <= 0) {  // held by nobody: leave it free
                atomicAdd(&refs[t], 1);
                paged_fault(PAGED_BAD_REFS);
            }
        } else if (t != -1) {
            paged_fault(PAGED_BAD_PAGE);
        }
    }
    if (tid == 0) len[a.slot] = now;
}

static int tree_batch(const ib_kv_batch* b, const char* who) {
    if (!b || !b->cu_q) return paged_refuse(who, "null pointer argument");
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_q < 0 || b->n_seqs > IB_KV_MAX_SLOTS ||
        b->n_tokens > (1 << 26))
        return paged_refuse(who, "bad batch sizes");
    return IB_OK;
}

// Whether [a, a + na) and [b, b + nb) of 32-bit values share any.
static bool meet(const void* a, int64_t na, const void* b, int64_t nb) {
    return bytes_meet(a, 4 * na, b, 4 * nb);
}

}  // namespace ib

using namespace ib;

extern "C" int ib_kv_tree_plan(const ib_kv_batch* batch, const int32_t* parents, int max_nodes,
                               int32_t* depth, uint32_t* mask, void* stream) {
    const char* who = "ib_kv_tree_plan";
    const int r = tree_batch(batch, who);
    if (r != IB_OK) return r;
    if (max_nodes < 1 || max_nodes > IB_KV_MAX_NODES)
        return paged_refuse(who, "max_nodes must be in [1, 1024]");
    const int64_t n = batch->n_tokens, nm = n * ((max_nodes + 31) / 32);
    if (n == 0 || batch->n_seqs == 0) return IB_OK;
    if (!parents || !depth || !mask) return paged_refuse(who, "null pointer argument");
    if (meet(depth, n, parents, n) || meet(mask, nm, parents, n) || meet(depth, n, mask, nm))
        return paged_refuse(who, "parents, depth and mask must not overlap");
    IB_CUDA_CHECK(launch_pdl(tree_plan_kernel, dim3(batch->n_seqs), dim3(TREE_THREADS), 0, as_stream(stream),
                             false, batch->cu_q, batch->slots, batch->n_tokens, parents, max_nodes, depth, mask));
    return IB_OK;
}

static int tree_verify(const ib_kv_batch* batch, int max_nodes, const int32_t* parents,
                       const int32_t* tokens, const int32_t* best, int32_t* path, int32_t* n_path,
                       int32_t* next, void* stream, const char* who) {
    const int r = tree_batch(batch, who);
    if (r != IB_OK) return r;
    if (max_nodes < 1 || max_nodes > IB_KV_MAX_NODES)
        return paged_refuse(who, "max_nodes must be in [1, 1024]");
    if (batch->n_seqs == 0) return IB_OK;
    // (lists of no nodes may be null)
    if ((batch->n_tokens && (!parents || !tokens || !best || !path)) || !n_path || !next)
        return paged_refuse(who, "null pointer argument");
    const int64_t T = batch->n_tokens, B = batch->n_seqs;
    const void* const out[3] = {path, n_path, next};
    const int64_t out_n[3] = {T, B, B};
    for (int i = 0; i < 3; ++i) {
        bool bad = meet(out[i], out_n[i], parents, T) || meet(out[i], out_n[i], tokens, T) ||
                   meet(out[i], out_n[i], best, T);
        for (int k = 0; k < i; ++k) bad = bad || meet(out[i], out_n[i], out[k], out_n[k]);
        if (bad) return paged_refuse(who, "the results must not overlap the lists or one another");
    }
    IB_CUDA_CHECK(launch_pdl(tree_verify_kernel, dim3(batch->n_seqs), dim3(32), 0, as_stream(stream), false,
                             batch->cu_q, batch->slots, batch->n_tokens, max_nodes, parents, tokens, best,
                             path, n_path, next));
    return IB_OK;
}

extern "C" int ib_kv_tree_verify(const ib_kv_batch* batch, const int32_t* parents, const int32_t* tokens,
                                 const int32_t* best, int32_t* path, int32_t* n_path, int32_t* next,
                                 void* stream) {
    return tree_verify(batch, IB_KV_MAX_NODES, parents, tokens, best, path, n_path, next, stream,
                       "ib_kv_tree_verify");
}

extern "C" int ib_kv_tree_verify_max(const ib_kv_batch* batch, int max_nodes, const int32_t* parents,
                                     const int32_t* tokens, const int32_t* best, int32_t* path,
                                     int32_t* n_path, int32_t* next, void* stream) {
    return tree_verify(batch, max_nodes, parents, tokens, best, path, n_path, next, stream,
                       "ib_kv_tree_verify_max");
}

static int tree_accept(const ib_kv_pages* pages, const ib_kv_seqs* seqs, const ib_kv_batch* batch,
                       int max_nodes, const int32_t* path, const int32_t* n_path, void* stream,
                       const char* who) {
    const int r = paged_check_batch(pages, seqs, batch, 0, pages ? pages->n_kv_heads : 0, who);
    if (r != IB_OK) return r;
    if (max_nodes < 1 || max_nodes > IB_KV_MAX_NODES)
        return paged_refuse(who, "max_nodes must be in [1, 1024]");
    if (batch->n_seqs == 0) return IB_OK;
    if ((batch->n_tokens && !path) || !n_path) return paged_refuse(who, "null pointer argument");
    const PagedView w = paged_view(pages, seqs, batch, pages->n_kv_heads);
    cudaStream_t st = as_stream(stream);
    IB_CUDA_CHECK(launch_pdl(tree_move_kernel, dim3(batch->n_seqs * ACCEPT_CTAS), dim3(ACCEPT_THREADS), 0, st,
                             true, w, max_nodes, pool_bytes(pages), path, n_path));
    IB_CUDA_CHECK(launch_pdl(tree_give_back_kernel, dim3(batch->n_seqs), dim3(GIVE_THREADS), 0, st, true, w,
                             max_nodes, seqs->table, seqs->len, seqs->refs, path, n_path));
    return IB_OK;
}

extern "C" int ib_kv_tree_accept(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                 const ib_kv_batch* batch, const int32_t* path, const int32_t* n_path,
                                 void* stream) {
    return tree_accept(pages, seqs, batch, IB_KV_MAX_NODES, path, n_path, stream, "ib_kv_tree_accept");
}

extern "C" int ib_kv_tree_accept_max(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                     const ib_kv_batch* batch, int max_nodes, const int32_t* path,
                                     const int32_t* n_path, void* stream) {
    return tree_accept(pages, seqs, batch, max_nodes, path, n_path, stream, "ib_kv_tree_accept_max");
}
