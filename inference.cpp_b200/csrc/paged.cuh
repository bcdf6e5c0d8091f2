// The paged KV cache as kernels see it: the pool of pages, the sequences' tables and a
// batch of new tokens (ib_kv_pages, ib_kv_seqs, ib_kv_batch of ib_cuda.h), with the
// checks of what lies in device memory.  Table rows, lengths and cu_q are written by the
// caller's kernels, so the host cannot check them: every value is clamped or skipped here
// before it becomes an address, and a bad one is recorded for ib_check_fault.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"

namespace ib {

constexpr int kSMs = 148;  // of a B200: how a call's work is cut, and so its workspace, follow it

// Codes of the paged kernels' fault word.
enum {
    PAGED_BAD_SLOT = 71,   // a slot outside [0, n_slots)
    PAGED_BAD_PAGE = 72,   // a table entry outside [-1, n_pages)
    PAGED_BAD_LEN = 73,    // len or cu_q out of order or out of range
    PAGED_BAD_REFS = 74,   // a reference count that a release would take below zero
    PAGED_BAD_ROPE = 75,   // a position behind the end of the RoPE table
    PAGED_BAD_WAIT = 76,   // a pipeline wait expired
    PAGED_SHARED = 77,     // a new token in a page that others hold too
    PAGED_BAD_TREE = 78    // a node, parent, depth or accepted path that cannot be
};

// Unsigned division by a number that the host prepares (page sizes need not be powers of
// two): n / d = (n * m) >> 32 >> s for n < 2^31, with s = floor(log2 d) and
// m = ceil(2^(32 + s) / d).  m d exceeds 2^(32 + s) by less than d < 2^(s + 1), so n times
// the excess stays below 2^(32 + s) and the quotient is exact.  Powers of two, whose m would
// not fit 32 bits, are a plain shift (m = 0).
struct FastDiv {
    uint32_t d, m, s;
    __host__ static FastDiv make(uint32_t d) {
        FastDiv f{d, 0, 0};
        while ((1ull << (f.s + 1)) <= d) ++f.s;
        if (d & (d - 1)) f.m = (uint32_t)(((1ull << (32 + f.s)) + d - 1) / d);
        return f;
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
        if (m == 0) return n >> s;
        return (uint32_t)(((uint64_t)n * m) >> 32) >> s;
    }
};

// One layer of the pool plus the sequences and the batch: a kernel argument.
struct PagedView {
    const int32_t* table;
    const int32_t* len;
    const int32_t* refs;
    const int32_t* cu_q;
    const int32_t* slots;  // null: sequence b is slot b
    int n_slots, max_pages, n_pages;
    int n_seqs, n_tokens;
    int max_nodes;  // of a sequence's tree; 0: the new tokens are no trees
    int H, Hkv, HD, page_size;
    FastDiv ps;     // of page_size
    FastDiv group;  // of H / Hkv
};

// Each translation unit's kernels record their first fault here: of values in device memory, which
// were passed over, and of waits that ran out, after which results are missing.  One does not hide
// the other.
struct PagedFaults {
    int value, wait;
};
static __device__ PagedFaults g_paged_faults;

// New tokens [q0, q0 + n) of sequence b, L positions in all, table row `row`.
struct SeqInfo {
    int q0, n, L;
    const int32_t* row;
};

__device__ __forceinline__ void paged_fault(int code) { atomicCAS(&g_paged_faults.value, 0, code); }

__device__ __forceinline__ SeqInfo seq_info(const PagedView& w, int b) {
    SeqInfo s;
    const int a = w.cu_q[b], e = w.cu_q[b + 1];
    const int slot = w.slots ? w.slots[b] : b;
    s.q0 = min(max(a, 0), w.n_tokens);
    s.n = min(max(e, s.q0), w.n_tokens) - s.q0;
    if (s.q0 != a || s.q0 + s.n != e) paged_fault(PAGED_BAD_LEN);
    if (slot < 0 || slot >= w.n_slots) {
        if (slot == -1) s.n = 0;  // left out of the step: its rows are nobody's
        else paged_fault(PAGED_BAD_SLOT);
        s.L = 0;
        s.row = w.table;
        return s;
    }
    const int cap = w.max_pages * w.page_size;  // at most 2^28 (paged_check)
    const int L = w.len[slot];
    s.L = min(max(L, 0), cap);
    if (s.L != L) paged_fault(PAGED_BAD_LEN);
    s.row = w.table + (size_t)slot * w.max_pages;
    if (w.max_nodes && s.n > w.max_nodes) {  // a tree that the masks have no room for: left out
        paged_fault(PAGED_BAD_TREE);
        s.n = 0;
    }
    return s;
}

// Nodes [q0, q0 + n) of sequence b's tree, from the batch alone (at most `most`, else recorded and
// none); the same range as seq_info's.
__device__ __forceinline__ int tree_nodes(const int32_t* cu_q, const int32_t* slots, int n_tokens, int b,
                                          int most, int& q0) {
    const int a = cu_q[b], e = cu_q[b + 1];
    q0 = min(max(a, 0), n_tokens);
    const int n = min(max(e, q0), n_tokens) - q0;
    if (q0 != a || q0 + n != e) paged_fault(PAGED_BAD_LEN);
    if (slots && slots[b] == -1) return 0;  // its rows are nobody's
    if (n <= most) return n;
    paged_fault(PAGED_BAD_TREE);
    return 0;
}

// Page of table entry e, or -1 (nothing there; out of range is recorded too).
__device__ __forceinline__ int page_at(const PagedView& w, int e) {
    if (e >= 0 && e < w.n_pages) return e;
    if (e != -1) paged_fault(PAGED_BAD_PAGE);
    return -1;
}

// Runs a set-up once per device; a failure is returned and tried again by the next call.
struct DeviceOnce {
    std::atomic<uint64_t> done{0};  // a bit per device
    template <typename F>
    cudaError_t run(F f) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
        e = f();
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
        return e;
    }
};

// The code to report of two: an expired wait before any value, else the first.
static inline int paged_fault_worse(int a, int b) {
    return a == PAGED_BAD_WAIT || b == PAGED_BAD_WAIT ? (int)PAGED_BAD_WAIT : a ? a : b;
}

// Reads and clears this translation unit's record.
static inline int paged_fault_take_here(int* code) {
    PagedFaults v = {0, 0};
    const PagedFaults none = {0, 0};
    IB_CUDA_CHECK(cudaMemcpyFromSymbol(&v, g_paged_faults, sizeof(v)));
    if (v.value || v.wait) IB_CUDA_CHECK(cudaMemcpyToSymbol(g_paged_faults, &none, sizeof(v)));
    *code = paged_fault_worse(v.value, v.wait);
    return IB_OK;
}

// Host side (paged.cu): checks of the structs and the kernels' view of them.
int paged_check(const ib_kv_pages* p, const ib_kv_seqs* s, const char* who);
int paged_check_batch(const ib_kv_pages* p, const ib_kv_seqs* s, const ib_kv_batch* b, int layer,
                      int n_heads, const char* who);
int paged_check_tree(const ib_kv_batch* b, const ib_kv_tree* t, const char* who);
int paged_refuse(const char* who, const char* what);  // sets the error, returns IB_ERR_INVALID
// Whether any of n rows of wa floats, sa apart from a, shares a float with one of wb, sb apart from b
// (rows of different strides: whether their whole ranges meet).
bool paged_rows_overlap(const float* a, int64_t sa, int64_t wa, const float* b, int64_t sb, int64_t wb,
                        int64_t n);
// Whether [a, a + na) and [b, b + nb) share a byte.
static inline bool bytes_meet(const void* a, int64_t na, const void* b, int64_t nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}
PagedView paged_view(const ib_kv_pages* p, const ib_kv_seqs* s, const ib_kv_batch* b, int n_heads,
                     const ib_kv_tree* t = nullptr);
int paged_fault_take(int* code);            // paged.cu
int paged_attention_fault_take(int* code);  // paged_attention.cu
int paged_tree_fault_take(int* code);       // paged_tree.cu

// The pool as bytes: layer l, page p at l * layer_bytes + p * page_bytes.
struct PoolBytes {
    uint8_t *k, *v;
    int n_layers, n_kv_heads, row_bytes;  // row: head_dim elements
    int64_t page_bytes, layer_bytes;
};
PoolBytes pool_bytes(const ib_kv_pages* p);

}  // namespace ib
