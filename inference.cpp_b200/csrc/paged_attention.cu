// ib_attention_paged: causal GQA attention of a batch of new tokens over the paged cache.
#include <cuda_fp16.h>

#include <string>

#include "common.cuh"
#include "kv.cuh"
#include "paged.cuh"

namespace ib {

int paged_attention_fault_take(int* code) { return paged_fault_take_here(code); }

// One warp per (token, head): positions one after another, lanes share head_dim, running
// maximum and sum.
template <typename KV>
__global__ void __launch_bounds__(128)
    attn_paged_kernel(const PagedView w, const float* __restrict__ q, int64_t q_stride,
                      float* __restrict__ out, int64_t out_stride, const KV* __restrict__ kp,
                      const KV* __restrict__ vp, float scale) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int t = row / w.H, h = row % w.H;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < w.n_seqs; i += 128) seq_info(w, i);  // records bad values
    if (t >= w.n_tokens) return;
    int b = -1;
    for (int i = 0; i < w.n_seqs; ++i)
        if (t >= w.cu_q[i] && t < w.cu_q[i + 1]) b = i;
    if (b < 0) return;
    const SeqInfo s = seq_info(w, b);
    const int pos = s.L - s.n + (t - s.q0);
    float qv[8], acc[8] = {}, m = -INFINITY, l = 0.f;
    const int hk = h / (w.H / w.Hkv);
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        qv[i] = d < w.HD ? q[t * q_stride + (int64_t)h * w.HD + d] : 0.f;
    }
    for (int p = 0; p <= pos; ++p) {
        const int col = (int)w.ps.div((uint32_t)p);
        const int page = page_at(w, s.row[col]);
        if (page < 0) continue;
        const size_t base = (((size_t)page * w.Hkv + hk) * w.page_size + (p - col * w.page_size)) * w.HD;
        float x = 0.f;
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d < w.HD) x += qv[i] * kv_at(kp, base + d);
        }
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x *= scale;
        const float mn = fmaxf(m, x);
        const float c = expf(m - mn), e = expf(x - mn);
        l = l * c + e;
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d < w.HD) acc[i] = acc[i] * c + e * kv_at(vp, base + d);
        }
        m = mn;
    }
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < w.HD)
            out[t * out_stride + (int64_t)h * w.HD + d] = m == -INFINITY && l == 0.f ? 0.f : acc[i] / l;
    }
}

}  // namespace ib

using namespace ib;

extern "C" size_t ib_attention_paged_workspace(const ib_kv_pages* pages, const ib_kv_seqs* seqs,
                                               const ib_kv_batch* batch, int n_heads) {
    if (paged_check_batch(pages, seqs, batch, 0, n_heads, "ib_attention_paged_workspace") != IB_OK)
        return 0;
    return 256;
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
    IB_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0 &&
                   workspace_bytes >= ib_attention_paged_workspace(pages, seqs, batch, n_heads),
               "ib_attention_paged: workspace missing, too small or not 256-byte aligned");
    const PagedView w = paged_view(pages, seqs, batch, n_heads);
    const int64_t rows = (int64_t)batch->n_tokens * n_heads;
    const int64_t off = (int64_t)layer * pages->n_pages * pages->n_kv_heads * pages->page_size *
                        pages->head_dim;
    const dim3 grid((unsigned)((rows + 3) / 4));
    cudaStream_t st = as_stream(stream);
    if (pages->type == IB_TYPE_F32)
        attn_paged_kernel<float><<<grid, 128, 0, st>>>(w, q, q_stride, out, out_stride,
                                                       (const float*)pages->k + off,
                                                       (const float*)pages->v + off, scale);
    else
        attn_paged_kernel<__half><<<grid, 128, 0, st>>>(w, q, q_stride, out, out_stride,
                                                        (const __half*)pages->k + off,
                                                        (const __half*)pages->v + off, scale);
    IB_LAUNCH_CHECK("attn_paged_kernel");
    return IB_OK;
}
