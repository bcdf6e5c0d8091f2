"""A whole model's layers over the paged KV cache: several sequences served at once with the
library's own operators (embedding, RMSNorm, quantized GEMM, kv_append, attention_paged, SwiGLU),
against the CPU oracle's forward pass of each sequence by itself.

Logits: within 1e-3 of the row's largest on FP32 pages, the bound that the model runner keeps
against the oracle, and 5e-3 on FP16 pages, the bound of its FP16 cache."""
import numpy as np
import pytest

from conftest import load_package

ib = load_package()
from inference_cpp_b200 import gguf_writer as gw  # noqa: E402

pytestmark = pytest.mark.gpu

CFGS = [
    gw.LlamaConfig("tiny-q4_0", 2, 64, 4, 2, 128, 256, 64, 10000.0, 1e-5, embed_type=ib.Q4_0,
                   linear_type=ib.Q4_0, attn_v_type=ib.Q5_1, ffn_down_type=ib.Q8_0,
                   output_type=ib.Q5_0),
    gw.LlamaConfig("tiny-k", 2, 256, 4, 1, 512, 300, 160, 500000.0, 1e-5, embed_type=ib.Q4_K,
                   linear_type=ib.Q4_K, attn_v_type=ib.Q6_K, ffn_down_type=ib.Q6_K,
                   output_type=ib.Q6_K, q6k_alternate=True),
]


class Served:
    """A model whose cache is a pool of pages."""

    def __init__(self, cuda, cfg, tensors, type_, n_slots, page, n_pages):
        self.cuda, self.cfg, self.n_slots = cuda, cfg, n_slots
        self.w = {n: (t, r, c, cuda.from_numpy(np.ascontiguousarray(d)).cuda())
                  for n, (t, r, c, d) in tensors.items()}
        self.pages = ib.KVPages.empty(cfg.n_layers, n_pages, cfg.n_kv_heads, page, cfg.head_dim, type_)
        self.seqs = ib.KVSeqs.empty(n_slots, -(-cfg.ctx // page), n_pages)
        HD = cfg.head_dim
        ang = np.arange(cfg.ctx)[:, None] / cfg.rope_theta ** (np.arange(HD // 2) * 2.0 / HD)[None]
        self.rope = cuda.from_numpy(np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)).cuda()

    def norm(self, x, name):
        y = self.cuda.empty_like(x)
        ib.rmsnorm(x, self.w[name][3], y, x.shape[0], self.cfg.dim, self.cfg.rms_eps)
        return y

    def linear(self, x, name):
        t, rows, cols, data = self.w[name]
        return ib.gemm_q(t, data, x, x.shape[0], rows, cols).view(x.shape[0], rows)

    def step(self, work):
        """work: [(slot, token ids)].  The logits of every sequence's last token, and status."""
        cuda, cfg = self.cuda, self.cfg
        i32 = lambda v: cuda.tensor(v, dtype=cuda.int32, device="cuda")  # noqa: E731
        slots = i32([s for s, _ in work])
        n_new = [len(ids) for _, ids in work]
        cu = [0]
        for n in n_new:
            cu.append(cu[-1] + n)
        T, H, Hkv, HD = cu[-1], cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        ids = i32([t for _, x in work for t in x])
        status = ib.kv_extend(self.pages, self.seqs, slots, i32(n_new))
        batch = ib.KVBatch(i32(cu), T, max_q=max(n_new),
                           slots=ib.kv_granted(self.pages, slots, status))
        t, rows, cols, table = self.w["token_embd.weight"]
        x = ib.embedding_q(t, table, ids, cfg.vocab, cfg.dim).view(T, cfg.dim)
        ws = ib.attention_paged_workspace(self.pages, self.seqs, batch, H)
        for layer in range(cfg.n_layers):
            p = f"blk.{layer}."
            y = self.norm(x, p + "attn_norm.weight")
            q = self.linear(y, p + "attn_q.weight").view(T, H, HD)
            k = self.linear(y, p + "attn_k.weight").view(T, Hkv, HD)
            v = self.linear(y, p + "attn_v.weight").view(T, Hkv, HD)
            ib.kv_append(self.pages, self.seqs, batch, layer, q, k, v, self.rope, q_out=q)
            o = ib.attention_paged(self.pages, self.seqs, batch, layer, q, HD ** -0.5, workspace=ws)
            ib.add(x, self.linear(o.view(T, H * HD), p + "attn_output.weight"), x.numel())
            y = self.norm(x, p + "ffn_norm.weight")
            g, u = self.linear(y, p + "ffn_gate.weight"), self.linear(y, p + "ffn_up.weight")
            ib.silu(g, g.numel())
            ib.mul(g, u, g.numel())
            ib.add(x, self.linear(g, p + "ffn_down.weight"), x.numel())
        last = x[[c - 1 for c in cu[1:]]].contiguous()
        logits = self.linear(self.norm(last, "output_norm.weight"), "output.weight")
        return logits.cpu().numpy(), status.tolist()


def close(got, want, rtol):
    return bool(np.all(np.abs(got - want) <= rtol * np.abs(want).max()))


@pytest.mark.parametrize("type_,rtol", [(ib.F32, 1e-3), (ib.F16, 5e-3)], ids=["f32", "f16"])
@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)
def test_a_model_served_from_pages(cuda, port, cfg, type_, rtol):
    tensors = {n: (t, r, c, d) for n, t, r, c, d in gw.synth_tensors(cfg, 2024, ib.synth_host)}
    om = port.model(cfg, tensors)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, cfg.vocab, n).tolist() for n in (8, 23, 1)]
    n_new = 12
    want = [om.generate(np.array(p, dtype=np.int32), n_new, want_logits=True) for p in prompts]
    m = Served(cuda, cfg, tensors, type_, 5, 4, 40)
    slots = [3, 0, 2]

    def check(b, i, row):  # the i-th new token of sequence b is chosen from this row
        tokens, logits = want[b]
        assert close(row, logits[i], rtol), (b, i)
        return int(tokens[len(prompts[b]) + i])

    # the long prompt in two chunks, the others beside it
    a, st = m.step([(slots[0], prompts[0]), (slots[1], prompts[1][:15])])
    b, st2 = m.step([(slots[1], prompts[1][15:]), (slots[2], prompts[2])])
    assert st == [1, 1] and st2 == [1, 1]
    nxt = [check(0, 0, a[0]), check(1, 0, b[0]), check(2, 0, b[1])]
    for i in range(1, 5):
        out, st = m.step([(s, [t]) for s, t in zip(slots, nxt)])
        assert st == [1, 1, 1]
        nxt = [check(j, i, out[j]) for j in range(3)]
    # a fork goes on as its parent; the parent leaves, and what is left moves together
    one = cuda.tensor([slots[1]], dtype=cuda.int32, device="cuda")
    child = cuda.tensor([4], dtype=cuda.int32, device="cuda")
    assert ib.kv_fork(m.pages, m.seqs, one, child).tolist() == [1]
    out, st = m.step([(s, [t]) for s, t in zip(slots + [4], nxt + [nxt[1]])])
    assert st == [1] * 4
    check(1, 5, out[3])
    nxt = [check(j, 5, out[j]) for j in range(3)]
    ib.kv_release(m.pages, m.seqs, one)
    ib.kv_compact(m.pages, m.seqs)
    slots[1] = 4
    for i in range(6, n_new):
        out, st = m.step([(s, [t]) for s, t in zip(slots, nxt)])
        assert st == [1, 1, 1]
        nxt = [check(j, i, out[j]) for j in range(3)]
    assert ib.check_fault() == 0
