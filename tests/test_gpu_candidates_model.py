"""A model's layers over the paged cache, decoding from several candidates at once: trees of drafted
tokens (plan, append, attention, verification, accept) against the CPU oracle's greedy decoding, and a
beam search (selection, reorder) against the oracle's logits of every prefix.

Logits: within 1e-3 of the row's largest on FP32 pages and 5e-3 on FP16 pages, as in
test_gpu_paged_model.py.  A log probability is a difference of a logit and a log sum that is off by no more
than the largest logit error: a step's scores by twice that, and a beam's sum by twice that a step."""
import random

import numpy as np
import pytest

from conftest import load_package
from test_gpu_paged import i32
from test_gpu_paged_model import CFGS, Served, close

ib = load_package()
from inference_cpp_b200 import gguf_writer as gw  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("type_,rtol", [(ib.F32, 1e-3), (ib.F16, 5e-3)], ids=["f32", "f16"])
MODELS = pytest.mark.parametrize("cfg", CFGS, ids=lambda c: c.name)


class Candidates(Served):
    """The same model; the new tokens of a step are trees, and every node's logits come back."""

    def tree_step(self, work):
        """work: [(slot, tokens, parents)].  (batch, tokens, parents, logits of all nodes)."""
        cuda, cfg = self.cuda, self.cfg
        slots = i32(cuda, [s for s, _, _ in work])
        cu = [0]
        for _, ids, _ in work:
            cu.append(cu[-1] + len(ids))
        T, H, Hkv, HD = cu[-1], cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        ids = i32(cuda, [t for _, x, _ in work for t in x])
        parents = i32(cuda, [p for _, _, x in work for p in x])
        new = i32(cuda, [len(x) for _, x, _ in work])
        assert ib.kv_extend(self.pages, self.seqs, slots, new).tolist() == [1] * len(work)
        batch = ib.KVBatch(i32(cuda, cu), T, max_q=max(len(x) for _, x, _ in work), slots=slots)
        tree = ib.kv_tree(batch, parents)
        t, rows, cols, table = self.w["token_embd.weight"]
        x = ib.embedding_q(t, table, ids, cfg.vocab, cfg.dim).view(T, cfg.dim)
        ws = ib.attention_paged_workspace(self.pages, self.seqs, batch, H, tree=tree)
        for layer in range(cfg.n_layers):
            p = f"blk.{layer}."
            y = self.norm(x, p + "attn_norm.weight")
            q = self.linear(y, p + "attn_q.weight").view(T, H, HD)
            k = self.linear(y, p + "attn_k.weight").view(T, Hkv, HD)
            v = self.linear(y, p + "attn_v.weight").view(T, Hkv, HD)
            ib.kv_append(self.pages, self.seqs, batch, layer, q, k, v, self.rope, q_out=q, tree=tree)
            o = ib.attention_paged(self.pages, self.seqs, batch, layer, q, HD ** -0.5, workspace=ws, tree=tree)
            ib.add(x, self.linear(o.view(T, H * HD), p + "attn_output.weight"), x.numel())
            y = self.norm(x, p + "ffn_norm.weight")
            g, u = self.linear(y, p + "ffn_gate.weight"), self.linear(y, p + "ffn_up.weight")
            ib.silu(g, g.numel())
            ib.mul(g, u, g.numel())
            ib.add(x, self.linear(g, p + "ffn_down.weight"), x.numel())
        logits = self.linear(self.norm(x, "output_norm.weight"), "output.weight")
        return batch, ids, parents, logits


@TYPES
@MODELS
def test_drafted_trees_decode_as_the_greedy_oracle(cuda, port, cfg, type_, rtol):
    tensors = {n: (t, r, c, d) for n, t, r, c, d in gw.synth_tensors(cfg, 2024, ib.synth_host)}
    om = port.model(cfg, tensors)
    rng = random.Random(7)
    prompts = [np.random.default_rng(5).integers(0, cfg.vocab, n).tolist() for n in (8, 23, 1)]
    n_new = 16
    want = [om.generate(np.array(p, dtype=np.int32), n_new, want_logits=True) for p in prompts]
    text = [[int(t) for t in tokens] for tokens, _ in want]
    m = Candidates(cuda, cfg, tensors, type_, 5, 4, 60)
    slots, stored, taken = [3, 0, 2], [], 0
    out, st = m.step([(s, p[:-1]) for s, p in zip(slots, prompts) if len(p) > 1])
    assert st == [1] * 2
    stored = [len(p) - 1 for p in prompts]  # the next token's place
    while min(s - len(p) for s, p in zip(stored, prompts)) < n_new - 6:
        work = []
        for b, s in enumerate(slots):
            n = rng.choice([1, 4, 7, 12])
            parents = [-1] + [rng.randint(max(0, i - 4), i - 1) for i in range(1, n)]
            depth, tokens, right = [0], [text[b][stored[b]]], [True]
            for i in range(1, n):
                p = parents[i]
                depth.append(depth[p] + 1)
                at = stored[b] + depth[i]
                # the text's own token on some branches, and not twice behind one node
                good = right[p] and at < len(text[b]) and rng.random() < 0.6
                tokens.append(text[b][at] if good else rng.randrange(cfg.vocab))
                right.append(right[p] and at < len(text[b]) and tokens[-1] == text[b][at])
            work.append((s, tokens, parents))
        batch, ids, parents, logits = m.tree_step(work)
        best = ib.beam_select(logits, k=1).token.flatten()
        path, n_path, nxt = ib.kv_tree_verify(batch, parents, ids, best)
        ib.kv_tree_accept(m.pages, m.seqs, batch, path, n_path)
        rows, cu = logits.cpu().numpy(), batch.cu_q.tolist()
        for b in range(3):
            nodes = path[cu[b]:cu[b] + n_path[b].item()].tolist()
            assert nodes[0] == 0
            for j, c in enumerate(nodes):  # node c stands at place stored + j, its row is of the next one
                at = stored[b] + j
                assert work[b][1][c] == text[b][at]
                i = at + 1 - len(prompts[b])
                if 0 <= i < n_new:
                    assert close(rows[cu[b] + c], want[b][1][i], rtol), (b, at)
            stored[b] += len(nodes)
            taken += len(nodes) - 1
            if stored[b] < len(text[b]):
                assert nxt[b].item() == text[b][stored[b]]
            assert m.seqs.len[slots[b]].item() == stored[b]
            if stored[b] >= len(text[b]) - 1:
                return  # the oracle's text is used up
    assert taken > 3  # some drafts were right
    assert ib.check_fault() == 0


@TYPES
@MODELS
def test_beam_search_against_the_oracles_logits(cuda, port, cfg, type_, rtol):
    tensors = {n: (t, r, c, d) for n, t, r, c, d in gw.synth_tensors(cfg, 2024, ib.synth_host)}
    om = port.model(cfg, tensors)
    B, steps, end = 3, 6, 5
    prompts = [np.random.default_rng(6).integers(0, cfg.vocab, n).tolist() for n in (11, 6)]
    m = Candidates(cuda, cfg, tensors, type_, 7, 4, 60)
    slots = [6, 1, 3, 0, 4, 2]
    first = [slots[0], slots[3]]

    def ref_row(tokens):
        _, lg = om.generate(np.array(tokens, dtype=np.int32), 1, want_logits=True)
        x = np.array(lg[0], dtype=np.float64)
        return x - x.max() - np.log(np.exp(x - x.max()).sum()), np.abs(x).max()

    rows, st = m.step(list(zip(first, prompts)))
    assert st == [1, 1]
    # every group's other beams begin as copies without a score
    par = i32(cuda, [slots[0]] * 2 + [slots[3]] * 2)
    assert ib.kv_fork(m.pages, m.seqs, par, i32(cuda, [slots[i] for i in (1, 2, 4, 5)])).tolist() == [1] * 4
    logits = cuda.from_numpy(rows).cuda().repeat_interleave(B, 0)
    scores = cuda.tensor([0.0, -np.inf, -np.inf] * 2, dtype=cuda.float32, device="cuda")
    text = [list(p) for p in prompts for _ in range(B)]
    total, off = [0.0] * 6, 0.0
    dslots = i32(cuda, slots)
    for step in range(steps):
        choice = ib.beam_select(logits, scores, beams=B)
        status = ib.kv_reorder(m.pages, m.seqs, dslots, choice.row.flatten())
        assert status.tolist() == [1] * 6
        token, row = choice.token.flatten().tolist(), choice.row.flatten().tolist()
        tables = [ref_row(t) for t in text]
        off += 2 * rtol * max(t[1] for t in tables) + 1e-6
        for g in range(2):
            alive = range(g * B, g * B + (1 if step == 0 else B))
            best = np.sort(np.concatenate([total[r] + tables[r][0] for r in alive]))[::-1][:B]
            mine = [total[r] + tables[r][0][t] for t, r in zip(token[g * B:g * B + B], row[g * B:g * B + B])]
            got = choice.score[g].cpu().numpy()
            assert np.all(np.abs(got - np.array(mine)) <= off), (step, g)
            assert np.all(np.abs(np.array(mine) - best) <= 2 * off), (step, g)
        total = [total[r] + tables[r][0][t] for t, r in zip(token, row)]
        text = [text[r] + [t] for t, r in zip(token, row)]
        scores = choice.score.flatten().clone()
        out, st = m.step([(s, [t]) for s, t in zip(slots, token)])
        assert st == [1] * 6
        logits = cuda.from_numpy(out).cuda()
    assert m.seqs.len.tolist()[5] == 0
    assert [m.seqs.len[s].item() for s in slots] == [len(t) for t in text]
    # ended beams keep their score and take no others
    ended = i32(cuda, [1, 0, 0, 1, 1, 1])
    choice = ib.beam_select(logits, scores, beams=B, ended=ended, end_token=end)
    assert sorted(choice.score[1].tolist()) == sorted(scores[3:].tolist()) and choice.token[1].tolist() == [end] * 3
    assert ib.check_fault() == 0
