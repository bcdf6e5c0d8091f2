"""Cases of the operators for decoding from several candidates over the paged KV cache: a tree of
drafted tokens (its plan and append, attention, verification and the keeping of the accepted
path) and beam search (selection over beams and vocabulary, reordering of the beams' states).

`own = False` computes the operators in elementary torch operations; `own = True` calls the
package.  A case is a dict of plain values; its ragged lengths, trees and page layout come from
its "shape" number, the values of its tensors from the seed given to prepare().

Layouts (both sides): pool k, v [layer][page][kv head][position in page][head_dim]; table
[slot][page of the sequence] of page numbers, -1 where there is none; len [slot]; refs [page],
zero for a free page.  A sequence's n new tokens are the last n of its len positions; in a tree
they are its nodes, each with a parent among the nodes before it, or -1: what follows the context.
depth [token]: ancestors of a node; mask [token][word]: bit c of word c / 32 where node c of the
same sequence is the node itself or one of its ancestors.
"""
import math
import random

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16}
_BYTES = {"f32": 4, "f16": 2}
_LAYER = 1  # the layer that attention and append work on, of two


def _package():
    """This repository's package (its directory name is not an identifier)."""
    import importlib.util
    import os
    import sys
    name = "inference_cpp_b200"
    if name not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        d = os.path.join(root, "inference.cpp_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
        mod.init(0)
    return sys.modules[name]


# ---- cases ---------------------------------------------------------------------------

def _tree(op, name, cache, heads, kv_heads, head_dim, page, seqs, nodes, kv, shape, pad=0, evicted=0,
          roots=1, reach=6, layers=2, tokens=0):
    """seqs sequences with a tree of nodes[0] .. nodes[1] nodes each, behind kv positions; a node's
    parent is among the `reach` before it; `roots` nodes follow the context; pad rows behind the
    last sequence; `evicted` pages behind each sequence's first one given back; tokens: how many
    different ones the drafts are made of (verification)."""
    return {"name": name, "op": op, "cache": cache, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "seqs": seqs, "n_min": nodes[0], "n_max": nodes[1],
            "kv_min": kv[0], "kv_max": kv[1], "shape": shape, "pad": pad, "evicted": evicted,
            "roots": roots, "reach": reach, "layers": layers, "tokens": tokens}


def _beam(name, logits, groups, beams, vocab, k, shape, banned=0.0, ended=0.0, stride=0):
    """banned: share of the vocabulary that a mask forbids (-inf); ended: share of the beams that
    have ended; stride: elements between rows (0: vocab)."""
    return {"name": name, "op": "beam", "logits": logits, "groups": groups, "beams": beams,
            "vocab": vocab, "k": k, "shape": shape, "banned": banned, "ended": ended,
            "stride": stride or vocab}


def _reorder(name, cache, layers, kv_heads, head_dim, page, groups, beams, kv, new, shape):
    """groups prompts of kv positions, `beams` beams on each that have gone on by `new` tokens."""
    return {"name": name, "op": "reorder", "cache": cache, "layers": layers, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "groups": groups, "beams": beams, "kv_min": kv[0],
            "kv_max": kv[1], "new": new, "shape": shape}


def listed():
    return [
        # one short story, seven drafted tokens looked at in one step: latency alone
        _tree("attention", "tree-short-f32", "f32", 6, 6, 48, 16, 1, (7, 7), (130, 130), 1, reach=3),
        # a busy server's verification step (32 heads on 8), contexts of every length
        _tree("attention", "tree-batch-f16", "f16", 32, 8, 128, 16, 32, (12, 24), (200, 4096), 2, pad=5),
        # large trees behind two long documents on the FP32 cache (32 heads on 4)
        _tree("attention", "tree-long-f32", "f32", 32, 4, 64, 64, 2, (33, 63), (20001, 32000), 3,
              evicted=7),
        # the step's first layer: the trees' plan, and the nodes' K and V at their depths
        _tree("append", "tree-append-short-f32", "f32", 6, 6, 48, 16, 1, (7, 7), (130, 130), 4, reach=3),
        _tree("append", "tree-append-batch-f16", "f16", 32, 8, 128, 16, 64, (16, 64), (200, 4096), 5,
              pad=9, reach=9),
        # what the model confirms of a tree stays in the cache, the rest goes
        _tree("accept", "accept-short-f32", "f32", 6, 6, 48, 16, 1, (7, 7), (130, 130), 6, layers=6,
              reach=3, tokens=2),
        _tree("accept", "accept-batch-f16", "f16", 32, 8, 128, 16, 32, (16, 64), (200, 2000), 7,
              layers=32, reach=9, tokens=3),
        # four beams of a small vocabulary: latency alone
        _beam("beam-few-f32", "f32", 1, 4, 32000, 4, 8),
        # a batch of eight beams each over a large vocabulary
        _beam("beam-batch-f32", "f32", 16, 8, 128256, 8, 9, banned=0.02, ended=0.06),
        # the ten likeliest continuations of each row: what a tree is drafted from
        _beam("rows-top-f16", "f16", 192, 1, 32003, 10, 10, stride=32016),
        # four beams on one prompt
        _reorder("reorder-few-f32", "f32", 4, 8, 128, 16, 1, 4, (333, 333), 9, 11),
        # sixteen prompts with eight beams each on a full server
        _reorder("reorder-batch-f16", "f16", 22, 4, 64, 64, 16, 8, (100, 2000), 40, 12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "accept", "beam", "beam",
                     "reorder"])
    cache = rng.choice(["f16", "f32"])
    shape = rng.randrange(1000, 1 << 30)
    if op == "beam":
        groups = _log_int(rng, 1, 256)
        beams = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
        vocab = _log_int(rng, 200, 152000)
        while groups * beams * vocab > 16 * 8 * 128256:
            groups, vocab = max(1, groups // 2), max(200, vocab - vocab // 5)
        k = rng.choice([1, beams, 2 * beams, rng.randrange(1, 41)])
        return _beam("", cache, groups, beams, vocab, k, shape, rng.choice([0.0, 0.3, 0.98]),
                     rng.choice([0.0, 0.2]), vocab + rng.choice([0, 0, rng.randrange(1, 70)]))
    kv_heads = rng.choice([1, 2, 4, 6, 8])
    head_dim = rng.choice([48, 64, 80, 96, 128, 128, 128])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    if op == "reorder":
        layers = _log_int(rng, 1, 32)
        groups, beams = _log_int(rng, 1, 24), rng.choice([2, 3, 4, 5, 8, 16])
        new = _log_int(rng, 1, 200)
        position = 2 * layers * kv_heads * head_dim * _BYTES[cache]
        top = max(2, min(2000, int(1.5e9 // position) // groups - beams * (new + 2 * page)))
        while groups * beams * (new + 2 * page) * position > 1.5e9 and (groups > 1 or beams > 2):
            groups, beams = max(1, groups // 2), max(2, beams - 1)
        return _reorder("", cache, layers, kv_heads, head_dim, page, groups, beams,
                        (max(1, top // _log_int(rng, 1, 20)), top), new, shape)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    seqs = _log_int(rng, 1, 64)
    n_max = _log_int(rng, 2, 128)
    n_min = rng.choice([1, max(1, n_max // 2), n_max])
    size = _BYTES[cache]
    top = _log_int(rng, 16, 32000)  # longest context
    layers = _log_int(rng, 2, 32) if op == "accept" else 2
    # what the listed cases cost at most: K and V of 270 MB in a layer, 2e10 operations
    per = 2 * layers * kv_heads * head_dim * size
    while seqs * (top + n_max + page) * per > (1.5e9 if op == "accept" else 5e8):
        seqs, top = max(1, seqs - seqs // 4), max(16, top - top // 4)
    while op == "attention" and 4.0 * head_dim * heads * seqs * n_max * top > 2e10 and n_max > 1:
        n_max = max(1, n_max // 2)
    n_min = min(n_min, n_max)
    low = _log_int(rng, 1, top)
    pad = rng.choice([0, 0, rng.randrange(1, 40)])
    evicted = rng.choice([0, 0, 0, rng.randrange(1, 30)]) if op == "attention" else 0
    return _tree(op, "", cache, heads, kv_heads, head_dim, page, seqs, (n_min, n_max), (low, top),
                 shape, pad, evicted, rng.choice([1, 1, 3]) if op != "accept" else 1,
                 _log_int(rng, 1, 20), layers, rng.choice([1, 2, 3, 8]) if op == "accept" else 0)


# ---- layouts from a case alone -------------------------------------------------------

def _tree_layout(case):
    """Nodes, contexts, parents of every node, table rows and the number of pages of the pool."""
    rng = random.Random(case["shape"])
    n = case["seqs"]
    ctx = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(n)]
    nodes = [rng.randint(case["n_min"], case["n_max"]) for _ in range(n)]
    parents = [[-1 if i < case["roots"] else rng.randint(max(0, i - case["reach"]), i - 1)
                for i in range(k)] for k in nodes]
    page = case["page"]
    per = [-(-(c + k) // page) for c, k in zip(ctx, nodes)]
    pages = sum(per) + 7
    free = list(range(pages))
    rng.shuffle(free)
    rows, at = [], 0
    for b in range(n):
        row = free[at:at + per[b]]
        at += per[b]
        # pages 1 .. evicted were given back; those of the nodes and the two before are kept
        for j in range(1, min(1 + case["evicted"], ctx[b] // page - 2)):
            row[j] = -1
        rows.append(row)
    return nodes, ctx, parents, rows, pages


def _ancestors(parents):
    """Bit c of entry i: node c is i or one of its ancestors."""
    m = []
    for i, p in enumerate(parents):
        m.append((1 << i) | (m[p] if p >= 0 else 0))
    return m


def _drafts(case, nodes):
    """Drafted tokens, and what the model has chosen behind each node."""
    rng = random.Random(case["shape"] + 2)
    make = lambda: [[rng.randrange(case["tokens"]) for _ in range(k)] for k in nodes]  # noqa: E731
    return make(), make()


def _path(parents, tokens, best):
    path = [0]
    for c in range(1, len(parents)):  # parents come before their children, the first match counts
        if parents[c] == path[-1] and tokens[c] == best[path[-1]]:
            path.append(c)
    return path


def _reorder_layout(case):
    """Table rows, lengths and reference counts of the beams, and their parents (entries of the
    same list)."""
    rng = random.Random(case["shape"])
    page, beams = case["page"], case["beams"]
    lens, rows, parents, at = [], [], [], 0
    plan = []
    for g in range(case["groups"]):
        prompt = rng.randint(case["kv_min"], case["kv_max"])
        total = prompt + case["new"]
        shared = prompt // page  # whole pages of the prompt are one for all beams
        head = list(range(at, at + shared))
        at += shared
        for b in range(beams):
            more = -(-total // page) - shared
            plan.append((head, list(range(at, at + more))))
            at += more
            lens.append(total)
            # the likelier beams have more children
            parents.append(g * beams + min(int(rng.expovariate(2.5 / beams)), beams - 1))
    pages = at + 5
    names = list(range(pages))
    rng.shuffle(names)
    refs = [0] * pages
    for head, tail in plan:
        row = [names[x] for x in head + tail]
        rows.append(row)
        for x in row:
            refs[x] += 1
    return lens, rows, refs, parents, pages


def work(case):
    op = case["op"]
    if op == "beam":
        rows = case["groups"] * case["beams"]
        n = rows * case["vocab"]
        return {"bytes": n * _BYTES[case["logits"]] + 8 * rows + 12 * case["groups"] * case["k"],
                "flops": 3 * n}
    size = _BYTES[case["cache"]]
    if op == "reorder":
        lens, rows, _, parents, _ = _reorder_layout(case)
        # every parent's partial page goes to one child as it is
        copies = len(parents) - len(set(parents))
        part = sum(lens[p] % case["page"] for p in parents) / len(parents) * copies
        per_pos = 2 * case["layers"] * case["kv_heads"] * case["head_dim"] * size
        return {"bytes": int(2 * part * per_pos) + 8 * sum(map(len, rows)), "flops": 0}
    nodes, ctx, parents, rows, _ = _tree_layout(case)
    H, Hkv, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    tokens, words = sum(nodes), -(-case["n_max"] // 32)
    if op == "append":
        return {"bytes": tokens * (D * (8 * H + Hkv * 2 * (4 + size)) + 4 * D + 8 + 4 * words),
                "flops": 3 * tokens * D * (H + Hkv)}
    if op == "accept":
        drafts, best = _drafts(case, nodes)
        moved = sum(sum(1 for j, c in enumerate(_path(p, t, b)) if c != j)
                    for p, t, b in zip(parents, drafts, best))
        return {"bytes": 4 * case["layers"] * Hkv * D * size * moved + 12 * tokens, "flops": 0}
    bytes_, pairs = tokens * (8 * H * D + 4 * words), 0
    for n, c, p, row in zip(nodes, ctx, parents, rows):
        there = c - sum(1 for x in row if x < 0) * page
        bytes_ += 2 * size * Hkv * D * (there + n) + 4 * len(row)
        pairs += n * there + sum(bin(m).count("1") for m in _ancestors(p))
    return {"bytes": bytes_, "flops": 4 * D * H * pairs}


# ---- inputs --------------------------------------------------------------------------

def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _table(rows, slots, width, device):
    t = torch.full((slots, width), -1, dtype=torch.int32)
    for i, row in enumerate(rows):
        t[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
    return t.to(device)


def _books(s, table, lens, refs):
    """table, len and refs as parts of one tensor, and a copy of it."""
    parts = [table.flatten(), lens, refs]
    at = [0]
    for x in parts:
        at.append(at[-1] + -(-x.numel() // 64) * 64)
    s["books"] = torch.zeros(at[-1], dtype=torch.int32, device=table.device)
    for x, a in zip(parts, at):
        s["books"][a:a + x.numel()] = x
    s["table"] = s["books"][:table.numel()].view(table.shape)
    s["len"] = s["books"][at[1]:at[1] + lens.numel()]
    s["refs"] = s["books"][at[2]:at[2] + refs.numel()]
    s["books_before"] = s["books"].clone()


def _inputs(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "beam":
        rows, V = case["groups"] * case["beams"], case["vocab"]
        x = 2.5 * torch.randn(rows, case["stride"], generator=gen, device=dev)
        if case["banned"]:
            ban = torch.rand(V, generator=gen, device=dev) < case["banned"]
            x[:, :V].masked_fill_(ban, float("-inf"))
            x[:, ::97] = torch.finfo(_DTYPE[case["logits"]]).min  # and as other masks write it
        s["logits"] = x.to(_DTYPE[case["logits"]])[:, :V]
        u = torch.rand(rows, generator=gen, device=dev)
        s["scores"] = torch.where(u < 0.02, float("-inf"), -25 * u) if case["beams"] > 1 else -25 * u
        end = torch.rand(rows, generator=gen, device=dev) < case["ended"]
        s["ended"] = end.int() if case["ended"] else None
        return s
    dt, Hkv, D, page = _DTYPE[case["cache"]], case["kv_heads"], case["head_dim"], case["page"]

    def pool(pages):
        shape = (case["layers"], pages, Hkv, page, D)
        return [torch.randn(shape, generator=gen, device=dev, dtype=dt) for _ in range(2)]

    if case["op"] == "reorder":
        lens, rows, refs, parents, pages = _reorder_layout(case)
        s["k"], s["v"] = pool(pages)
        order = list(range(len(rows)))  # the slots of the list's entries
        random.Random(case["shape"] + 1).shuffle(order)
        by_slot, by_len = [None] * len(rows), [0] * len(rows)
        for i, slot in enumerate(order):
            by_slot[slot], by_len[slot] = rows[i], lens[i]
        s["table"] = _table(by_slot, len(rows), max(map(len, rows)) + 1, dev)
        s["len"], s["refs"] = _int32(by_len, dev), _int32(refs, dev)
        s["slots"], s["parents"] = _int32(order, dev), _int32(parents, dev)
        return s
    nodes, ctx, parents, rows, pages = _tree_layout(case)
    n = case["seqs"]
    order = list(range(n + 3))  # the batch's rows of the table, among slots not in the batch
    random.Random(case["shape"] + 1).shuffle(order)
    order = order[:n]
    by_slot, lens = [[] for _ in range(n + 3)], [0] * (n + 3)
    for b, slot in enumerate(order):
        by_slot[slot], lens[slot] = rows[b], ctx[b] + nodes[b]
    cu = [0]
    for x in nodes:
        cu.append(cu[-1] + x)
    tokens, words = cu[-1] + case["pad"], -(-case["n_max"] // 32)
    s.update(nodes=nodes, ctx=ctx, order=order, cu=cu, tokens=tokens, words=words)
    s["k"], s["v"] = pool(pages)
    refs = [0] * pages
    for row in rows:
        for x in row:
            if x >= 0:
                refs[x] += 1
    _books(s, _table(by_slot, n + 3, max(map(len, rows)) + 1, dev), _int32(lens, dev),
           _int32(refs, dev))
    s["cu_q"], s["slots"] = _int32(cu, dev), _int32(order, dev)
    flat = [x for p in parents for x in p] + [-1] * case["pad"]
    s["parent"] = _int32(flat, dev)
    s["depth"] = torch.zeros(tokens, dtype=torch.int32, device=dev)
    s["mask"] = torch.zeros(tokens, words, dtype=torch.int32, device=dev)
    if case["op"] == "attention":
        sets = [m for p in parents for m in _ancestors(p)]
        s["depth"][:cu[-1]] = _int32([bin(m).count("1") - 1 for m in sets], dev)
        s["mask"][:cu[-1]] = torch.tensor([[(m >> (32 * w)) & 0xffffffff for w in range(words)] for m in sets],
                                          dtype=torch.int64).to(dev).to(torch.int32)
        s["q"] = 1.5 * torch.randn(tokens, case["heads"], D, generator=gen, device=dev)
        s["out"] = torch.zeros(tokens, case["heads"], D, device=dev)
        s["scale"] = 1.0 / math.sqrt(D)
    elif case["op"] == "append":
        # the projections' output: q, k and v of a token next to each other
        s["qkv"] = torch.randn(tokens, case["heads"] + 2 * Hkv, D, generator=gen, device=dev)
        s["out"] = torch.zeros(tokens, case["heads"], D, device=dev)
        pos = torch.arange(max(lens), dtype=torch.float64, device=dev)
        freq = 500000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device=dev) * 2 / D)
        ang = pos[:, None] * freq[None, :]
        s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    else:
        drafts, best = _drafts(case, nodes)
        s["draft"] = _int32([x for t in drafts for x in t] + [0] * case["pad"], dev)
        s["best"] = _int32([x for t in best for x in t] + [0] * case["pad"], dev)
        s["path"] = torch.full((tokens,), -1, dtype=torch.int32, device=dev)
        s["n_path"], s["next"] = (torch.zeros(n, dtype=torch.int32, device=dev) for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the handles, workspace and output buffers that a serving program keeps
        ib = _package()
        if case["op"] == "beam":
            dev, shape = s["logits"].device, (case["groups"], case["k"])
            s["out"] = ib.BeamChoice(torch.empty(shape, device=dev),
                                     torch.empty(shape, dtype=torch.int32, device=dev),
                                     torch.empty(shape, dtype=torch.int32, device=dev))
            s["workspace"] = ib.beam_select_workspace(s["logits"], case["beams"], case["k"])
            return s
        s["pages"] = ib.KVPages(s["k"], s["v"])
        s["seqs"] = ib.KVSeqs(s["table"], s["len"], s["refs"])
        if case["op"] == "reorder":
            s["status"] = torch.empty_like(s["slots"])
            s["workspace"] = ib.kv_reorder_workspace(s["seqs"], s["slots"].numel())
            return s
        s["batch"] = ib.KVBatch(s["cu_q"], s["tokens"], max_q=case["n_max"], slots=s["slots"])
        s["tree"] = ib.KVTree(s["parent"], s["depth"], s["mask"], case["n_max"])
        if case["op"] == "attention":
            s["workspace"] = ib.attention_paged_workspace(s["pages"], s["seqs"], s["batch"],
                                                          case["heads"], tree=s["tree"])
        elif case["op"] == "append":
            s["q"], s["kn"], s["vn"] = s["qkv"].split([case["heads"], case["kv_heads"],
                                                       case["kv_heads"]], dim=1)
    return s


# ---- one pass ------------------------------------------------------------------------

def run(s):
    return {"attention": _run_attention, "append": _run_append, "accept": _run_accept,
            "beam": _run_beam, "reorder": _run_reorder}[s["case"]["op"]](s)


def _batched(s, x, fill=0):
    """Rows of the batch's tokens as [sequence][node][...]."""
    n_max = s["case"]["n_max"]
    at = s["cu_q"][:-1, None].long() + torch.arange(n_max, device=x.device)
    there = at < s["cu_q"][1:, None]
    y = x[at.clamp(max=x.shape[0] - 1)]
    return torch.where(there.view(there.shape + (1,) * (x.dim() - 1)), y, torch.full_like(y, fill)), there, at


def _run_attention(s):
    if own:
        _package().attention_paged(s["pages"], s["seqs"], s["batch"], _LAYER, s["q"], s["scale"],
                                   out=s["out"], workspace=s["workspace"], tree=s["tree"])
        return s["out"]
    case = s["case"]
    H, Hkv, D, page, n = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["n_max"]
    G, B, dev = H // Hkv, case["seqs"], s["q"].device
    q, there, at = _batched(s, s["q"])                     # [seqs, nodes, heads, D]
    words = _batched(s, s["mask"])[0]
    bits = (words[..., None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1
    sees = bits.flatten(-2).bool()                         # [seqs, nodes, nodes (32 words)]
    ids = s["table"][s["slots"].long()].long()             # [seqs, pages]
    P = ids.shape[1]
    # [seqs, pages, kv heads, page, D] -> [seqs, kv heads, positions, D]
    k, v = (x[_LAYER, ids.clamp(min=0)].float().transpose(1, 2).reshape(B, Hkv, P * page, D)
            for x in (s["k"], s["v"]))
    pos = torch.arange(P * page, device=dev)
    count = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    node = pos[None, :] - (s["len"][s["slots"].long()].long() - count)[:, None]
    paged = (ids >= 0).repeat_interleave(page, dim=1)
    inner = torch.gather(sees, 2, node.clamp(0, sees.shape[2] - 1)[:, None, :].expand(B, n, P * page))
    keep = ((node < 0)[:, None, :] | (inner & (node < count[:, None])[:, None, :])) & paged[:, None, :]
    q = q.view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    sc = torch.matmul(q, k.transpose(2, 3)).view(B, Hkv, G, n, P * page) * s["scale"]
    sc = sc.masked_fill(~keep[:, None, None], float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1)
    o = torch.matmul(p.view(B, Hkv, G * n, P * page), v).view(B, Hkv, G, n, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    s["out"][at[there]] = o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)[there]
    return s["out"]


def _closure(parent):
    """[seqs][node][node]: whether the second is the first or one of its ancestors."""
    B, n = parent.shape
    dev = parent.device
    x = (parent[..., None] == torch.arange(n, device=dev)).float() + torch.eye(n, device=dev)
    for _ in range(max(1, (n - 1).bit_length())):  # chains twice as long each time
        x = (torch.matmul(x, x) > 0).float()
    return x


def _run_append(s):
    if own:
        ib = _package()
        ib.kv_tree(s["batch"], s["parent"], out=s["tree"])
        ib.kv_append(s["pages"], s["seqs"], s["batch"], _LAYER, s["q"], s["kn"], s["vn"],
                     s["rope"], q_out=s["out"], tree=s["tree"])
        return [s["depth"], s["mask"], s["out"], s["k"], s["v"]]
    case, dev = s["case"], s["qkv"].device
    H, Hkv, page, n = case["heads"], case["kv_heads"], case["page"], case["n_max"]
    parent, there, at = _batched(s, s["parent"], -1)
    anc = _closure(parent)
    rows = at[there]
    depth = (anc.sum(-1) - 1).int()[there]
    full = torch.zeros(*anc.shape[:2], 32 * s["words"], dtype=torch.int64, device=dev)
    full[..., :n] = anc.long()
    words = (full.view(*anc.shape[:2], s["words"], 32) << torch.arange(32, device=dev)).sum(-1)
    s["depth"][rows], s["mask"][rows] = depth, words.to(torch.int32)[there]
    count = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    start = (s["len"][s["slots"].long()].long() - count)[:, None].expand(there.shape)[there]
    x = s["qkv"][rows]
    cs = s["rope"][start + depth.long()][:, None]
    a, b = x[:, :H + Hkv, 0::2], x[:, :H + Hkv, 1::2]
    turned = torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1).flatten(-2)
    s["out"][rows] = turned[:, :H]
    pos = start + torch.arange(n, device=dev).expand(there.shape)[there]
    slot = s["slots"].long()[:, None].expand(there.shape)[there]
    ids = s["table"][slot, torch.div(pos, page, rounding_mode="floor")].long()
    s["k"][_LAYER][ids, :, pos % page] = turned[:, H:].to(s["k"].dtype)
    s["v"][_LAYER][ids, :, pos % page] = x[:, H + Hkv:].to(s["v"].dtype)
    return [s["depth"], s["mask"], s["out"], s["k"], s["v"]]


def _run_accept(s):
    s["books"].copy_(s["books_before"])  # the room of the nodes is there again
    outputs = [s["path"], s["n_path"], s["next"], s["table"], s["len"], s["refs"], s["k"], s["v"]]
    if own:
        ib = _package()
        ib.kv_tree_verify(s["batch"], s["parent"], s["draft"], s["best"], path=s["path"],
                          n_path=s["n_path"], next=s["next"])
        ib.kv_tree_accept(s["pages"], s["seqs"], s["batch"], s["path"], s["n_path"])
        return outputs
    case, dev = s["case"], s["k"].device
    n, page = case["n_max"], case["page"]
    parent, there, at = _batched(s, s["parent"], -2)
    draft, best = _batched(s, s["draft"])[0], _batched(s, s["best"])[0]
    node = torch.arange(n, device=dev)
    match = (parent >= 0) & (draft == best.gather(1, parent.clamp(min=0).long()))
    before = (parent[:, :, None] == parent[:, None, :]) & match[:, None, :] & (node[None, :] < node[:, None])
    good = (match & ~before.any(-1)) | (node == 0)
    taken = ((_closure(parent) * (~good).float()[:, None, :]).sum(-1) == 0) & there
    m = taken.sum(1)
    path = torch.sort(torch.where(taken, node, n + node), dim=1).values
    on = node < m[:, None]
    s["path"][at[there]] = torch.where(on, path, torch.full_like(path, -1)).int()[there]
    s["n_path"].copy_(m)
    s["next"].copy_(best.gather(1, path.gather(1, m[:, None] - 1))[:, 0])
    slot = s["slots"].long()
    count = (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    start = s["len"][slot].long() - count
    src = start[:, None] + torch.where(on, path, torch.zeros_like(path))
    dst = start[:, None] + torch.where(on, node, torch.zeros_like(node))
    place = lambda p: (s["table"][slot[:, None], torch.div(p, page, rounding_mode="floor")].long(), p % page)  # noqa: E731
    (pi, pr), (qi, qr) = place(src), place(dst)
    for x in (s["k"], s["v"]):
        x[:, qi, :, qr] = x[:, pi, :, pr]
    now = start + m
    table = s["table"][slot]
    cols = torch.arange(table.shape[1], device=dev)
    gone = (cols >= -torch.div(-now, page, rounding_mode="floor")[:, None]) & (table >= 0)
    s["refs"].index_add_(0, table.clamp(min=0).flatten().long(), -gone.flatten().int())
    s["table"][slot] = torch.where(gone, torch.full_like(table, -1), table)
    s["len"][slot] = now.int()
    return outputs


_END = 2  # what an ended beam goes on with


def _run_beam(s):
    case = s["case"]
    if own:
        return list(_package().beam_select(s["logits"], s["scores"], beams=case["beams"], k=case["k"],
                                           ended=s["ended"], end_token=_END, out=s["out"],
                                           workspace=s["workspace"]))
    x = s["logits"].float() + 0.0
    rows, V = x.shape
    dev, G, B, k = x.device, case["groups"], case["beams"], case["k"]
    # the k largest of a row, equal ones in order: numbers that sort as the values do, then the place
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    key = (order << 32) | (0xffffffff - torch.arange(V, device=dev))
    most = min(k, V)
    token = 0xffffffff - (torch.topk(key, most, dim=1).values & 0xffffffff)
    # in 64 bits: candidates of different beams may be close
    y = x.double()
    top = y.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(y - top).sum(1, keepdim=True))
    value = s["scores"].double()[:, None] + y.gather(1, token) - lse
    value = torch.where(value.isnan(), torch.full_like(value, float("-inf")), value)
    if s["ended"] is not None:
        end = (s["ended"] != 0)[:, None]
        first = torch.arange(most, device=dev) == 0
        kept = torch.where(first, s["scores"].double()[:, None], torch.full_like(value, float("-inf")))
        value = torch.where(end, kept, value)
        token = torch.where(end, torch.full_like(token, _END), token)
    if B * most < k:  # fewer candidates than places
        value = torch.nn.functional.pad(value.view(G, -1), (0, k - B * most), value=float("-inf"))
        token = torch.nn.functional.pad(token.view(G, -1), (0, k - B * most))
    # equal ones in order of beam and token: a row's candidates are in that order already
    value, token = value.view(G, -1), token.view(G, -1)
    value, at = torch.sort(value, dim=1, descending=True, stable=True)
    value, at = value[:, :k], at[:, :k]
    real = value > float("-inf")
    row = torch.arange(G, device=dev)[:, None] * B + torch.div(at, most, rounding_mode="floor")
    none = torch.full_like(row, -1)
    return [value.float(), torch.where(real, token.gather(1, at), none).int(),
            torch.where(real, row, none).int()]


def _run_reorder(s):
    if own:
        _package().kv_reorder(s["pages"], s["seqs"], s["slots"], s["parents"], status=s["status"],
                              workspace=s["workspace"])
        return [s["status"], s["table"], s["len"], s["refs"], s["k"], s["v"]]
    case = s["case"]
    page, slots, par = case["page"], s["slots"].long(), s["parents"].long()
    table, lens, refs = s["table"], s["len"], s["refs"]
    dev, n = table.device, slots.numel()
    entry = torch.arange(n, device=dev)
    old, new, L = table[slots], table[slots[par]], lens[slots[par]]
    full, part = torch.div(L, page, rounding_mode="floor"), L % page
    cols = torch.arange(table.shape[1], device=dev)
    # a partial last page stays with its slot where that goes on, else with the first that takes it
    rank = torch.where(par == entry, -1, entry)
    first = torch.full((n,), n, device=dev).scatter_reduce_(0, par, rank, "amin")
    copy = (part > 0) & (first[par] != rank)
    lost = copy[:, None] & (cols[None, :] == full[:, None])
    kept = torch.where(lost, torch.full_like(new, -1), new)
    count = torch.zeros_like(refs)
    for rows, sign in ((old, -1), (kept, 1)):
        count.index_add_(0, rows.clamp(min=0).flatten().long(), sign * (rows >= 0).flatten().int())
    refs += count
    free = torch.sort((refs > 0).int(), stable=True).indices  # free pages first, lowest first
    at = torch.cumsum(copy.int(), 0) - 1
    page_of = free[at.clamp(min=0)].int()
    row = torch.where(lost, page_of[:, None], new)
    refs.index_add_(0, page_of.long(), copy.int())
    # rows of the copied pages: src to dst, others to themselves
    where = full.clamp(max=table.shape[1] - 1).long()[:, None]
    src = new.gather(1, where)[:, 0].clamp(min=0).long()
    dst = torch.where(copy, page_of.long(), src)
    some = torch.nonzero(copy)[:, 0]
    src, dst = src[some], dst[some]
    keep = torch.arange(page, device=dev)[None, :] < part[some][:, None]
    for x in (s["k"], s["v"]):
        for layer in range(x.shape[0]):
            x[layer, dst] = torch.where(keep[:, None, :, None], x[layer, src], x[layer, dst])
    table[slots] = row
    lens[slots] = L
    return [torch.ones_like(s["slots"]), table, lens, refs, s["k"], s["v"]]


# ---- the definition in 64 bits -------------------------------------------------------

def exact(case, seed):
    """Attention, append and the scores of a selection from their definitions in 64 bits; what
    moves values or chooses among them has none."""
    if case["op"] not in ("attention", "append", "beam"):
        return None
    s = _inputs(case, seed)
    f8 = torch.float64
    if case["op"] == "beam":
        B, k = case["beams"], case["k"]
        out = []
        for g in range(case["groups"]):
            offers = []
            for r in range(g * B, g * B + B):
                if s["ended"] is not None and int(s["ended"][r]):
                    offers.append(s["scores"][r:r + 1].to(f8))
                else:
                    offers.append(torch.log_softmax(s["logits"][r].to(f8), 0) + s["scores"][r].to(f8))
            offers = torch.cat(offers)
            offers = offers[offers > float("-inf")].sort(descending=True).values[:k]
            out.append(torch.cat([offers, offers.new_full((k - offers.numel(),), float("-inf"))]))
        return [torch.stack(out), None, None]
    nodes, ctx, parents, rows, _ = _tree_layout(case)
    page, D, H, Hkv = case["page"], case["head_dim"], case["heads"], case["kv_heads"]
    dev = s["k"].device
    if case["op"] == "append":
        x = s["qkv"].to(f8)
        out = torch.zeros(s["tokens"], H, D, dtype=f8, device=dev)
        k, v = s["k"].to(f8), s["v"].to(f8)
        turn = torch.view_as_complex(s["rope"].to(f8).contiguous())
        for b, (n, c) in enumerate(zip(nodes, ctx)):
            at = slice(s["cu"][b], s["cu"][b] + n)
            depth = []
            for p in parents[b]:
                depth.append(depth[p] + 1 if p >= 0 else 0)
            z = torch.view_as_complex(x[at].reshape(n, H + 2 * Hkv, D // 2, 2).contiguous())
            z = z * turn[torch.tensor(depth, device=dev) + c][:, None]
            z = torch.view_as_real(z).reshape(n, H + 2 * Hkv, D)
            out[at] = z[:, :H]
            for i in range(n):
                to, r = rows[b][(c + i) // page], (c + i) % page
                k[_LAYER, to, :, r] = z[i, H:H + Hkv]
                v[_LAYER, to, :, r] = x[at][i, H + Hkv:]
        return [None, None, out, k, v]
    out = torch.zeros(s["tokens"], H, D, dtype=f8, device=dev)
    for b, (n, c) in enumerate(zip(nodes, ctx)):
        where = [p for p in range(0, c + n, page) if rows[b][p // page] >= 0]
        at_pos = torch.cat([torch.arange(p, min(c + n, p + page)) for p in where])
        ids = torch.tensor([rows[b][p // page] for p in where], device=dev)
        seen = torch.zeros(n, c + n, dtype=torch.bool)
        seen[:, :c] = True
        for i, p in enumerate(parents[b]):
            if p >= 0:
                seen[i, c:] = seen[p, c:]
            seen[i, c + i] = True
        seen = seen[:, at_pos].to(dev)
        q = s["q"][s["cu"][b]:s["cu"][b] + n].to(f8) * s["scale"]
        for h in range(H):
            kk = s["k"][_LAYER, ids, h // (H // Hkv)].reshape(-1, D)[:at_pos.numel()].to(f8)
            vv = s["v"][_LAYER, ids, h // (H // Hkv)].reshape(-1, D)[:at_pos.numel()].to(f8)
            logit = (q[:, h] @ kk.t()).masked_fill(~seen, float("-inf"))
            out[s["cu"][b]:s["cu"][b] + n, h] = torch.softmax(logit, 1) @ vv
    return out
