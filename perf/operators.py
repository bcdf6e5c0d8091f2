"""Cases of the paged KV cache operators: attention over pages, the append that fills them,
and the page bookkeeping (fork with extend and release, compact).

`own = False` computes the operators in elementary torch operations; `own = True` calls the
package.  A case is a dict of plain values; its ragged lengths and page layout come from its
"shape" number, the values of its tensors from the seed given to prepare().

Layouts (both sides): pool k, v [layer][page][kv head][position in page][head_dim]; table
[slot][page of the sequence] of page numbers, -1 where there is none; len [slot]; refs [page],
zero for a free page.  A sequence's n new tokens are the last n of its len positions.
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

def _attention(name, cache, heads, kv_heads, head_dim, page, seqs, q, kv, shape, pad=0, evicted=0,
               chunks=0, chunk=0):
    """seqs sequences with q tokens each, `chunks` of them with `chunk` tokens instead; pad rows
    behind the last sequence; `evicted` pages behind each sequence's first one given back."""
    return {"name": name, "op": "attention", "cache": cache, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "seqs": seqs, "q_min": q[0], "q_max": q[1],
            "kv_min": kv[0], "kv_max": kv[1], "shape": shape, "pad": pad, "evicted": evicted,
            "chunks": chunks, "chunk": chunk}


def _append(name, cache, heads, kv_heads, head_dim, page, seqs, q, kv, shape, pad=0):
    return {"name": name, "op": "append", "cache": cache, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "seqs": seqs, "q_min": q[0], "q_max": q[1],
            "kv_min": kv[0], "kv_max": kv[1], "shape": shape, "pad": pad, "evicted": 0,
            "chunks": 0, "chunk": 0}


def _fork(name, cache, layers, kv_heads, head_dim, page, parents, children, kv, new, shape):
    return {"name": name, "op": "fork", "cache": cache, "layers": layers, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "parents": parents, "children": children,
            "kv_min": kv[0], "kv_max": kv[1], "new": new, "shape": shape}


def _compact(name, cache, layers, kv_heads, head_dim, page, pages, seqs, kv, shape):
    return {"name": name, "op": "compact", "cache": cache, "layers": layers, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "pages": pages, "seqs": seqs, "kv_min": kv[0],
            "kv_max": kv[1], "shape": shape}


def listed():
    return [
        # one short story being continued token by token: latency alone
        _attention("attn-token-short-f32", "f32", 6, 6, 48, 16, 1, (1, 1), (17, 17), 1),
        # a busy server's decode step (32 heads on 8), contexts of every length
        _attention("attn-token-batch-f16", "f16", 32, 8, 128, 16, 64, (1, 1), (200, 4096), 2),
        # two very long documents being answered (64 heads on 8)
        _attention("attn-token-long-f16", "f16", 64, 8, 128, 64, 2, (1, 1), (100001, 131072), 3),
        # a chunk of a long prompt behind what earlier chunks stored
        _attention("attn-chunk-f16", "f16", 32, 8, 128, 32, 1, (2048, 2048), (8192, 8192), 4),
        # prompt chunks and single tokens in one padded step of a server that gives old pages back
        _attention("attn-mixed-f16", "f16", 32, 8, 128, 16, 30, (1, 4), (300, 4000), 5, pad=13,
                   evicted=20, chunks=2, chunk=509),
        # prompts of a small model (32 heads on 4) on the FP32 cache, pages of an odd size
        _attention("attn-chunk-f32", "f32", 32, 4, 64, 24, 3, (200, 701), (900, 1999), 6),
        # a decode step's new tokens
        _append("append-token-f16", "f16", 32, 8, 128, 16, 64, (1, 1), (200, 4096), 7),
        # a step full of prompt tokens, padded
        _append("append-prompt-f32", "f32", 32, 8, 128, 16, 9, (300, 1300), (1300, 4000), 8, pad=5),
        # four candidates continued from one prompt, generation after generation
        _fork("fork-few-f32", "f32", 4, 8, 128, 16, 1, 4, (333, 333), 9, 9),
        # the same on a full server
        _fork("fork-batch-f16", "f16", 22, 4, 64, 64, 16, 96, (100, 2000), 40, 10),
        # a small pool after a few sequences left
        _compact("compact-few-f32", "f32", 4, 8, 128, 16, 300, 8, (50, 500), 11),
        # a large pool at half its load, gathered to give its upper part back
        _compact("compact-pool-f16", "f16", 22, 4, 64, 16, 6000, 40, (100, 2048), 12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "fork", "compact"])
    cache = rng.choice(["f16", "f32"])
    kv_heads = rng.choice([1, 2, 4, 6, 8])
    head_dim = rng.choice([48, 64, 80, 96, 128, 128, 128])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    shape = rng.randrange(1000, 1 << 30)
    if op in ("attention", "append"):
        heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
        seqs = _log_int(rng, 1, 96)
        top = _log_int(rng, 16, 32768)  # longest context; all contexts within 200 thousand positions
        top = max(16, min(top, 200000 // seqs))
        low = _log_int(rng, 8, top)
        q_max = rng.choice([1, 1, 4, _log_int(rng, 2, 2048)])
        q_max = max(1, min(q_max, low, 4096 // seqs))
        q_min = rng.choice([1, q_max])
        pad = rng.choice([0, 0, rng.randrange(1, 40)])
        if op == "append":
            return _append("", cache, heads, kv_heads, head_dim, page, seqs, (q_min, q_max),
                           (low, top), shape, pad)
        # at most what the largest listed chunk costs: 4 head_dim flops per head, token and position
        while 4.0 * head_dim * heads * seqs * q_max * top > 2e11 and q_max > 1:
            q_max //= 2
        q_min = min(q_min, q_max)
        evicted = rng.choice([0, 0, 0, rng.randrange(1, 30)])
        return _attention("", cache, heads, kv_heads, head_dim, page, seqs, (q_min, q_max),
                          (low, top), shape, pad, evicted)
    layers = _log_int(rng, 1, 32)
    page_bytes = 2 * layers * kv_heads * page * head_dim * _BYTES[cache]
    most = max(40, min(6000, int(2.5e9 // page_bytes)))  # pages of a pool of 2.5 GB
    if op == "fork":
        parents = _log_int(rng, 1, 24)
        children = _log_int(rng, 1, 128)
        new = _log_int(rng, 1, 64)
        per_child = 2 + new // page
        children = max(1, min(children, (most // 2) // per_child))
        top = max(page, min(2000, (most // 2) // parents * page))
        return _fork("", cache, layers, kv_heads, head_dim, page, parents, children,
                     (max(1, top // _log_int(rng, 1, 20)), top), new, shape)
    pages = _log_int(rng, 40, most)
    seqs = _log_int(rng, 1, 48)
    top = max(1, min(4096, int(pages * rng.uniform(0.1, 0.9)) // seqs * page))
    return _compact("", cache, layers, kv_heads, head_dim, page, pages, seqs,
                    (max(1, top // 8), top), shape)


# ---- layouts from a case alone -------------------------------------------------------

def _batch_layout(case):
    """(q lengths, contexts, table rows, pool pages) of an attention or append case."""
    rng = random.Random(case["shape"])
    n = case["seqs"]
    ctx = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(n)]
    q = [min(c, rng.randint(case["q_min"], case["q_max"])) for c in ctx]
    for b in range(case["chunks"]):
        at = (b * n) // case["chunks"]
        q[at] = case["chunk"]
        ctx[at] = max(ctx[at], q[at])
    per = [-(-c // case["page"]) for c in ctx]
    pages = sum(per) + 7
    free = list(range(pages))
    rng.shuffle(free)
    rows, at = [], 0
    for b in range(n):
        row = free[at:at + per[b]]
        at += per[b]
        # pages 1 .. evicted were given back; those of the new tokens and the two before are kept
        last = (ctx[b] - q[b]) // case["page"] - 2
        for j in range(1, min(1 + case["evicted"], last)):
            row[j] = -1
        rows.append(row)
    return q, ctx, rows, pages


def _fork_layout(case):
    """Parents in the first slots, the previous generation's children in the others."""
    rng = random.Random(case["shape"])
    p, c, page = case["parents"], case["children"], case["page"]
    lens = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(p)]
    per = [-(-x // page) for x in lens]
    of = [rng.randrange(p) for _ in range(c)]       # this generation's parents
    was = [rng.randrange(p) for _ in range(c)]      # the previous one's
    fresh = [-(-(lens[i] + case["new"]) // page) - lens[i] // page for i in of]
    old = [-(-(lens[i] + case["new"]) // page) - lens[i] // page for i in was]
    pages = sum(per) + max(sum(fresh), sum(old)) + 9
    free = list(range(pages))
    rng.shuffle(free)
    rows, at = [], 0
    for b in range(p):
        rows.append(free[at:at + per[b]])
        at += per[b]
    refs = [0] * pages
    for row in rows:
        for x in row:
            refs[x] += 1
    all_lens = list(lens)
    for i, parent in enumerate(was):
        full = lens[parent] // page
        row = rows[parent][:full] + free[at:at + old[i]]
        at += old[i]
        rows.append(row)
        all_lens.append(lens[parent] + case["new"])
        for x in row:
            refs[x] += 1
    return all_lens, rows, refs, of, pages


def _compact_layout(case):
    rng = random.Random(case["shape"])
    page, pages = case["page"], case["pages"]
    free = list(range(pages))
    rng.shuffle(free)
    lens, rows, refs = [], [], [0] * pages
    for b in range(case["seqs"]):
        n = rng.randint(case["kv_min"], case["kv_max"])
        need = -(-n // page)
        share = rng.randrange(0, need) if b and rng.random() < 0.3 else 0
        head = rows[rng.randrange(b)][:share] if share else []  # a prefix shared with another
        need -= len(head)
        if need > len(free):
            need = len(free)
            n = (len(head) + need) * page
        row = head + [free.pop() for _ in range(need)]
        lens.append(n)
        rows.append(row)
        for x in row:
            refs[x] += 1
    return lens, rows, refs


def _moves(refs):
    live = sum(1 for r in refs if r)
    return live, sum(1 for r in refs[live:] if r)


def work(case):
    size = _BYTES[case["cache"]]
    if case["op"] in ("attention", "append"):
        q, ctx, rows, _ = _batch_layout(case)
        H, Hkv, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        tokens = sum(q)
        if case["op"] == "append":
            return {"bytes": tokens * D * (8 * H + Hkv * 2 * (4 + size)) + 4 * D * tokens,
                    "flops": 3 * tokens * D * (H + Hkv)}
        bytes_, pairs = 8 * tokens * H * D, 0
        for n, c, row in zip(q, ctx, rows):
            gone = sum(1 for x in row if x < 0) * page
            bytes_ += 2 * size * Hkv * D * (c - gone) + 4 * len(row)
            pairs += n * (c - n - gone) + n * (n + 1) // 2
        return {"bytes": bytes_, "flops": 4 * D * H * pairs}
    per_pos = 2 * case["layers"] * case["kv_heads"] * case["head_dim"] * size
    if case["op"] == "fork":
        lens, rows, refs, of, pages = _fork_layout(case)
        part = sum(lens[i] % case["page"] for i in of)
        ids = sum(len(rows[i]) for i in of) + sum(len(r) for r in rows[case["parents"]:])
        return {"bytes": 2 * part * per_pos + 4 * (2 * ids + pages), "flops": 0}
    lens, rows, refs = _compact_layout(case)
    _, moved = _moves(refs)
    return {"bytes": 2 * moved * case["page"] * per_pos + 4 * (3 * len(refs) + 2 * sum(map(len, rows))),
            "flops": 0}


# ---- inputs --------------------------------------------------------------------------

def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _table(rows, slots, width, device):
    t = torch.full((slots, width), -1, dtype=torch.int32)
    for i, row in enumerate(rows):
        t[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
    return t.to(device)


def _pool(gen, layers, pages, case, device):
    shape = (layers, pages, case["kv_heads"], case["page"], case["head_dim"])
    dt = _DTYPE[case["cache"]]
    return [torch.randn(shape, generator=gen, device=device, dtype=dt) for _ in range(2)]


def _inputs(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    s = {"case": case}
    page, Hkv, D = case["page"], case["kv_heads"], case["head_dim"]
    if case["op"] in ("attention", "append"):
        q, ctx, rows, pages = _batch_layout(case)
        n, H = case["seqs"], case["heads"]
        order = list(range(n + 3))  # the batch's rows of the table, among slots not in the batch
        random.Random(case["shape"] + 1).shuffle(order)
        order = order[:n]
        width = max(map(len, rows)) + 1
        by_slot, lens = [[] for _ in range(n + 3)], [0] * (n + 3)
        for b, slot in enumerate(order):
            by_slot[slot], lens[slot] = rows[b], ctx[b]
        cu = [0]
        for x in q:
            cu.append(cu[-1] + x)
        tokens = cu[-1] + case["pad"]
        s.update(q_lens=q, ctx=ctx, order=order, cu=cu, tokens=tokens)
        s["k"], s["v"] = _pool(gen, 2, pages, case, dev)
        s["table"], s["len"] = _table(by_slot, n + 3, width, dev), _int32(lens, dev)
        refs = [0] * pages
        for row in rows:
            for x in row:
                if x >= 0:
                    refs[x] += 1
        s["refs"] = _int32(refs, dev)
        s["cu_q"], s["slots"] = _int32(cu, dev), _int32(order, dev)
        if case["op"] == "attention":
            s["q"] = 1.5 * torch.randn(tokens, H, D, generator=gen, device=dev)
            s["out"] = torch.zeros(tokens, H, D, device=dev)
            s["scale"] = 1.0 / math.sqrt(D)
        else:
            # the projections' output: q, k and v of a token next to each other
            s["qkv"] = torch.randn(tokens, H + 2 * Hkv, D, generator=gen, device=dev)
            s["out"] = torch.zeros(tokens, H, D, device=dev)
            half = D // 2
            pos = torch.arange(max(ctx), dtype=torch.float64, device=dev)
            freq = 500000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) * 2 / D)
            ang = pos[:, None] * freq[None, :]
            s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    elif case["op"] == "fork":
        lens, rows, refs, of, pages = _fork_layout(case)
        slots = len(rows)
        s["k"], s["v"] = _pool(gen, case["layers"], pages, case, dev)
        s["table"] = _table(rows, slots, max(map(len, rows)) + 2, dev)
        s["len"], s["refs"] = _int32(lens, dev), _int32(refs, dev)
        s["parents"] = _int32(of, dev)
        s["children"] = _int32(range(case["parents"], slots), dev)
        s["new"] = _int32([case["new"]] * case["children"], dev)
    else:
        lens, rows, refs = _compact_layout(case)
        s["k"], s["v"] = _pool(gen, case["layers"], case["pages"], case, dev)
        s["table"] = _table(rows, len(rows) + 2, max(map(len, rows)) + 1, dev)
        s["len"], s["refs"] = _int32(lens + [0, 0], dev), _int32(refs, dev)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the handles, workspace and output buffers that a serving program keeps
        ib = _package()
        Hkv, dev = case["kv_heads"], s["k"].device
        s["pages"] = ib.KVPages(s["k"], s["v"])
        s["seqs"] = ib.KVSeqs(s["table"], s["len"], s["refs"])
        if case["op"] in ("attention", "append"):
            s["batch"] = ib.KVBatch(s["cu_q"], s["tokens"], max_q=max(s["q_lens"]), slots=s["slots"])
        if case["op"] == "attention":
            s["workspace"] = ib.attention_paged_workspace(s["pages"], s["seqs"], s["batch"],
                                                          case["heads"])
        elif case["op"] == "append":
            H = case["heads"]
            s["q"], s["kn"], s["vn"] = s["qkv"].split([H, Hkv, Hkv], dim=1)
        elif case["op"] == "fork":
            s["status"] = [torch.empty(case["children"], dtype=torch.int32, device=dev)
                           for _ in range(2)]
        elif case["op"] == "compact":
            # the other half of a double-buffered table
            s["seqs_out"] = ib.KVSeqs(torch.empty_like(s["table"]), s["len"],
                                      torch.empty_like(s["refs"]))
            s["plan"] = ib.kv_compact_plan(s["pages"])
    return s


# ---- one pass ------------------------------------------------------------------------

def run(s):
    return {"attention": _run_attention, "append": _run_append, "fork": _run_fork,
            "compact": _run_compact}[s["case"]["op"]](s)


def _run_attention(s):
    if own:
        _package().attention_paged(s["pages"], s["seqs"], s["batch"], _LAYER, s["q"], s["scale"],
                                   out=s["out"], workspace=s["workspace"])
        return s["out"]
    case = s["case"]
    H, Hkv, D, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    G = H // Hkv
    for b, slot in enumerate(s["order"]):
        n, c, at = s["q_lens"][b], s["ctx"][b], s["cu"][b]
        ids = s["table"][slot, :-(-c // page)].long()
        there = (ids >= 0).repeat_interleave(page)[:c]
        ids = ids.clamp(min=0)
        # [pages, kv heads, page, D] -> [kv heads, positions, D]
        k = s["k"][_LAYER, ids].float().transpose(0, 1).reshape(Hkv, -1, D)[:, :c]
        v = s["v"][_LAYER, ids].float().transpose(0, 1).reshape(Hkv, -1, D)[:, :c]
        pos = torch.arange(c, device=k.device)
        new = torch.arange(c - n, c, device=k.device)
        keep = there[None, :] & (pos[None, :] <= new[:, None])      # [tokens, positions]
        q = s["q"][at:at + n].view(n, Hkv, G, D).permute(1, 2, 0, 3)  # [kv heads, group, tokens, D]
        for g in range(Hkv):
            sc = torch.matmul(q[g], k[g].t()) * s["scale"]
            sc = sc.masked_fill(~keep, float("-inf"))
            p = torch.exp(sc - sc.amax(-1, keepdim=True))
            o = torch.matmul(p, v[g]) / p.sum(-1, keepdim=True)
            s["out"][at:at + n].view(n, Hkv, G, D)[:, g] = o.transpose(0, 1)
    return s["out"]


def _run_append(s):
    if own:
        _package().kv_append(s["pages"], s["seqs"], s["batch"], _LAYER, s["q"], s["kn"], s["vn"],
                             s["rope"], q_out=s["out"])
        return [s["out"], s["k"], s["v"]]
    case = s["case"]
    H, Hkv, page = case["heads"], case["kv_heads"], case["page"]

    def rotate(x, cs):
        a, b = x[..., 0::2], x[..., 1::2]
        c, d = cs[:, None, :, 0], cs[:, None, :, 1]
        return torch.stack([a * c - b * d, a * d + b * c], -1).flatten(-2)

    for b, slot in enumerate(s["order"]):
        n, c, at = s["q_lens"][b], s["ctx"][b], s["cu"][b]
        pos = torch.arange(c - n, c, device=s["k"].device)
        ids, rows = s["table"][slot, pos // page].long(), pos % page
        x, cs = s["qkv"][at:at + n], s["rope"][c - n:c]
        s["out"][at:at + n] = rotate(x[:, :H], cs)
        s["k"][_LAYER][ids, :, rows] = rotate(x[:, H:H + Hkv], cs).to(s["k"].dtype)
        s["v"][_LAYER][ids, :, rows] = x[:, H + Hkv:].to(s["v"].dtype)
    return [s["out"], s["k"], s["v"]]


def _run_fork(s):
    """The last generation leaves, a new one is forked and gets room for its new tokens."""
    if own:
        ib = _package()
        ib.kv_release(s["pages"], s["seqs"], s["children"])
        ib.kv_fork(s["pages"], s["seqs"], s["parents"], s["children"], status=s["status"][0])
        ib.kv_extend(s["pages"], s["seqs"], s["children"], s["new"], status=s["status"][1])
        return [s["status"][0], s["status"][1], s["table"], s["len"], s["refs"], s["k"], s["v"]]
    page = s["case"]["page"]
    table, lens, refs, par, chi = s["table"], s["len"], s["refs"], s["parents"].long(), \
        s["children"].long()
    width = table.shape[1]
    cols = torch.arange(width, device=table.device)
    # release
    used = table[chi]
    held = used >= 0
    refs -= torch.zeros_like(refs).index_add_(0, used.clamp(min=0).flatten().long(),
                                              held.flatten().int())
    table[chi] = -1
    # fork: whole pages are shared, the partial last one is copied
    n = lens[par]
    full, part = torch.div(n, page, rounding_mode="floor"), n % page
    # pages in the order of need: the partial pages child by child, then the new ones
    grown = -torch.div(-(n + s["new"]), page, rounding_mode="floor")
    first = (part > 0).int()
    more = grown - full - first
    free = torch.sort((refs > 0).int(), stable=True).indices  # free pages first, lowest first
    row = torch.where(cols[None, :] < full[:, None], table[par], torch.full_like(used, -1))
    at = torch.cumsum(first, 0) - first
    total = first.sum()
    at_more = total + torch.cumsum(more, 0) - more
    own_col = (cols[None, :] == full[:, None]) & (part[:, None] > 0)
    row = torch.where(own_col, free[at.clamp(max=free.numel() - 1)][:, None].int(), row)
    k_new = cols[None, :] - (full + first)[:, None]
    new_col = (k_new >= 0) & (cols[None, :] < grown[:, None])
    row = torch.where(new_col, free[(at_more[:, None] + k_new).clamp(0, free.numel() - 1)].int(), row)
    some = torch.nonzero(part > 0)[:, 0]
    src = table[par[some], full[some].long()].long()
    dst = row[some, full[some].long()].long()
    keep = torch.arange(page, device=table.device)[None, :] < part[some][:, None]
    for x in (s["k"], s["v"]):
        for layer in range(x.shape[0]):
            x[layer, dst] = torch.where(keep[:, None, :, None], x[layer, src], x[layer, dst])
    table[chi] = row
    held = row >= 0
    refs += torch.zeros_like(refs).index_add_(0, row.clamp(min=0).flatten().long(),
                                              held.flatten().int())
    lens[chi] = n + s["new"]
    one = torch.ones_like(par, dtype=torch.int32)
    return [one, one.clone(), table, lens, refs, s["k"], s["v"]]


def _run_compact(s):
    if own:
        ib = _package()
        plan = ib.kv_compact(s["pages"], s["seqs"], out=s["seqs_out"], plan=s["plan"])
        return [plan.map, plan.n_live, s["seqs_out"].table, s["seqs_out"].refs, s["k"], s["v"]]
    refs, table = s["refs"], s["table"]
    live = refs > 0
    index = torch.arange(refs.numel(), device=refs.device)
    n_live = live.sum()
    src = torch.nonzero(live & (index >= n_live))[:, 0]
    dst = torch.nonzero(~live & (index < n_live))[:, 0]
    to = torch.where(live, index, torch.full_like(index, -1))
    to[src] = dst
    refs_out = refs.clone()
    refs_out[dst] = refs[src]
    refs_out[src] = 0
    table_out = torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table)
    for x in (s["k"], s["v"]):
        x[:, dst] = x[:, src]
    return [to.int(), n_live.int(), table_out, refs_out, s["k"], s["v"]]


# ---- the definition in 64 bits -------------------------------------------------------

def exact(case, seed):
    """Attention and append from their definitions in 64 bits; the bookkeeping moves values
    without computing any, so its outputs have none."""
    if case["op"] not in ("attention", "append"):
        return None
    s = _inputs(case, seed)
    f8, page, D = torch.float64, case["page"], case["head_dim"]
    H, Hkv = case["heads"], case["kv_heads"]
    table = s["table"].tolist()
    if case["op"] == "append":
        x = s["qkv"].to(f8)
        out = torch.zeros(s["tokens"], H, D, dtype=f8, device=x.device)
        k, v = s["k"].to(f8), s["v"].to(f8)
        turn = torch.view_as_complex(s["rope"].to(f8).contiguous())
        for b, slot in enumerate(s["order"]):
            c, n = s["ctx"][b], s["q_lens"][b]
            rows = slice(s["cu"][b], s["cu"][b] + n)
            z = torch.view_as_complex(x[rows].reshape(n, H + 2 * Hkv, D // 2, 2).contiguous())
            z = torch.view_as_real(z * turn[c - n:c, None, :]).reshape(n, H + 2 * Hkv, D)
            out[rows] = z[:, :H]
            p = c - n
            while p < c:  # page by page
                stop = min(c, (p // page + 1) * page)
                i, a = table[slot][p // page], p % page
                t0, t1 = p - (c - n), stop - (c - n)
                k[_LAYER, i, :, a:a + stop - p] = z[t0:t1, H:H + Hkv].transpose(0, 1)
                v[_LAYER, i, :, a:a + stop - p] = x[rows][t0:t1, H + Hkv:].transpose(0, 1)
                p = stop
        return [out, k, v]
    out = torch.zeros(s["tokens"], H, D, dtype=f8, device=s["q"].device)
    for b, slot in enumerate(s["order"]):
        n, c, at = s["q_lens"][b], s["ctx"][b], s["cu"][b]
        q = s["q"][at:at + n].to(f8) * s["scale"]
        where = [p for p in range(0, c, page) if table[slot][p // page] >= 0]
        at_pos = torch.cat([torch.arange(p, min(c, p + page)) for p in where]).to(q.device)
        ids = torch.tensor([table[slot][p // page] for p in where], device=q.device)
        for h in range(H):
            kk = s["k"][_LAYER, ids, h // (H // Hkv)].reshape(-1, D)[:at_pos.numel()].to(f8)
            vv = s["v"][_LAYER, ids, h // (H // Hkv)].reshape(-1, D)[:at_pos.numel()].to(f8)
            logit = torch.einsum("td,pd->tp", q[:, h], kk)
            seen = at_pos[None, :] <= torch.arange(c - n, c, device=q.device)[:, None]
            top = torch.where(seen, logit, torch.full_like(logit, -1e300)).max(dim=1).values
            w = torch.where(seen, torch.exp(logit - top[:, None]), torch.zeros_like(logit))
            out[at:at + n, h] = torch.einsum("tp,pd->td", w, vv) / w.sum(1)[:, None]
    return out
