"""Trees of drafted tokens over the paged cache: the plan (depths and masks), append at a node's
depth, attention over context and ancestors, greedy verification and the keeping of the accepted
path, each against a plain restatement (whole numbers in Python, values in 64 bits).

Attention's tolerance per output element is the causal operator's (test_gpu_paged.py): products of
FP32 operands keep 2^-20, so |out - ref| <= ((2 A + 1) 2^-20 + sqrt(L) 2^-24) sum p |v| with
A = scale * the largest sum |q_d k_d| of a position that the row sees."""
import math
import random

import pytest

from conftest import load_package
from test_gpu_paged import Book, i32, make, pool, rope_table, seqs_of

ib = load_package()
pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("type_", [ib.F32, ib.F16], ids=["f32", "f16"])


def random_tree(rng, n, roots=1, reach=6):
    return [-1 if i < roots else rng.randint(max(0, i - reach), i - 1) for i in range(n)]


def ancestors(parents):
    """Node sets: a node and its ancestors."""
    sets = []
    for i, p in enumerate(parents):
        sets.append({i} | (sets[p] if p >= 0 else set()))
    return sets


def flat(parents, pad=0, fill=-1):
    return [x for p in parents for x in p] + [fill] * pad


def plan_of(cuda, batch, parents, pad=0, max_nodes=0):
    return ib.kv_tree(batch, i32(cuda, flat(parents, pad)), max_nodes)


# ---- plan ------------------------------------------------------------------------------

@pytest.mark.parametrize("nodes,max_nodes,pad", [([1], 1, 0), ([7, 0, 33, 1], 33, 3), ([32, 31], 32, 0),
                                                 ([1024, 5, 700], 1024, 2), ([65, 64], 200, 1)])
def test_plan(cuda, nodes, max_nodes, pad):
    rng = random.Random(sum(nodes))
    parents = [random_tree(rng, n, rng.choice([1, 2]), rng.choice([1, 4, 40])) for n in nodes]
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    T = cu[-1] + pad
    batch = ib.KVBatch(i32(cuda, cu), T, max_q=max(nodes))
    words = -(-max_nodes // 32)
    tree = ib.KVTree(i32(cuda, flat(parents, pad, 12345)), cuda.full((T,), 9, dtype=cuda.int32, device="cuda"),
                     cuda.full((T, words), 9, dtype=cuda.int32, device="cuda"), max_nodes)
    assert ib.kv_tree(batch, tree.parents, out=tree) is tree
    depth, mask = tree.depth.tolist(), tree.mask.tolist()
    for b, p in enumerate(parents):
        for i, a in enumerate(ancestors(p)):
            t = cu[b] + i
            assert depth[t] == len(a) - 1
            assert sum((w & 0xffffffff) << (32 * j) for j, w in enumerate(mask[t])) == sum(1 << c for c in a)
    for t in range(cu[-1], T):  # rows of nobody
        assert depth[t] == 9 and mask[t] == [9] * words
    assert ib.check_fault() == 0


def test_plan_records_what_cannot_be(cuda):
    cu = i32(cuda, [0, 3, 7])
    for parents, want in (([-1, 1, 0, -1, 0, 1, 2], [0, 0, 1, 0, 1, 2, 3]),
                          ([-1, 0, 5, -2, 0, 4, 2], [0, 1, 0, 0, 1, 0, 1 + 0])):
        tree = ib.kv_tree(ib.KVBatch(cu, 7), i32(cuda, parents), 4)
        want_mask = []
        for b, e in ((0, 3), (3, 7)):
            fixed = [p if -1 <= p < i else -1 for i, p in enumerate(parents[b:e])]
            want_mask += [sum(1 << c for c in a) for a in ancestors(fixed)]
        assert [m[0] for m in tree.mask.tolist()] == want_mask
        with pytest.raises(RuntimeError, match="78"):
            ib.check_fault()
    # more nodes than the masks have room for; a sequence left out
    tree = ib.kv_tree(ib.KVBatch(cu, 7), i32(cuda, [-1, 0, 1, -1, 0, 1, 2]), 3)
    assert tree.depth.tolist() == [0, 1, 2, 0, 0, 0, 0] and tree.mask[3:].abs().max().item() == 0
    with pytest.raises(RuntimeError, match="78"):
        ib.check_fault()
    tree = ib.kv_tree(ib.KVBatch(cu, 7, slots=i32(cuda, [-1, 4])), i32(cuda, [-1, 0, 1, -1, 0, 1, 2]))
    assert tree.depth.tolist() == [0, 0, 0, 0, 1, 2, 3]
    ib.kv_tree(ib.KVBatch(i32(cuda, [0, 9]), 7), i32(cuda, [-1] * 7))
    with pytest.raises(RuntimeError, match="73"):
        ib.check_fault()


# ---- append ----------------------------------------------------------------------------

@TYPES
@pytest.mark.parametrize("H,Hkv,HD,page,nodes,ctx,pad,sl", [
    (4, 2, 128, 16, [5, 1, 9], [1, 16, 40], 0, True),
    (6, 6, 48, 7, [33, 0, 2, 12], [3, 5, 0, 140], 4, True),
    (3, 3, 256, 100, [70], [333], 7, False),
])
def test_append_at_depths(cuda, type_, H, Hkv, HD, page, nodes, ctx, pad, sl):
    """As kv_append, with the angles of L - n + depth: bit for bit what kv_append makes of each node
    as a single token at that position."""
    rng = random.Random(HD)
    total = [c + n for c, n in zip(ctx, nodes)]
    seqs, batch, table, slots, n_pages, cu = make(cuda, rng, page, nodes, total, pad, sl)
    pages = pool(cuda, 2, n_pages, Hkv, page, HD, type_, 9)
    T = batch.n_tokens
    qkv = cuda.randn(T, H + 2 * Hkv, HD, generator=cuda.Generator(device="cuda").manual_seed(4), device="cuda")
    q, k, v = qkv.split([H, Hkv, Hkv], dim=1)
    rope = rope_table(cuda, max(total + [1]), HD)
    parents = [random_tree(rng, n, 1, 5) for n in nodes]
    tree = plan_of(cuda, batch, parents, pad)
    # the wanted rows, a token at a time, each a sequence of its own on a page of its own
    alone = pool(cuda, 1, T, Hkv, 1, HD, type_, 9)
    where = [(b, i) for b in range(len(nodes)) for i in range(nodes[b])]
    lens = [ctx[b] + tree.depth[cu[b] + i].item() + 1 for b, i in where]
    width = max(lens + [1])
    tab = cuda.full((len(where), width), -1, dtype=cuda.int32, device="cuda")
    for t, n in enumerate(lens):
        tab[t, n - 1] = t
    want_q = cuda.full((T, H, HD), 7.0, device="cuda")
    ib.kv_append(alone, ib.KVSeqs(tab, i32(cuda, lens), i32(cuda, [1] * T)),
                 ib.KVBatch(i32(cuda, range(len(where) + 1)), len(where), max_q=1), 0,
                 *(x[:len(where)] for x in (q, k, v)), rope, q_out=want_q[:len(where)])
    want = [pages.k.clone(), pages.v.clone()]
    for t, (b, i) in enumerate(where):
        pos = ctx[b] + i
        for x, y in zip(want, (alone.k, alone.v)):
            x[1, table[slots[b]][pos // page], :, pos % page] = y[0, t, :, 0]
    out = cuda.full((T, H, HD), 7.0, device="cuda")
    ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, q_out=out, tree=tree)
    assert cuda.equal(out, want_q)
    assert cuda.equal(pages.k, want[0]) and cuda.equal(pages.v, want[1])
    # a chain is what kv_append does without a tree
    chain = plan_of(cuda, batch, [[i - 1 for i in range(n)] for n in nodes], pad)
    a = ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, q_out=cuda.zeros_like(out), tree=chain)
    k0 = pages.k.clone()
    b = ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, q_out=cuda.zeros_like(out))
    assert cuda.equal(a, b) and cuda.equal(k0, pages.k)
    assert ib.check_fault() == 0


def test_append_passes_over_bad_depths(cuda):
    pages = pool(cuda, 1, 3, 1, 4, 8, ib.F32, 0, fill=1.0)
    seqs = ib.KVSeqs(i32(cuda, [0, 1]).view(1, 2), i32(cuda, [7]), i32(cuda, [1, 1, 0]))
    batch = ib.KVBatch(i32(cuda, [0, 3]), 3)
    x = cuda.full((3, 1, 8), 5.0, device="cuda")
    tree = ib.KVTree(i32(cuda, [-1, 0, 1]), i32(cuda, [0, 2, -1]), cuda.ones(3, 1, dtype=cuda.int32, device="cuda"), 3)
    out = ib.kv_append(pages, seqs, batch, 0, x, x, x, rope_table(cuda, 16, 8), q_out=cuda.zeros_like(x), tree=tree)
    assert bool((out[0] != 0).all()) and not bool((out[1:] != 0).any())
    assert [pages.v[0, 1, 0, r, 0].item() for r in range(4)] == [5.0, 1.0, 1.0, 1.0]
    with pytest.raises(RuntimeError, match="78"):
        ib.check_fault()
    # angles go by the depth, not by the place: a long tree at the end of the table of rotations
    flat_tree = plan_of(cuda, batch, [[-1, -1, -1]])
    out = ib.kv_append(pages, seqs, batch, 0, x, x, x, rope_table(cuda, 5, 8), q_out=cuda.zeros_like(x), tree=flat_tree)
    assert bool((out != 0).any(-1).all()) and cuda.equal(out[0], out[2])
    assert ib.check_fault() == 0


# ---- attention -------------------------------------------------------------------------

def tree_ref(cuda, pages, layer, table, slots, cu, nodes, ctx, parents, q, scale):
    """(out, tolerance) in 64 bits; rows of nobody are NaN in out."""
    H, HD = q.shape[1], q.shape[2]
    G, page, f8 = H // pages.n_kv_heads, pages.page_size, cuda.float64
    out = cuda.full(q.shape, float("nan"), dtype=f8, device="cuda")
    tol = cuda.zeros(q.shape, dtype=f8, device="cuda")
    for b, s in enumerate(slots):
        n, c = nodes[b], ctx[b]
        if n == 0:
            continue
        pos = [p for p in range(c + n) if table[s][p // page] >= 0]
        rows = slice(cu[b], cu[b] + n)
        if not pos:
            out[rows] = 0
            continue
        ids = cuda.tensor([table[s][p // page] for p in pos], device="cuda")
        at = cuda.tensor([p % page for p in pos], device="cuda")
        k = pages.k[layer][ids, :, at].to(f8)
        v = pages.v[layer][ids, :, at].to(f8)
        seen = cuda.tensor([[p < c or p - c in a for p in pos] for a in ancestors(parents[b])], device="cuda")
        for h in range(H):
            kk, vv, qq = k[:, h // G].nan_to_num(0, 0, 0), v[:, h // G].nan_to_num(0, 0, 0), q[rows, h].to(f8)
            sc = (qq @ kk.t() * scale).masked_fill(~seen, -math.inf)
            A = (qq.abs() @ kk.abs().t() * abs(scale)).masked_fill(~seen, 0).amax(1, keepdim=True)
            top = sc.amax(1, keepdim=True).clamp(min=-1e300)
            p = cuda.exp(sc - top)
            l = p.sum(1, keepdim=True)
            p = cuda.where(l > 0, p / l, cuda.zeros_like(p))
            out[rows, h] = p @ vv
            tol[rows, h] = ((2 * A + 1) * 2.0 ** -20 + math.sqrt(c + n) * 2.0 ** -24) * (p @ vv.abs())
    return out, tol


def run_tree(cuda, type_, H, Hkv, HD, page, nodes, ctx, pad=0, with_slots=True, holes=0.0, seed=0,
             spoil=False, max_nodes=0, max_q=None, roots=1, reach=6, scale=None, parents=None, q_size=1.5):
    rng = random.Random(seed + HD * 7 + page)
    total = [c + n for c, n in zip(ctx, nodes)]
    seqs, batch, table, slots, n_pages, cu = make(cuda, rng, page, nodes, total, pad, with_slots)
    pages = pool(cuda, 2, n_pages, Hkv, page, HD, type_, seed + 1)
    for row in table:
        for j in range(len(row)):
            if rng.random() < holes:
                row[j] = -1
    seqs.table.copy_(cuda.tensor(table, dtype=cuda.int32))
    if max_q is not None:
        batch = ib.KVBatch(batch.cu_q, batch.n_tokens, max_q=max_q, slots=batch.slots)
    if spoil:  # whatever no sequence holds
        held = cuda.zeros(n_pages, page, dtype=cuda.bool, device="cuda")
        for s, n in zip(slots, total):
            for p in range(n):
                if table[s][p // page] >= 0:
                    held[table[s][p // page], p % page] = True
        bad = cuda.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")
        for x in (pages.k, pages.v):
            fill = bad[cuda.randint(0, 3, x.shape, device="cuda")].to(x.dtype)
            x.copy_(cuda.where(held[None, :, None, :, None], x, fill))
    parents = parents or [random_tree(rng, n, roots, reach) for n in nodes]
    tree = plan_of(cuda, batch, parents, pad, max_nodes or max(nodes + [1]))
    T = batch.n_tokens
    scale = 1.0 / math.sqrt(HD) if scale is None else scale
    buf = q_size * cuda.randn(T, H + 2 * Hkv, HD, generator=cuda.Generator(device="cuda").manual_seed(seed + 2),
                              device="cuda")
    q = buf[:, :H]  # rows apart
    obuf = cuda.full((T, H + 1, HD), 3.0, device="cuda")
    out = obuf[:, :H]
    ib.attention_paged(pages, seqs, batch, 1, q, scale, out=out, tree=tree)
    ref, tol = tree_ref(cuda, pages, 1, table, slots, cu, nodes, ctx, parents, q, scale)
    mine = ~ref.isnan()
    err = (out.double() - ref).abs()
    worst = (err / tol.clamp(min=1e-300))[mine & (tol > 0)]
    assert bool((err <= tol)[mine].all()), \
        f"{worst.max().item() if worst.numel() else err[mine].max().item()} of the tolerance"
    assert bool((out[~mine] == 3.0).all()) and bool((obuf[:, H] == 3.0).all())
    assert ib.check_fault() == 0
    return pages, seqs, batch, tree, q, out, scale, table, slots


SHAPES = [(6, 6, 48, 16), (32, 8, 128, 16), (32, 4, 64, 24), (4, 4, 8, 1), (8, 1, 256, 64),
          (7, 1, 80, 100), (24, 2, 96, 7), (16, 8, 136, 32), (5, 5, 16, 128)]


@TYPES
@pytest.mark.parametrize("H,Hkv,HD,page", SHAPES)
def test_attention_small_trees(cuda, type_, H, Hkv, HD, page):
    ctx = [0, 1, 2, 15, 16, 17, 63, 64, 130, 700]
    run_tree(cuda, type_, H, Hkv, HD, page, [1, 3, 2, 4, 5, 1, 7, 0, 6, 5], ctx, pad=2)


@TYPES
@pytest.mark.parametrize("H,Hkv,HD,page", SHAPES)
def test_attention_large_trees(cuda, type_, H, Hkv, HD, page):
    run_tree(cuda, type_, H, Hkv, HD, page, [1, 33, 0, 5, 130, 64], [500, 33, 9, 66, 401, 64], pad=5)


@TYPES
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 96, 128, 129, 257, 1024])
def test_attention_every_number_of_nodes(cuda, type_, n):
    run_tree(cuda, type_, 8, 2, 64, 16, [n, n], [0, 190], seed=n, reach=max(6, n // 8))


@TYPES
@pytest.mark.parametrize("G", [1, 2, 3, 5, 16])
def test_attention_groups(cuda, type_, G):
    run_tree(cuda, type_, 2 * G, 2, 128, 16, [12, 17, 40], [200, 77, 1300], seed=G)


@TYPES
def test_attention_shapes_of_trees(cuda, type_):
    n, c = 70, 131
    shapes = {"chain": [i - 1 for i in range(n)], "star": [-1] + [0] * (n - 1), "roots": [-1] * n,
              "binary": [-1] + [(i - 1) // 2 for i in range(1, n)]}
    for parents in shapes.values():
        a = run_tree(cuda, type_, 8, 2, 128, 16, [n], [c], parents=[parents])
    # a chain is causal attention
    pages, seqs, batch, tree, q, out, scale, _, _ = run_tree(cuda, type_, 8, 2, 128, 16, [n], [c],
                                                             parents=[shapes["chain"]])
    plain = ib.attention_paged(pages, seqs, batch, 1, q, scale)
    size = pages.v.abs().max()
    assert bool(((plain - out).abs() <= 2.0 ** -17 * size).all())


@TYPES
def test_attention_long_contexts_are_split(cuda, type_):
    run_tree(cuda, type_, 8, 2, 128, 64, [5], [20001])
    run_tree(cuda, type_, 8, 2, 128, 64, [40, 3], [9001, 12000])
    run_tree(cuda, type_, 16, 2, 64, 16, [64], [15000])


@TYPES
@pytest.mark.parametrize("nodes", [[1, 2, 4, 0], [150, 1, 66, 9], [20, 12, 30, 9]])
def test_attention_holes_and_empty_rows(cuda, type_, nodes):
    ctx = [400, 33, 70, 12]
    run_tree(cuda, type_, 8, 2, 64, 16, nodes, ctx, holes=0.4, seed=5)
    run_tree(cuda, type_, 8, 2, 128, 5, nodes, ctx, holes=0.4, seed=6, spoil=True)
    run_tree(cuda, type_, 8, 2, 64, 16, nodes, ctx, holes=1.0)  # nothing to see: zeros


@TYPES
@pytest.mark.parametrize("page", [1, 2, 5, 7, 12, 100])
@pytest.mark.parametrize("HD", [64, 96])
def test_attention_odd_pages(cuda, type_, page, HD):
    nodes, ctx = [50, 1, 130, 20], [400, 70, 333, 40]
    run_tree(cuda, type_, 8, 2, HD, page, nodes, ctx, holes=0.3, seed=page)
    run_tree(cuda, type_, 8, 2, HD, page, nodes, ctx, holes=0.3, seed=page, spoil=True)


@TYPES
@pytest.mark.parametrize("n,H,HD", [(6, 4, 64), (40, 8, 128), (140, 8, 128), (100, 2, 64), (20, 8, 48), (9, 2, 256),
                                    (60, 4, 136)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_attention_rows_do_not_see_other_branches(cuda, type_, n, H, HD, what):
    """A node's K and V are not finite: every node but its descendants and itself is as without it."""
    c = 50
    pages, seqs, batch, tree, q, out, scale, table, slots = run_tree(cuda, type_, H, 2, HD, 16, [n], [c])
    sets = ancestors(tree.parents.tolist())
    for bad in (n // 2, 0, n - 1):
        page, at = table[slots[0]][(c + bad) // 16], (c + bad) % 16
        keep = [x[1, page, :, at].clone() for x in (pages.k, pages.v)]
        for x in (pages.k, pages.v):
            x[1, page, :, at] = what
        again = cuda.empty_like(q.contiguous())
        ib.attention_paged(pages, seqs, batch, 1, q, scale, out=again, tree=tree)
        for i in range(n):
            if bad in sets[i]:
                assert not bool(again[i].isfinite().any()), (bad, i)
            else:
                assert cuda.equal(again[i], out[i]), (bad, i)
        for x, y in zip((pages.k, pages.v), keep):
            x[1, page, :, at] = y


@TYPES
def test_attention_bits_of_later_nodes_do_not_count(cuda, type_):
    """Masks of the caller's own: garbage above a node's own bit, and a node that sees nothing."""
    for n, H in ((6, 4), (40, 8), (90, 4)):
        pages, seqs, batch, tree, q, out, scale, table, slots = run_tree(cuda, type_, H, 2, 64, 16, [n], [37], seed=n)
        own = cuda.arange(n, device="cuda")
        words = tree.mask.shape[1]
        keep = cuda.zeros(n, words * 32, dtype=cuda.int64, device="cuda")
        keep[own[:, None] >= cuda.arange(words * 32, device="cuda")[None, :]] = 1
        keep = (keep.view(n, words, 32) << cuda.arange(32, device="cuda")).sum(-1).to(cuda.int32)
        noisy = ib.KVTree(tree.parents, tree.depth, (tree.mask & keep) | ~keep, tree.max_nodes)
        assert cuda.equal(ib.attention_paged(pages, seqs, batch, 1, q, scale, tree=noisy), out)
        none = ib.KVTree(tree.parents, tree.depth, cuda.zeros_like(tree.mask), tree.max_nodes)
        seqs.table.fill_(-1)
        seqs.table[slots[0], 2] = table[slots[0]][2]  # positions 32 .. 47: the tree begins at 37
        seqs.table[slots[0], 2 if n < 16 else 3] = table[slots[0]][3 if n >= 16 else 2]
        got = ib.attention_paged(pages, seqs, batch, 1, q, scale, tree=none)
        assert bool(got.isfinite().all())
        seqs.table.fill_(-1)
        seqs.table[slots[0], 3:] = cuda.tensor(table[slots[0]][3:], dtype=cuda.int32)
        got = ib.attention_paged(pages, seqs, batch, 1, q, scale, tree=none)
        assert not bool(got.any())
    assert ib.check_fault() == 0


@TYPES
def test_attention_wide_range_of_values(cuda, type_):
    run_tree(cuda, type_, 4, 2, 64, 16, [5, 70, 20], [300, 300, 90], q_size=40.0)
    run_tree(cuda, type_, 8, 2, 128, 16, [5, 70, 20], [300, 300, 90], scale=-0.7)
    run_tree(cuda, type_, 8, 2, 128, 16, [5, 70, 20], [300, 300, 90], scale=0.0)


@TYPES
def test_attention_hints_and_workspace_do_not_change_results(cuda, type_):
    for hint in (0, 1, 4, 60, 10 ** 6):  # a wrong hint is slower, not wrong
        run_tree(cuda, type_, 8, 2, 128, 16, [15, 1, 50], [300, 77, 20], max_q=hint)
    run_tree(cuda, type_, 8, 2, 128, 16, [15, 1, 50], [300, 77, 20], max_nodes=1000)
    pages, seqs, batch, tree, q, out, scale, _, _ = run_tree(cuda, type_, 8, 2, 128, 16, [30, 1, 50], [300, 3000, 20])
    ws = ib.attention_paged_workspace(pages, seqs, batch, 8, tree=tree)
    for fill in (0, 255):
        ws.fill_(fill)
        again = cuda.empty_like(out.contiguous())
        ib.attention_paged(pages, seqs, batch, 1, q, scale, out=again, workspace=ws, tree=tree)
        assert cuda.equal(again, out)
    inplace = q.contiguous().clone()
    ib.attention_paged(pages, seqs, batch, 1, inplace, scale, out=inplace, workspace=ws, tree=tree)
    assert cuda.equal(inplace, out)


def test_attention_leaves_out_trees_that_are_too_large(cuda):
    for n, most in ((9, 8), (80, 40)):
        pages, seqs, batch, tree, q, out, scale, _, _ = run_tree(cuda, ib.F16, 8, 2, 64, 16, [4, n], [30, 50])
        small = ib.kv_tree(batch, tree.parents, most)
        with pytest.raises(RuntimeError, match="78"):
            ib.check_fault()
        got = ib.attention_paged(pages, seqs, batch, 1, q, scale, out=cuda.full_like(q.contiguous(), 3.0), tree=small)
        assert bool((got[4:] == 3.0).all())
        assert bool(((got[:4] - out[:4]).abs() <= 2.0 ** -17 * pages.v.abs().max()).all())
        with pytest.raises(RuntimeError, match="78"):
            ib.check_fault()


# ---- verify and accept -----------------------------------------------------------------

def path_of(parents, tokens, best):
    path = [0]
    while True:
        c = next((c for c in range(path[-1] + 1, len(parents))
                  if parents[c] == path[-1] and tokens[c] == best[path[-1]]), None)
        if c is None:
            return path
        path.append(c)


@pytest.mark.parametrize("nodes,pad", [([1], 0), ([5, 0, 33, 64, 1], 3), ([1024, 7], 0), ([40] * 70, 1)])
def test_verify(cuda, nodes, pad):
    for seed, values in enumerate((1, 2, 3, 40)):
        rng = random.Random(seed + len(nodes))
        parents = [random_tree(rng, n, rng.choice([1, 2]), rng.choice([1, 3, 30])) for n in nodes]
        tokens = [[rng.randrange(values) for _ in range(n)] for n in nodes]
        best = [[rng.randrange(values) for _ in range(n)] for n in nodes]
        cu = [0]
        for n in nodes:
            cu.append(cu[-1] + n)
        batch = ib.KVBatch(i32(cuda, cu), cu[-1] + pad)
        out = [cuda.full((m,), 77, dtype=cuda.int32, device="cuda") for m in (cu[-1] + pad, len(nodes), len(nodes))]
        path, n_path, nxt = ib.kv_tree_verify(batch, i32(cuda, flat(parents, pad)), i32(cuda, flat(tokens, pad)),
                                              i32(cuda, flat(best, pad)), *out)
        for b, n in enumerate(nodes):
            want = path_of(parents[b], tokens[b], best[b]) if n else []
            assert path[cu[b]:cu[b] + n].tolist() == want + [-1] * (n - len(want))
            assert n_path[b].item() == len(want) and nxt[b].item() == (best[b][want[-1]] if n else -1)
        assert path[cu[-1]:].tolist() == [77] * pad
    assert ib.check_fault() == 0


def test_verify_of_odd_input(cuda):
    """Parents that are none (their own, later ones) are never followed; sequences left out."""
    parents = [-1, 1, 0, 5, 2, 0]
    batch = ib.KVBatch(i32(cuda, [0, 6, 6, 7]), 7, slots=i32(cuda, [3, 1, -1]))
    path, n_path, nxt = ib.kv_tree_verify(batch, i32(cuda, parents + [-1]), i32(cuda, [4] * 7), i32(cuda, [4] * 7))
    assert path.tolist() == [0, 2, 4, -1, -1, -1, -1] and n_path.tolist() == [3, 0, 0]
    assert nxt.tolist() == [4, -1, -1]
    assert ib.check_fault() == 0
    n = ib.KV_MAX_NODES + 1
    z = cuda.zeros(n, dtype=cuda.int32, device="cuda")
    path, n_path, nxt = ib.kv_tree_verify(ib.KVBatch(i32(cuda, [0, n]), n), z, z, z)
    assert n_path.tolist() == [0] and nxt.tolist() == [-1] and bool((path == -1).all())
    with pytest.raises(RuntimeError, match="78"):
        ib.check_fault()


@TYPES
@pytest.mark.parametrize("layers,Hkv,HD,page,nodes,ctx", [
    (1, 1, 8, 1, [5, 3], [0, 9]), (3, 2, 128, 16, [7, 0, 64, 1, 20], [16, 4, 100, 31, 15]),
    (2, 3, 24, 5, [33, 12], [2, 44]), (40, 8, 128, 64, [40, 40, 40], [5, 64, 200]),
    (2, 1, 256, 7, [300], [10]),
])
def test_accept(cuda, type_, layers, Hkv, HD, page, nodes, ctx):
    rng = random.Random(page)
    total = [c + n for c, n in zip(ctx, nodes)]
    book = Book(len(nodes) + 2, max(-(-t // page) for t in total) + 1, sum(-(-t // page) for t in total) + 9, page)
    slots = rng.sample(range(len(nodes) + 2), len(nodes))
    assert book.extend(slots, total) == [1] * len(nodes)
    seqs = seqs_of(cuda, book)
    pages = pool(cuda, layers, len(book.refs), Hkv, page, HD, type_, 3)
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    paths = [sorted(rng.sample(range(n), rng.randrange(0, n + 1))) if n else [] for n in nodes]
    paths[-1] = [0] + [i for i in range(2, nodes[-1], 3)]
    want = [pages.k.clone(), pages.v.clone()]
    for b, path in enumerate(paths):
        row = book.table[slots[b]]
        for x in want:
            rows = [x[:, row[(ctx[b] + c) // page], :, (ctx[b] + c) % page].clone() for c in path]
            for j, y in enumerate(rows):
                x[:, row[(ctx[b] + j) // page], :, (ctx[b] + j) % page] = y
        if nodes[b]:
            L = ctx[b] + len(path)
            for j in range(-(-L // page), -(-total[b] // page)):
                book.refs[row[j]] -= 1
                row[j] = -1
            book.len[slots[b]] = L
    batch = ib.KVBatch(i32(cuda, cu), cu[-1] + 2, slots=i32(cuda, slots))
    ib.kv_tree_accept(pages, seqs, batch, i32(cuda, [x for n, p in zip(nodes, paths) for x in p + [-1] * (n - len(p))] + [0, 0]),
                      i32(cuda, map(len, paths)))
    assert cuda.equal(pages.k, want[0]) and cuda.equal(pages.v, want[1])
    assert seqs.len.tolist() == book.len and seqs.refs.tolist() == book.refs and seqs.table.tolist() == book.table
    assert ib.check_fault() == 0


def test_accept_passes_over_what_cannot_be(cuda):
    def fresh():
        book = Book(3, 6, 20, 4)
        book.extend([0, 1, 2], [11, 9, 6])
        return book, seqs_of(cuda, book), pool(cuda, 2, 20, 1, 4, 8, ib.F32, 0)

    cu = i32(cuda, [0, 6, 9, 11])

    def run(path, n_path, change=None, slots=None):
        book, seqs, pages = fresh()
        if change:
            change(book, seqs)
        k = pages.k.clone()
        ib.kv_tree_accept(pages, seqs, ib.KVBatch(cu, 11, slots=slots), i32(cuda, path), i32(cuda, n_path))
        return book, seqs, pages, k

    good = [0, 1, -1, -1, -1, -1, 0, -1, -1, 0, 1]
    # n_path that cannot be: nothing changes for that sequence
    for n in (-1, 7):
        book, seqs, pages, k = run(good, [n, 1, 2])
        assert seqs.len.tolist() == [11, 7, 6] and seqs.table[0].tolist() == book.table[0]
        with pytest.raises(RuntimeError, match="78"):
            ib.check_fault()
    # entries that are none of a path end it
    for path, m in (([0, 0, 2], 1), ([0, 6, 2], 1), ([-1, 1, 2], 0), ([0, 3, 2], 2)):
        book, seqs, pages, k = run(path + [-1] * 3 + good[6:], [3, 1, 2])
        assert seqs.len.tolist() == [5 + m, 7, 6]
        with pytest.raises(RuntimeError, match="78"):
            ib.check_fault()
    # left out
    book, seqs, pages, k = run(good, [2, 1, 2], slots=i32(cuda, [-1, 1, -1]))
    assert seqs.len.tolist() == [11, 7, 6] and cuda.equal(k, pages.k) and ib.check_fault() == 0
    book, seqs, pages, k = run(good, [2, 1, 2], slots=i32(cuda, [3, 1, 2]))
    assert seqs.len.tolist() == [11, 7, 6]
    with pytest.raises(RuntimeError, match="71"):
        ib.check_fault()

    # a page that others hold is not written, and its holder keeps it
    def share(book, seqs):
        seqs.refs[book.table[0][1]] = 2

    moved = [1, 3, 5, -1, -1, -1] + good[6:]
    book, seqs, pages, k = run(moved, [3, 1, 2], share)
    assert cuda.equal(k[:, book.table[0][1]], pages.k[:, book.table[0][1]])
    with pytest.raises(RuntimeError, match="77"):
        ib.check_fault()

    # fewer positions than new tokens, a page that is not there, entries that are none
    def short(book, seqs):
        seqs.len[0] = 5

    book, seqs, pages, k = run(moved, [3, 1, 2], short)
    assert seqs.len.tolist() == [5, 7, 6]
    with pytest.raises(RuntimeError, match="73"):
        ib.check_fault()

    def hole(book, seqs):
        seqs.table[0, 1] = -1

    book, seqs, pages, k = run(moved, [3, 1, 2], hole)
    assert seqs.len.tolist() == [8, 7, 6] and ib.check_fault() == 0

    def none(book, seqs):
        seqs.table[0, 2] = 20

    run([0, -1, -1, -1, -1, -1] + good[6:], [1, 1, 2], none)
    with pytest.raises(RuntimeError, match="72"):
        ib.check_fault()


# ---- together --------------------------------------------------------------------------

@TYPES
def test_a_step_captured_and_replayed(cuda, type_):
    """Extend, plan, append, attention, verify and accept in one graph, replayed with other trees and
    lengths, against the same calls made one by one; two graphs of workspaces of their own on two
    streams."""
    H, Hkv, HD, page, n, N = 8, 2, 128, 16, 3, 40
    nodes = [24, 3, 40]
    T = 70
    cu = [0, 24, 27, 67]
    rope = rope_table(cuda, 4000, HD)

    def state(seed):
        rng = random.Random(seed)
        book = Book(n, 100, 400, page)
        book.extend([0, 1, 2], [700, 33, 90])
        gen = cuda.Generator(device="cuda").manual_seed(seed)
        s = dict(seqs=seqs_of(cuda, book), pages=pool(cuda, 2, 400, Hkv, page, HD, type_, seed))
        s["batch"] = ib.KVBatch(i32(cuda, cu), T, max_q=N)
        s["new"], s["slots"] = i32(cuda, nodes), i32(cuda, range(n))
        s["parents"] = cuda.zeros(T, dtype=cuda.int32, device="cuda")
        s["tokens"], s["best"] = cuda.zeros_like(s["parents"]), cuda.zeros_like(s["parents"])
        s["tree"] = ib.KVTree(s["parents"], cuda.zeros_like(s["parents"]),
                              cuda.zeros(T, 2, dtype=cuda.int32, device="cuda"), N)
        s["qkv"] = cuda.randn(T, H + 2 * Hkv, HD, generator=gen, device="cuda")
        s["out"] = cuda.zeros(T, H, HD, device="cuda")
        s["rot"], s["status"] = cuda.zeros_like(s["out"]), cuda.zeros(n, dtype=cuda.int32, device="cuda")
        s["ws"] = ib.attention_paged_workspace(s["pages"], s["seqs"], s["batch"], H, tree=s["tree"])
        s["path"], s["n_path"], s["next"] = (cuda.zeros(m, dtype=cuda.int32, device="cuda") for m in (T, n, n))
        return s

    def draft(s, seed):
        rng = random.Random(seed)
        par = flat([random_tree(rng, m, 1, 4) for m in nodes], T - cu[-1])
        for name, v in (("parents", par), ("tokens", [rng.randrange(2) for _ in range(T)]),
                        ("best", [rng.randrange(2) for _ in range(T)])):
            s[name].copy_(i32(cuda, v))

    def step(s):
        ib.kv_extend(s["pages"], s["seqs"], s["slots"], s["new"], status=s["status"])
        ib.kv_tree(s["batch"], s["parents"], out=s["tree"])
        q, k, v = s["qkv"].split([H, Hkv, Hkv], dim=1)
        ib.kv_append(s["pages"], s["seqs"], s["batch"], 1, q, k, v, rope, q_out=s["rot"], tree=s["tree"])
        ib.attention_paged(s["pages"], s["seqs"], s["batch"], 1, s["rot"], 0.09, out=s["out"], workspace=s["ws"],
                           tree=s["tree"])
        ib.kv_tree_verify(s["batch"], s["parents"], s["tokens"], s["best"], s["path"], s["n_path"], s["next"])
        ib.kv_tree_accept(s["pages"], s["seqs"], s["batch"], s["path"], s["n_path"])

    live, plain, graphs = [state(5), state(6)], [state(5), state(6)], []
    for s in live:
        draft(s, 99)
        side = cuda.cuda.Stream()
        side.wait_stream(cuda.cuda.current_stream())
        before = [s["seqs"].table.clone(), s["seqs"].len.clone(), s["seqs"].refs.clone(), s["pages"].k.clone(),
                  s["pages"].v.clone()]
        with cuda.cuda.stream(side):
            step(s)  # first use outside the capture
        cuda.cuda.synchronize()
        for x, y in zip((s["seqs"].table, s["seqs"].len, s["seqs"].refs, s["pages"].k, s["pages"].v), before):
            x.copy_(y)
        g = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(g, stream=side):
            step(s)
        graphs.append((g, side))
    for i in range(4):
        for a, b, (g, side) in zip(live, plain, graphs):
            draft(a, i)
            draft(b, i)
            side.wait_stream(cuda.cuda.current_stream())
        for g, side in graphs:
            with cuda.cuda.stream(side):
                g.replay()
        for b in plain:
            step(b)
        cuda.cuda.synchronize()
        for a, b in zip(live, plain):
            for x in ("out", "rot", "path", "n_path", "next", "status"):
                assert cuda.equal(a[x], b[x]), (i, x)
            assert a["status"].tolist() == [1] * n
            for x in ("table", "len", "refs"):
                assert cuda.equal(getattr(a["seqs"], x), getattr(b["seqs"], x))
            assert cuda.equal(a["pages"].k, b["pages"].k) and cuda.equal(a["pages"].v, b["pages"].v)
    assert ib.check_fault() == 0


@TYPES
@pytest.mark.parametrize("H,Hkv,HD", [(8, 2, 128), (12, 1, 64), (24, 2, 96)])
def test_attention_at_the_lengths_where_tiles_are_cut(cuda, type_, H, Hkv, HD):
    """Few sequences, so that pieces are as short as they get, of contexts about the shortest one that
    is cut; many short ones, so that pieces hold several tiles."""
    for c in (1, 500, 639, 640, 641, 703, 704, 705, 767, 768, 769, 833, 896, 897, 1025, 1500):
        run_tree(cuda, type_, H, Hkv, HD, 16, [40], [c], seed=c)
    run_tree(cuda, type_, H, Hkv, HD, 16, [30, 41, 27], [700, 6000, 800], seed=4)
    rng = random.Random(HD)
    run_tree(cuda, type_, H, Hkv, HD, 16, [rng.randint(10, 40) for _ in range(150)],
             [rng.choice([0, 3, 100, 300, 900]) for _ in range(150)], seed=5)


@TYPES
@pytest.mark.parametrize("n", [2, 40, 150])
def test_attention_of_sequences_without_positions(cuda, type_, n):
    """A length of zero: the tree's rows see nothing and are zeros, written once."""
    pages, seqs, batch, tree, q, out, scale, _, _ = run_tree(cuda, type_, 8, 2, 64, 16, [n, 5, n], [900, 80, 10])
    slot = batch.slots[2].item()
    before = out.clone()
    seqs.len[slot] = 0
    ib.attention_paged(pages, seqs, batch, 1, q, scale, out=out, tree=tree)
    assert cuda.equal(out[:n + 5], before[:n + 5]) and not bool(out[n + 5:2 * n + 5].any())
    assert ib.check_fault() == 0


@TYPES
def test_a_step_on_a_given_stream(cuda, type_):
    """Every call of a step with stream=, where what it makes itself is of that stream's memory pool."""
    H, Hkv, HD, page, nodes, ctx = 8, 2, 64, 16, [40, 3, 60], [900, 33, 5]
    cu, T = [0, 40, 43, 103], 103
    rope = rope_table(cuda, 2000, HD)
    results = []
    for given in (False, True):
        book = Book(3, 80, 300, page)
        book.extend([0, 1, 2], ctx)
        seqs, pages = seqs_of(cuda, book), pool(cuda, 2, 300, Hkv, page, HD, type_, 3)
        qkv = cuda.randn(T, H + 2 * Hkv, HD, generator=cuda.Generator(device="cuda").manual_seed(1), device="cuda")
        q, k, v = qkv.split([H, Hkv, Hkv], dim=1)
        rng = random.Random(8)
        parents = i32(cuda, flat([random_tree(rng, n) for n in nodes]))
        tokens, best = (i32(cuda, [rng.randrange(2) for _ in range(T)]) for _ in range(2))
        batch, slots = ib.KVBatch(i32(cuda, cu), T, max_q=60), i32(cuda, [0, 1, 2])
        new = i32(cuda, nodes)
        side = cuda.cuda.Stream()
        side.wait_stream(cuda.cuda.current_stream())
        kw = dict(stream=side.cuda_stream) if given else {}
        ib.kv_extend(pages, seqs, slots, new, **kw)
        tree = ib.kv_tree(batch, parents, **kw)
        rot = ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, tree=tree, **kw)
        out = ib.attention_paged(pages, seqs, batch, 1, rot, 0.1, tree=tree, **kw)
        path, n_path, nxt = ib.kv_tree_verify(batch, parents, tokens, best, **kw)
        ib.kv_tree_accept(pages, seqs, batch, path, n_path, **kw)
        cuda.cuda.synchronize()
        results.append([out.clone(), path, n_path, nxt, seqs.table, seqs.len, seqs.refs, pages.k, pages.v])
    for a, b in zip(*results):
        assert cuda.equal(a, b)
    assert ib.check_fault() == 0


def make_long(cuda, rng, page, *args, **kw):
    """As make, with rows of the table for more than 64000 positions: what few trees over short rows
    take another kernel for."""
    seqs, batch, table, slots, n_pages, cu = make_short(cuda, rng, page, *args, **kw)
    more = -(-64001 // page) - len(table[0])
    table = [row + [-1] * more for row in table]
    seqs = ib.KVSeqs(cuda.tensor(table, dtype=cuda.int32, device="cuda"), seqs.len, seqs.refs)
    return seqs, batch, table, slots, n_pages, cu


make_short = make
BRANCHES = [(40, 8, 128), (140, 8, 128), (100, 2, 64), (20, 8, 48), (90, 4, 96)]


@TYPES
@pytest.mark.parametrize("case", ["nan", "inf", "bits", "shapes", "small", "holes", "pages", "values", "groups", "number", "lengths"])
def test_attention_over_long_tables(cuda, type_, case, monkeypatch):
    """The tests above on the kernels that few trees over short tables do not reach."""
    import sys
    monkeypatch.setattr(sys.modules[__name__], "make", make_long)
    if case in ("nan", "inf"):
        for n, H, HD in BRANCHES:
            test_attention_rows_do_not_see_other_branches(cuda, type_, n, H, HD, float(case))
    elif case == "bits":
        test_attention_bits_of_later_nodes_do_not_count(cuda, type_)
    elif case == "shapes":
        test_attention_shapes_of_trees(cuda, type_)
    elif case == "small":
        for shape in SHAPES:
            test_attention_small_trees(cuda, type_, *shape)
            test_attention_large_trees(cuda, type_, *shape)
    elif case == "holes":
        for nodes in ([1, 2, 4, 0], [150, 1, 66, 9], [20, 12, 30, 9], [40, 50, 60, 70]):
            test_attention_holes_and_empty_rows(cuda, type_, nodes)
    elif case == "pages":
        for page in (1, 2, 5, 7, 12, 100):
            test_attention_odd_pages(cuda, type_, page, 96)
    elif case == "values":
        test_attention_wide_range_of_values(cuda, type_)
    elif case == "groups":
        for G in (1, 3, 16):
            test_attention_groups(cuda, type_, G)
    elif case == "number":
        for n in (5, 9, 17, 31, 32, 33, 63, 64, 65, 96, 128, 129):
            test_attention_every_number_of_nodes(cuda, type_, n)
    else:
        for H, Hkv, HD in ((8, 2, 128), (12, 1, 64)):
            for c in (1, 127, 128, 129, 300, 511, 512, 513, 767, 768, 769, 1025):
                run_tree(cuda, type_, H, Hkv, HD, 16, [40], [c], seed=c)
        for n in (2, 40, 150):
            test_attention_of_sequences_without_positions(cuda, type_, n)


@TYPES
@pytest.mark.parametrize("H,Hkv,HD", [(8, 2, 128), (6, 6, 48), (4, 1, 256)])
def test_attention_of_few_rows_however_it_is_cut(cuda, type_, H, Hkv, HD):
    """Few rows over tables of about 192 positions, below which nothing is cut, and about the lengths of one
    and more parts, few trees and many."""
    for page in (1, 16, 64):
        for total in (127, 128, 129, 176, 191, 192, 193, 208, 256, 257):
            run_tree(cuda, type_, H, Hkv, HD, page, [3], [total - 3], seed=total)
    run_tree(cuda, type_, H, Hkv, HD, 16, [2, 4, 1], [1021, 1022, 2100], seed=2)
    run_tree(cuda, type_, H, Hkv, HD, 16, [1 + i % 4 for i in range(90)], [(37 * i) % 1300 for i in range(90)], seed=3)


@TYPES
@pytest.mark.parametrize("HD", [64, 128])
def test_attention_with_empty_sequences_between_others(cuda, type_, HD):
    """Trees whose rows see nothing between trees of queries of very different sizes: one and two in a row,
    one kv head, so that a tile is a sequence, and contexts of two and four key tiles."""
    H, page, n, B = 8, 16, 6, 600
    rng = random.Random(HD)
    empty = [b % 5 in (1, 3, 4) for b in range(B)]
    nodes = [n] * B
    ctx = [rng.choice([rng.randint(123, 250), rng.randint(379, 506)]) for _ in range(B)]
    seqs, batch, table, slots, n_pages, cu = make(cuda, rng, page, nodes, [c + n for c in ctx], 0, True)
    pages = pool(cuda, 2, n_pages, 1, page, HD, type_, 3)
    for b in range(B):
        if empty[b]:
            seqs.len[slots[b]] = 0
    parents = [random_tree(rng, n) for _ in nodes]
    tree = plan_of(cuda, batch, parents, 0, n)
    size = cuda.tensor([2.0 ** rng.randint(-5, 5) for _ in nodes], device="cuda").repeat_interleave(n)
    q = cuda.randn(B * n, H, HD, generator=cuda.Generator(device="cuda").manual_seed(HD), device="cuda")
    q = q * size[:, None, None]
    scale = 1.0 / math.sqrt(HD)
    ref, tol = tree_ref(cuda, pages, 1, table, slots, cu, [0 if e else n for e in empty], ctx, parents, q, scale)
    there = ~ref.isnan()
    for _ in range(20):
        out = ib.attention_paged(pages, seqs, batch, 1, q, scale, out=cuda.full_like(q, 3.0), tree=tree)
        assert bool(((out.double() - ref).abs() <= tol)[there].all())
        assert not bool(out[~there].any())
    assert ib.check_fault() == 0


@TYPES
@pytest.mark.parametrize("max_q", [0, 1, 7, 20])
def test_a_hint_leaves_no_tree_out(cuda, type_, max_q):
    """More nodes in all than one tree may have, with no hint, one that is too small and a right one."""
    nodes, ctx = [20, 0] + [17] * 60, [100, 3] + [(29 * b) % 300 for b in range(60)]
    pages, seqs, batch, tree, q, out, scale, _, _ = run_tree(cuda, type_, 8, 2, 64, 16, nodes, ctx, max_q=20, max_nodes=20)
    batch = ib.KVBatch(batch.cu_q, batch.n_tokens, max_q=max_q, slots=batch.slots)
    other = ib.kv_tree(batch, tree.parents)
    assert cuda.equal(other.depth, tree.depth) and cuda.equal(other.mask[:, :1], tree.mask)
    assert not bool(other.mask[:, 1:].any())
    got = ib.attention_paged(pages, seqs, batch, 1, q, scale, tree=other)
    assert bool(((got - out).abs() <= 2.0 ** -17 * pages.v.abs().max()).all())
    assert ib.check_fault() == 0


@TYPES
@pytest.mark.parametrize("n,most", [(9, 8), (40, 32), (1030, 1024), (1025, 1000)])
def test_a_step_with_a_tree_that_is_too_large(cuda, type_, n, most):
    """Left out of plan, append and attention, it has no path, and nothing of it stays in the cache."""
    H, Hkv, HD, page = 4, 2, 64, 16
    nodes, ctx = [5, n, 7], [30, 50, 11]
    cu, T = [0, 5, 5 + n, 12 + n], 12 + n
    book = Book(3, 90, 200, page)
    book.extend([0, 1, 2], ctx)
    seqs, pages = seqs_of(cuda, book), pool(cuda, 2, 200, Hkv, page, HD, type_, 3)
    k, v = pages.k.clone(), pages.v.clone()
    batch, new = ib.KVBatch(i32(cuda, cu), T), i32(cuda, nodes)
    assert ib.kv_extend(pages, seqs, i32(cuda, [0, 1, 2]), new).tolist() == [1, 1, 1]
    table = seqs.table.clone()
    parents = i32(cuda, [-1, 0, 0, 1, 2] + [i - 1 for i in range(n)] + [-1, 0, 1, 2, 3, 4, 5])
    tokens = i32(cuda, [4] * T)
    tree = ib.kv_tree(batch, parents, most)
    qkv = cuda.randn(T, H + 2 * Hkv, HD, generator=cuda.Generator(device="cuda").manual_seed(1), device="cuda")
    q, kn, vn = qkv.split([H, Hkv, Hkv], dim=1)
    rope = rope_table(cuda, 2000, HD)
    for layer in range(2):
        rot = ib.kv_append(pages, seqs, batch, layer, q, kn, vn, rope, tree=tree)
        out = ib.attention_paged(pages, seqs, batch, layer, rot, 0.1, tree=tree, out=cuda.full((T, H, HD), 3.0, device="cuda"))
        assert bool((out[5:5 + n] == 3.0).all()) and not bool((out[:5] == 3.0).any())
    path, n_path, nxt = ib.kv_tree_verify(batch, parents, tokens, tokens, tree=tree)
    assert n_path.tolist() == [3, 0, 7] and nxt.tolist() == [4, -1, 4]
    assert path.tolist() == [0, 1, 3, -1, -1] + [-1] * n + list(range(7))
    with pytest.raises(RuntimeError, match="78"):
        ib.check_fault()
    mine = n_path.clone()
    mine[1] = 3  # and a path of the caller's own
    path[5:8] = i32(cuda, [0, 1, 2])
    refs = seqs.refs.clone()
    for paths in (n_path, mine):
        seqs.table.copy_(table)
        seqs.refs.copy_(refs)
        seqs.len.copy_(i32(cuda, [c + m for c, m in zip(ctx, nodes)]))
        ib.kv_tree_accept(pages, seqs, batch, path, paths, tree=tree)
        assert seqs.len.tolist() == [33, 50, 18]
        with pytest.raises(RuntimeError, match="78"):
            ib.check_fault()
        kept = [[x if j < -(-L // page) else -1 for j, x in enumerate(row)] for row, L in zip(table.tolist(), (33, 50, 18))]
        assert seqs.table.tolist() == kept
        held = [x for row in kept for x in row if x >= 0]
        assert seqs.refs.tolist() == [int(p in held) for p in range(200)]
    for b in range(3):  # what was there before the step is as it was
        for p in range(ctx[b]):
            at = table[b, p // page].item()
            assert cuda.equal(pages.k[:, at, :, p % page], k[:, at, :, p % page])
            assert cuda.equal(pages.v[:, at, :, p % page], v[:, at, :, p % page])


@TYPES
def test_accept_by_the_counts_before_the_call(cuda, type_):
    """Sequences forked with their nodes: a page that one of the two gives back in the call is not written
    by the other, in any layer."""
    page, ctx, n, pairs = 4, 5, 11, 64
    book = Book(2 * pairs, 4, 4 * pairs + 8, page)
    assert book.extend(range(pairs), [ctx + n] * pairs) == [1] * pairs
    status, copies = book.fork(range(pairs), range(pairs, 2 * pairs))
    assert status == [1] * pairs and not copies
    pages = pool(cuda, 24, 4 * pairs + 8, 2, page, 64, type_, 1)
    k, v = pages.k.clone(), pages.v.clone()
    cu = i32(cuda, range(0, 2 * pairs * n + 1, n))
    long, short = [1, 3, 4, 7, 8, 10], [0]  # entries for pages 1 and 2; 2 and 3 are given back by the others
    path = i32(cuda, [x for p in (long, short) for _ in range(pairs) for x in p + [-1] * (n - len(p))])
    n_path = i32(cuda, [len(long)] * pairs + [len(short)] * pairs)
    for order in (range(2 * pairs), [b // 2 + pairs * (b % 2) for b in range(2 * pairs)]):
        slots = i32(cuda, order)
        seqs = seqs_of(cuda, book)
        batch = ib.KVBatch(cu, 2 * pairs * n, slots=slots)
        rows = slots.long()  # of the lists, which go by slots
        ib.kv_tree_accept(pages, seqs, batch, path.view(-1, n)[rows].flatten().contiguous(), n_path[rows].contiguous())
        assert cuda.equal(pages.k, k) and cuda.equal(pages.v, v)
        with pytest.raises(RuntimeError, match="77"):
            ib.check_fault()
        assert seqs.len.tolist() == [ctx + len(long)] * pairs + [ctx + len(short)] * pairs
        for b in range(2 * pairs):
            keep = 3 if b < pairs else 2
            assert seqs.table[b].tolist() == book.table[b][:keep] + [-1] * (4 - keep)
            held = book.table[b % pairs]
            assert [seqs.refs[p].item() for p in held] == [2, 2, 1, 0]


@TYPES
def test_a_step_without_tokens(cuda, type_):
    """Every sequence left out, or none with a new token: each call of the step is allowed and changes nothing."""
    H, Hkv, HD, page = 4, 2, 64, 16
    book = Book(3, 9, 30, page)
    book.extend([0, 1, 2], [30, 50, 11])
    seqs, pages = seqs_of(cuda, book), pool(cuda, 2, 30, Hkv, page, HD, type_, 3)
    k, v = pages.k.clone(), pages.v.clone()
    none = i32(cuda, [])
    for slots in (None, i32(cuda, [-1, -1, -1])):
        batch = ib.KVBatch(i32(cuda, [0, 0, 0, 0]), 0, slots=slots)
        tree = ib.kv_tree(batch, none)
        q = cuda.zeros(0, H, HD, device="cuda")
        kn = cuda.zeros(0, Hkv, HD, device="cuda")
        ib.kv_append(pages, seqs, batch, 1, q, kn, kn, rope_table(cuda, 100, HD), tree=tree)
        assert ib.attention_paged(pages, seqs, batch, 1, q, 0.1, tree=tree).shape == q.shape
        for kw in ({}, dict(tree=tree)):
            path, n_path, nxt = ib.kv_tree_verify(batch, none, none, none, **kw)
            assert path.numel() == 0 and n_path.tolist() == [0] * 3 and nxt.tolist() == [-1] * 3
            ib.kv_tree_accept(pages, seqs, batch, path, n_path, **kw)
        assert seqs.len.tolist() == book.len and seqs.refs.tolist() == book.refs and seqs.table.tolist() == book.table
    assert cuda.equal(pages.k, k) and cuda.equal(pages.v, v)
    assert ib.check_fault() == 0
