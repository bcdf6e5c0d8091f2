"""The paged KV cache on the GPU: bookkeeping (extend, fork, release, compact), append and
attention, each against a plain restatement (whole numbers in Python, values in 64 bits), and
a serving run of them together against the contiguous cache's operators.

Attention's tolerance, per output element: a product of FP32 operands is kept to 2^-20 of its
size (FP16 or TF32 parts: hi hi + hi lo + lo hi), so a score is off by at most 2^-20 A with
A = scale * sum |q_d k_d| (rounding of its sum and of the exponent's argument included: their
2^-24 parts have random signs).  A weight e^s is then off by 2^-20 A of itself, in numerator
and denominator, the products p v by another 2^-20 and a sum over L positions by sqrt(L) 2^-24:
    |out - ref| <= ((2 A + 1) 2^-20 + sqrt(L) 2^-24) * sum p |v|.
"""
import math
import random

import numpy as np
import pytest

from conftest import load_package

ib = load_package()
pytestmark = pytest.mark.gpu


# ---- a cache in Python -----------------------------------------------------------------

class Book:
    """The bookkeeping's rules, restated on lists."""

    def __init__(self, n_slots, max_pages, n_pages, page):
        self.table = [[-1] * max_pages for _ in range(n_slots)]
        self.len = [0] * n_slots
        self.refs = [0] * n_pages
        self.page, self.max_pages = page, max_pages

    def lowest(self, n):
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        return free[:n] if len(free) >= n else None

    def extend(self, slots, n_new):
        status, seen, short = [], set(), False
        plan = []
        for s, n in zip(slots, n_new):
            if not 0 <= s < len(self.len) or s in seen:
                status.append(-1)
                continue
            seen.add(s)
            if n < 0:
                status.append(-1)
                continue
            L = self.len[s]
            if L + n > self.max_pages * self.page:
                status.append(0)
                continue
            a, b = -(-L // self.page), -(-(L + n) // self.page)
            got = [] if b == a else None if short else self.lowest(b - a)
            if got is None:
                short = True
                status.append(0)
                continue
            for j, p in enumerate(got):
                self.table[s][a + j] = p
                self.refs[p] = 1
            plan.append((s, L + n))
            status.append(1)
        for s, L in plan:
            self.len[s] = L
        return status

    def fork(self, parents, children):
        status, seen, short, copies = [], set(), False, []
        start = list(self.len)
        for p, c in zip(parents, children):
            ok = 0 <= c < len(self.len) and c not in seen
            if 0 <= c < len(self.len):
                seen.add(c)
            if not ok or not 0 <= p < len(self.len) or p == c or start[c] != 0:
                status.append(-1)
                continue
            L = start[p]
            full, part = L // self.page, L % self.page
            last = self.table[p][full] if part else -1
            if last >= 0:
                got = None if short else self.lowest(1)
                if got is None:
                    short = True
                    status.append(0)
                    continue
                self.table[c][full] = got[0]
                self.refs[got[0]] = 1
                copies.append((last, got[0], part))
            status.append(1)
            for j in range(full):
                t = self.table[p][j]
                self.table[c][j] = t
                if t >= 0:
                    self.refs[t] += 1
            self.len[c] = L
        return status, copies

    def release(self, slots):
        for s in slots:
            for j in range(-(-self.len[s] // self.page)):
                t = self.table[s][j]
                if t >= 0:
                    self.refs[t] -= 1
                self.table[s][j] = -1
            self.len[s] = 0

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(live)
        holes = [p for p in range(n) if self.refs[p] <= 0]
        movers = [p for p in live if p >= n]
        to = {p: p for p in live}
        for a, b in zip(movers, holes):
            to[a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(t, -1) if t >= 0 else t for t in row] for row in self.table]
        return n, list(zip(movers, holes)), [to.get(p, -1) for p in range(len(self.refs))]


def i32(cuda, v):
    return cuda.tensor(list(v), dtype=cuda.int32, device="cuda")


def seqs_of(cuda, book):
    return ib.KVSeqs(cuda.tensor(book.table, dtype=cuda.int32, device="cuda"),
                     i32(cuda, book.len), i32(cuda, book.refs))


def same(book, seqs):
    assert seqs.len.tolist() == book.len
    assert seqs.refs.tolist() == book.refs
    assert seqs.table.tolist() == book.table


def pool(cuda, layers, n_pages, Hkv, page, HD, type_, seed, fill=None):
    gen = cuda.Generator(device="cuda").manual_seed(seed)
    pages = ib.KVPages.empty(layers, n_pages, Hkv, page, HD, type_)
    for x in (pages.k, pages.v):
        if fill is None:
            x.copy_(cuda.randn(x.shape, generator=gen, device="cuda"))
        else:
            x.fill_(fill)
    return pages


# ---- bookkeeping -----------------------------------------------------------------------

def test_extend_hands_out_lowest_pages_in_order(cuda):
    book = Book(6, 9, 23, 4)
    for p in (0, 3, 4, 7, 22):
        book.refs[p] = 1
    seqs = seqs_of(cuda, book)
    pages = pool(cuda, 1, 23, 1, 4, 8, ib.F16, 0)
    for slots, new in (([2, 0, 5], [9, 1, 4]), ([0, 0, 2], [3, 1, 0]), ([1, 9, -1, 4], [0, 1, 1, -2]),
                       ([3], [36]), ([3], [37]), ([1, 4, 5], [33, 2, 0]), ([5, 0], [1, 30])):
        want = book.extend(slots, new)
        got = ib.kv_extend(pages, seqs, i32(cuda, slots), i32(cuda, new))
        assert got.tolist() == want, (slots, new)
        same(book, seqs)
    assert ib.check_fault() == 0


@pytest.mark.parametrize("seed", range(4))
def test_bookkeeping_random_runs(cuda, seed):
    rng = random.Random(seed)
    page = [1, 5, 16, 64][seed]
    n_slots, max_pages, n_pages = 40, 30, [300, 500, 9000, 20000][seed]
    book = Book(n_slots, max_pages, n_pages, page)
    seqs = seqs_of(cuda, book)
    pages = pool(cuda, 2, n_pages, 1, page, 8, ib.F16, seed)
    for step in range(40):
        what = rng.choice(["extend", "extend", "fork", "release", "compact"])
        some = [rng.randrange(-1, n_slots + 1) for _ in range(rng.randrange(1, 25))]
        if what == "extend":
            new = [rng.choice([0, 1, rng.randrange(0, 8 * page + 2), -1]) for _ in some]
            want = book.extend(some, new)
            assert ib.kv_extend(pages, seqs, i32(cuda, some), i32(cuda, new)).tolist() == want
        elif what == "fork":
            par = [rng.randrange(0, n_slots) for _ in some]
            k0, v0 = pages.k.clone(), pages.v.clone()
            want, copies = book.fork(par, some)
            assert ib.kv_fork(pages, seqs, i32(cuda, par), i32(cuda, some)).tolist() == want
            for a, b, part in copies:
                k0[:, b, :, :part], v0[:, b, :, :part] = k0[:, a, :, :part], v0[:, a, :, :part]
            assert cuda.equal(k0, pages.k) and cuda.equal(v0, pages.v)
        elif what == "release":
            some = [s for s in some if 0 <= s < n_slots]
            if some:
                book.release(some)
                ib.kv_release(pages, seqs, i32(cuda, some))
        else:
            k0, v0 = pages.k.clone(), pages.v.clone()
            n, moves, to = book.compact()
            plan = ib.kv_compact(pages, seqs)
            assert plan.info.tolist() == [n, len(moves)]
            assert plan.map.tolist() == to
            assert plan.moves.view(-1)[:2 * len(moves)].tolist() == [x for m in moves for x in m]
            for a, b in moves:
                k0[:, b], v0[:, b] = k0[:, a], v0[:, a]
            assert cuda.equal(k0, pages.k) and cuda.equal(v0, pages.v)
        same(book, seqs)
    assert ib.check_fault() == 0


@pytest.mark.parametrize("type_,layers,Hkv,page,HD", [(ib.F32, 3, 2, 5, 24), (ib.F16, 2, 8, 16, 128),
                                                      (ib.F16, 1, 3, 7, 8)])
def test_compact_into_other_arrays_keeps_the_old(cuda, type_, layers, Hkv, page, HD):
    rng = random.Random(page)
    n_pages = 211
    book = Book(9, 20, n_pages, page)
    ids = list(range(n_pages))
    rng.shuffle(ids)
    for s in range(7):
        n = rng.randrange(1, 15)
        for j in range(n):
            book.table[s][j] = ids.pop()
            book.refs[book.table[s][j]] = 1
        book.len[s] = n * page
    book.refs[book.table[2][0]] = 0  # given back early
    book.table[2][0] = -1
    seqs = seqs_of(cuda, book)
    pages = pool(cuda, layers, n_pages, Hkv, page, HD, type_, 5)
    k0, v0 = pages.k.clone(), pages.v.clone()
    before = [t.clone() for t in (seqs.table, seqs.refs)]
    out = ib.KVSeqs(cuda.full_like(seqs.table, 77), seqs.len, cuda.full_like(seqs.refs, 77))
    for _ in range(2):  # the sources keep their bytes: the same call again does the same
        plan = ib.kv_compact(pages, seqs, out=out)
        assert all(cuda.equal(a, b) for a, b in zip(before, (seqs.table, seqs.refs)))
    n, moves, to = book.compact()
    assert plan.info.tolist() == [n, len(moves)] and plan.map.tolist() == to
    assert out.table.tolist() == book.table and out.refs.tolist() == book.refs
    for a, b in moves:
        k0[:, b], v0[:, b] = k0[:, a], v0[:, a]
    assert cuda.equal(k0, pages.k) and cuda.equal(v0, pages.v)


def test_extend_of_a_list_larger_than_a_block(cuda):
    n = 3000
    book = Book(n, 3, 5000, 4)
    seqs, pages = seqs_of(cuda, book), pool(cuda, 1, 5000, 1, 4, 8, ib.F16, 0)
    rng = random.Random(3)
    slots = list(range(n))
    rng.shuffle(slots)
    for _ in range(3):  # the second and third run out of pages on the way
        new = [rng.randrange(0, 6) for _ in slots]
        want = book.extend(slots, new)
        assert ib.kv_extend(pages, seqs, i32(cuda, slots), i32(cuda, new)).tolist() == want
        same(book, seqs)
    assert 0 in want


def test_bookkeeping_records_bad_values(cuda):
    pages = pool(cuda, 1, 10, 1, 4, 8, ib.F16, 0)

    def fresh():
        b = Book(3, 4, 10, 4)
        b.extend([0, 1], [10, 4])
        return b

    def code_after(change, act):
        b = fresh()
        change(b)
        s = seqs_of(cuda, b)
        act(s)
        with pytest.raises(RuntimeError, match="paged KV cache") as e:
            ib.check_fault()
        assert ib.check_fault() == 0  # read and cleared
        return str(e.value)

    one = i32(cuda, [0])
    assert "71" in code_after(lambda b: None, lambda s: ib.kv_release(pages, s, i32(cuda, [3])))

    def bad_entry(b):
        b.table[0][1] = 10

    assert "72" in code_after(bad_entry, lambda s: ib.kv_release(pages, s, one))
    assert "72" in code_after(bad_entry, lambda s: ib.kv_fork(pages, s, one, i32(cuda, [2])))
    assert "72" in code_after(bad_entry, lambda s: ib.kv_compact(pages, s))

    def bad_len(b):
        b.len[0] = 17

    assert "73" in code_after(bad_len, lambda s: ib.kv_extend(pages, s, one, one))

    def bad_refs(b):
        b.refs[b.table[0][0]] = 0

    s = []
    assert "74" in code_after(bad_refs, lambda x: (s.append(x), ib.kv_release(pages, x, one)))
    assert s[0].refs.min().item() >= 0


# ---- append ----------------------------------------------------------------------------

def layout(rng, page, ctx, n_slots, extra_pages=3):
    """(table rows by slot, lens, slots of the batch, pages of the pool)."""
    per = [-(-c // page) for c in ctx]
    n_pages = sum(per) + extra_pages
    ids = list(range(n_pages))
    rng.shuffle(ids)
    slots = list(range(n_slots))
    rng.shuffle(slots)
    slots = slots[:len(ctx)]
    width = max(per + [1]) + 1
    table, lens = [[-1] * width for _ in range(n_slots)], [0] * n_slots
    for b, s in enumerate(slots):
        lens[s] = ctx[b]
        for j in range(per[b]):
            table[s][j] = ids.pop()
    return table, lens, slots, n_pages


def make(cuda, rng, page, q_lens, ctx, pad=0, with_slots=True):
    n = len(ctx)
    table, lens, slots, n_pages = layout(rng, page, ctx, n + 2 if with_slots else n)
    if not with_slots:
        order = sorted(range(n), key=lambda b: slots[b])
        slots, inv = list(range(n)), [slots[b] for b in range(n)]
        table, lens = [table[s] for s in inv], [lens[s] for s in inv]
        del order
    refs = [0] * n_pages
    for row in table:
        for t in row:
            if t >= 0:
                refs[t] += 1
    seqs = ib.KVSeqs(cuda.tensor(table, dtype=cuda.int32, device="cuda"), i32(cuda, lens),
                     i32(cuda, refs))
    cu = [0]
    for x in q_lens:
        cu.append(cu[-1] + x)
    batch = ib.KVBatch(i32(cuda, cu), cu[-1] + pad, max_q=max(q_lens + [0]),
                       slots=i32(cuda, slots) if with_slots else None)
    return seqs, batch, table, slots, n_pages, cu


def rope_table(cuda, n, HD):
    pos = np.arange(n)[:, None] * 500000.0 ** (-np.arange(HD // 2) * 2.0 / HD)[None, :]
    return cuda.from_numpy(np.stack([np.cos(pos), np.sin(pos)], -1).astype(np.float32)).cuda()


@pytest.mark.parametrize("type_", [ib.F32, ib.F16], ids=["f32", "f16"])
@pytest.mark.parametrize("H,Hkv,HD,page,q_lens,ctx,pad,sl", [
    (4, 2, 128, 16, [1, 1, 1], [1, 16, 17], 0, True),
    (6, 6, 48, 7, [3, 0, 9, 1], [3, 5, 40, 14], 4, True),
    (8, 1, 8, 1, [5, 2], [9, 2], 0, False),
    (3, 3, 256, 100, [250], [333], 7, False),
    (2, 1, 64, 24, [4, 3, 2], [2, 3, 0], 1, True),  # more new tokens than positions
    (1, 1, 16, 16, [1] * 70, list(range(1, 71)), 3, True),
])
def test_append(cuda, type_, H, Hkv, HD, page, q_lens, ctx, pad, sl):
    rng = random.Random(HD + page)
    seqs, batch, table, slots, n_pages, cu = make(cuda, rng, page, q_lens, ctx, pad, sl)
    pages = pool(cuda, 2, n_pages, Hkv, page, HD, type_, 9)
    T = batch.n_tokens
    gen = cuda.Generator(device="cuda").manual_seed(4)
    qkv = cuda.randn(T, H + 2 * Hkv, HD, generator=gen, device="cuda")
    q, k, v = qkv.split([H, Hkv, Hkv], dim=1)
    rope = rope_table(cuda, max(ctx + [1]), HD)
    want_k, want_v = pages.k.double().clone(), pages.v.double().clone()
    want_q = cuda.full((T, H, HD), 7.0, dtype=cuda.float64, device="cuda")
    size_k, size_q = want_k.abs(), want_q.abs()
    dt = pages.k.dtype
    for b, s in enumerate(slots):
        for i in range(q_lens[b]):
            t, pos = cu[b] + i, ctx[b] - q_lens[b] + i
            if pos < 0:
                continue
            c, sn = rope[pos, :, 0].double(), rope[pos, :, 1].double()
            x = qkv[t, :H + Hkv].double()
            y, size = cuda.empty_like(x), cuda.empty_like(x)
            y[:, 0::2] = x[:, 0::2] * c - x[:, 1::2] * sn
            y[:, 1::2] = x[:, 0::2] * sn + x[:, 1::2] * c
            size[:, 0::2] = size[:, 1::2] = x[:, 0::2].abs() + x[:, 1::2].abs()
            page_id = table[s][pos // page]
            want_q[t], size_q[t] = y[:H], size[:H]
            want_k[1, page_id, :, pos % page] = y[H:]
            size_k[1, page_id, :, pos % page] = size[H:]
            want_v[1, page_id, :, pos % page] = v[t].to(dt).double()
    out = cuda.full((T, H, HD), 7.0, device="cuda")
    ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, q_out=out)
    # two products and their sum: three FP32 roundings of at most |x0| + |x1|; FP16 pages add
    # half a step of the rounded value (and of the subnormal spacing)
    f32 = 3 * 2.0 ** -24
    assert bool(((out.double() - want_q).abs() <= f32 * size_q).all())
    half = 2.0 ** -11 if dt == cuda.float16 else 0.0
    tol = f32 * size_k * (1 + half) + half * want_k.abs() + (2.0 ** -25 if half else 0.0)
    assert bool(((pages.k.double() - want_k).abs() <= tol).all())
    assert cuda.equal(pages.v.double(), want_v)
    # in place, as a slice of the projection
    before = qkv.clone()
    ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, q_out=q)
    own = [t for b in range(len(ctx)) for i in range(q_lens[b])
           for t in [cu[b] + i] if ctx[b] - q_lens[b] + i >= 0]
    for t in range(T):
        assert cuda.equal(q[t], out[t] if t in own else before[t, :H])
    assert cuda.equal(qkv[:, H:], before[:, H:])
    assert ib.check_fault() == 0


def test_append_matches_the_contiguous_operators(cuda):
    H, Hkv, HD, page, T, start = 8, 2, 64, 16, 37, 21
    gen = cuda.Generator(device="cuda").manual_seed(1)
    q, k, v = (cuda.randn(T, h, HD, generator=gen, device="cuda") for h in (H, Hkv, Hkv))
    rope = rope_table(cuda, 64, HD)
    qc, kc_in = q.clone(), k.clone()
    ib.rope_batch(qc, kc_in, rope, H, Hkv, HD, start, T)
    kc, vc = cuda.zeros(Hkv, 64, HD, device="cuda"), cuda.zeros(Hkv, 64, HD, device="cuda")
    ib.kv_write_batch(kc, vc, kc_in, v, Hkv, HD, 64, start, T)
    pages = pool(cuda, 1, 4, Hkv, page, HD, ib.F32, 0, fill=0.0)
    table = i32(cuda, [2, 0, 3, 1]).view(1, 4)
    seqs = ib.KVSeqs(table, i32(cuda, [start + T]), i32(cuda, [1] * 4))
    out = ib.kv_append(pages, seqs, ib.KVBatch(i32(cuda, [0, T]), T), 0, q, k, v, rope)
    gather = [pages.k[0, table[0].long()].transpose(0, 1).reshape(Hkv, 64, HD),
              pages.v[0, table[0].long()].transpose(0, 1).reshape(Hkv, 64, HD)]
    # the rotation's two products may be contracted differently: one rounding of |x0| + |x1|
    for a, b in ((out, qc), (gather[0], kc)):
        assert bool(((a - b).abs() <= 2.0 ** -22 * (b.abs().max())).all())
    assert cuda.equal(gather[1], vc)


def test_append_passes_over_what_has_no_place(cuda):
    pages = pool(cuda, 1, 4, 1, 4, 8, ib.F32, 0, fill=1.0)
    x = cuda.full((3, 1, 8), 5.0, device="cuda")
    rope = rope_table(cuda, 8, 8)
    # the first token's page was given back: its q is rotated, nothing is written for it
    seqs = ib.KVSeqs(i32(cuda, [1, -1, 2]).view(1, 3), i32(cuda, [8]), i32(cuda, [0, 1, 1, 0]))
    out = cuda.zeros_like(x)
    batch = ib.KVBatch(i32(cuda, [0, 3]), 3)
    ib.kv_append(pages, seqs, batch, 0, x, x, x, rope, q_out=out)
    assert bool((pages.v == 1).all()) and bool((out != 0).any(-1).all())
    assert ib.check_fault() == 0
    # positions behind the table of rotations
    seqs.len.fill_(10)
    out.zero_()
    ib.kv_append(pages, seqs, batch, 0, x, x, x, rope, q_out=out)
    assert bool((out[0] != 0).any()) and not bool((out[1:] != 0).any())
    assert not bool((pages.v == 5).any())
    with pytest.raises(RuntimeError, match="75"):
        ib.check_fault()
    # a table entry that is no page
    seqs.table.copy_(i32(cuda, [1, 4, -7]).view(1, 3))
    seqs.len.fill_(8)
    ib.kv_append(pages, seqs, batch, 0, x, x, x, rope, q_out=out)
    assert bool((pages.v == 1).all())
    with pytest.raises(RuntimeError, match="72"):
        ib.check_fault()
    # a batch whose rows do not fit, and a slot that is none
    ib.kv_append(pages, seqs, ib.KVBatch(i32(cuda, [0, 4]), 3), 0, x, x, x, rope, q_out=out)
    with pytest.raises(RuntimeError, match="73"):
        ib.check_fault()
    ib.kv_append(pages, seqs, ib.KVBatch(i32(cuda, [0, 3]), 3, slots=i32(cuda, [1])), 0, x, x, x,
                 rope, q_out=out)
    with pytest.raises(RuntimeError, match="71"):
        ib.check_fault()


# ---- attention -------------------------------------------------------------------------

def attention_ref(cuda, pages, layer, table, slots, cu, q_lens, ctx, q, scale):
    """(out, tolerance) in 64 bits; rows of nobody are NaN in out."""
    H, HD = q.shape[1], q.shape[2]
    Hkv, page = pages.n_kv_heads, pages.page_size
    G = H // Hkv
    f8 = cuda.float64
    out = cuda.full(q.shape, float("nan"), dtype=f8, device="cuda")
    tol = cuda.zeros(q.shape, dtype=f8, device="cuda")
    for b, s in enumerate(slots):
        n, c = q_lens[b], ctx[b]
        if n == 0:
            continue
        pos = [p for p in range(c) if table[s][p // page] >= 0]
        rows = slice(cu[b], cu[b] + n)
        if not pos:
            out[rows] = 0
            continue
        ids = cuda.tensor([table[s][p // page] for p in pos], device="cuda")
        at = cuda.tensor([p % page for p in pos], device="cuda")
        pos = cuda.tensor(pos, device="cuda")
        k = pages.k[layer][ids, :, at].to(f8)      # [positions, Hkv, HD]
        v = pages.v[layer][ids, :, at].to(f8)
        seen = pos[None, :] <= cuda.arange(c - n, c, device="cuda")[:, None]
        for h in range(H):
            kk, vv, qq = k[:, h // G], v[:, h // G], q[rows, h].to(f8)
            sc = (qq @ kk.nan_to_num(0, 0, 0).t() * scale).masked_fill(~seen, -math.inf)
            A = (qq.abs() @ kk.nan_to_num(0, 0, 0).abs().t() * abs(scale))
            A = A.masked_fill(~seen, 0).amax(1, keepdim=True)
            top = sc.amax(1, keepdim=True).clamp(min=-1e300)
            p = cuda.exp(sc - top)
            l = p.sum(1, keepdim=True)
            p = cuda.where(l > 0, p / l, cuda.zeros_like(p))
            vv = vv.nan_to_num(0, 0, 0)
            out[rows, h] = p @ vv
            tol[rows, h] = ((2 * A + 1) * 2.0 ** -20 + math.sqrt(c) * 2.0 ** -24) * (p @ vv.abs())
    return out, tol


def run_attention(cuda, type_, H, Hkv, HD, page, q_lens, ctx, pad=0, with_slots=True, holes=0.0,
                  seed=0, spoil=False, max_q=None, q_size=1.5, scale=None):
    rng = random.Random(seed + HD * 7 + page)
    seqs, batch, table, slots, n_pages, cu = make(cuda, rng, page, q_lens, ctx, pad, with_slots)
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
        for s, n in zip(slots, ctx):
            for p in range(n):
                if table[s][p // page] >= 0:
                    held[table[s][p // page], p % page] = True
        bad = cuda.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")
        for x in (pages.k, pages.v):
            fill = bad[cuda.randint(0, 3, x.shape, device="cuda")].to(x.dtype)
            x.copy_(cuda.where(held[None, :, None, :, None], x, fill))
    T = batch.n_tokens
    gen = cuda.Generator(device="cuda").manual_seed(seed + 2)
    scale = 1.0 / math.sqrt(HD) if scale is None else scale
    buf = q_size * cuda.randn(T, H + 2 * Hkv, HD, generator=gen, device="cuda")
    q = buf[:, :H]  # rows apart
    obuf = cuda.full((T, H + 1, HD), 3.0, device="cuda")
    out = obuf[:, :H]
    ib.attention_paged(pages, seqs, batch, 1, q, scale, out=out)
    ref, tol = attention_ref(cuda, pages, 1, table, slots, cu, q_lens, ctx, q, scale)
    mine = ~ref.isnan()
    err = (out.double() - ref).abs()
    worst = (err / tol.clamp(min=1e-300))[mine & (tol > 0)]
    assert bool((err <= tol)[mine].all()), \
        f"{worst.max().item() if worst.numel() else err[mine].max().item()} of the tolerance"
    assert bool((out[~mine] == 3.0).all()) and bool((obuf[:, H] == 3.0).all())
    assert ib.check_fault() == 0
    return pages, seqs, batch, q, out, scale


TYPES = pytest.mark.parametrize("type_", [ib.F32, ib.F16], ids=["f32", "f16"])
SHAPES = [(6, 6, 48, 16), (32, 8, 128, 16), (32, 4, 64, 24), (4, 4, 8, 1), (8, 1, 256, 64),
          (7, 1, 80, 100), (24, 2, 96, 7), (16, 8, 136, 32), (5, 5, 16, 128)]


@TYPES
@pytest.mark.parametrize("H,Hkv,HD,page", SHAPES)
def test_attention_single_tokens(cuda, type_, H, Hkv, HD, page):
    ctx = [1, 2, 15, 16, 17, 63, 64, 65, 130, 700]
    run_attention(cuda, type_, H, Hkv, HD, page, [1] * len(ctx), ctx, pad=2)


@TYPES
@pytest.mark.parametrize("H,Hkv,HD,page", SHAPES)
def test_attention_chunks(cuda, type_, H, Hkv, HD, page):
    run_attention(cuda, type_, H, Hkv, HD, page, [1, 33, 0, 5, 130, 64], [500, 33, 9, 66, 401, 64],
                  pad=5)


@TYPES
@pytest.mark.parametrize("H,Hkv,HD,page", [(32, 8, 128, 16), (32, 4, 64, 24), (8, 8, 48, 5)])
def test_attention_long_chunk(cuda, type_, H, Hkv, HD, page):
    run_attention(cuda, type_, H, Hkv, HD, page, [517, 1, 300], [1500, 3001, 300])


@TYPES
@pytest.mark.parametrize("q_len", [1, 2, 3, 4, 5, 8, 16, 17, 31, 64, 65, 128, 129, 257])
def test_attention_every_number_of_new_tokens(cuda, type_, q_len):
    run_attention(cuda, type_, 8, 2, 64, 16, [q_len, q_len], [q_len, q_len + 190])


@TYPES
def test_attention_one_long_sequence_is_split(cuda, type_):
    run_attention(cuda, type_, 8, 2, 128, 64, [1], [20001])
    run_attention(cuda, type_, 8, 2, 128, 64, [70], [9001])


@TYPES
@pytest.mark.parametrize("q_lens", [[1, 1, 4, 0], [150, 1, 66, 9]])
def test_attention_holes_and_empty_rows(cuda, type_, q_lens):
    ctx = [400, 33, 70, 12]
    run_attention(cuda, type_, 8, 2, 64, 16, q_lens, ctx, holes=0.4, seed=5)
    run_attention(cuda, type_, 8, 2, 64, 16, q_lens, ctx, holes=1.0)  # nothing to see: zeros
    # more new tokens than positions: the first rows see nothing
    run_attention(cuda, type_, 8, 2, 128, 16, [9, 200, 3], [5, 130, 0], pad=1)


@TYPES
@pytest.mark.parametrize("page", [1, 2, 5, 7, 12, 100])
@pytest.mark.parametrize("HD", [64, 96])
def test_attention_odd_pages_with_holes(cuda, type_, page, HD):
    q_lens, ctx = [150, 1, 300, 40], [400, 70, 333, 40]
    run_attention(cuda, type_, 8, 2, HD, page, q_lens, ctx, holes=0.3, seed=page)
    run_attention(cuda, type_, 8, 2, HD, page, q_lens, ctx, holes=0.3, seed=page, spoil=True)


@TYPES
@pytest.mark.parametrize("q_lens", [[1, 1, 4], [150, 1, 66]])
def test_attention_ignores_what_no_sequence_holds(cuda, type_, q_lens):
    run_attention(cuda, type_, 8, 2, 128, 24, q_lens, [400, 33, 70], holes=0.3, spoil=True)


@TYPES
@pytest.mark.parametrize("n,H,HD", [(6, 4, 64), (140, 8, 128), (300, 2, 64), (40, 8, 48)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_attention_rows_do_not_see_later_positions(cuda, type_, n, H, HD, what):
    """The last token's K and V are not finite: every row before it is as without it."""
    ctx = n + 50
    pages, seqs, batch, q, out, scale = run_attention(cuda, type_, H, 2, HD, 16, [n], [ctx])
    slot = batch.slots[0].item()
    page = seqs.table[slot, (ctx - 1) // 16].item()
    for x in (pages.k, pages.v):
        x[1, page, :, (ctx - 1) % 16] = what
    again = cuda.empty_like(q.contiguous())
    ib.attention_paged(pages, seqs, batch, 1, q, scale, out=again)
    assert cuda.equal(again[:n - 1], out[:n - 1])
    assert not bool(again[n - 1].isfinite().any())


@TYPES
def test_attention_wide_range_of_values(cuda, type_):
    """Large scores (one position takes everything) and values far from 1."""
    H, Hkv, HD, page = 4, 2, 64, 16
    run_attention(cuda, type_, H, Hkv, HD, page, [1, 70], [300, 300], q_size=40.0)
    for size in (1e-4, 3e3):
        rng = random.Random(1)
        seqs, batch, table, slots, n_pages, cu = make(cuda, rng, page, [1, 70], [300, 200])
        pages = pool(cuda, 2, n_pages, Hkv, page, HD, type_, 3)
        pages.k.mul_(size)
        pages.v.mul_(1 / size)
        q = cuda.randn(71, H, HD, device="cuda") / size
        out = ib.attention_paged(pages, seqs, batch, 1, q, 0.125)
        ref, tol = attention_ref(cuda, pages, 1, table, slots, cu, [1, 70], [300, 200], q, 0.125)
        assert bool(((out.double() - ref).abs() <= tol).all()), size


@TYPES
@pytest.mark.parametrize("HD", [64, 128])
def test_attention_diagonal_over_several_key_tiles(cuda, type_, HD):
    """Without groups a tile's 256 rows see the ends of two and more key tiles in a row, all of
    which are looked through for values that are not finite."""
    for _ in range(3):
        run_attention(cuda, type_, 8, 8, HD, 16, [900, 40, 700], [1500, 2000, 700], spoil=True)
        run_attention(cuda, type_, 2, 2, HD, 128, [3000], [3100], spoil=True)


def test_attention_fp32_pages_past_the_fp16_range(cuda):
    rng = random.Random(1)
    seqs, batch, table, slots, n_pages, cu = make(cuda, rng, 16, [1, 70], [300, 200])
    for size in (1e9, 1e-9):
        pages = pool(cuda, 2, n_pages, 2, 16, 64, ib.F32, 3)
        pages.k.mul_(size)
        pages.v.mul_(size)
        q = cuda.randn(71, 4, 64, device="cuda") / size
        out = ib.attention_paged(pages, seqs, batch, 1, q, 0.125)
        ref, tol = attention_ref(cuda, pages, 1, table, slots, cu, [1, 70], [300, 200], q, 0.125)
        assert bool(((out.double() - ref).abs() <= tol).all()), size


@TYPES
def test_attention_hint_and_workspace_do_not_change_results(cuda, type_):
    H, Hkv, HD = 8, 2, 128
    for hint in (0, 1, 4, 200, 10 ** 6):  # a wrong hint is slower, not wrong
        run_attention(cuda, type_, H, Hkv, HD, 16, [150, 1, 20], [300, 77, 20], max_q=hint)
    a = run_attention(cuda, type_, H, Hkv, HD, 16, [150, 1, 20], [300, 3000, 20])
    pages, seqs, batch, q, out, scale = a
    ws = ib.attention_paged_workspace(pages, seqs, batch, H)
    for fill in (0, 255):  # it needs no initial value, and nothing is kept in it
        ws.fill_(fill)
        again = cuda.empty_like(out.contiguous())
        ib.attention_paged(pages, seqs, batch, 1, q, scale, out=again, workspace=ws)
        assert cuda.equal(again, out)


@TYPES
def test_attention_captured_and_replayed_with_other_lengths(cuda, type_):
    """One graph serves step after step: table, lengths and cu_q are read at replay."""
    H, Hkv, HD, page, n = 8, 2, 64, 16, 5
    book = Book(n, 80, 400, page)
    seqs = seqs_of(cuda, book)
    pages = pool(cuda, 2, 400, Hkv, page, HD, type_, 3)
    one = i32(cuda, [1] * n)
    first = [3, 16, 700, 64, 1000]
    slots = i32(cuda, range(n))
    ib.kv_extend(pages, seqs, slots, i32(cuda, first))
    batch = ib.KVBatch(i32(cuda, range(n + 1)), n, max_q=1)
    q = cuda.randn(n, H, HD, device="cuda")
    out = cuda.zeros(n, H, HD, device="cuda")
    status = cuda.zeros(n, dtype=cuda.int32, device="cuda")
    rope = rope_table(cuda, 80 * page, HD)
    kv = cuda.randn(n, 2 * Hkv, HD, device="cuda")
    rot = cuda.empty_like(q)

    def step(ws):
        ib.kv_extend(pages, seqs, slots, one, status=status)
        ib.kv_append(pages, seqs, batch, 1, q, kv[:, :Hkv], kv[:, Hkv:], rope, q_out=rot)
        ib.attention_paged(pages, seqs, batch, 1, rot, 0.125, out=out, workspace=ws)

    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.stream(side):
        ws = ib.attention_paged_workspace(pages, seqs, batch, H)
        step(ws)
        side.synchronize()
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=side):
            step(ws)
        for i in range(20):
            q.normal_()
            kv.normal_()
            graph.replay()
    side.synchronize()
    lens = [x + 21 for x in first]
    assert seqs.len.tolist() == lens and status.tolist() == [1] * n
    ref, tol = attention_ref(cuda, pages, 1, seqs.table.tolist(), list(range(n)),
                             list(range(n + 1)), [1] * n, lens, rot, 0.125)
    assert bool(((out.double() - ref).abs() <= tol).all())
    assert ib.check_fault() == 0


def test_attention_on_two_streams_at_once(cuda):
    jobs = []
    for i, (q_lens, ctx) in enumerate([([1] * 8, [3000] * 8), ([200, 90], [900, 1200])]):
        jobs.append(run_attention(cuda, ib.F16, 8, 2, 128, 16, q_lens, ctx, seed=i))
    streams = [cuda.cuda.Stream() for _ in jobs]
    outs = [[] for _ in jobs]
    cuda.cuda.synchronize()
    for _ in range(10):
        for i, (pages, seqs, batch, q, _, scale) in enumerate(jobs):
            with cuda.cuda.stream(streams[i]):
                outs[i].append(ib.attention_paged(pages, seqs, batch, 1, q, scale))
    # and on a stream named by its handle, from another current stream
    for i, (pages, seqs, batch, q, _, scale) in enumerate(jobs):
        o = cuda.zeros(q.shape, device="cuda")
        streams[i].wait_stream(cuda.cuda.current_stream())
        ib.attention_paged(pages, seqs, batch, 1, q, scale, out=o,
                           stream=streams[i].cuda_stream)
        outs[i].append(o)
    cuda.cuda.synchronize()
    for i, job in enumerate(jobs):
        assert all(cuda.equal(o, job[4]) for o in outs[i])


@TYPES
@pytest.mark.parametrize("n,H,Hkv,HD", [(700, 4, 1, 64), (1100, 2, 2, 128)])
def test_attention_many_sequences(cuda, type_, n, H, Hkv, HD):
    """More sequences than a planning CTA has threads, of every kind side by side."""
    rng = random.Random(n)
    q_lens = [rng.choice([0, 1, 1, 1, 2, 8, 9, 40]) for _ in range(n)]
    ctx = [x + rng.choice([0, 1, 30, 200]) for x in q_lens]
    q_lens[n - 3], ctx[n - 3] = 330, 700
    run_attention(cuda, type_, H, Hkv, HD, 16, q_lens, ctx, pad=3, seed=n)
    q_lens = [min(x, 2) for x in q_lens]
    run_attention(cuda, type_, H, Hkv, HD, 16, q_lens, ctx, pad=3, seed=n)


@TYPES
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30, -4.0])
def test_attention_scales(cuda, type_, scale):
    run_attention(cuda, type_, 8, 2, 64, 16, [1, 90, 3], [70, 300, 40], scale=scale)


@TYPES
@pytest.mark.parametrize("H,Hkv,HD", [(71, 1, 64), (33, 1, 128), (99, 3, 40), (300, 1, 8)])
def test_attention_large_groups(cuda, type_, H, Hkv, HD):
    run_attention(cuda, type_, H, Hkv, HD, 16, [1], [900])
    run_attention(cuda, type_, H, Hkv, HD, 16, [1, 0, 2, 7], [300, 5, 2, 130])


@TYPES
def test_attention_in_place(cuda, type_):
    for q_lens, ctx in (([1] * 9, [2000] * 9), ([400], [2000]), ([300, 1, 5], [700, 900, 1000])):
        pages, seqs, batch, q, out, scale = run_attention(cuda, type_, 8, 2, 128, 16, q_lens, ctx)
        for _ in range(3):
            x = q.clone()
            assert ib.attention_paged(pages, seqs, batch, 1, x, scale, out=x) is x
            assert cuda.equal(x, out)


@TYPES
def test_attention_mixed_batch_in_a_graph(cuda, type_):
    """The kernels of a mixed batch overlap; what is around them in the graph does not."""
    pages, seqs, batch, q, out, scale = run_attention(
        cuda, type_, 8, 2, 128, 16, [260, 1, 1, 5, 90, 1], [900, 4000, 33, 2500, 90, 1000])
    ws = ib.attention_paged_workspace(pages, seqs, batch, 8)
    x, y = cuda.empty_like(q.contiguous()), cuda.zeros(q.shape, device="cuda")
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.stream(side):
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=side):
            total = cuda.zeros_like(y)
            for i in range(3):  # one workspace, one after the other
                x.copy_(q)
                y.fill_(-1)
                ib.attention_paged(pages, seqs, batch, 1, x, scale, out=y, workspace=ws)
                x.zero_()
                total += y
        for _ in range(5):
            graph.replay()
    side.synchronize()
    assert cuda.equal(y, out) and cuda.equal(total, out + out + out)


def test_calls_on_another_stream_make_their_tensors_there(cuda):
    """What a call allocates and clears itself belongs to the stream that it runs on."""
    pages, seqs, batch, q, out, scale = run_attention(cuda, ib.F16, 8, 2, 64, 16, [3, 1], [50, 90])
    other = cuda.cuda.Stream()
    for i in range(2):  # memory of both streams to be handed out again (a new piece waits)
        got = ib.attention_paged(pages, seqs, batch, 1, q, scale, stream=other.cuda_stream)
        more = ib.attention_paged(pages, seqs, batch, 1, q, scale)
        cuda.cuda.synchronize()
        del got, more
    cuda.cuda._sleep(50_000_000)  # the current stream is busy for some 25 ms
    got = ib.attention_paged(pages, seqs, batch, 1, q, scale, stream=other.cuda_stream)
    cuda.cuda.synchronize()
    assert cuda.equal(got, out)
    slots = i32(cuda, [batch.slots[0].item()])
    kv = cuda.randn(4, 2, 64, device="cuda")
    rope = rope_table(cuda, 128, 64)
    want = ib.kv_append(pages, seqs, batch, 0, q, kv, kv, rope)
    none = cuda.zeros_like(slots)
    cuda.cuda.synchronize()
    cuda.cuda._sleep(50_000_000)
    new = ib.kv_append(pages, seqs, batch, 0, q, kv, kv, rope, stream=other.cuda_stream)
    status = ib.kv_extend(pages, seqs, slots, none, stream=other.cuda_stream)
    plan = ib.kv_compact(pages, seqs, stream=other.cuda_stream)
    trash = [cuda.full_like(t, 5) for t in (new, status, plan.map) for _ in range(4)]
    cuda.cuda.synchronize()
    assert cuda.equal(new, want) and status.tolist() == [1] and len(trash) == 12
    assert plan.info[0].item() == int((seqs.refs > 0).sum())


def test_attention_records_bad_values_and_reads_nothing_there(cuda):
    for q_len in (1, 100):
        pages, seqs, batch, q, out, scale = run_attention(cuda, ib.F16, 8, 2, 64, 16, [q_len], [300])
        slot = batch.slots[0].item()
        row = seqs.table[slot].clone()
        for bad in (2 ** 31 - 1, pages.n_pages, -2, -2 ** 31):
            seqs.table[slot, 3] = bad
            got = ib.attention_paged(pages, seqs, batch, 1, q, scale)
            with pytest.raises(RuntimeError, match="72"):
                ib.check_fault()
            seqs.table[slot, 3] = -1
            assert cuda.equal(got, ib.attention_paged(pages, seqs, batch, 1, q, scale))
        seqs.table[slot] = row
        seqs.len[slot] = 2 ** 31 - 1  # taken as a full row: the entries behind are -1
        ib.attention_paged(pages, seqs, batch, 1, q, scale)
        with pytest.raises(RuntimeError, match="73"):
            ib.check_fault()
        seqs.len[slot] = -5
        assert not bool(ib.attention_paged(pages, seqs, batch, 1, q, scale).any())
        with pytest.raises(RuntimeError, match="73"):
            ib.check_fault()
        seqs.len[slot] = 300
        for cu in ([0, q_len + 1], [-1, q_len], [2 ** 31 - 1, -2 ** 31], [5, 3]):
            ib.attention_paged(pages, seqs, ib.KVBatch(i32(cuda, cu), q_len, slots=batch.slots), 1,
                               q, scale)
            with pytest.raises(RuntimeError, match="73"):
                ib.check_fault()
        ib.attention_paged(pages, seqs, ib.KVBatch(i32(cuda, [0, q_len]), q_len,
                                                   slots=i32(cuda, [2 ** 30])), 1, q, scale)
        with pytest.raises(RuntimeError, match="71"):
            ib.check_fault()


@pytest.mark.parametrize("q_len", [1, 90])
def test_attention_pool_past_32_bit_offsets(cuda, q_len):
    """Pages whose elements lie past 2^32 of the layer's first."""
    H, Hkv, HD, page = 8, 8, 128, 128
    n_pages = 2 ** 32 // (Hkv * HD * page) + 9
    pages = ib.KVPages.empty(1, n_pages, Hkv, page, HD, ib.F16)
    rows = [[n_pages - 1, 0, n_pages - 5], [n_pages - 3, n_pages - 8, 2]]
    for row in rows:
        for t in row:
            pages.k[0, t].normal_()
            pages.v[0, t].normal_()
    seqs = ib.KVSeqs(cuda.tensor(rows, dtype=cuda.int32, device="cuda"), i32(cuda, [300, 257]),
                     cuda.ones(n_pages, dtype=cuda.int32, device="cuda"))
    q = cuda.randn(2 * q_len, H, HD, device="cuda")
    cu = [0, q_len, 2 * q_len]
    out = ib.attention_paged(pages, seqs, ib.KVBatch(i32(cuda, cu), 2 * q_len, max_q=q_len), 0, q,
                             0.09)
    ref, tol = attention_ref(cuda, pages, 0, rows, [0, 1], cu, [q_len] * 2, [300, 257], q, 0.09)
    assert bool(((out.double() - ref).abs() <= tol).all())
    x = cuda.randn(2 * q_len, Hkv, HD, device="cuda")
    ib.kv_append(pages, seqs, ib.KVBatch(i32(cuda, cu), 2 * q_len), 0, q, x, x,
                 rope_table(cuda, 300, HD))
    assert cuda.equal(pages.v[0, n_pages - 5, :, 300 - 257], x[q_len - 1].half())
    assert ib.check_fault() == 0


# ---- refusals --------------------------------------------------------------------------

def test_refusals(cuda):
    pages, seqs, batch, q, out, scale = run_attention(cuda, ib.F16, 8, 2, 64, 16, [3], [20])

    def refused(match, f, *a, **k):
        with pytest.raises((ValueError, RuntimeError), match=match):
            f(*a, **k)

    att = ib.attention_paged
    refused("dtype|float32", att, pages, seqs, batch, 1, q.half(), scale)
    refused("shape", att, pages, seqs, batch, 1, q[:2], scale)
    refused("shape", att, pages, seqs, batch, 1, q[:, :, :32], scale)
    refused("multiple of n_kv_heads", att, pages, seqs, batch, 1, q[:, :7], scale)
    refused("contiguous", att, pages, seqs, batch, 1, q.transpose(1, 2).contiguous().transpose(1, 2),
            scale)
    refused("layer", att, pages, seqs, batch, 2, q, scale)
    refused("layer", att, pages, seqs, batch, -1, q, scale)
    refused("cpu", att, pages, seqs, batch, 1, q.cpu(), scale)
    refused("workspace", att, pages, seqs, batch, 1, q, scale,
            workspace=cuda.empty(16, dtype=cuda.uint8, device="cuda"))
    odd = cuda.empty(3 * 8 * 64 + 1, device="cuda")[1:].view(3, 8, 64)
    refused("aligned", att, pages, seqs, batch, 1, odd, scale)
    refused("slots", att, pages, ib.KVSeqs(seqs.table[:1], seqs.len[:1], seqs.refs),
            ib.KVBatch(i32(cuda, [0, 1, 2, 3]), 3), 1, q, scale)
    refused("refs", att, pages, ib.KVSeqs(seqs.table, seqs.len, seqs.refs[:1]), batch, 1, q, scale)
    refused("head_dim", att, ib.KVPages(*[cuda.zeros(2, 4, 2, 16, 12, device="cuda")] * 2), ib.KVSeqs(
        seqs.table, seqs.len, seqs.refs[:4]), batch, 1, q[:, :, :12].contiguous(), scale)
    refused("dtype", ib.KVPages, q.bfloat16(), q.bfloat16())
    refused("shape", ib.KVPages, pages.k, pages.v[:1])
    refused("contiguous", ib.KVPages, pages.k.transpose(2, 3), pages.v.transpose(2, 3))
    refused("dtype", ib.KVBatch, batch.cu_q.long(), 3)
    refused("dtype", ib.kv_release, pages, seqs, batch.cu_q.long())
    refused("shape", ib.kv_extend, pages, seqs, i32(cuda, [0, 1]), i32(cuda, [1]))
    rope = rope_table(cuda, 20, 64)
    kv = cuda.zeros(3, 2, 64, device="cuda")
    refused("shape", ib.kv_append, pages, seqs, batch, 1, q, kv[:, :1], kv, rope)
    refused("shape", ib.kv_append, pages, seqs, batch, 1, q, kv, kv, rope[:, :16])
    # nothing to do is fine
    ib.kv_release(pages, seqs, i32(cuda, []))
    ib.kv_extend(pages, seqs, i32(cuda, []), i32(cuda, []))
    ib.kv_fork(pages, seqs, i32(cuda, []), i32(cuda, []))
    e = cuda.zeros(0, 8, 64, device="cuda")
    assert att(pages, seqs, ib.KVBatch(i32(cuda, [0]), 0), 1, e, scale).shape == e.shape
    assert ib.check_fault() == 0


# ---- together --------------------------------------------------------------------------

@TYPES
def test_a_serving_run(cuda, type_):
    """Prompts in chunks, single tokens, a fork, a release and a compaction, step after step
    in one pool; every step's attention is that of the contiguous operators on the sequence's
    own cache."""
    H, Hkv, HD, page, n_slots, MAX = 8, 2, 64, 16, 6, 400
    layers, layer = 2, 1
    scale = 1.0 / math.sqrt(HD)
    pages = pool(cuda, layers, 90, Hkv, page, HD, type_, 1, fill=float("nan"))
    seqs = ib.KVSeqs.empty(n_slots, MAX // page, 90)
    rope = rope_table(cuda, MAX, HD)
    dt = cuda.float32 if type_ == ib.F32 else cuda.float16
    flat = {}  # slot -> contiguous caches, rounded as the pages are
    gen = cuda.Generator(device="cuda").manual_seed(5)

    def step(work):  # [(slot, new tokens)]
        slots = i32(cuda, [s for s, _ in work])
        assert ib.kv_extend(pages, seqs, slots, i32(cuda, [n for _, n in work])).tolist() == \
            [1] * len(work)
        cu = [0]
        for _, n in work:
            cu.append(cu[-1] + n)
        T = cu[-1]
        batch = ib.KVBatch(i32(cuda, cu), T, slots=slots)
        qkv = cuda.randn(T, H + 2 * Hkv, HD, generator=gen, device="cuda")
        q, k, v = qkv.split([H, Hkv, Hkv], dim=1)
        rot = ib.kv_append(pages, seqs, batch, layer, q, k, v, rope)
        out = ib.attention_paged(pages, seqs, batch, layer, rot, scale)
        for b, (s, n) in enumerate(work):
            kc, vc, start = flat.get(s, (cuda.zeros(Hkv, MAX, HD, device="cuda"),
                                         cuda.zeros(Hkv, MAX, HD, device="cuda"), 0))
            rows = slice(cu[b], cu[b] + n)
            qq, kk = q[rows].contiguous(), k[rows].contiguous()
            ib.rope_batch(qq, kk, rope, H, Hkv, HD, start, n)
            ib.kv_write_batch(kc, vc, kk.to(dt).float(), v[rows].to(dt).float().contiguous(), Hkv,
                              HD, MAX, start, n)
            flat[s] = (kc, vc, start + n)
            want = cuda.empty(n, H, HD, device="cuda")
            ib.attention_batch(qq, kc, vc, want, H, Hkv, HD, MAX, start, n, scale)
            # both keep about 2^-20 of each product (the note above, A < 16); a rotated k that
            # the two round differently before FP16 is one FP16 step of one element apart
            tol = 2e-4 if type_ == ib.F32 else 2e-3
            assert bool(((out[rows] - want).abs() <= tol).all())

    step([(0, 70), (3, 1), (5, 33)])
    step([(0, 30), (5, 1), (3, 16)])
    assert ib.kv_fork(pages, seqs, i32(cuda, [0, 0]), i32(cuda, [1, 4])).tolist() == [1, 1]
    for c in (1, 4):
        flat[c] = (flat[0][0].clone(), flat[0][1].clone(), flat[0][2])
    step([(1, 1), (0, 2), (4, 5), (3, 1)])
    ib.kv_release(pages, seqs, i32(cuda, [5, 0]))
    del flat[5], flat[0]
    step([(4, 1), (1, 1), (0, 50)])
    ib.kv_release(pages, seqs, i32(cuda, [0]))
    del flat[0]
    used = seqs.refs > 0
    above = int(used[int(used.sum()):].sum())
    plan = ib.kv_compact(pages, seqs)
    assert int(plan.n_moves) == above > 0
    assert seqs.refs[:int(plan.n_live)].min().item() > 0
    step([(0, 1), (1, 1), (3, 1), (4, 1)])
    step([(2, 200), (1, 1)])
    ib.kv_release(pages, seqs, i32(cuda, range(n_slots)))
    assert not bool(seqs.refs.any()) and bool((seqs.table == -1).all())
    assert ib.check_fault() == 0


# ---- the largest FP32 values -------------------------------------------------------------

LARGEST = 3.4028234663852886e38  # every FP32 value within 2^-12 of it rounds up in TF32


@pytest.mark.parametrize("n,H,HD", [(6, 4, 64), (140, 8, 128), (300, 2, 64), (40, 8, 48), (5, 4, 256),
                                    (90, 4, 256)])
@pytest.mark.parametrize("what", [LARGEST, -LARGEST, 3.4023e38])
def test_attention_rows_do_not_see_later_largest_values(cuda, n, H, HD, what):
    """The last token's K and V are the type's largest: every row before it is as without it."""
    ctx = n + 50
    pages, seqs, batch, q, out, scale = run_attention(cuda, ib.F32, H, 2, HD, 16, [n], [ctx])
    page = seqs.table[batch.slots[0].item(), (ctx - 1) // 16].item()
    for x in (pages.k, pages.v):
        x[1, page, :, (ctx - 1) % 16] = what
    again = cuda.empty_like(q.contiguous())
    ib.attention_paged(pages, seqs, batch, 1, q, scale, out=again)
    assert cuda.equal(again[:n - 1], out[:n - 1])


@pytest.mark.parametrize("HD", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 70])
def test_attention_of_the_largest_values(cuda, n, HD):
    """Seen values of that size are kept like any other: q, K and V at the top of the range, in
    products that stay in it."""
    rng = random.Random(n)
    ctx = n + 20
    seqs, batch, table, slots, n_pages, cu = make(cuda, rng, 16, [n], [ctx])
    gen = cuda.Generator(device="cuda").manual_seed(n)

    def check(pages, q, scale):
        out = ib.attention_paged(pages, seqs, batch, 1, q, scale)
        ref, tol = attention_ref(cuda, pages, 1, table, slots, cu, [n], [ctx], q, scale)
        assert bool(out.isfinite().all()) and bool(((out.double() - ref).abs() <= tol).all())

    # K: one component of the largest size against a q whose products stay in range
    pages = pool(cuda, 2, n_pages, 2, 16, HD, ib.F32, 3)
    sign = cuda.randn(pages.k.shape[:-1], generator=gen, device="cuda").sign()
    pages.k.zero_()
    pages.k[..., 3] = sign * LARGEST
    q = cuda.zeros(n, 4, HD, device="cuda")
    q[..., 3] = cuda.rand(n, 4, generator=gen, device="cuda") * 2.0 ** -100
    check(pages, q, 2.0 ** -27)
    # q: the same the other way round
    pages.k[..., 3] = sign * 2.0 ** -100
    q[..., 3] = LARGEST
    check(pages, q, 2.0 ** -27)
    # V: the first position takes the weight, with products that cannot add up past the range
    pages = pool(cuda, 2, n_pages, 2, 16, HD, ib.F32, 3)
    pages.k.zero_()
    pages.k[1, table[slots[0]][0], :, 0, 0] = 100.0
    pages.v[1, table[slots[0]][0], :, 0] = LARGEST * cuda.randn(2, HD, generator=gen, device="cuda").sign()
    q = cuda.zeros(n, 4, HD, device="cuda")
    q[..., 0] = 2.0
    check(pages, q, 1.0)
    assert ib.check_fault() == 0


# ---- sequences that got no room ------------------------------------------------------------

def test_granted(cuda):
    pages = pool(cuda, 1, 4, 1, 4, 8, ib.F16, 0)
    slots, status = list(range(700)), [(i * 7) % 3 - 1 for i in range(700)]
    want = [s if st == 1 else -1 for s, st in zip(slots, status)]
    a = i32(cuda, slots)
    assert ib.kv_granted(pages, a, i32(cuda, status)).tolist() == want
    assert a.tolist() == slots
    assert ib.kv_granted(pages, a, i32(cuda, status), out=a) is a and a.tolist() == want
    assert ib.kv_granted(pages, i32(cuda, []), i32(cuda, [])).tolist() == []
    with pytest.raises(ValueError, match="shape"):
        ib.kv_granted(pages, a, i32(cuda, [1]))
    with pytest.raises(ValueError, match="dtype"):
        ib.kv_granted(pages, a, a.long())


@TYPES
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [9, 130, 1, 40], [40, 300, 64, 90]])
def test_a_step_leaves_out_what_got_no_room(cuda, type_, q_lens):
    """Entry 1 and the last of a step get no room: whatever kernel takes the step, their cache
    and their rows stay as they were, and the others' are as in a step without them."""
    H, Hkv, HD, page = 8, 2, 64, 16
    first = [50, 33, 70, 20]
    book = Book(4, 40, 60, page)
    assert book.extend(range(4), first) == [1] * 4
    seqs = seqs_of(cuda, book)
    pages = pool(cuda, 2, 60, Hkv, page, HD, type_, 3)
    slots = i32(cuda, [2, 0, 3, 1])  # entry b is slot slots[b]
    status = i32(cuda, [1, 0, 1, -1])
    grow = [n if st == 1 else 0 for n, st in zip(q_lens, [1, 0, 1, -1])]
    assert book.extend([2, 0, 3, 1], grow) == [1] * 4
    seqs = seqs_of(cuda, book)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    T = cu[-1]
    granted = ib.kv_granted(pages, slots, status)
    batch = ib.KVBatch(i32(cuda, cu), T, max_q=max(q_lens), slots=granted)
    gen = cuda.Generator(device="cuda").manual_seed(7)
    qkv = cuda.randn(T, H + 2 * Hkv, HD, generator=gen, device="cuda")
    q, k, v = qkv.split([H, Hkv, Hkv], dim=1)
    rope = rope_table(cuda, 640, HD)
    k0, v0 = pages.k.clone(), pages.v.clone()
    rot = ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, q_out=cuda.full_like(q, 3.0))
    out = ib.attention_paged(pages, seqs, batch, 1, rot, 0.125, out=cuda.full_like(q, 5.0))
    for b in (1, 3):
        rows = slice(cu[b], cu[b + 1])
        assert bool((rot[rows] == 3).all()) and bool((out[rows] == 5).all())
        for t in book.table[[2, 0, 3, 1][b]]:
            if t >= 0:
                assert cuda.equal(pages.k[:, t], k0[:, t]) and cuda.equal(pages.v[:, t], v0[:, t])
    # the same step of entries 0 and 2 alone
    keep = cuda.cat([cuda.arange(cu[b], cu[b + 1], device="cuda") for b in (0, 2)])
    n0 = q_lens[0]
    pages2 = ib.KVPages(k0, v0)
    batch2 = ib.KVBatch(i32(cuda, [0, n0, n0 + q_lens[2]]), n0 + q_lens[2],
                        max_q=max(n0, q_lens[2]), slots=i32(cuda, [2, 3]))
    rot2 = ib.kv_append(pages2, seqs, batch2, 1, q[keep], k[keep], v[keep], rope)
    assert cuda.equal(rot2, rot[keep])
    assert cuda.equal(pages2.k, pages.k) and cuda.equal(pages2.v, pages.v)
    ctx = [book.len[2], book.len[3]]
    ref, tol = attention_ref(cuda, pages, 1, book.table, [2, 3], [0, n0, n0 + q_lens[2]],
                             [n0, q_lens[2]], ctx, rot2, 0.125)
    assert bool(((out[keep].double() - ref).abs() <= tol).all())
    assert ib.check_fault() == 0


def test_a_captured_step_whose_pool_runs_out(cuda):
    """Forks share their prefix; step after step of one graph the pool runs out for one after the
    other.  Nothing that a sequence has stored changes, and every length is what was granted."""
    H, Hkv, HD, page, n_pages = 4, 2, 32, 4, 14
    book = Book(5, 16, n_pages, page)
    book.extend([0], [10])  # pages 0 .. 2
    seqs, pages = seqs_of(cuda, book), pool(cuda, 1, n_pages, Hkv, page, HD, ib.F32, 1)
    children = [1, 2, 3, 4]
    want, copies = book.fork([0] * 4, children)
    assert want == [1] * 4
    status = ib.kv_fork(pages, seqs, i32(cuda, [0] * 4), i32(cuda, children))
    slots = ib.kv_granted(pages, i32(cuda, children), status)
    ones, status = i32(cuda, [1] * 4), i32(cuda, [0] * 4)
    granted = i32(cuda, [0] * 4)
    batch = ib.KVBatch(i32(cuda, range(5)), 4, max_q=1, slots=granted)
    x = cuda.zeros(4, H + 2 * Hkv, HD, device="cuda")
    rope = rope_table(cuda, 64, HD)
    out = cuda.zeros(4, H, HD, device="cuda")

    def step(ws, new=ones):
        ib.kv_extend(pages, seqs, slots, new, status=status)
        ib.kv_granted(pages, slots, status, out=granted)
        q = ib.kv_append(pages, seqs, batch, 0, x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], rope)
        ib.attention_paged(pages, seqs, batch, 0, q, 0.2, out=out, workspace=ws)

    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    kept = [[] for _ in range(5)]  # V rows that each child has stored
    short = 0
    with cuda.cuda.stream(side):
        ws = ib.attention_paged_workspace(pages, seqs, batch, H)
        step(ws, new=i32(cuda, [-1] * 4))  # refused, all of it: nothing changes
        side.synchronize()
        same(book, seqs)
        assert status.tolist() == granted.tolist() == [-1] * 4 and not bool(out.any())
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=side):
            step(ws)
        for i in range(30):
            x.fill_(i + 1.0)
            out.fill_(-1.0)
            graph.replay()
            side.synchronize()
            got = book.extend(children, [1] * 4)
            assert status.tolist() == got
            same(book, seqs)
            for j, c in enumerate(children):
                assert bool((out[j] == -1).all()) == (got[j] != 1)
                if got[j] == 1:
                    kept[c].append(i + 1.0)
                else:
                    short += 1
                for p, val in enumerate(kept[c], start=10):
                    t = book.table[c][p // page]
                    assert bool((pages.v[0, t, :, p % page] == val).all())
    assert 0 < short < 120
    assert ib.check_fault() == 0


@TYPES
def test_append_never_writes_a_shared_page(cuda, type_):
    """A step that ignores the status of an extend without room: the sequence's last tokens are
    taken for the new ones, but pages that forks share keep what they hold, and it is recorded."""
    H, Hkv, HD, page = 4, 2, 32, 4
    book = Book(3, 4, 4, page)
    assert book.extend([0], [8]) == [1]
    assert book.fork([0, 0], [1, 2])[0] == [1, 1]
    assert book.extend([1], [8]) == [1]  # the last free pages
    assert book.extend([2], [3]) == [0]
    seqs, pages = seqs_of(cuda, book), pool(cuda, 2, 4, Hkv, page, HD, type_, 2)
    k0, v0 = pages.k.clone(), pages.v.clone()
    x = cuda.randn(3, H + 2 * Hkv, HD, device="cuda")
    q, k, v = x.split([H, Hkv, Hkv], dim=1)
    rope = rope_table(cuda, 16, HD)
    batch = ib.KVBatch(i32(cuda, [0, 3]), 3, slots=i32(cuda, [2]))
    out = ib.kv_append(pages, seqs, batch, 1, q, k, v, rope, q_out=cuda.zeros_like(q))
    assert cuda.equal(pages.k, k0) and cuda.equal(pages.v, v0) and bool(out.any(-1).all())
    with pytest.raises(RuntimeError, match="held by other sequences.*77"):
        ib.check_fault()
    # its own pages are written
    batch = ib.KVBatch(i32(cuda, [0, 3]), 3, slots=i32(cuda, [1]))
    ib.kv_append(pages, seqs, batch, 1, q, k, v, rope)
    t = book.table[1][3]
    assert cuda.equal(pages.v[1, t, :, 1:4], v.to(pages.v.dtype).transpose(0, 1))
    assert ib.check_fault() == 0


def test_an_expired_wait_is_not_hidden_by_bad_values(cuda):
    """Results are missing after an expired wait: it is reported before values that were passed
    over, whichever kernel recorded them and in whatever order, and named as attention's."""
    pages, seqs = pool(cuda, 1, 4, 1, 4, 8, ib.F16, 0), ib.KVSeqs.empty(2, 2, 4)

    def bad_slot():
        ib.kv_release(pages, seqs, i32(cuda, [7]))

    def wait():  # records a bad table entry first
        ib.call("ib_kv_wait_selftest", None)

    for acts in ([wait], [bad_slot, wait], [wait, bad_slot]):
        for act in acts:
            act()
        with pytest.raises(RuntimeError, match="attention_paged.*76"):
            ib.check_fault()
        assert ib.check_fault() == 0  # all of it read and cleared
    bad_slot()
    with pytest.raises(RuntimeError, match="slot was out of range.*71"):
        ib.check_fault()
    assert ib.check_fault() == 0


def test_compact_into_sequences_with_lengths_of_their_own(cuda):
    """The second half of a double buffer: what the call leaves in `out` is a whole cache."""
    book = Book(4, 6, 20, 4)
    for s, n in ((0, 9), (1, 16), (2, 5), (3, 21)):
        book.extend([s], [n])
    book.release([1])
    seqs, pages = seqs_of(cuda, book), pool(cuda, 1, 20, 1, 4, 8, ib.F16, 1)
    old = [t.clone() for t in (seqs.table, seqs.len, seqs.refs)]
    book.compact()
    out = ib.KVSeqs.empty(4, 6, 20)
    ib.kv_compact(pages, seqs, out=out)
    same(book, out)
    assert all(cuda.equal(a, b) for a, b in zip(old, (seqs.table, seqs.len, seqs.refs)))
    # the same on a stream of its own, while the current one is busy
    other, again = cuda.cuda.Stream(), ib.KVSeqs.empty(4, 6, 20)
    plan = ib.kv_compact_plan(pages)
    cuda.cuda.synchronize()
    cuda.cuda._sleep(50_000_000)
    ib.kv_compact(pages, seqs, out=again, plan=plan, stream=other.cuda_stream)
    other.synchronize()
    with cuda.cuda.stream(other):
        same(book, again)
    cuda.cuda.synchronize()
    assert ib.check_fault() == 0


# ---- head_dim above 128: kernels of its own --------------------------------------------------

WIDE_HD = pytest.mark.parametrize("H,Hkv,HD", [(8, 2, 136), (4, 2, 256), (3, 3, 200), (16, 1, 256)])


@TYPES
@WIDE_HD
def test_large_head_dim_holes_and_spoiled_memory(cuda, type_, H, Hkv, HD):
    for page in (1, 7, 16, 100):
        q_lens, ctx = [150, 1, 40, 9, 0, 3], [700, 300, 333, 12, 5, 65]
        run_attention(cuda, type_, H, Hkv, HD, page, q_lens, ctx, pad=2, holes=0.3, seed=page,
                      spoil=True)
    run_attention(cuda, type_, H, Hkv, HD, 16, [1, 60, 4], [400, 90, 12], holes=1.0)
    # more new tokens than positions: the first rows see nothing
    run_attention(cuda, type_, H, Hkv, HD, 16, [9, 200, 3], [5, 130, 0], pad=1)


@TYPES
@WIDE_HD
def test_large_head_dim_cut_over_many_pieces(cuda, type_, H, Hkv, HD):
    run_attention(cuda, type_, H, Hkv, HD, 32, [300], [2500], spoil=True)
    run_attention(cuda, type_, H, Hkv, HD, 16, [1], [9001])
    run_attention(cuda, type_, H, Hkv, HD, 16, [1] * 40, [50 * i + 1 for i in range(40)])
    run_attention(cuda, type_, H, Hkv, HD, 24, [257, 1, 33, 1, 8], [900, 4000, 33, 2500, 1000])


@TYPES
@pytest.mark.parametrize("n,H,HD", [(6, 4, 256), (140, 8, 136), (90, 4, 256), (40, 8, 200)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_large_head_dim_rows_do_not_see_later_positions(cuda, type_, n, H, HD, what):
    test_attention_rows_do_not_see_later_positions(cuda, type_, n, H, HD, what)


@TYPES
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30, -4.0])
@pytest.mark.parametrize("HD", [136, 256])
def test_large_head_dim_scales(cuda, type_, scale, HD):
    run_attention(cuda, type_, 8, 2, HD, 16, [1, 90, 3], [70, 300, 40], scale=scale)


@TYPES
@pytest.mark.parametrize("HD", [136, 256])
def test_large_head_dim_in_place_hints_and_workspace(cuda, type_, HD):
    for q_lens, ctx in (([1] * 9, [2000] * 9), ([400], [2000]), ([300, 1, 5], [700, 900, 1000])):
        pages, seqs, batch, q, out, scale = run_attention(cuda, type_, 8, 2, HD, 16, q_lens, ctx)
        ws = ib.attention_paged_workspace(pages, seqs, batch, 8)
        for fill in (0, 255):
            ws.fill_(fill)
            x = q.clone()
            assert ib.attention_paged(pages, seqs, batch, 1, x, scale, out=x, workspace=ws) is x
            assert cuda.equal(x, out)
    for hint in (0, 1, 4, 200, 10 ** 6):
        run_attention(cuda, type_, 8, 2, HD, 16, [150, 1, 20], [300, 77, 20], max_q=hint)


@TYPES
@pytest.mark.parametrize("HD", [136, 256])
def test_large_head_dim_mixed_batch_in_a_graph(cuda, type_, HD):
    pages, seqs, batch, q, out, scale = run_attention(
        cuda, type_, 8, 2, HD, 16, [260, 1, 1, 5, 90, 1], [900, 4000, 33, 2500, 90, 1000])
    ws = ib.attention_paged_workspace(pages, seqs, batch, 8)
    x, y = cuda.empty_like(q.contiguous()), cuda.zeros(q.shape, device="cuda")
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.stream(side):
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=side):
            total = cuda.zeros_like(y)
            for i in range(3):
                x.copy_(q)
                y.fill_(-1)
                ib.attention_paged(pages, seqs, batch, 1, x, scale, out=y, workspace=ws)
                x.zero_()
                total += y
        for _ in range(5):
            graph.replay()
    side.synchronize()
    assert cuda.equal(y, out) and cuda.equal(total, out + out + out)
    assert ib.check_fault() == 0


@TYPES
@pytest.mark.parametrize("HD", [136, 256])
def test_large_head_dim_bad_values(cuda, type_, HD):
    for q_len in (1, 100):
        pages, seqs, batch, q, out, scale = run_attention(cuda, type_, 8, 2, HD, 16, [q_len], [300])
        slot = batch.slots[0].item()
        for bad in (2 ** 31 - 1, pages.n_pages, -2, -2 ** 31):
            seqs.table[slot, 3] = bad
            got = ib.attention_paged(pages, seqs, batch, 1, q, scale)
            with pytest.raises(RuntimeError, match="72"):
                ib.check_fault()
            seqs.table[slot, 3] = -1
            assert cuda.equal(got, ib.attention_paged(pages, seqs, batch, 1, q, scale))
        assert ib.check_fault() == 0
