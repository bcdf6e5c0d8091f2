"""Beam search over the paged cache: the selection over beams and vocabulary against its definition in
64 bits, and the reordering of the beams' states against its rules on lists.

Tolerance of a score, in units of 2^-24 (a rounding of FP32): the result is rounded once (|v|); of the
log sum, a weight e^(x - m) has a rounded argument, |x - m| of the weight, which the weights average to
at most A = sum p (max x - x), and expf's 2 of its steps (4); a thread adds 16 weights in a step of 4096
values and rescales its sum once, by a factor with the same errors as a weight (16 + 4 + 2, and A
again); S steps at most:  |score - ref| <= (|v| + (S + 1) (A + 24)) 2^-24."""
import math
import random

import numpy as np
import pytest

from conftest import load_package
from test_gpu_paged import Book, i32, pool, same, seqs_of

ib = load_package()
pytestmark = pytest.mark.gpu


# ---- selection -------------------------------------------------------------------------

def want_of(logits, scores, ended, beams, k, end_token):
    """(score, token, row, tolerance) in 64 bits; logits a numpy array of its own type."""
    x = logits.astype(np.float64)
    rows, V = x.shape
    steps = -(-V // 4096)
    res = []
    with np.errstate(all="ignore"):
        for g in range(rows // beams):
            cand = []
            for r in range(g * beams, (g + 1) * beams):
                s = 0.0 if scores is None else float(scores[r])
                if ended is not None and ended[r]:
                    if s > -math.inf:
                        cand.append((-s, r, end_token, 0.0))
                    continue
                m = x[r].max()
                e = np.exp(x[r] - m)
                total = e.sum()
                v = s - np.log(total) + (x[r] - m)
                if not np.isfinite(total) or not s > -math.inf:
                    continue
                A = float(np.nansum(e * np.where(np.isfinite(x[r]), m - x[r], 0)) / total)
                few = np.argsort(-x[r], kind="stable")[:k]
                cand += [(-v[t], r, int(t), A) for t in few if x[r, t] > -math.inf]
            cand.sort(key=lambda c: c[:3])
            cand = cand[:k]
            res.append([[-c[0] for c in cand] + [-math.inf] * (k - len(cand)),
                        [c[2] for c in cand] + [-1] * (k - len(cand)),
                        [c[1] for c in cand] + [-1] * (k - len(cand)),
                        [(abs(c[0]) + (steps + 1) * (c[3] + 24)) * 2.0 ** -24 for c in cand] + [0.0] * (k - len(cand))])
    return [np.array([r[i] for r in res]) for i in range(4)]


def check(cuda, logits, scores=None, ended=None, beams=1, k=None, end_token=0, exact_places=True, **kw):
    out = ib.beam_select(logits, scores, beams=beams, k=k, ended=ended, end_token=end_token, **kw)
    cpu = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    score, token, row, tol = want_of(cpu(logits), cpu(scores), cpu(ended), beams, k or beams, end_token)
    got = cpu(out.score).astype(np.float64)
    assert (np.isneginf(got) == np.isneginf(score)).all()
    fine = np.isfinite(score)
    err = np.abs(got[fine] - score[fine])
    assert (err <= tol[fine]).all(), (err / tol[fine]).max()
    if exact_places:
        assert (cpu(out.token) == token).all() and (cpu(out.row) == row).all()
    assert ib.check_fault() == 0
    return out


def random_logits(cuda, rows, vocab, dt, seed, stride=0, size=2.5):
    gen = cuda.Generator(device="cuda").manual_seed(seed)
    x = size * cuda.randn(rows, stride or vocab, generator=gen, device="cuda")
    return x.to(dt)[:, :vocab]


DT = pytest.mark.parametrize("dt", ["float32", "float16"])


@DT
@pytest.mark.parametrize("groups,beams,vocab,k,stride", [
    (1, 1, 1, 1, 0), (1, 1, 1, 4, 0), (2, 3, 2, 3, 0), (1, 4, 32000, 4, 0), (3, 5, 4095, 5, 4101),
    (2, 2, 4096, 8, 0), (2, 2, 4097, 9, 0), (5, 8, 32003, 16, 32011), (1, 1, 128256, 128, 0), (300, 1, 257, 1, 0),
    (7, 16, 1000, 32, 1001), (1, 64, 5000, 64, 0), (2, 1, 152064, 40, 0), (40, 1, 31, 40, 33), (1, 1024, 300, 5, 0),
    (1, 2, 9000, 127, 0)])
def test_select(cuda, dt, groups, beams, vocab, k, stride):
    dt = getattr(cuda, dt)
    x = random_logits(cuda, groups * beams, vocab, dt, vocab + k, stride)
    scores = -20 * cuda.rand(groups * beams, device="cuda", generator=cuda.Generator(device="cuda").manual_seed(k))
    check(cuda, x, scores, beams=beams, k=k)
    check(cuda, x, None, beams=beams, k=k)


@DT
def test_select_ties_go_to_the_lowest(cuda, dt):
    """Equal rows with equal scores, equal values in a row, zeros of both signs."""
    dt = getattr(cuda, dt)
    x = cuda.zeros(4, 9000, device="cuda", dtype=dt)
    for k in (1, 3, 100, 128):
        out = check(cuda, x, beams=2, k=k)
        assert out.token.tolist() == [list(range(k))] * 2 and out.row.tolist() == [[0] * k, [2] * k]
    x[:, 1::2] = -0.0
    out = check(cuda, x, beams=4, k=5)
    assert out.token.tolist() == [[0, 1, 2, 3, 4]]
    x = cuda.randint(0, 3, (6, 20000), device="cuda", generator=cuda.Generator(device="cuda").manual_seed(1)).to(dt)
    x[3:] = x[:3]
    check(cuda, x, beams=6, k=40)
    check(cuda, x, beams=1, k=128)


@DT
def test_select_masked_and_bad_values(cuda, dt):
    dt = getattr(cuda, dt)
    low = cuda.finfo(dt).min
    x = random_logits(cuda, 8, 5000, dt, 3)
    x[0, :] = -math.inf                      # nothing to offer
    x[1, 7] = math.nan                       # no sum
    x[2, 9] = math.inf
    x[3, :] = low                            # the type's lowest value everywhere
    x[4, :] = -math.inf
    x[4, 4999] = -3.0                        # one token
    x[5, :4990] = -math.inf                  # ten
    x[6, :] = low
    x[6, 40:44] = 1.0
    scores = cuda.tensor([-1.0, -1.0, -1.0, -2.0, -0.5, -3.0, -4.0, -math.inf], device="cuda")
    for k in (1, 5, 12, 40):
        check(cuda, x, scores, beams=8, k=k)
        check(cuda, x, scores, beams=1, k=k)
    scores[4] = math.nan
    out = ib.beam_select(x, scores, beams=8, k=8)
    assert 4 not in out.row.tolist()[0] and out.row.tolist()[0][0] == 5
    out = check(cuda, cuda.full((2, 100), -math.inf, device="cuda", dtype=dt), beams=2, k=3)
    assert out.token.tolist() == [[-1] * 3] and out.row.tolist() == [[-1] * 3]


@DT
def test_select_values_in_order(cuda, dt):
    """Orders that a threshold does not help with: rising, falling, the largest at a slice's end."""
    dt = getattr(cuda, dt)
    up = cuda.linspace(-8, 8, 20000, device="cuda").to(dt)
    x = cuda.stack([up, up.flip(0), cuda.roll(up, 1), cuda.roll(up, -9999)])
    for k in (1, 8, 128):
        check(cuda, x, cuda.tensor([0.0, -0.25, -0.5, -0.125], device="cuda"), beams=4, k=k)
        many = x.repeat(200, 1)  # whole rows to a slice
        out = ib.beam_select(many, beams=4, k=k)
        one = ib.beam_select(x, beams=4, k=k)
        # the four rows hold the same values in different places: their log sums are equal in exact
        # arithmetic, and which of them wins is rounding's choice, so the values won are compared
        at = lambda o, y: y[o.row.long(), o.token.long()]  # noqa: E731
        assert cuda.equal(at(out, many), at(one, x).expand(200, k))


@DT
def test_select_ended_beams(cuda, dt):
    dt = getattr(cuda, dt)
    x = random_logits(cuda, 12, 700, dt, 8)
    scores = -6 * cuda.rand(12, device="cuda", generator=cuda.Generator(device="cuda").manual_seed(2))
    ended = i32(cuda, [0, 1, 0, 1, 1, 1, -7, 0, 0, 0, 0, 2])
    x[1] = math.nan  # not read
    scores[4] = -math.inf
    for k in (1, 4, 9):
        check(cuda, x, scores, ended, beams=4, k=k, end_token=2)
    out = check(cuda, x, scores, cuda.ones_like(ended), beams=4, k=4, end_token=699)
    assert (out.token == 699).sum().item() == 11


def test_select_as_argmax(cuda):
    x = random_logits(cuda, 33, 32003, cuda.float32, 5)
    best = ib.beam_select(x, k=1).token.flatten()
    one = cuda.zeros(1, dtype=cuda.int32, device="cuda")
    for r in (0, 17, 32):
        ib.argmax(x[r].contiguous(), 32003, one)
        assert best[r].item() == one.item()


def test_select_close_candidates_of_different_beams(cuda):
    """Beams whose candidates differ by less than FP32 tells apart: the order is that of 64 bits."""
    x = random_logits(cuda, 2, 3000, cuda.float32, 6)
    x[1] = x[0]
    x[1, 5] = x[0].max() - 12.0          # moves the second row's sum by some 1e-7 of itself
    x[0, 5] = x[0].max() - 11.0
    lse = cuda.logsumexp(x.double(), 1)
    assert 1e-8 < (lse[0] - lse[1]).item() < 1e-5
    out = check(cuda, x, beams=2, k=8)
    assert out.row.tolist() == [[1, 0] * 4]


def test_select_streams_graphs_and_workspaces(cuda):
    xs = [random_logits(cuda, 12, 40000, cuda.float32, s) for s in (1, 2)]
    want = [ib.beam_select(x, beams=4, k=6) for x in xs]
    held = []
    for x in xs:
        side = cuda.cuda.Stream()
        side.wait_stream(cuda.cuda.current_stream())
        out = ib.BeamChoice(*(cuda.full_like(t, 9) for t in want[0]))
        ws = ib.beam_select_workspace(x, 4, 6)
        ws.fill_(255)
        buf = cuda.zeros_like(x)
        g = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(g, stream=side):
            ib.beam_select(buf, beams=4, k=6, out=out, workspace=ws)
        held.append((g, side, out, buf, ws))
    for turn in range(3):
        for i, (g, side, out, buf, ws) in enumerate(held):
            buf.copy_(xs[(i + turn) % 2])
            side.wait_stream(cuda.cuda.current_stream())
            with cuda.cuda.stream(side):
                g.replay()
        cuda.cuda.synchronize()
        for i, h in enumerate(held):
            for a, b in zip(h[2], want[(i + turn) % 2]):
                assert cuda.equal(a, b)
    assert ib.check_fault() == 0


# ---- reorder ---------------------------------------------------------------------------

def reorder(book, slots, parents):
    """The rules on lists; returns status and the copies (from, to, rows)."""
    N, n = len(book.len), len(slots)
    seen, accepted, status = set(), [], [-1] * n
    for i, (s, p) in enumerate(zip(slots, parents)):
        if not 0 <= s < N:
            continue
        first = s not in seen
        seen.add(s)
        if not first or not -1 <= p < n or (p >= 0 and not 0 <= slots[p] < N):
            continue
        accepted.append(i)
        status[i] = 1
    old = {s: (list(book.table[s]), book.len[s]) for s in range(N)}
    given = {slots[i] for i in accepted}
    for s in given:
        for t in old[s][0]:
            if t >= 0:
                book.refs[t] -= 1
        book.table[s], book.len[s] = [-1] * book.max_pages, 0
    takers, need = {}, []
    for i in accepted:
        if parents[i] < 0:
            continue
        src = slots[parents[i]]
        row, L = old[src]
        full = L // book.page
        for t in row[:full]:
            if t >= 0:
                book.refs[t] += 1
        book.table[slots[i]][:full] = row[:full]
        book.len[slots[i]] = L
        if L % book.page and row[full] >= 0:
            takers.setdefault(src, []).append(i)
    for src, some in takers.items():
        heir = None
        if src in given:
            heir = next((i for i in some if slots[i] == src), some[0])
            L = old[src][1]
            book.table[slots[heir]][L // book.page] = old[src][0][L // book.page]
            book.refs[old[src][0][L // book.page]] += 1
        need += [i for i in some if i != heir]
    copies = []
    free = [p for p, r in enumerate(book.refs) if r <= 0]
    for place, i in enumerate(sorted(need)):
        s, src = slots[i], slots[parents[i]]
        L = old[src][1]
        col = L // book.page
        if place >= len(free):
            status[i] = 0
            for t in book.table[s]:
                if t >= 0:
                    book.refs[t] -= 1
            book.table[s], book.len[s] = [-1] * book.max_pages, 0
            continue
        book.table[s][col] = free[place]
        book.refs[free[place]] = 1
        copies.append((old[src][0][col], free[place], L % book.page))
    return status, copies


def run_reorder(cuda, book, seqs, pages, slots, parents, **kw):
    k0, v0 = pages.k.clone(), pages.v.clone()
    want, copies = reorder(book, slots, parents)
    got = ib.kv_reorder(pages, seqs, i32(cuda, slots), i32(cuda, parents), **kw)
    assert got.tolist() == want
    same(book, seqs)
    for x, y in ((k0, pages.k), (v0, pages.v)):
        src = [x[:, a, :, :part].clone() for a, _, part in copies]
        for (a, b, part), rows in zip(copies, src):
            x[:, b, :, :part] = rows
        assert cuda.equal(x, y)
    return want


@pytest.mark.parametrize("type_,layers,Hkv,HD,page", [(ib.F32, 3, 2, 24, 5), (ib.F16, 2, 8, 128, 16),
                                                      (ib.F16, 1, 3, 8, 1), (ib.F32, 33, 1, 64, 64)])
def test_reorder_of_beams(cuda, type_, layers, Hkv, HD, page):
    """Beams of two prompts, step after step, with all kinds of parents."""
    rng = random.Random(page)
    book = Book(9, 12, 90, page)
    pages = pool(cuda, layers, 90, Hkv, page, HD, type_, 1)
    seqs = seqs_of(cuda, book)
    slots = [3, 1, 8, 0, 5, 2]
    new = [2 * page + 3] * 3 + [page] * 3
    assert ib.kv_extend(pages, seqs, i32(cuda, slots), i32(cuda, new)).tolist() == book.extend(slots, new)
    for step in range(25):
        parents = [rng.choice([0, 1, 2]) for _ in range(3)] + [rng.choice([3, 4, 5]) for _ in range(3)]
        parents = {0: list(range(6)), 1: [1, 2, 0, 4, 5, 3], 2: [0, 0, 0, 5, 5, 5]}.get(step, parents)
        assert run_reorder(cuda, book, seqs, pages, slots, parents) == [1] * 6
        one = [1] * 6
        if max(book.len) < 12 * page:
            assert ib.kv_extend(pages, seqs, i32(cuda, slots), i32(cuda, one)).tolist() == book.extend(slots, one)
        same(book, seqs)
    assert ib.check_fault() == 0


@pytest.mark.parametrize("seed", range(6))
def test_reorder_random(cuda, seed):
    """Any lists: repeated and missing slots, parents that are none, little room, pages given back."""
    rng = random.Random(seed)
    page = [1, 4, 7, 16, 3, 5][seed]
    N, W, P = [(12, 9, 60), (40, 20, 500), (12, 9, 50), (9, 5, 20000), (300, 6, 9000), (7, 4, 16)][seed]
    book = Book(N, W, P, page)
    pages = pool(cuda, 2, P, 2, page, 8, ib.F16, seed)
    seqs = seqs_of(cuda, book)
    for step in range(30):
        some = rng.sample(range(N), rng.randrange(1, N + 1))
        new = [rng.randrange(0, 2 * page + 1) for _ in some]
        assert ib.kv_extend(pages, seqs, i32(cuda, some), i32(cuda, new)).tolist() == book.extend(some, new)
        n = rng.randrange(1, N + 4)
        slots = rng.sample(range(N), min(n, N))
        if step % 3 == 0:
            slots = [s if rng.random() < 0.8 else rng.randrange(-1, N + 1) for s in slots]
        n = len(slots)
        parents = [rng.randrange(n) if rng.random() < 0.9 else rng.choice([-1, -1, -2, n]) for _ in slots]
        if step % 7 == 3:  # pages given back early
            for s in rng.sample(range(N), 2):
                if book.len[s] and book.table[s][0] >= 0 and book.refs[book.table[s][0]] == 1:
                    book.refs[book.table[s][0]] = 0
                    book.table[s][0] = -1
            seqs.table.copy_(cuda.tensor(book.table, dtype=cuda.int32))
            seqs.refs.copy_(i32(cuda, book.refs))
        run_reorder(cuda, book, seqs, pages, slots, parents)
        if step % 9 == 8:
            gone = rng.sample(range(N), N // 2)
            book.release(gone)
            ib.kv_release(pages, seqs, i32(cuda, gone))
    assert ib.check_fault() == 0


def test_reorder_without_room(cuda):
    """Copies that there is no page for: the first in the list are served, the others end empty and hold
    nothing; what takes no copy is served all the same."""
    book = Book(7, 5, 12, 4)
    book.extend([0, 1, 2], [18, 8, 11])  # 5, 2 and 3 pages of 12
    seqs, pages = seqs_of(cuda, book), pool(cuda, 2, 12, 2, 4, 8, ib.F16, 1)
    want = run_reorder(cuda, book, seqs, pages, [6, 5, 0, 4, 3, 1, 2], [2, 2, 2, 2, 5, 5, 6])
    assert want == [1, 1, 1, 0, 1, 1, 1] and book.len == [18, 8, 11, 8, 0, 18, 18]
    run_reorder(cuda, book, seqs, pages, [4, 0, 1], [1, 1, 1])
    assert ib.check_fault() == 0


def test_reorder_of_many(cuda):
    n = 3000
    rng = random.Random(3)
    book = Book(n, 3, 7000, 4)
    seqs, pages = seqs_of(cuda, book), pool(cuda, 1, 7000, 1, 4, 8, ib.F16, 0)
    slots = list(range(n))
    rng.shuffle(slots)
    new = [rng.randrange(0, 9) for _ in slots]
    ib.kv_extend(pages, seqs, i32(cuda, slots), i32(cuda, new))
    book.extend(slots, new)
    for _ in range(3):
        run_reorder(cuda, book, seqs, pages, slots, [rng.randrange(n) for _ in slots])
    assert ib.check_fault() == 0


def test_reorder_records_bad_values_and_needs_no_initial_workspace(cuda):
    pages = pool(cuda, 1, 12, 1, 4, 8, ib.F16, 0)

    def fresh():
        b = Book(4, 4, 12, 4)
        b.extend([0, 1, 2], [10, 4, 7])
        return b

    for fill in (0, 255):
        b = fresh()
        s = seqs_of(cuda, b)
        ws = ib.kv_reorder_workspace(s, 3)
        ws.fill_(fill)
        run_reorder(cuda, b, s, pages, [0, 1, 2], [2, 2, 0], workspace=ws)
    for change, code in ((lambda b: b.len.__setitem__(0, 17), "73"), (lambda b: b.len.__setitem__(0, -1), "73"),
                         (lambda b: b.table[0].__setitem__(1, 12), "72"), (lambda b: b.table[0].__setitem__(2, -9), "72"),
                         (lambda b: b.refs.__setitem__(b.table[1][0], 0), "74")):
        b = fresh()
        change(b)
        s = seqs_of(cuda, b)
        ib.kv_reorder(pages, s, i32(cuda, [0, 1, 2]), i32(cuda, [1, 0, 0]))
        with pytest.raises(RuntimeError, match=code):
            ib.check_fault()
        assert s.refs.min().item() >= 0
    # a length that cannot be refuses the entries it concerns, and no others
    b = fresh()
    b.len[0] = 17
    s = seqs_of(cuda, b)
    assert ib.kv_reorder(pages, s, i32(cuda, [0, 1, 2]), i32(cuda, [1, 0, 2])).tolist() == [-1, -1, 1]
    with pytest.raises(RuntimeError, match="73"):
        ib.check_fault()


def test_reorder_follows_a_selection(cuda):
    """The rows of a selection are the parents: beams without a candidate end empty."""
    book = Book(6, 5, 40, 4)
    book.extend([0, 1, 2, 3, 4, 5], [6] * 6)
    seqs, pages = seqs_of(cuda, book), pool(cuda, 2, 40, 1, 4, 8, ib.F32, 0)
    x = cuda.full((6, 50), -math.inf, device="cuda")
    x[1, 3], x[4, 7:20] = 1.0, 0.5
    out = ib.beam_select(x, beams=3)
    assert out.row.tolist() == [[1, -1, -1], [4, 4, 4]] and out.token.tolist() == [[3, -1, -1], [7, 8, 9]]
    run_reorder(cuda, book, seqs, pages, list(range(6)), out.row.flatten().tolist())
    assert seqs.len.tolist() == [6, 0, 0, 6, 6, 6]


def test_a_beam_step_captured_and_replayed(cuda):
    """Extend, select and reorder in one graph, replayed with other logits, against the same calls made
    one by one; two graphs with workspaces of their own on two streams."""
    groups, beams, V, page = 2, 3, 5000, 4
    n = groups * beams

    def state(seed):
        book = Book(n, 60, 300, page)
        book.extend(list(range(n)), [5, 6, 7, 3, 4, 8])
        s = dict(seqs=seqs_of(cuda, book), pages=pool(cuda, 2, 300, 1, page, 8, ib.F16, seed))
        s["slots"], s["one"] = i32(cuda, range(n)), i32(cuda, [1] * n)
        s["x"] = cuda.zeros(n, V, device="cuda")
        s["scores"], s["ended"] = cuda.zeros(n, device="cuda"), i32(cuda, [0, 0, 0, 0, 1, 0])
        s["out"] = ib.BeamChoice(*(cuda.zeros(groups, beams, dtype=t, device="cuda")
                                   for t in (cuda.float32, cuda.int32, cuda.int32)))
        s["ext"], s["status"] = i32(cuda, [0] * n), i32(cuda, [0] * n)
        s["ws"] = ib.beam_select_workspace(s["x"], beams), ib.kv_reorder_workspace(s["seqs"], n)
        return s

    def step(s):
        ib.kv_extend(s["pages"], s["seqs"], s["slots"], s["one"], status=s["ext"])
        out = ib.beam_select(s["x"], s["scores"], beams=beams, ended=s["ended"], end_token=2, out=s["out"],
                             workspace=s["ws"][0])
        ib.kv_reorder(s["pages"], s["seqs"], s["slots"], out.row.view(-1), status=s["status"], workspace=s["ws"][1])
        s["scores"].copy_(out.score.view(-1))

    def held(s):
        return [s["seqs"].table, s["seqs"].len, s["seqs"].refs, s["pages"].k, s["pages"].v, s["scores"]]

    live, plain, graphs = [state(1), state(2)], [state(1), state(2)], []
    for s in live:
        before = [x.clone() for x in held(s)]
        side = cuda.cuda.Stream()
        side.wait_stream(cuda.cuda.current_stream())
        with cuda.cuda.stream(side):
            step(s)  # first use outside the capture
        cuda.cuda.synchronize()
        for x, y in zip(held(s), before):
            x.copy_(y)
        g = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(g, stream=side):
            step(s)
        graphs.append((g, side))
    for i in range(6):
        for k, (a, b) in enumerate(zip(live, plain)):
            x = 3 * cuda.randn(n, V, generator=cuda.Generator(device="cuda").manual_seed(10 * i + k), device="cuda")
            a["x"].copy_(x), b["x"].copy_(x)
        for g, side in graphs:
            side.wait_stream(cuda.cuda.current_stream())
            with cuda.cuda.stream(side):
                g.replay()
        cuda.cuda.synchronize()
        for a, b in zip(live, plain):
            step(b)
            assert a["status"].tolist() == [1] * n
            for x, y in zip(held(a) + list(a["out"]), held(b) + list(b["out"])):
                assert cuda.equal(x, y)
    assert ib.check_fault() == 0


def test_select_and_reorder_on_a_given_stream(cuda):
    """What a call makes itself is of the launch stream's memory pool; results are the same."""
    book = Book(4, 5, 30, 4)
    book.extend([0, 1, 2, 3], [6] * 4)
    seqs, pages = seqs_of(cuda, book), pool(cuda, 2, 30, 1, 4, 8, ib.F32, 0)
    x = cuda.randn(4, 3001, generator=cuda.Generator(device="cuda").manual_seed(3), device="cuda")
    want = ib.beam_select(x, beams=2)
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    got = ib.beam_select(x, beams=2, stream=side.cuda_stream)
    status = ib.kv_reorder(pages, seqs, i32(cuda, [0, 1, 2, 3]), i32(cuda, want.row.flatten().tolist()),
                           stream=side.cuda_stream)
    side.synchronize()
    for a, b in zip(got, want):
        assert cuda.equal(a, b)
    reorder(book, [0, 1, 2, 3], want.row.flatten().tolist())
    same(book, seqs)
    assert status.tolist() == [1] * 4 and ib.check_fault() == 0


@DT
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 4096), (1, 4097), (147, 4100), (149, 20000), (304, 15427), (360, 9000),
                                        (700, 5000)])
def test_select_however_the_rows_are_cut(cuda, dt, rows, vocab):
    """Numbers of rows and values about those where the number of slices changes."""
    check(cuda, random_logits(cuda, rows, vocab, getattr(cuda, dt), rows), k=min(7, vocab))


@pytest.mark.parametrize("n,max_pages", [(1, 3), (32, 128), (33, 128), (32, 129), (31, 40), (60, 300)])
def test_reorder_of_few_and_many(cuda, n, max_pages):
    """About the bounds where the rows go with the plan; slots named twice and entries refused among them."""
    rng = random.Random(n + max_pages)
    page = 4
    book = Book(n + 3, max_pages, (n + 3) * max_pages // 2 + 40, page)
    seqs, pages = seqs_of(cuda, book), pool(cuda, 2, len(book.refs), 2, page, 8, ib.F32, 0)
    slots = rng.sample(range(n + 3), n)
    new = [rng.randrange(0, max_pages * page // 3 + 1) for _ in slots]
    assert ib.kv_extend(pages, seqs, i32(cuda, slots), i32(cuda, new)).tolist() == book.extend(slots, new)
    for turn in range(6):
        parents = [rng.randrange(-1, n) for _ in slots]
        names = list(slots)
        if turn > 2 and n > 2:
            names[rng.randrange(n)] = names[rng.randrange(n)]
            names[rng.randrange(n)] = rng.choice([-1, n + 3, names[0]])
            parents[rng.randrange(n)] = n
        run_reorder(cuda, book, seqs, pages, names, parents)
    assert ib.check_fault() == 0


@pytest.mark.parametrize("vocab", [300, 5000, 40000])
def test_select_orders_a_row_by_its_logits(cuda, vocab):
    """Values that 64 bits do not tell apart once the log sum is taken off (logits next to zero, large scores):
    a row's order is that of its logits, and with k = 1 the choice is the first maximum."""
    x = cuda.full((2, vocab), -3.0, device="cuda")
    at = [2, 7, vocab // 2, vocab - 300 + 50, vocab - 1]
    x[:, at] = cuda.tensor([1e-30, 3e-30, 2e-30, -1e-30, 3e-30], device="cuda")
    order = [at[1], at[4], at[2], at[0], at[3]]
    one = cuda.zeros(1, dtype=cuda.int32, device="cuda")
    ib.argmax(x[0].contiguous(), vocab, one)
    assert one.item() == at[1]
    for scores in (None, cuda.tensor([-1.5, -4.0], device="cuda"), cuda.tensor([1e25, 1e24], device="cuda")):
        for k in (1, 2, 5):
            out = ib.beam_select(x, scores, k=k)
            assert out.token.tolist() == [order[:k]] * 2 and out.row.tolist() == [[0] * k, [1] * k]
        out = ib.beam_select(x, scores, beams=2, k=10)
        if scores is not None and scores[0] > 1e24:  # all of the first row's values are above the second's
            assert out.token.tolist() == [order + [0, 1, 3, 4, 5]] and out.row.tolist() == [[0] * 10]
        else:
            assert out.token.tolist() == [order * 2] and out.row.tolist() == [[0] * 5 + [1] * 5]
    # many rows of them: the kernel's slow path
    out = ib.beam_select(x.repeat(400, 1), beams=800, k=128)
    assert out.row.tolist() == [[i // 5 for i in range(128)]] and out.token.tolist() == [(order * 26)[:128]]
    assert ib.check_fault() == 0


@DT
def test_select_signed_zeros_are_equal(cuda, dt):
    """Ended rows that offer 0 and -0, and logits of both: the lowest row and token win."""
    ones = cuda.ones(64, dtype=cuda.int32, device="cuda")
    x = cuda.zeros(64, 100, dtype=getattr(cuda, dt), device="cuda")
    for at in (0, 3, 63):
        scores = cuda.zeros(64, device="cuda")
        scores[at] = -0.0
        for k in (1, 8, 9):
            out = ib.beam_select(x, scores, beams=64, k=k, ended=ones, end_token=5)
            assert out.row.tolist() == [list(range(k))] and out.token.tolist() == [[5] * k]
            assert not bool(out.score.any())
    x[:, ::2] = -0.0
    out = ib.beam_select(x, beams=64, k=8)
    assert out.row.tolist() == [[0] * 8] and out.token.tolist() == [list(range(8))]
    assert ib.check_fault() == 0


def test_select_weights_of_a_log_sum(cuda):
    """The weights e^t of a row's log sum, t from 0 down: rows of 256 zeros, one among each 16 values, and t.
    With w the weights' share of the sum, |error| <= |v| 2^-24 (the result's rounding) + w (4 + 2 |t|) 2^-24 (a
    weight: 2^-22 of the instruction, two roundings of its argument) + 8 2^-24 (a thread's sum)."""
    t = -np.concatenate([np.geomspace(1e-7, 100, 1500), np.linspace(0, 20, 500), [87.0, 88.0, 103.0, 104.0, 1e4, 3e38]])
    t = t.astype(np.float32)
    x = cuda.tensor(t, device="cuda")[:, None].repeat(1, 4096)
    x[:, 0:1024:4] = 0.0
    out = ib.beam_select(x, k=1)
    t = t.astype(np.float64)
    weight = 15 * np.exp(t)
    want = -(math.log(256) + np.log1p(weight))
    got = out.score.flatten().cpu().numpy().astype(np.float64)
    tol = (np.abs(want) + weight / (1 + weight) * (4 + 2 * np.abs(t)) + 8) * 2.0 ** -24
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    assert not bool(out.token.any()) and ib.check_fault() == 0
