"""Argument checks of the tree and beam operators, which need no GPU: a refused call returns before any
CUDA call, so the pointers here are only numbers."""
import ctypes

import pytest

from conftest import load_package
from test_paged_cpu import BAD_BATCH, BAD_POOL, PTR, _cpp, batch, pages, ref, seqs

ib = load_package()
FAR = PTR + (1 << 24)


def tree(**k):
    d = dict(max_nodes=8, depth=PTR, mask=PTR)
    d.update(k)
    return ib._CKVTree(*[d[f] for f, _ in ib._CKVTree._fields_])


def attention(p=None, s=None, b=None, t=None, layer=0, H=4, q=PTR, qs=256, out=PTR, os_=256, ws=PTR,
              size=1 << 40):
    return ib.lib().ib_attention_paged_tree(ref(p or pages()), ref(s or seqs()), ref(b or batch()),
                                            ref(t or tree()), layer, H, q, qs, out, os_, 0.1, ws, size, None)


def append(p=None, s=None, b=None, t=None, layer=0, H=4, q=PTR, qs=256, k=PTR, ks=128, v=PTR, vs=128, o=PTR,
           os_=256, rope=PTR, n=64):
    return ib.lib().ib_kv_append_tree(ref(p or pages()), ref(s or seqs()), ref(b or batch()), ref(t or tree()),
                                      layer, H, q, qs, k, ks, v, vs, o, os_, rope, n, None)


BAD_TREE = [dict(t=tree(max_nodes=0)), dict(t=tree(max_nodes=-1)), dict(t=tree(max_nodes=1025)),
            dict(t=tree(depth=None)), dict(t=tree(mask=None))]


@pytest.mark.parametrize("bad", BAD_POOL + BAD_BATCH + BAD_TREE + [
    dict(out=None), dict(out=PTR + 8), dict(os_=252), dict(os_=258), dict(ws=None), dict(ws=PTR + 16),
    dict(size=0), dict(out=PTR + 16), dict(os_=260)])
def test_attention_refuses(bad):
    assert attention(**bad) == ib.IB_ERR_INVALID
    assert "ib_attention_paged_tree" in ib.last_error()


@pytest.mark.parametrize("bad", BAD_POOL + BAD_BATCH + BAD_TREE + [
    dict(k=None), dict(v=None), dict(o=None), dict(rope=None), dict(k=PTR + 4), dict(v=PTR + 8),
    dict(o=PTR + 4), dict(rope=PTR + 4), dict(ks=130), dict(vs=-4), dict(os_=252), dict(n=-1),
    dict(o=PTR + 16)])
def test_append_refuses(bad):
    assert append(**bad) == ib.IB_ERR_INVALID
    assert "ib_kv_append_tree" in ib.last_error()


def test_null_structs_and_types():
    L, p, s, b, t = ib.lib(), ref(pages()), ref(seqs()), ref(batch()), ref(tree())
    for a in ((None, s, b, t), (p, None, b, t), (p, s, None, t), (p, s, b, None)):
        assert L.ib_attention_paged_tree(*a, 0, 4, PTR, 256, PTR, 256, 0.1, PTR, 1 << 40, None) == ib.IB_ERR_INVALID
        assert L.ib_attention_paged_tree_workspace(*a, 4) == 0
        assert L.ib_kv_append_tree(*a, 0, 4, PTR, 256, PTR, 128, PTR, 128, PTR, 256, PTR, 64, None) == \
            ib.IB_ERR_INVALID
    for type_ in (ib.Q8_0, ib.I16, 30):
        assert attention(p=pages(type=type_)) == ib.IB_ERR_UNSUPPORTED
        assert append(p=pages(type=type_)) == ib.IB_ERR_UNSUPPORTED
        assert L.ib_kv_reorder(ref(pages(type=type_)), s, 1, PTR, FAR, FAR + 64, PTR, 1 << 30, None) == \
            ib.IB_ERR_UNSUPPORTED
        assert L.ib_kv_tree_accept(ref(pages(type=type_)), s, b, PTR, PTR, None) == ib.IB_ERR_UNSUPPORTED
        assert L.ib_beam_select(type_, PTR, 10, None, None, 0, 1, 1, 10, 1, FAR, FAR, FAR, PTR, 1 << 30, None) == \
            ib.IB_ERR_UNSUPPORTED
    # an empty batch is no work
    assert attention(b=batch(n_tokens=0)) == ib.IB_OK
    assert append(b=batch(n_seqs=0)) == ib.IB_OK
    assert L.ib_kv_tree_plan(ref(batch(n_tokens=0)), None, 4, None, None, None) == ib.IB_OK
    assert L.ib_kv_tree_verify(ref(batch(n_seqs=0)), None, None, None, None, None, None, None) == ib.IB_OK
    assert L.ib_kv_tree_accept(p, s, ref(batch(n_seqs=0)), None, None, None) == ib.IB_OK
    assert L.ib_kv_reorder(p, s, 0, None, None, None, None, 0, None) == ib.IB_OK
    assert L.ib_beam_select(ib.F32, None, 10, None, None, 0, 0, 1, 10, 1, None, None, None, None, 0, None) == ib.IB_OK


BAD_LISTS = [dict(cu_q=None), dict(n_seqs=-1), dict(n_tokens=-1), dict(max_q=-1), dict(n_seqs=16385),
             dict(n_tokens=(1 << 26) + 1)]


@pytest.mark.parametrize("bad", BAD_LISTS)
def test_plan_and_verify_refuse_bad_batches(bad):
    L, b = ib.lib(), ref(batch(**bad))
    for x in (b, None):
        assert L.ib_kv_tree_plan(x, PTR, 4, FAR, FAR + (1 << 20), None) == ib.IB_ERR_INVALID
        assert "ib_kv_tree_plan" in ib.last_error()
        assert L.ib_kv_tree_verify(x, PTR, PTR, PTR, FAR, FAR + (1 << 20), FAR + (1 << 21), None) == ib.IB_ERR_INVALID
        assert "ib_kv_tree_verify" in ib.last_error()


def test_plan_refuses():
    L, b = ib.lib(), ref(batch(n_tokens=5))
    for n in (0, -3, 1025):
        assert L.ib_kv_tree_plan(b, PTR, n, FAR, FAR + 4096, None) == ib.IB_ERR_INVALID
    for i in range(3):
        a = [PTR, FAR, FAR + 4096]
        a[i] = None
        assert L.ib_kv_tree_plan(b, a[0], 4, a[1], a[2], None) == ib.IB_ERR_INVALID
    # five nodes, two words each
    for parents, depth, mask in ((PTR, PTR, FAR), (PTR, FAR, PTR), (PTR, PTR + 16, FAR), (PTR, FAR, PTR - 36),
                                 (PTR, FAR, FAR), (PTR, FAR, FAR - 36), (PTR, FAR, FAR + 16)):
        assert L.ib_kv_tree_plan(b, parents, 40, depth, mask, None) == ib.IB_ERR_INVALID
        assert "overlap" in ib.last_error()


def test_verify_refuses():
    L, b = ib.lib(), ref(batch(n_tokens=5, n_seqs=2))
    good = [PTR, PTR, PTR, FAR, FAR + 4096, FAR + 8192]
    for i in range(6):
        a = list(good)
        a[i] = None
        assert L.ib_kv_tree_verify(b, *a, None) == ib.IB_ERR_INVALID
    for i, at in ((3, PTR + 16), (3, PTR - 16), (4, PTR + 16), (4, PTR - 4), (5, PTR), (4, FAR + 16), (4, FAR - 4),
                  (5, FAR + 4096 + 4), (5, FAR)):
        a = list(good)
        a[i] = at
        assert L.ib_kv_tree_verify(b, *a, None) == ib.IB_ERR_INVALID
        assert "overlap" in ib.last_error()


@pytest.mark.parametrize("bad", BAD_POOL + [dict(b=batch(cu_q=None)), dict(b=batch(n_seqs=-1)),
                                            dict(b=batch(n_tokens=-1)), dict(b=batch(n_seqs=5))])
def test_accept_refuses(bad):
    L = ib.lib()
    a = [ref(bad.get("p") or pages()), ref(bad.get("s") or seqs()), ref(bad.get("b") or batch())]
    assert L.ib_kv_tree_accept(*a, PTR, PTR, None) == ib.IB_ERR_INVALID
    assert "ib_kv_tree_accept" in ib.last_error()


def test_accept_refuses_null():
    L, a = ib.lib(), [ref(pages()), ref(seqs()), ref(batch())]
    for i in range(3):
        x = list(a)
        x[i] = None
        assert L.ib_kv_tree_accept(*x, PTR, PTR, None) == ib.IB_ERR_INVALID
    assert L.ib_kv_tree_accept(*a, None, PTR, None) == ib.IB_ERR_INVALID
    assert L.ib_kv_tree_accept(*a, PTR, None, None) == ib.IB_ERR_INVALID


@pytest.mark.parametrize("bad", BAD_POOL)
def test_reorder_refuses_bad_pools(bad):
    p, s = ref(bad.get("p") or pages()), ref(bad.get("s") or seqs())
    assert ib.lib().ib_kv_reorder(p, s, 1, PTR, FAR, FAR + 64, PTR, 1 << 30, None) == ib.IB_ERR_INVALID


def test_reorder_refuses():
    L, p, s = ib.lib(), ref(pages()), ref(seqs())
    need = L.ib_kv_reorder_workspace(s, 5)
    assert need >= 5 * 4 * 4
    ok = [PTR, FAR, FAR + 64]
    for n in (-1, 16385):
        assert L.ib_kv_reorder(p, s, n, *ok, PTR, need, None) == ib.IB_ERR_INVALID
        assert L.ib_kv_reorder_workspace(s, n) == 0
    for i in range(3):
        a = list(ok)
        a[i] = None
        assert L.ib_kv_reorder(p, s, 5, *a, PTR, need, None) == ib.IB_ERR_INVALID
    for ws, size in ((None, need), (PTR + 16, need), (PTR, need - 1)):
        assert L.ib_kv_reorder(p, s, 5, *ok, ws, size, None) == ib.IB_ERR_INVALID
        assert "workspace" in ib.last_error()
    for lists in ((PTR, FAR, PTR), (FAR, PTR, PTR), (PTR, FAR, PTR + 16), (FAR, PTR, PTR - 16)):
        assert L.ib_kv_reorder(p, s, 5, *lists, PTR, need, None) == ib.IB_ERR_INVALID
        assert "overlap" in ib.last_error()
    assert L.ib_kv_reorder_workspace(None, 5) == 0
    assert L.ib_kv_reorder_workspace(ref(seqs(max_pages=0)), 5) == 0
    assert L.ib_kv_reorder_workspace(s, 0) >= 1


def test_beam_select_refuses():
    L = ib.lib()
    good = dict(type=ib.F32, x=PTR, stride=100, scores=None, ended=None, end=0, groups=2, beams=3, vocab=100, k=4,
                a=FAR, b=FAR + 4096, c=FAR + 8192, ws=PTR, size=1 << 30)

    def call(**bad):
        d = dict(good, **bad)
        return L.ib_beam_select(*d.values(), None)

    for bad in (dict(x=None), dict(a=None), dict(b=None), dict(c=None), dict(stride=99), dict(stride=-100),
                dict(groups=-1), dict(beams=0), dict(beams=1025), dict(groups=1 << 20), dict(vocab=0),
                dict(vocab=(1 << 28) + 1), dict(k=0), dict(k=129), dict(x=PTR + 2), dict(type=ib.F16, x=PTR + 1),
                dict(ws=None), dict(ws=PTR + 16), dict(size=0)):
        assert call(**bad) == ib.IB_ERR_INVALID, bad
        assert "ib_beam_select" in ib.last_error()
    for a in ((2, 0, 100, 4), (-1, 3, 100, 4), (2, 3, 0, 4), (2, 3, 100, 0), (2, 3, 100, 129)):
        assert L.ib_beam_select_workspace(*a) == 0
    assert L.ib_beam_select_workspace(2, 3, 100, 4) > 0
    assert call(size=L.ib_beam_select_workspace(2, 3, 100, 4) - 1) == ib.IB_ERR_INVALID


def test_results_must_not_overlap_a_selections_inputs():
    L = ib.lib()
    n = L.ib_beam_select_workspace(2, 3, 100, 4)
    far = [FAR + (i << 20) for i in range(8)]

    def call(x=far[0], scores=far[1], ended=far[2], a=far[3], b=far[4], c=far[5], ws=far[6]):
        return L.ib_beam_select(ib.F32, x, 100, scores, ended, 0, 2, 3, 100, 4, a, b, c, ws, n, None)

    for bad in (dict(a=far[0]), dict(b=far[0] + 4 * 599), dict(c=far[1]), dict(a=far[2] + 4 * 5), dict(b=far[3] + 28),
                dict(c=far[4]), dict(a=far[6]), dict(c=far[6] + n - 4), dict(ws=far[0]), dict(ws=far[1] - n + 256)):
        assert call(**bad) == ib.IB_ERR_INVALID, bad
        assert "overlap" in ib.last_error()


def test_python_handles_refuse():
    torch = pytest.importorskip("torch")
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="cpu"):
        ib.KVTree(z, z, torch.zeros(4, 1, dtype=torch.int32), 4)
    for n in (0, 1025):
        with pytest.raises(ValueError, match="max_nodes"):
            ib.KVTree(z, z, z, n)
    for x, what in ((torch.zeros(4, 9), "logits"), (torch.zeros(4, 9, dtype=torch.bfloat16), "logits"),
                    (torch.zeros(9), "logits")):
        with pytest.raises(ValueError, match=what):
            ib.beam_select(x)


def test_struct_layout():
    assert ctypes.sizeof(ib._CKVTree) == 24
    assert ib._CKVTree.depth.offset == 8 and ib._CKVTree.mask.offset == 16


def test_roles_of_the_tree_kernel_come_to_their_ends(tmp_path):
    """The programs of its warps in random orders: waits, slots, masks and looks as the kernel has them."""
    assert "runs, 0 stuck, 0 faults" in _cpp(tmp_path, "split_ring_test")


def test_the_search_finds_looks_that_are_not_counted(tmp_path):
    """The same with warps that count only their own looks at a slot: some order never ends."""
    assert "runs, 0 stuck, 0 faults" not in _cpp(tmp_path, "split_ring_test", "forget")


def test_rows_factors_of_the_tree_kernel_are_their_segments_own(tmp_path):
    """Every order of its softmax groups and MMAs over short batches, segments without key tiles among them."""
    assert " 0 faults, 0 orders without an end" in _cpp(tmp_path, "split_scales_test")


def test_the_search_finds_factors_of_another_segment(tmp_path):
    """The same where segments without key tiles are counted as the others are."""
    assert " 0 faults" not in _cpp(tmp_path, "split_scales_test", "all")


def test_verify_and_accept_refuse_a_bad_limit():
    L, b = ib.lib(), ref(batch(n_tokens=5, n_seqs=2))
    for most in (0, -1, 1025):
        assert L.ib_kv_tree_verify_max(b, most, PTR, PTR, PTR, FAR, FAR + 4096, FAR + 8192, None) == ib.IB_ERR_INVALID
        assert "ib_kv_tree_verify_max: max_nodes" in ib.last_error()
        assert L.ib_kv_tree_accept_max(ref(pages()), ref(seqs()), b, most, PTR, PTR, None) == ib.IB_ERR_INVALID
        assert "ib_kv_tree_accept_max: max_nodes" in ib.last_error()
    assert L.ib_kv_tree_verify_max(b, 8, PTR, PTR, PTR, PTR, FAR, FAR + 4096, None) == ib.IB_ERR_INVALID
    assert L.ib_kv_tree_accept_max(ref(pages()), ref(seqs()), None, 8, PTR, PTR, None) == ib.IB_ERR_INVALID
