"""The paged KV cache's argument checks, which need no GPU: a refused call returns before any
CUDA call, so the pointers here are only numbers."""
import ctypes

import pytest

from conftest import load_package

ib = load_package()
PTR = 0x10000


def pages(**k):
    d = dict(type=ib.F16, n_layers=2, n_pages=8, n_kv_heads=2, page_size=16, head_dim=64, k=PTR,
             v=PTR)
    d.update(k)
    return ib._CKVPages(*[d[f] for f, _ in ib._CKVPages._fields_])


def seqs(**k):
    d = dict(n_slots=4, max_pages=4, table=PTR, len=PTR, refs=PTR)
    d.update(k)
    return ib._CKVSeqs(*[d[f] for f, _ in ib._CKVSeqs._fields_])


def batch(**k):
    d = dict(n_seqs=2, n_tokens=3, max_q=2, cu_q=PTR, slots=PTR)
    d.update(k)
    return ib._CKVBatch(*[d[f] for f, _ in ib._CKVBatch._fields_])


def ref(x):
    return None if x is None else ctypes.byref(x)


def attention(p=None, s=None, b=None, layer=0, H=4, q=PTR, qs=256, out=PTR, os_=256, ws=PTR,
              size=1 << 40):
    return ib.lib().ib_attention_paged(ref(p or pages()), ref(s or seqs()), ref(b or batch()), layer,
                                       H, q, qs, out, os_, 0.1, ws, size, None)


def append(p=None, s=None, b=None, layer=0, H=4, q=PTR, qs=256, k=PTR, ks=128, v=PTR, vs=128,
           o=PTR, os_=256, rope=PTR, n=64):
    return ib.lib().ib_kv_append(ref(p or pages()), ref(s or seqs()), ref(b or batch()), layer, H, q,
                                 qs, k, ks, v, vs, o, os_, rope, n, None)


BAD_POOL = [dict(p=pages(k=None)), dict(p=pages(v=None)), dict(p=pages(k=PTR + 8)),
            dict(p=pages(n_layers=0)), dict(p=pages(n_pages=0)), dict(p=pages(n_pages=2 ** 20 + 1)),
            dict(p=pages(n_kv_heads=0)), dict(p=pages(page_size=0)), dict(p=pages(page_size=4097)),
            dict(p=pages(head_dim=0)), dict(p=pages(head_dim=20)), dict(p=pages(head_dim=264)),
            dict(s=seqs(table=None)), dict(s=seqs(len=None)), dict(s=seqs(refs=None)),
            dict(s=seqs(n_slots=0)), dict(s=seqs(n_slots=16385)), dict(s=seqs(max_pages=0)),
            dict(s=seqs(max_pages=2 ** 24 + 1))]
BAD_BATCH = [dict(b=batch(cu_q=None)), dict(b=batch(n_seqs=-1)), dict(b=batch(n_tokens=-1)),
             dict(b=batch(max_q=-1)), dict(b=batch(slots=None, n_seqs=5)), dict(layer=-1),
             dict(layer=2), dict(H=0), dict(H=3), dict(b=batch(n_tokens=2 ** 28 + 1)),
             dict(q=None), dict(q=PTR + 4), dict(qs=254), dict(qs=-256)]


@pytest.mark.parametrize("bad", BAD_POOL + BAD_BATCH + [
    dict(out=None), dict(out=PTR + 8), dict(os_=252), dict(os_=258), dict(ws=None),
    dict(ws=PTR + 16), dict(size=0)])
def test_attention_refuses(bad):
    assert attention(**bad) == ib.IB_ERR_INVALID
    assert "ib_attention_paged" in ib.last_error()


@pytest.mark.parametrize("bad", BAD_POOL + BAD_BATCH + [
    dict(k=None), dict(v=None), dict(o=None), dict(rope=None), dict(k=PTR + 4), dict(v=PTR + 8),
    dict(o=PTR + 4), dict(rope=PTR + 4), dict(ks=130), dict(vs=-4), dict(os_=252), dict(n=-1)])
def test_append_refuses(bad):
    assert append(**bad) == ib.IB_ERR_INVALID
    assert "ib_kv_append" in ib.last_error()


@pytest.mark.parametrize("bad", BAD_POOL)
def test_bookkeeping_refuses_bad_pools(bad):
    L, p, s = ib.lib(), ref(bad.get("p") or pages()), ref(bad.get("s") or seqs())
    assert L.ib_kv_extend(p, s, 1, PTR, PTR, PTR, None) == ib.IB_ERR_INVALID
    assert L.ib_kv_fork(p, s, 1, PTR, PTR, PTR, None) == ib.IB_ERR_INVALID
    assert L.ib_kv_release(p, s, 1, PTR, None) == ib.IB_ERR_INVALID
    assert L.ib_kv_compact(p, s, PTR, PTR, PTR, PTR, PTR, None) == ib.IB_ERR_INVALID


def test_bookkeeping_refuses_bad_lists():
    L, p, s = ib.lib(), ref(pages()), ref(seqs())
    for n in (-1, 16385):
        assert L.ib_kv_extend(p, s, n, PTR, PTR, PTR, None) == ib.IB_ERR_INVALID
        assert L.ib_kv_fork(p, s, n, PTR, PTR, PTR, None) == ib.IB_ERR_INVALID
        assert L.ib_kv_release(p, s, n, PTR, None) == ib.IB_ERR_INVALID
    for i in range(3):
        a = [PTR] * 3
        a[i] = None
        assert L.ib_kv_extend(p, s, 1, *a, None) == ib.IB_ERR_INVALID
        assert L.ib_kv_fork(p, s, 1, *a, None) == ib.IB_ERR_INVALID
    assert L.ib_kv_release(p, s, 1, None, None) == ib.IB_ERR_INVALID
    for i in range(5):
        a = [PTR] * 5
        a[i] = None
        assert L.ib_kv_compact(p, s, *a, None) == ib.IB_ERR_INVALID
    # empty lists are no work
    assert L.ib_kv_extend(p, s, 0, PTR, PTR, PTR, None) == ib.IB_OK
    assert L.ib_kv_fork(p, s, 0, PTR, PTR, PTR, None) == ib.IB_OK
    assert L.ib_kv_release(p, s, 0, PTR, None) == ib.IB_OK


def test_types_and_null_structs():
    L = ib.lib()
    for t in (ib.Q8_0, ib.Q4_K, ib.I16, 30):
        assert attention(p=pages(type=t)) == ib.IB_ERR_UNSUPPORTED
        assert append(p=pages(type=t)) == ib.IB_ERR_UNSUPPORTED
    p, s, b = ref(pages()), ref(seqs()), ref(batch())
    for a in ((None, s, b), (p, None, b), (p, s, None)):
        assert L.ib_attention_paged(*a, 0, 4, PTR, 256, PTR, 256, 0.1, PTR, 1 << 40, None) == \
            ib.IB_ERR_INVALID
        assert L.ib_attention_paged_workspace(*a, 4) == 0
    assert L.ib_kv_release(None, s, 1, PTR, None) == ib.IB_ERR_INVALID
    # an empty batch is no work
    assert attention(b=batch(n_tokens=0)) == ib.IB_OK
    assert append(b=batch(n_seqs=0)) == ib.IB_OK


def test_python_handles_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="cpu"):
        ib.KVPages.empty(1, 2, 1, 4, 8, ib.F16, device="cpu")
    with pytest.raises(ValueError, match="cpu"):
        ib.KVSeqs.empty(2, 3, 4, device="cpu")
    with pytest.raises(ValueError, match="F32 or F16"):
        ib.KVPages.empty(1, 2, 1, 4, 8, ib.Q8_0)
    with pytest.raises(ValueError, match="cpu"):
        ib.KVBatch(torch.zeros(2, dtype=torch.int32), 1)


def _cpp(tmp_path, name, *args):
    """Compiles tests/cpp/<name>.cpp against the kernels' host-side headers and runs it."""
    import os
    import shutil
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / name)
    r = subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-I",
                        os.path.join(root, "inference.cpp_b200", "csrc"),
                        os.path.join(root, "tests", "cpp", name + ".cpp"), "-o", exe],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe, *args], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    return r.stdout


def test_copies_of_the_tensor_kernel_never_lose_a_wait(tmp_path):
    """Every interleaving of the copying warps, the TMA and the MMAs, with the kernel's own
    assignment of look barriers to ring slots."""
    assert "0 of the patterns" in _cpp(tmp_path, "copy_ring_test")


def test_the_search_finds_a_shared_look_barrier(tmp_path):
    """The same search on one look barrier for all slots: two careful key tiles in a row can
    lap a warp."""
    assert "2 key tiles, careful 3: a wait that never ends" in _cpp(tmp_path, "copy_ring_test", "shared")


def test_granted_refuses_bad_lists():
    L = ib.lib()
    for n in (-1, 16385):
        assert L.ib_kv_granted(n, PTR, PTR, PTR, None) == ib.IB_ERR_INVALID
    for i in range(3):
        a = [PTR] * 3
        a[i] = None
        assert L.ib_kv_granted(1, *a, None) == ib.IB_ERR_INVALID
        assert "ib_kv_granted" in ib.last_error()
    assert L.ib_kv_granted(0, None, None, None, None) == ib.IB_OK


STEP = 4 * (256 + 2 * 128)  # bytes between rows of one projection's q (4 x 64), k and v (2 x 64)
QKV = dict(q=PTR, qs=512, k=PTR + 1024, ks=512, v=PTR + 1024 + 512, vs=512)


@pytest.mark.parametrize("bad", [
    dict(o=PTR, os_=256),                       # in place, rows of another step
    dict(o=PTR + 16, os_=512),                  # beside q's rows by four elements
    dict(o=PTR - 16, os_=512), dict(o=PTR + STEP, os_=512), dict(o=PTR - 2 * STEP, os_=512),
    dict(o=PTR + 1024, os_=512),                # k and v
    dict(o=PTR + 1024 + 512, os_=512),          # v, and the next row's q
    dict(o=PTR + 2 * STEP + 1008, os_=256),     # another step, over the last row's end
])
def test_append_refuses_rows_that_overlap(bad):
    assert append(**QKV, **bad) == ib.IB_ERR_INVALID
    assert "ib_kv_append" in ib.last_error() and "overlap" in ib.last_error()


@pytest.mark.parametrize("bad", [dict(os_=260), dict(out=PTR + 16), dict(out=PTR - 1008),
                                 dict(out=PTR + 2048), dict(qs=0), dict(qs=0, out=PTR + 1008),
                                 dict(qs=512, os_=512, out=PTR + 1008),
                                 dict(qs=512, os_=512, out=PTR + 2048 - 16)])
def test_attention_refuses_rows_that_overlap(bad):
    assert attention(**bad) == ib.IB_ERR_INVALID
    assert "ib_attention_paged" in ib.last_error() and "overlap" in ib.last_error()


@pytest.mark.parametrize("entry", ["ib_kv_extend", "ib_kv_fork"])
def test_status_must_not_overlap_the_lists(entry):
    f, p, s = getattr(ib.lib(), entry), ref(pages()), ref(seqs())
    far = PTR + (1 << 20)
    for lists in ((PTR, far, PTR), (far, PTR, PTR), (PTR, far, PTR + 4 * 4), (far, PTR, PTR - 4 * 4),
                  (PTR, PTR, PTR)):
        assert f(p, s, 5, *lists, None) == ib.IB_ERR_INVALID
        assert entry in ib.last_error() and "overlap" in ib.last_error()


def test_granted_must_not_overlap_its_lists():
    f, far = ib.lib().ib_kv_granted, PTR + (1 << 20)
    for slots, status, out in ((PTR, far, PTR + 4), (PTR, far, PTR - 16), (far, PTR, PTR),
                               (PTR, PTR, PTR), (PTR, PTR + 16, PTR)):
        assert f(5, slots, status, out, None) == ib.IB_ERR_INVALID
        assert "ib_kv_granted" in ib.last_error() and "overlap" in ib.last_error()


def test_a_failed_lookup_is_tried_again(tmp_path):
    _cpp(tmp_path, "lookup_test")
