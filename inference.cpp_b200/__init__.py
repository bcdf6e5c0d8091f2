"""Python mirror of the B200 backend's C ABI (include/ib_cuda.h).

The function names and argument meaning follow the reference's C++ backend
interface `inference::cuda` (include/ops/cuda_backend.hpp:17-64): gemv,
gemv_i16, gemm, gemm_i16, rmsnorm, silu, mul, add, embedding*, kv_write*, rope*,
attention*.  Device memory is held in torch tensors (plumbing only); every
operation runs through libib_cuda.so, and a failing call raises RuntimeError
with the library's message, as the reference's check() throws
std::runtime_error (src/ops/cuda_backend.cpp:76-85).

The directory name is not a Python identifier; load it with
`importlib.util.spec_from_file_location("inference_cpp_b200", ".../__init__.py")`
(tests/conftest.py and __graft_entry__.py do this).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os
import typing

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libib_cuda.so")
HEADER_DIR = os.path.join(os.path.dirname(HERE), "include")

# GGUF tensor types (reference include/core/tensor.hpp:16-37)
F32, F16, Q4_0, Q5_0, Q5_1, Q8_0, Q4_K, Q6_K, I16 = 0, 1, 2, 6, 7, 8, 12, 14, 17
# formats the reference sizes but does not decode (its dequantisers throw): decoded here
# from the published GGUF layouts
Q4_1, Q2_K, Q3_K, Q5_K = 3, 10, 11, 13
EXTRA_QUANT_TYPES = (Q4_1, Q2_K, Q3_K, Q5_K)
QUANT_TYPES = (Q4_0, Q5_0, Q5_1, Q8_0, Q4_K, Q6_K)
TYPE_NAMES = {F32: "F32", F16: "F16", Q4_0: "Q4_0", Q5_0: "Q5_0", Q5_1: "Q5_1",
              Q8_0: "Q8_0", Q4_K: "Q4_K", Q6_K: "Q6_K", I16: "I16", Q4_1: "Q4_1",
              Q2_K: "Q2_K", Q3_K: "Q3_K", Q5_K: "Q5_K"}
TYPE_BY_NAME = {v: k for k, v in TYPE_NAMES.items()}
BLOCK_ELEMS = {Q4_0: 32, Q5_0: 32, Q5_1: 32, Q8_0: 32, Q4_K: 256, Q6_K: 256, F32: 1, F16: 1,
               Q4_1: 32, Q2_K: 256, Q3_K: 256, Q5_K: 256}
BLOCK_BYTES = {Q4_0: 18, Q5_0: 22, Q5_1: 24, Q8_0: 34, Q4_K: 144, Q6_K: 210, F32: 4, F16: 2,
               Q4_1: 20, Q2_K: 84, Q3_K: 110, Q5_K: 176}
COMM_DEFAULT_TIMEOUT_MS = 300000  # IB_COMM_DEFAULT_TIMEOUT_MS
# byte alignment the GEMV entry points require of a weight base
GEMV_ALIGN = {Q4_0: 2, Q5_0: 2, Q5_1: 8, Q8_0: 2, Q4_K: 16, Q6_K: 2,
              Q4_1: 4, Q2_K: 4, Q3_K: 2, Q5_K: 16}

IB_OK = 0
IB_ERR_INVALID, IB_ERR_CUDA, IB_ERR_UNSUPPORTED, IB_ERR_OOM, IB_ERR_TIMEOUT, IB_ERR_COMM = range(1, 7)

_c = ctypes
_vp, _i, _i64, _f, _sz, _u64 = _c.c_void_p, _c.c_int, _c.c_int64, _c.c_float, _c.c_size_t, _c.c_uint64

# name -> argtypes (restype is int unless listed in _RESTYPE)
SIGNATURES = {
    "ib_last_error": [],
    "ib_version": [],
    "ib_type_info": [_i, _vp, _vp],
    "ib_init": [_i],
    "ib_available": [],
    "ib_device_name": [_c.c_char_p, _sz],
    "ib_memory_info": [_vp, _vp],
    "ib_sync": [],
    "ib_check_fault": [_vp],
    "ib_shutdown": [],
    "ib_alloc": [_vp, _sz],
    "ib_free": [_vp],
    "ib_upload": [_vp, _vp, _sz, _vp],
    "ib_download": [_vp, _vp, _sz, _vp],
    "ib_memset": [_vp, _i, _sz, _vp],
    "ib_dequant_f32": [_i, _vp, _vp, _i64, _i64, _vp],
    "ib_dequant_i16": [_i, _vp, _vp, _vp, _i64, _i64, _vp],
    "ib_gemv_q": [_i, _vp, _vp, _vp, _i64, _i64, _vp],
    "ib_gemv_q_noalloc": [_i, _vp, _vp, _vp, _i64, _i64, _vp],
    "ib_slab_bytes": [_i, _i64, _vp],
    "ib_limb_slab": [_i, _vp, _i64, _vp, _vp],
    "ib_gemv_q_slab": [_i, _vp, _vp, _vp, _i64, _i64, _vp],
    "ib_gemv_q_slab_chained": [_i, _vp, _vp, _vp, _i64, _i64, _vp],
    "ib_comm_unique_id": [_vp],
    "ib_comm_init": [_i, _i, _vp, _i, _vp],
    "ib_comm_init_timeout": [_i, _i, _vp, _i, _i64, _vp],
    "ib_comm_failed": [_vp, _vp],
    "ib_comm_abort": [_vp],
    "ib_peer_setup_check": [_i, _i, _i, _i, _i, _vp, _vp, _vp, _vp],
    "ib_model_tp_exchange_time": [_vp, _i, _vp],
    "ib_model_set_kv_type": [_vp, _i],
    "ib_model_kv_type": [_vp, _vp],
    "ib_comm_allreduce_f32": [_vp, _vp, _i64, _vp],
    "ib_comm_free": [_vp],
    "ib_tp_shard": [_i, _vp, _i64, _i64, _i, _i, _i, _vp],
    "ib_gemm_q": [_i, _vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "ib_gemm_set_path": [_i],
    "ib_gemm_planes_bytes": [_i64, _i64],
    "ib_gemm_prepare_planes": [_i, _vp, _i64, _i64, _vp, _vp],
    "ib_gemm_planes": [_vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "ib_model_set_prefill_planes": [_vp, _i],
    "ib_embedding_q": [_i, _vp, _vp, _vp, _i, _i64, _i64, _vp],
    "ib_gemv": [_vp, _vp, _vp, _i, _i, _vp],
    "ib_gemv_i16": [_vp, _vp, _vp, _vp, _i, _i, _vp],
    "ib_gemm": [_vp, _vp, _vp, _i, _i, _i, _vp],
    "ib_gemm_i16": [_vp, _vp, _vp, _vp, _i, _i, _i, _vp],
    "ib_rmsnorm": [_vp, _vp, _vp, _i, _i, _f, _vp],
    "ib_silu": [_vp, _i, _vp],
    "ib_mul": [_vp, _vp, _i, _vp],
    "ib_add": [_vp, _vp, _i, _vp],
    "ib_embedding": [_vp, _i, _vp, _i, _vp],
    "ib_embedding_i16": [_vp, _vp, _i, _vp, _i, _vp],
    "ib_embedding_batch": [_vp, _vp, _vp, _i, _i, _vp],
    "ib_embedding_batch_i16": [_vp, _vp, _vp, _vp, _i, _i, _vp],
    "ib_kv_write": [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp],
    "ib_kv_write_batch": [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp],
    "ib_rope": [_vp, _vp, _vp, _i, _i, _i, _i, _vp],
    "ib_rope_batch": [_vp, _vp, _vp, _i, _i, _i, _i, _i, _vp],
    "ib_attention": [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _f, _vp],
    "ib_attention_batch": [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _f, _vp],
    "ib_attention_split_part_bytes": [_i, _i],
    "ib_attention_split": [_vp, _vp, _vp, _vp, _i, _i, _i, _i, _vp, _f, _vp, _vp, _vp],
    "ib_kv_extend": [_vp, _vp, _i, _vp, _vp, _vp, _vp],
    "ib_kv_fork": [_vp, _vp, _i, _vp, _vp, _vp, _vp],
    "ib_kv_granted": [_i, _vp, _vp, _vp, _vp],
    "ib_kv_release": [_vp, _vp, _i, _vp, _vp],
    "ib_kv_compact": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "ib_kv_wait_selftest": [_vp],
    "ib_kv_append": [_vp, _vp, _vp, _i, _i, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i,
                     _vp],
    "ib_attention_paged_workspace": [_vp, _vp, _vp, _i],
    "ib_attention_paged": [_vp, _vp, _vp, _i, _i, _vp, _i64, _vp, _i64, _f, _vp, _sz, _vp],
    "ib_kv_reorder_workspace": [_vp, _i],
    "ib_kv_reorder": [_vp, _vp, _i, _vp, _vp, _vp, _vp, _sz, _vp],
    "ib_kv_tree_plan": [_vp, _vp, _i, _vp, _vp, _vp],
    "ib_kv_append_tree": [_vp, _vp, _vp, _vp, _i, _i, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64,
                          _vp, _i, _vp],
    "ib_attention_paged_tree_workspace": [_vp, _vp, _vp, _vp, _i],
    "ib_attention_paged_tree": [_vp, _vp, _vp, _vp, _i, _i, _vp, _i64, _vp, _i64, _f, _vp, _sz,
                                _vp],
    "ib_kv_tree_verify": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "ib_kv_tree_verify_max": [_vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "ib_kv_tree_accept": [_vp, _vp, _vp, _vp, _vp, _vp],
    "ib_kv_tree_accept_max": [_vp, _vp, _vp, _i, _vp, _vp, _vp],
    "ib_beam_select_workspace": [_i, _i, _i, _i],
    "ib_beam_select": [_i, _vp, _i64, _vp, _vp, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _sz, _vp],
    "ib_argmax": [_vp, _i, _vp, _vp],
    "ib_synth_host": [_i, _i64, _i64, _u64, _f, _vp, _i],
    "ib_synth_device": [_i, _i64, _i64, _u64, _f, _vp, _vp],
    "ib_synth_values_host": [_i64, _u64, _f, _vp],
}
_RESTYPE = {"ib_last_error": _c.c_char_p, "ib_attention_split_part_bytes": _c.c_size_t,
            "ib_gemm_planes_bytes": _c.c_size_t, "ib_attention_paged_workspace": _c.c_size_t,
            "ib_attention_paged_tree_workspace": _c.c_size_t,
            "ib_kv_reorder_workspace": _c.c_size_t, "ib_beam_select_workspace": _c.c_size_t}

_lib = None


def lib() -> ctypes.CDLL:
    """Load libib_cuda.so (raises if it has not been built: there is no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"libib_cuda.so not found at {LIB_PATH}; run inference.cpp_b200/build.py")
        L = ctypes.CDLL(LIB_PATH)
        for name, argt in SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = argt
            fn.restype = _RESTYPE.get(name, _i)
        _lib = L
    return _lib


def last_error() -> str:
    # messages can quote names read from a file, which need not be valid UTF-8
    return (lib().ib_last_error() or b"").decode("utf-8", errors="replace")


def check(status: int, what: str = "") -> None:
    if status != IB_OK:
        raise RuntimeError(last_error() or f"{what} failed with status {status}")


def call(name: str, *args) -> None:
    check(getattr(lib(), name)(*args), name)


def packed_nbytes(type_: int, rows: int, cols: int) -> int:
    return rows * (cols // BLOCK_ELEMS[type_]) * BLOCK_BYTES[type_]


# ---------------------------------------------------------------------------
# torch-facing helpers (device memory as torch tensors; pointers go to the C ABI)
# ---------------------------------------------------------------------------

def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(stream) -> int | None:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream or None
    return stream


def init(device: int = 0) -> None:
    call("ib_init", device)


def available() -> bool:
    return bool(lib().ib_available())


def device_name() -> str:
    buf = ctypes.create_string_buffer(256)
    call("ib_device_name", buf, 256)
    return buf.value.decode()


def memory_info() -> tuple[int, int]:
    f, t = ctypes.c_size_t(), ctypes.c_size_t()
    call("ib_memory_info", ctypes.byref(f), ctypes.byref(t))
    return f.value, t.value


def sync() -> None:
    call("ib_sync")


def check_fault() -> int:
    """Raises if a bounded pipeline wait expired since the last check, or a kernel of the paged
    cache passed over a bad value."""
    code = ctypes.c_int()
    call("ib_check_fault", ctypes.byref(code))
    return code.value


def dequantize(type_: int, W, rows: int, cols: int, out=None, stream=None):
    import torch
    if out is None:
        out = torch.empty(rows * cols, dtype=torch.float32, device=W.device)
    call("ib_dequant_f32", type_, _ptr(W), _ptr(out), rows, cols, _stream(stream))
    return out


def dequantize_i16(type_: int, W, rows: int, cols: int, stream=None):
    import torch
    q = torch.empty(rows * cols, dtype=torch.int16, device=W.device)
    s = torch.empty(rows, dtype=torch.float32, device=W.device)
    call("ib_dequant_i16", type_, _ptr(W), _ptr(q), _ptr(s), rows, cols, _stream(stream))
    return q, s


def gemv_q(type_: int, W, x, rows: int, cols: int, y=None, stream=None):
    import torch
    if y is None:
        y = torch.empty(rows, dtype=torch.float32, device=x.device)
    call("ib_gemv_q", type_, _ptr(W), _ptr(x), _ptr(y), rows, cols, _stream(stream))
    return y


NOALLOC_MAX_COLS = 32768


def gemv_q_noalloc(type_: int, W, x, y, rows: int, cols: int, stream=None):
    """ib_gemv_q with its scratch in a static device array: y must be given (the
    call allocates nothing); cols <= NOALLOC_MAX_COLS."""
    call("ib_gemv_q_noalloc", type_, _ptr(W), _ptr(x), _ptr(y), rows, cols, _stream(stream))
    return y


def limb_slab(type_: int, x, cols: int, slab=None, stream=None):
    """Exact int8 limb split of x for GEMVs on weights of `type_`'s family."""
    import torch
    if slab is None:
        n = ctypes.c_size_t()
        call("ib_slab_bytes", type_, cols, ctypes.byref(n))
        slab = torch.empty(n.value, dtype=torch.uint8, device=x.device)
    call("ib_limb_slab", type_, _ptr(x), cols, _ptr(slab), _stream(stream))
    return slab


def gemv_q_slab(type_: int, W, slab, rows: int, cols: int, y=None, stream=None,
                chained: bool = False):
    """chained: ib_gemv_q_slab_chained (the launch may stream its weights while the
    previous kernel on the stream runs; no earlier kernel may write W)."""
    import torch
    if y is None:
        y = torch.empty(rows, dtype=torch.float32, device=W.device)
    call("ib_gemv_q_slab_chained" if chained else "ib_gemv_q_slab", type_, _ptr(W), _ptr(slab),
         _ptr(y), rows, cols, _stream(stream))
    return y


def tp_shard(type_: int, data, rows: int, cols: int, axis: int, rank: int, world: int):
    """Host shard of a packed [rows, cols] tensor (numpy uint8/float32 array)."""
    import numpy as np
    src = np.ascontiguousarray(data)
    n = packed_nbytes(type_, rows, cols) // world
    dst = np.empty(n, dtype=np.uint8)
    call("ib_tp_shard", type_, src.ctypes.data, rows, cols, axis, rank, world, dst.ctypes.data)
    return dst


class Comm:
    """NCCL communicator for tensor parallelism (one process per GPU), in NCCL's
    non-blocking mode: initialisation and every later call settle within timeout_ms or
    raise (IB_ERR_TIMEOUT), and the communicator is then aborted."""

    def __init__(self, rank: int, world: int, uid: bytes, device: int = 0,
                 timeout_ms: int = COMM_DEFAULT_TIMEOUT_MS):
        buf = (ctypes.c_uint8 * 128).from_buffer_copy(uid)
        h = ctypes.c_void_p()
        call("ib_comm_init_timeout", rank, world, buf, device, timeout_ms, ctypes.byref(h))
        self.h, self.rank, self.world = h, rank, world

    @property
    def failed(self) -> bool:
        f = ctypes.c_int()
        call("ib_comm_failed", self.h, ctypes.byref(f))
        return bool(f.value)

    def abort(self):
        call("ib_comm_abort", self.h)

    @staticmethod
    def unique_id() -> bytes:
        buf = (ctypes.c_uint8 * 128)()
        call("ib_comm_unique_id", buf)
        return bytes(buf)

    def allreduce(self, t, stream=None):
        call("ib_comm_allreduce_f32", self.h, _ptr(t), t.numel(), _stream(stream))
        return t

    def close(self):
        if self.h:
            call("ib_comm_free", self.h)
            self.h = None


GATHER_FN = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                             ctypes.c_size_t)


def peer_setup_check(rank: int, world: int, gather, local_status: int = 0, fail_rank: int = -1,
                     fail_step: int = 0):
    """The tensor-parallel peer-memory set-up protocol with a stand-in IPC layer over
    `gather(bytes) -> list of world bytes objects` (ib_peer_setup_check).  Returns
    (status code, error text or "", mappings made, mappings released)."""
    def cb(_ctx, mine, out, n):
        try:
            parts = gather(ctypes.string_at(mine, n))
            blob = b"".join(parts)
            if len(blob) != n * world:
                return 1
            ctypes.memmove(out, blob, len(blob))
            return 0
        except Exception:  # a rank that left: the protocol reports the failure
            return 1
    fn = GATHER_FN(cb)
    opened, closed = ctypes.c_int(), ctypes.c_int()
    rc = lib().ib_peer_setup_check(rank, world, local_status, fail_rank, fail_step,
                                   ctypes.cast(fn, ctypes.c_void_p), None, ctypes.byref(opened),
                                   ctypes.byref(closed))
    return rc, (last_error() if rc else ""), opened.value, closed.value


def gemm_prepare_planes(type_: int, W, rows: int, cols: int, stream=None):
    """The packed weights decoded once into FP16 hi/lo planes (a uint8 CUDA tensor of
    ib_gemm_planes_bytes bytes) for gemm_planes."""
    import torch
    P = torch.empty(lib().ib_gemm_planes_bytes(rows, cols), dtype=torch.uint8, device="cuda")
    call("ib_gemm_prepare_planes", type_, _ptr(W), rows, cols, _ptr(P), _stream(stream))
    return P


def gemm_planes(P, X, T: int, rows: int, cols: int, Y=None, stream=None):
    import torch
    if Y is None:
        Y = torch.empty(T * rows, dtype=torch.float32, device="cuda")
    call("ib_gemm_planes", _ptr(P), _ptr(X), _ptr(Y), T, rows, cols, _stream(stream))
    return Y


def gemm_q(type_: int, W, X, T: int, rows: int, cols: int, Y=None, stream=None):
    import torch
    if Y is None:
        Y = torch.empty(T * rows, dtype=torch.float32, device=X.device)
    call("ib_gemm_q", type_, _ptr(W), _ptr(X), _ptr(Y), T, rows, cols, _stream(stream))
    return Y


GEMM_TENSOR_CORES, GEMM_CUDA_CORES, GEMM_TC_STAGED, GEMM_TC_PLANES = 0, 1, 2, 3


def gemm_set_path(path: int) -> None:
    """Kernel behind gemm_q (process-wide): GEMM_TENSOR_CORES (tcgen05, automatic choice;
    default), GEMM_CUDA_CORES, or one tcgen05 kernel: GEMM_TC_STAGED (weights decoded per
    tile in the kernel) or GEMM_TC_PLANES (weights decoded once into FP16 planes, TMA)."""
    call("ib_gemm_set_path", path)


def embedding_q(type_: int, table, ids, vocab: int, dim: int, out=None, stream=None):
    import torch
    T = ids.numel()
    if out is None:
        out = torch.empty(T * dim, dtype=torch.float32, device=ids.device)
    call("ib_embedding_q", type_, _ptr(table), _ptr(ids), _ptr(out), T, vocab, dim, _stream(stream))
    return out


# Reference-named FP32 / INT16 operators (include/ops/cuda_backend.hpp:31-64).
def gemv(W, x, y, M, N, stream=None):
    call("ib_gemv", _ptr(W), _ptr(x), _ptr(y), M, N, _stream(stream))


def gemv_i16(W, row_scale, x, y, M, N, stream=None):
    call("ib_gemv_i16", _ptr(W), _ptr(row_scale), _ptr(x), _ptr(y), M, N, _stream(stream))


def gemm(W, X, Y, T, M, K, stream=None):
    call("ib_gemm", _ptr(W), _ptr(X), _ptr(Y), T, M, K, _stream(stream))


def gemm_i16(W, row_scale, X, Y, T, M, K, stream=None):
    call("ib_gemm_i16", _ptr(W), _ptr(row_scale), _ptr(X), _ptr(Y), T, M, K, _stream(stream))


def rmsnorm(x, w, out, rows, dim, eps, stream=None):
    call("ib_rmsnorm", _ptr(x), _ptr(w), _ptr(out), rows, dim, eps, _stream(stream))


def silu(x, n, stream=None):
    call("ib_silu", _ptr(x), n, _stream(stream))


def mul(a, b, n, stream=None):
    call("ib_mul", _ptr(a), _ptr(b), n, _stream(stream))


def add(a, b, n, stream=None):
    call("ib_add", _ptr(a), _ptr(b), n, _stream(stream))


def embedding(table, id_, out, dim, stream=None):
    call("ib_embedding", _ptr(table), id_, _ptr(out), dim, _stream(stream))


def embedding_i16(table, row_scale, id_, out, dim, stream=None):
    call("ib_embedding_i16", _ptr(table), _ptr(row_scale), id_, _ptr(out), dim, _stream(stream))


def embedding_batch(table, ids, out, T, dim, stream=None):
    call("ib_embedding_batch", _ptr(table), _ptr(ids), _ptr(out), T, dim, _stream(stream))


def embedding_batch_i16(table, row_scale, ids, out, T, dim, stream=None):
    call("ib_embedding_batch_i16", _ptr(table), _ptr(row_scale), _ptr(ids), _ptr(out), T, dim,
         _stream(stream))


def kv_write(kc, vc, k, v, n_heads, head_dim, max_seq, pos, stream=None):
    call("ib_kv_write", _ptr(kc), _ptr(vc), _ptr(k), _ptr(v), n_heads, head_dim, max_seq, pos,
         _stream(stream))


def kv_write_batch(kc, vc, k, v, n_heads, head_dim, max_seq, start, T, stream=None):
    call("ib_kv_write_batch", _ptr(kc), _ptr(vc), _ptr(k), _ptr(v), n_heads, head_dim, max_seq,
         start, T, _stream(stream))


def rope(q, k, table, n_heads, n_kv_heads, head_dim, pos, stream=None):
    call("ib_rope", _ptr(q), _ptr(k), _ptr(table), n_heads, n_kv_heads, head_dim, pos,
         _stream(stream))


def rope_batch(q, k, table, n_heads, n_kv_heads, head_dim, start, T, stream=None):
    call("ib_rope_batch", _ptr(q), _ptr(k), _ptr(table), n_heads, n_kv_heads, head_dim, start, T,
         _stream(stream))


def attention(q, kc, vc, out, n_heads, n_kv_heads, head_dim, max_seq, pos, scale, stream=None):
    call("ib_attention", _ptr(q), _ptr(kc), _ptr(vc), _ptr(out), n_heads, n_kv_heads, head_dim,
         max_seq, pos, scale, _stream(stream))


def attention_split(q, kc, vc, out, n_heads, n_kv_heads, head_dim, max_seq, pos_dev, scale,
                    part, counters, stream=None):
    """Decode attention through the decode step's split kernel; the position is read
    from the int32 device word pos_dev.  part: attention_split_part_bytes(n_heads,
    head_dim) bytes of scratch; counters: n_kv_heads zeroed int32, left zeroed."""
    call("ib_attention_split", _ptr(q), _ptr(kc), _ptr(vc), _ptr(out), n_heads, n_kv_heads,
         head_dim, max_seq, _ptr(pos_dev), scale, _ptr(part), _ptr(counters), _stream(stream))


def attention_split_part_bytes(n_heads, head_dim):
    return lib().ib_attention_split_part_bytes(n_heads, head_dim)


def attention_batch(q, kc, vc, out, n_heads, n_kv_heads, head_dim, max_seq, start, T, scale,
                    stream=None):
    call("ib_attention_batch", _ptr(q), _ptr(kc), _ptr(vc), _ptr(out), n_heads, n_kv_heads,
         head_dim, max_seq, start, T, scale, _stream(stream))


def argmax(x, n, out, stream=None):
    call("ib_argmax", _ptr(x), n, _ptr(out), _stream(stream))


# ---------------------------------------------------------------------------
# paged KV cache (ib_kv_*, ib_attention_paged)
# ---------------------------------------------------------------------------

@functools.cache
def _torch():
    import torch
    return torch


@functools.cache
def _raw_stream():
    """Device index -> handle of its current stream, without building a Stream object where torch
    offers that (a tenth of a microsecond instead of two, on calls of ten)."""
    fast = getattr(_torch()._C, "_cuda_getCurrentRawStream", None)
    return fast or (lambda index: _torch().cuda.current_stream(index).cuda_stream)


@functools.cache
def _entry(name):
    return getattr(lib(), name)


def _call(name, *args):  # call(), without looking the function up again
    status = _entry(name)(*args)
    if status != IB_OK:
        check(status, name)


class _CKVPages(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("n_layers", ctypes.c_int32),
                ("n_pages", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("k", ctypes.c_void_p), ("v", ctypes.c_void_p)]


class _CKVSeqs(ctypes.Structure):
    _fields_ = [("n_slots", ctypes.c_int32), ("max_pages", ctypes.c_int32),
                ("table", ctypes.c_void_p), ("len", ctypes.c_void_p), ("refs", ctypes.c_void_p)]


class _CKVBatch(ctypes.Structure):
    _fields_ = [("n_seqs", ctypes.c_int32), ("n_tokens", ctypes.c_int32),
                ("max_q", ctypes.c_int32), ("cu_q", ctypes.c_void_p), ("slots", ctypes.c_void_p)]


def _paged_tensor(t, name, dtype, shape, device):
    """t as the paged calls take it: a contiguous CUDA tensor; -1 in shape is any size."""
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.dim() != len(shape) or any(w not in (-1, g) for g, w in zip(t.shape, shape)):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name}: on {t.device}, expected {device or 'a CUDA device'}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: not contiguous")
    return t


def _tensor_ptr(t, name, dtype, shape, dev):
    """Pointer of such a tensor (None: none), without the messages' work where it is one."""
    if t is None:
        return None
    if not (t.dtype is dtype and t.shape == shape and t.device == dev and t.is_contiguous()):
        _paged_tensor(t, name, dtype, shape, dev)
    return t.data_ptr()


class KVPages:
    """A pool of KV pages: k and v each [n_layers, n_pages, n_kv_heads, page_size, head_dim],
    float32 or float16 CUDA tensors (kept here; the calls work on them in place)."""

    def __init__(self, k, v):
        import torch
        if k.dtype not in (torch.float32, torch.float16):
            raise ValueError(f"k: dtype {k.dtype}, expected float32 or float16")
        self.k = _paged_tensor(k, "k", k.dtype, (-1,) * 5, None)
        self.v = _paged_tensor(v, "v", k.dtype, k.shape, k.device)
        self.device = k.device
        self.type = F32 if k.dtype == torch.float32 else F16
        self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self._c = _CKVPages(self.type, self.n_layers, self.n_pages, self.n_kv_heads,
                            self.page_size, self.head_dim, k.data_ptr(), v.data_ptr())
        self._p = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, n_layers, n_pages, n_kv_heads, page_size, head_dim, type_=F32, device="cuda"):
        import torch
        dt = {F32: torch.float32, F16: torch.float16}.get(type_)
        if dt is None:
            raise ValueError(f"pages must be F32 or F16, not {TYPE_NAMES.get(type_, type_)}")
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dt, device=device),
                   torch.empty(shape, dtype=dt, device=device))


class KVSeqs:
    """The sequences of a pool: table [n_slots, max_pages] (-1: no page), len [n_slots] and
    refs [n_pages], int32 CUDA tensors (kept here; the calls work on them in place)."""

    def __init__(self, table, len, refs):
        import torch
        self.table = _paged_tensor(table, "table", torch.int32, (-1, -1), None)
        self.device = table.device
        self.n_slots, self.max_pages = table.shape
        self.len = _paged_tensor(len, "len", torch.int32, (self.n_slots,), self.device)
        self.refs = _paged_tensor(refs, "refs", torch.int32, (-1,), self.device)
        self.n_refs = refs.numel()
        self._c = _CKVSeqs(self.n_slots, self.max_pages, table.data_ptr(), len.data_ptr(),
                           refs.data_ptr())
        self._p = ctypes.addressof(self._c)

    @classmethod
    def empty(cls, n_slots, max_pages, n_pages, device="cuda"):
        import torch
        return cls(torch.full((n_slots, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_slots, dtype=torch.int32, device=device),
                   torch.zeros(n_pages, dtype=torch.int32, device=device))


class KVBatch:
    """A step's new tokens: rows cu_q[b] .. cu_q[b + 1] of its n_tokens rows are the last
    tokens of sequence b (slot slots[b], or slot b; -1: left out of the step, kv_granted).  cu_q,
    slots: int32 CUDA tensors.  max_q: the most tokens of one sequence where known (chooses
    kernels only)."""

    def __init__(self, cu_q, n_tokens, max_q=0, slots=None):
        import torch
        self.cu_q = _paged_tensor(cu_q, "cu_q", torch.int32, (-1,), None)
        self.device = cu_q.device
        self.n_seqs, self.n_tokens = cu_q.numel() - 1, int(n_tokens)
        self.slots = slots
        if slots is not None:
            _paged_tensor(slots, "slots", torch.int32, (self.n_seqs,), self.device)
        self._c = _CKVBatch(self.n_seqs, self.n_tokens, int(max_q), cu_q.data_ptr(), _ptr(slots))
        self._p = ctypes.addressof(self._c)


def _paged_stream(pages, stream, *others):
    """The stream to launch on, after checking that everything is on the current device."""
    dev = pages.device
    for o in others:
        if o.device != dev:
            raise ValueError(f"arguments on {dev} and {o.device}")
    cuda, index = _torch().cuda, dev.index
    if cuda.current_device() != index:
        raise ValueError(f"the pages are on {dev}, the current device is "
                         f"cuda:{cuda.current_device()}")
    return (_raw_stream()(index) or None) if stream is None else stream


def _allocating(pages, stream):
    """Context for the tensors that a call makes: of the launch stream's memory pool, where they
    may be handed out again, in stream order, once they are dropped."""
    if stream is None:
        return contextlib.nullcontext()
    cuda = _torch().cuda
    return cuda.stream(cuda.ExternalStream(stream, pages.device) if stream else
                       cuda.default_stream(pages.device))


def _seqs_of(pages, seqs):
    if seqs.n_refs != pages.n_pages:
        raise ValueError(f"refs: {seqs.n_refs} entries for {pages.n_pages} pages")
    return seqs._p


def _paged_list(pages, t, name, n):
    """Pointer of a contiguous int32 list of n entries on the pages' device."""
    if t.dtype is _torch().int32 and t.shape == (n,) and t.device == pages.device \
            and t.is_contiguous():
        return t.data_ptr()
    if t.dtype != _torch().int32:
        raise ValueError(f"{name}: dtype {t.dtype}, expected torch.int32")
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected ({n},)")
    if t.device != pages.device or not t.is_contiguous():
        raise ValueError(f"{name}: on {t.device}, contiguous {t.is_contiguous()}; expected "
                         f"contiguous on {pages.device}")
    return t.data_ptr()


def kv_extend(pages, seqs, slots, n_new, status=None, stream=None):
    """Room for n_new[i] more tokens of each slot; returns status (1 done, 0 no room,
    -1 refused), int32 tensors on the pages' device.  A step must not go on with a sequence that
    got no room (its last tokens would be written over): kv_granted makes the batch's slots."""
    if status is None:
        with _allocating(pages, stream):
            status = _torch().empty_like(slots)
    n = slots.numel()
    a, b, c = (_paged_list(pages, slots, "slots", n), _paged_list(pages, n_new, "n_new", n),
               _paged_list(pages, status, "status", n))
    st = _paged_stream(pages, stream, seqs)
    _call("ib_kv_extend", pages._p, _seqs_of(pages, seqs), n, a, b, c, st)
    return status


def kv_fork(pages, seqs, parents, children, status=None, stream=None):
    """children[i] becomes a copy of parents[i], sharing its whole pages; returns status."""
    if status is None:
        with _allocating(pages, stream):
            status = _torch().empty_like(parents)
    n = parents.numel()
    a, b, c = (_paged_list(pages, parents, "parents", n),
               _paged_list(pages, children, "children", n),
               _paged_list(pages, status, "status", n))
    st = _paged_stream(pages, stream, seqs)
    _call("ib_kv_fork", pages._p, _seqs_of(pages, seqs), n, a, b, c, st)
    return status


def kv_granted(pages, slots, status, out=None, stream=None):
    """slots with -1 where status (of kv_extend, or of kv_fork for its children) is not 1: the
    slots of a step's batch, or of the kv_extend behind a kv_fork.  out may be slots."""
    n = slots.numel()
    if out is None:
        with _allocating(pages, stream):
            out = _torch().empty_like(slots)
    a, b, c = (_paged_list(pages, slots, "slots", n), _paged_list(pages, status, "status", n),
               _paged_list(pages, out, "out", n))
    _call("ib_kv_granted", n, a, b, c, _paged_stream(pages, stream))
    return out


def kv_release(pages, seqs, slots, stream=None):
    """The slots give up their pages."""
    n = slots.numel()
    a = _paged_list(pages, slots, "slots", n)
    st = _paged_stream(pages, stream, seqs)
    _call("ib_kv_release", pages._p, _seqs_of(pages, seqs), n, a, st)


def _workspace(pages, workspace):
    """(pointer, bytes) of a caller's workspace on the pages' device."""
    if workspace.device != pages.device or not workspace.is_contiguous():
        raise ValueError(f"workspace: on {workspace.device}, contiguous "
                         f"{workspace.is_contiguous()}; expected contiguous on {pages.device}")
    return workspace.data_ptr(), workspace.nbytes


def kv_reorder_workspace(seqs, n):
    """Scratch for kv_reorder calls with n slots, one at a time (a uint8 CUDA tensor)."""
    size = lib().ib_kv_reorder_workspace(seqs._p, n)
    if size == 0:
        raise ValueError(last_error())
    return _torch().empty(size, dtype=_torch().uint8, device=seqs.device)


def kv_reorder(pages, seqs, slots, parents, status=None, workspace=None, stream=None):
    """slots[i] becomes what slots[parents[i]] held, all at once (-1: it is left empty): the states
    of a beam search behind beam_select, whose rows are the parents.  Whole pages are shared, a
    partial last page goes to one of those that take it and is copied for the others.  Returns
    status (1 done, 0 no page for the copy: left empty, -1 refused: as it was).  workspace:
    kv_reorder_workspace(), allocated for the call when None."""
    n = slots.numel()
    st = _paged_stream(pages, stream, seqs)
    if status is None or workspace is None:
        with _allocating(pages, stream):
            status = _torch().empty_like(slots) if status is None else status
            workspace = kv_reorder_workspace(seqs, n) if workspace is None else workspace
    a, b, c = (_paged_list(pages, slots, "slots", n), _paged_list(pages, parents, "parents", n),
               _paged_list(pages, status, "status", n))
    _call("ib_kv_reorder", pages._p, _seqs_of(pages, seqs), n, a, b, c, *_workspace(pages, workspace),
          st)
    return status


class KVCompactPlan:
    """What kv_compact did: map [n_pages] (new index of each page, -1 for a free one), info
    {pages in use, pages moved} and the moves' (old, new) pairs."""

    def __init__(self, pages):
        import torch
        n = pages.n_pages
        self.map = torch.empty(n, dtype=torch.int32, device=pages.device)
        self.moves = torch.empty(n, dtype=torch.int32, device=pages.device)
        self.info = torch.empty(2, dtype=torch.int32, device=pages.device)
        self.n_live, self.n_moves = self.info[0], self.info[1]
        self.n_pages, self.device = n, pages.device


def kv_compact_plan(pages):
    return KVCompactPlan(pages)


def kv_compact(pages, seqs, out=None, plan=None, stream=None):
    """Moves the used pages to the lowest indices; the renamed table and refs, and the lengths, go
    to `out` (a KVSeqs; default: seqs itself; it may share arrays with seqs).  Returns the
    plan."""
    out = seqs if out is None else out
    if plan is None:
        with _allocating(pages, stream):
            plan = KVCompactPlan(pages)
    st = _paged_stream(pages, stream, seqs, out, plan)
    if out.table.shape != seqs.table.shape or plan.n_pages != pages.n_pages:
        raise ValueError("out or plan of another cache")
    _seqs_of(pages, out)
    _call("ib_kv_compact", pages._p, _seqs_of(pages, seqs), out.table.data_ptr(),
         out.refs.data_ptr(), plan.map.data_ptr(), plan.moves.data_ptr(), plan.info.data_ptr(),
         st)
    if out.len.data_ptr() != seqs.len.data_ptr():
        with _allocating(pages, stream):  # on the launch stream
            out.len.copy_(seqs.len)
    return plan


def _paged_rows(t, name, tokens, heads, head_dim, device):
    """(pointer, row stride, heads) of a float32 [tokens, heads, head_dim] tensor whose rows may
    be apart (slices of a projection's output); heads None: any number."""
    shape = t.shape
    if t.dtype != _torch().float32 or t.device != device:
        raise ValueError(f"{name}: {t.dtype} on {t.device}, expected float32 on {device}")
    if len(shape) != 3 or shape[0] != tokens or shape[2] != head_dim \
            or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name}: shape {tuple(shape)}, expected "
                         f"({tokens}, {heads or 'heads'}, {head_dim})")
    row, head, one = t.stride()
    heads = shape[1]
    if one != 1 or (head != head_dim and heads != 1):
        raise ValueError(f"{name}: the heads of a token are not contiguous")
    return t.data_ptr(), row if tokens > 1 else heads * head_dim, heads


class _CKVTree(ctypes.Structure):
    _fields_ = [("max_nodes", ctypes.c_int32), ("depth", ctypes.c_void_p), ("mask", ctypes.c_void_p)]


KV_MAX_NODES = 1024  # IB_KV_MAX_NODES


class KVTree:
    """The trees of a batch whose new tokens are drafts: parents [n_tokens] (an earlier node of the
    same sequence, or -1: what follows the context), depth [n_tokens] and mask [n_tokens,
    (max_nodes + 31) // 32] (bit c % 32 of word c // 32: node c is the row's own or an ancestor),
    int32 CUDA tensors, kept here; kv_tree fills depth and mask from the parents."""

    def __init__(self, parents, depth, mask, max_nodes):
        import torch
        max_nodes = int(max_nodes)
        if not 1 <= max_nodes <= KV_MAX_NODES:
            raise ValueError(f"max_nodes: {max_nodes}, expected 1 .. {KV_MAX_NODES}")
        self.parents = _paged_tensor(parents, "parents", torch.int32, (-1,), None)
        self.device, self.n_tokens, self.max_nodes = parents.device, parents.shape[0], max_nodes
        self.depth = _paged_tensor(depth, "depth", torch.int32, (self.n_tokens,), self.device)
        self.mask = _paged_tensor(mask, "mask", torch.int32,
                                  (self.n_tokens, (max_nodes + 31) // 32), self.device)
        self._c = _CKVTree(max_nodes, depth.data_ptr(), mask.data_ptr())
        self._p = ctypes.addressof(self._c)


def _tree_of(pages, batch, tree):
    if tree.device != pages.device:
        raise ValueError(f"arguments on {pages.device} and {tree.device}")
    if tree.n_tokens != batch.n_tokens:
        raise ValueError(f"tree: {tree.n_tokens} nodes for {batch.n_tokens} tokens")
    return tree._p


def _max_nodes_of(pages, batch, tree):
    _tree_of(pages, batch, tree)
    return tree.max_nodes


def kv_tree(batch, parents, max_nodes=0, out=None, stream=None):
    """The trees of a batch's new tokens from their parents: once a step, for every layer's
    kv_append and attention_paged.  max_nodes: the most nodes of one sequence, which the masks have
    room for (0: what the batch can have, its n_tokens up to KV_MAX_NODES; its max_q is a hint and
    bounds nothing); a sequence with more is left out of the step and recorded.  out: a KVTree of
    such a batch, whose depth and mask are filled again.  Returns the KVTree."""
    torch, T = _torch(), batch.n_tokens
    st = _paged_stream(batch, stream)
    p = _paged_list(batch, parents, "parents", T)
    if out is None:
        max_nodes = int(max_nodes) or min(T, KV_MAX_NODES) or 1
        with _allocating(batch, stream):
            out = KVTree(parents, torch.zeros(T, dtype=torch.int32, device=batch.device),
                         torch.zeros(T, (max_nodes + 31) // 32, dtype=torch.int32,
                                     device=batch.device), max_nodes)
    elif out.n_tokens != T or out.device != batch.device or max_nodes not in (0, out.max_nodes):
        raise ValueError("out: a tree of another batch")
    _call("ib_kv_tree_plan", batch._p, p, out.max_nodes, out.depth.data_ptr(), out.mask.data_ptr(),
          st)
    out.parents = parents
    return out


def kv_tree_verify(batch, parents, tokens, best, path=None, n_path=None, next=None, stream=None,
                   tree=None):
    """Greedy verification of the batch's trees.  tokens: the nodes' tokens (node 0's is certain),
    best: what the model chose behind each node (beam_select with k = 1), int32 [n_tokens].
    Returns path [n_tokens] (the confirmed nodes of a sequence, in its rows, -1 behind them),
    n_path and next [n_seqs] (the token behind the last confirmed node; -1: no nodes).  tree: the
    step's; a sequence with more nodes than its max_nodes, which the step has left out, has none."""
    torch, T, n = _torch(), batch.n_tokens, batch.n_seqs
    most = KV_MAX_NODES if tree is None else _max_nodes_of(batch, batch, tree)
    st = _paged_stream(batch, stream)
    if path is None or n_path is None or next is None:
        with _allocating(batch, stream):
            make = lambda m: torch.full((m,), -1, dtype=torch.int32, device=batch.device)  # noqa: E731
            path = make(T) if path is None else path
            n_path = make(n) if n_path is None else n_path
            next = make(n) if next is None else next
    _call("ib_kv_tree_verify_max", batch._p, most, _paged_list(batch, parents, "parents", T),
          _paged_list(batch, tokens, "tokens", T), _paged_list(batch, best, "best", T),
          _paged_list(batch, path, "path", T), _paged_list(batch, n_path, "n_path", n),
          _paged_list(batch, next, "next", n), st)
    return path, n_path, next


def kv_tree_accept(pages, seqs, batch, path, n_path, stream=None, tree=None):
    """Of the batch's new tokens only the path stays in the cache: its K and V move together in
    every layer, the lengths follow, and the pages behind them are given back.  path, n_path: as
    kv_tree_verify returns them, or the caller's own.  tree: the step's; of a sequence with more
    nodes than its max_nodes, which the step has left out, nothing stays."""
    st = _paged_stream(pages, stream, seqs, batch)
    most = KV_MAX_NODES if tree is None else _max_nodes_of(pages, batch, tree)
    _call("ib_kv_tree_accept_max", pages._p, _seqs_of(pages, seqs), batch._p, most,
          _paged_list(pages, path, "path", batch.n_tokens),
          _paged_list(pages, n_path, "n_path", batch.n_seqs), st)


def kv_append(pages, seqs, batch, layer, q, k, v, rope_table, q_out=None, stream=None, tree=None):
    """RoPE on q and k and the write of k and v into the layer's pages.  q [tokens, heads,
    head_dim], k and v [tokens, kv heads, head_dim] float32 (rows may be slices);
    rope_table [positions, head_dim / 2, 2].  tree: the new tokens are nodes of trees (kv_tree),
    rotated by their depths.  Returns q_out."""
    torch = _torch()
    T, HD, Hkv, dev = batch.n_tokens, pages.head_dim, pages.n_kv_heads, pages.device
    if q_out is None:
        with _allocating(pages, stream):
            q_out = torch.empty(q.shape, dtype=torch.float32, device=dev)
    qp, qs, H = _paged_rows(q, "q", T, None, HD, dev)
    kp, ks, _ = _paged_rows(k, "k", T, Hkv, HD, dev)
    vp, vs, _ = _paged_rows(v, "v", T, Hkv, HD, dev)
    op, os_, _ = _paged_rows(q_out, "q_out", T, H, HD, dev)
    n = rope_table.shape[0]
    rope = _tensor_ptr(rope_table, "rope_table", torch.float32, (n, HD // 2, 2), dev)
    st = _paged_stream(pages, stream, seqs, batch)
    args = (layer, H, qp, qs, kp, ks, vp, vs, op, os_, rope, n, st)
    if tree is None:
        _call("ib_kv_append", pages._p, _seqs_of(pages, seqs), batch._p, *args)
    else:
        _call("ib_kv_append_tree", pages._p, _seqs_of(pages, seqs), batch._p,
              _tree_of(pages, batch, tree), *args)
    return q_out


def attention_paged_workspace(pages, seqs, batch, n_heads, tree=None):
    """Scratch for attention_paged calls of this shape, one at a time (a uint8 CUDA tensor)."""
    import torch
    if tree is None:
        n = lib().ib_attention_paged_workspace(pages._p, seqs._p, batch._p, n_heads)
    else:
        n = lib().ib_attention_paged_tree_workspace(pages._p, seqs._p, batch._p,
                                                    _tree_of(pages, batch, tree), n_heads)
    if n == 0:
        raise ValueError(last_error())
    return torch.empty(n, dtype=torch.uint8, device=pages.device)


def attention_paged(pages, seqs, batch, layer, q, scale, out=None, workspace=None, stream=None,
                    tree=None):
    """Causal attention of the batch's new tokens over the layer's pages.  q, out [tokens,
    heads, head_dim] float32 (rows may be slices).  workspace: attention_paged_workspace(),
    allocated for the call when None.  tree: the new tokens are nodes of trees (kv_tree): each sees
    the context, its ancestors and itself; the workspace is then one made with the tree.  Returns
    out (rows of nobody: as they were)."""
    torch = _torch()
    T, HD, dev = batch.n_tokens, pages.head_dim, pages.device
    qp, qs, H = _paged_rows(q, "q", T, None, HD, dev)
    if out is None:
        with _allocating(pages, stream):
            out = torch.zeros(q.shape, dtype=torch.float32, device=dev)
    op, os_, _ = _paged_rows(out, "out", T, H, HD, dev)
    st = _paged_stream(pages, stream, seqs, batch)
    if workspace is None:
        with _allocating(pages, stream):
            workspace = attention_paged_workspace(pages, seqs, batch, H, tree)
    elif workspace.device != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace: on {workspace.device}, expected contiguous on {dev}")
    args = (layer, H, qp, qs, op, os_, scale, workspace.data_ptr(), workspace.nbytes, st)
    if tree is None:
        _call("ib_attention_paged", pages._p, _seqs_of(pages, seqs), batch._p, *args)
    else:
        _call("ib_attention_paged_tree", pages._p, _seqs_of(pages, seqs), batch._p,
              _tree_of(pages, batch, tree), *args)
    return out


# ---------------------------------------------------------------------------
# beam search (ib_beam_select; the beams' states follow with kv_reorder)
# ---------------------------------------------------------------------------

class BeamChoice(typing.NamedTuple):
    """What beam_select chose, [groups, k], largest first: score float32, token and row int32
    (-inf, -1, -1 where there was no candidate)."""
    score: typing.Any
    token: typing.Any
    row: typing.Any


def _beam_shape(logits, beams, k):
    """(type, rows, vocab, groups, k) of a selection."""
    torch, dtype = _torch(), logits.dtype
    type_ = F32 if dtype is torch.float32 else F16 if dtype is torch.float16 else None
    if type_ is None or logits.dim() != 2 or not logits.is_cuda:
        raise ValueError(f"logits: {dtype} {tuple(logits.shape)} on {logits.device}, expected "
                         f"float32 or float16 [rows, vocab] on a CUDA device")
    rows, vocab = logits.shape
    if beams < 1 or rows % beams:
        raise ValueError(f"beams: {beams}, expected a divisor of {rows} rows")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("logits: the values of a row are not contiguous")
    return type_, rows, vocab, rows // beams, beams if k is None else int(k)


def beam_select_workspace(logits, beams=1, k=None):
    """Scratch for beam_select calls of this shape, one at a time (a uint8 CUDA tensor)."""
    _, _, vocab, groups, k = _beam_shape(logits, beams, k)
    n = lib().ib_beam_select_workspace(groups, beams, vocab, k)
    if n == 0:
        raise ValueError(last_error())
    return _torch().empty(n, dtype=_torch().uint8, device=logits.device)


def beam_select(logits, scores=None, beams=1, k=None, ended=None, end_token=0, out=None,
                workspace=None, stream=None):
    """The k (default: beams) best continuations of each group of `beams` rows of the logits [rows,
    vocab] (float32 or float16, rows may be apart): scores[row] + log_softmax(logits[row])[token],
    equal ones in the order of row and token.  ended [rows] int32: a row with a value other than 0
    offers (end_token, scores[row]) alone.  -inf and NaN are no candidates.  Returns a BeamChoice
    (out: one to be filled).  With beams = 1, the rows' top k; with k = 1, their argmax.
    workspace: beam_select_workspace(), allocated for the call when None."""
    torch = _torch()
    type_, rows, vocab, groups, k = _beam_shape(logits, beams, k)
    dev, f32, i32 = logits.device, torch.float32, torch.int32
    st = _paged_stream(logits, stream)
    if out is None or workspace is None:
        with _allocating(logits, stream):
            if out is None:
                out = BeamChoice(torch.empty(groups, k, device=dev),
                                 *(torch.empty(groups, k, dtype=i32, device=dev) for _ in range(2)))
            if workspace is None:
                workspace = beam_select_workspace(logits, beams, k)
    score, token, row = out
    per_row, per_group = (rows,), (groups, k)
    _call("ib_beam_select", type_, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab,
          _tensor_ptr(scores, "scores", f32, per_row, dev), _tensor_ptr(ended, "ended", i32, per_row, dev),
          end_token, groups, beams, vocab, k, _tensor_ptr(score, "out.score", f32, per_group, dev),
          _tensor_ptr(token, "out.token", i32, per_group, dev),
          _tensor_ptr(row, "out.row", i32, per_group, dev), *_workspace(logits, workspace), st)
    return out


# ---------------------------------------------------------------------------
# synthetic weights
# ---------------------------------------------------------------------------

def synth_host(type_: int, rows: int, cols: int, seed: int, std: float = 0.02, threads: int = 0):
    """Packed blocks (numpy uint8) of a [rows, cols] N(0, std) tensor quantised to type_."""
    import numpy as np
    if type_ == F32:
        out = np.empty(rows * cols, dtype=np.float32)
    else:
        out = np.empty(packed_nbytes(type_, rows, cols), dtype=np.uint8)
    call("ib_synth_host", type_, rows, cols, seed, std, out.ctypes.data, threads)
    return out


def synth_values(n: int, seed: int, std: float = 0.02):
    import numpy as np
    out = np.empty(n, dtype=np.float32)
    call("ib_synth_values_host", n, seed, std, out.ctypes.data)
    return out


def synth_device(type_: int, rows: int, cols: int, seed: int, std: float = 0.02, out=None,
                 device="cuda", stream=None):
    import torch
    if out is None:
        n = rows * cols * 4 if type_ == F32 else packed_nbytes(type_, rows, cols)
        out = torch.empty(n, dtype=torch.uint8, device=device)
    call("ib_synth_device", type_, rows, cols, seed, std, _ptr(out), _stream(stream))
    return out


# ---------------------------------------------------------------------------
# native model runner (ib_model_*): the generate_cuda counterpart
# ---------------------------------------------------------------------------
NATIVE, INT16, FP32 = 0, 1, 2
PRECISIONS = {"native": NATIVE, "int16": INT16, "fp32": FP32}


class ModelConfig(ctypes.Structure):
    _fields_ = [("n_layers", ctypes.c_int32), ("dim", ctypes.c_int32),
                ("n_heads", ctypes.c_int32), ("n_kv_heads", ctypes.c_int32),
                ("ffn", ctypes.c_int32), ("vocab", ctypes.c_int32),
                ("max_seq", ctypes.c_int32), ("rope_theta", ctypes.c_float),
                ("rms_eps", ctypes.c_float), ("precision", ctypes.c_int32)]


class GenerationStats(ctypes.Structure):
    _fields_ = [("init_ms", ctypes.c_double), ("prefill_ms", ctypes.c_double),
                ("decode_ms", ctypes.c_double), ("generated", ctypes.c_int32)]


SIGNATURES.update({
    "ib_model_create": [_vp, _i, _vp],
    "ib_model_create_tp": [_vp, _i, _vp, _vp],
    "ib_tp_wait_selftest": [_i, _vp, _vp],
    "ib_model_load_gguf_tp": [_c.c_char_p, _i, _i, _i, _vp, _vp],
    "ib_model_set_tensor": [_vp, _c.c_char_p, _i, _i64, _i64, _vp, _i],
    "ib_model_finalize": [_vp],
    "ib_model_load_gguf": [_c.c_char_p, _i, _i, _i, _vp],
    "ib_model_free": [_vp],
    "ib_model_prefill": [_vp, _vp, _i, _i, _vp, _vp],
    "ib_model_decode": [_vp, _c.c_int32, _i, _vp, _vp],
    "ib_model_generate": [_vp, _vp, _i, _i, _c.c_int32, _vp, _vp, _vp],
    "ib_model_set_graph": [_vp, _i],
    "ib_model_set_fused": [_vp, _i],
    "ib_model_uses_fused": [_vp, _vp],
    "ib_model_set_persistent": [_vp, _i],
    "ib_model_get_config": [_vp, _vp],
    "ib_model_decode_path": [_vp, _vp],
    "ib_model_weight_bytes": [_vp, _vp],
    "ib_model_decode_loop": [_vp, _c.c_int32, _i, _i, _vp],
    "ib_model_stream": [_vp, _vp],
    "ib_model_step_kernels": [_vp, _vp],
})


class Model:
    """A Llama model held on one GPU by the native runner."""

    def __init__(self, handle, vocab: int):
        self.h = ctypes.c_void_p(handle)
        self.vocab = vocab

    @classmethod
    def create(cls, cfg, precision: int = NATIVE, device: int = 0, max_seq: int | None = None,
               comm: "Comm | None" = None):
        """comm: split the model over the communicator's ranks (tensor parallelism)."""
        c = ModelConfig(cfg.n_layers, cfg.dim, cfg.n_heads, cfg.n_kv_heads, cfg.ffn, cfg.vocab,
                        max_seq or cfg.ctx, cfg.rope_theta, cfg.rms_eps, precision)
        h = ctypes.c_void_p()
        if comm is None:
            call("ib_model_create", ctypes.byref(c), device, ctypes.byref(h))
        else:
            call("ib_model_create_tp", ctypes.byref(c), device, comm.h, ctypes.byref(h))
        return cls(h.value, cfg.vocab)

    @classmethod
    def from_tensors(cls, cfg, tensors: dict, precision: int = NATIVE, device: int = 0,
                     max_seq: int | None = None, comm: "Comm | None" = None):
        """tensors: {gguf name: (type, rows, cols, numpy bytes or CUDA tensor)}."""
        m = cls.create(cfg, precision, device, max_seq, comm)
        for name, (t, r, c, data) in tensors.items():
            m.set_tensor(name, t, r, c, data)
        m.finalize()
        return m

    @classmethod
    def from_gguf(cls, path: str, precision: int = NATIVE, device: int = 0, max_seq: int = 0,
                  comm: "Comm | None" = None):
        h = ctypes.c_void_p()
        if comm is None:
            call("ib_model_load_gguf", path.encode(), precision, device, max_seq, ctypes.byref(h))
        else:
            call("ib_model_load_gguf_tp", path.encode(), precision, device, max_seq, comm.h,
                 ctypes.byref(h))
        from .gguf_writer import _read_vocab  # type: ignore
        return cls(h.value, _read_vocab(path))

    def set_tensor(self, name, type_, rows, cols, data):
        on_dev = 0
        if hasattr(data, "data_ptr"):
            ptr, on_dev = data.data_ptr(), 1 if data.is_cuda else 0
        else:
            ptr = data.ctypes.data
        call("ib_model_set_tensor", self.h, name.encode(), type_, rows, cols, ptr, on_dev)

    def finalize(self):
        call("ib_model_finalize", self.h)

    def set_graph(self, enabled: bool):
        call("ib_model_set_graph", self.h, 1 if enabled else 0)

    def set_fused(self, enabled: bool):
        call("ib_model_set_fused", self.h, 1 if enabled else 0)

    def uses_fused(self) -> bool:
        f = ctypes.c_int()
        call("ib_model_uses_fused", self.h, ctypes.byref(f))
        return bool(f.value)

    def set_persistent(self, enabled: bool):
        """The persistent decode step (one kernel per token) when the model supports it."""
        call("ib_model_set_persistent", self.h, 1 if enabled else 0)

    def decode_path(self) -> str:
        """Which decode step runs: "persistent" (one kernel per token), "fused" per-op
        kernels, or the "separate" kernels."""
        p = ctypes.c_int()
        call("ib_model_decode_path", self.h, ctypes.byref(p))
        return {0: "separate", 1: "fused", 2: "persistent"}[p.value]

    def set_prefill_planes(self, enabled: bool):
        """Keep every packed linear's weights decoded as FP16 hi/lo planes (4 bytes per
        weight) for the prompt GEMMs, or release them."""
        call("ib_model_set_prefill_planes", self.h, 1 if enabled else 0)

    def set_kv_type(self, type_: int):
        """KV cache element type: F32 (default) or F16.  On a finalized model the caches
        start empty again (prefill before decoding)."""
        call("ib_model_set_kv_type", self.h, type_)

    def kv_type(self) -> int:
        t = ctypes.c_int()
        call("ib_model_kv_type", self.h, ctypes.byref(t))
        return t.value

    def tp_exchange_us(self, rounds: int = 64) -> float:
        """Device time of one exchange round of the fused tensor-parallel step, in
        isolation (collective: every rank calls it with the same rounds)."""
        us = ctypes.c_float()
        call("ib_model_tp_exchange_time", self.h, rounds, ctypes.byref(us))
        return us.value

    def weight_bytes(self) -> int:
        n = ctypes.c_size_t()
        call("ib_model_weight_bytes", self.h, ctypes.byref(n))
        return n.value

    def prefill(self, ids, start: int = 0, want_logits: bool = False):
        import numpy as np
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        lg = np.empty(self.vocab, np.float32) if want_logits else None
        nxt = ctypes.c_int32()
        call("ib_model_prefill", self.h, ids.ctypes.data, ids.size, start,
             lg.ctypes.data if want_logits else None, ctypes.byref(nxt))
        return (nxt.value, lg) if want_logits else nxt.value

    def decode(self, token: int, pos: int, want_logits: bool = False):
        import numpy as np
        lg = np.empty(self.vocab, np.float32) if want_logits else None
        nxt = ctypes.c_int32()
        call("ib_model_decode", self.h, int(token), int(pos),
             lg.ctypes.data if want_logits else None, ctypes.byref(nxt))
        return (nxt.value, lg) if want_logits else nxt.value

    def decode_loop(self, token: int, pos: int, n_steps: int):
        """n_steps greedy steps on the device; returns the generated ids."""
        import numpy as np
        out = np.empty(max(n_steps, 1), np.int32)
        call("ib_model_decode_loop", self.h, int(token), int(pos), int(n_steps), out.ctypes.data)
        return out[:n_steps]

    def stream(self) -> int:
        s = ctypes.c_void_p()
        call("ib_model_stream", self.h, ctypes.byref(s))
        return s.value or 0

    def step_kernels(self) -> int:
        n = ctypes.c_int()
        call("ib_model_step_kernels", self.h, ctypes.byref(n))
        return n.value

    def generate(self, prompt, max_tokens: int, eos: int = -1):
        import numpy as np
        prompt = np.ascontiguousarray(prompt, dtype=np.int32)
        out = np.empty(prompt.size + max_tokens, np.int32)
        n = ctypes.c_int()
        st = GenerationStats()
        call("ib_model_generate", self.h, prompt.ctypes.data, prompt.size, max_tokens, eos,
             out.ctypes.data, ctypes.byref(n), ctypes.byref(st))
        return out[:n.value], st

    def close(self):
        if self.h:
            lib().ib_model_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
