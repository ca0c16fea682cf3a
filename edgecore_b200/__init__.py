"""edgecore_b200 -- B200 (sm_100a) implementation of EdgeCore's inference hot path.

The product is the C library ``libedgecore_b200.so`` (include/edgecore.h and
include/edgecore_b200.h).  This package builds it (``build.py``), loads it with
ctypes, and mirrors the reference entry points for Python callers:

* ``gemm_int8``, ``gemm_fp16_fp32``, ``gemm_bf16_fp32`` -- reference
  src/kernels.c:129-168, on the GPU;
* ``Model`` -- ``gpt2_load`` / ``gpt2_forward`` / ``gpt2_free`` (reference
  src/gpt2.c:161-805) plus the greedy/device-resident extensions.

Arrays may be numpy arrays (host) or objects exposing ``data_ptr()`` (device
tensors); the library classifies each pointer.  There is no CPU fallback: if
the shared library is missing or fails to load, every call raises.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
from pathlib import Path
from typing import Any

import numpy as np

__all__ = ["load_library", "Model", "gemm_int8", "gemm_fp16_fp32", "gemm_bf16_fp32",
           "quantize_rows", "linear_int8", "gemm_async", "device_error_take", "attention_force_split", "reference_math", "argmax_key", "argmax_key_decode",
           "tree_attention", "tree_attention_work", "tree_commit", "kv_copy", "sample", "tree_mask", "LIB_PATH"]

LIB_PATH = Path(__file__).resolve().parent / "libedgecore_b200.so"
_LIB: C.CDLL | None = None

_vp, _i, _f = C.c_void_p, C.c_int, C.c_float


def _declare(lib: C.CDLL) -> None:
    sig = {
        "ec_last_error": (C.c_char_p, []),
        "ec_version": (C.c_char_p, []),
        "ec_model_open": (_vp, [C.c_char_p, _i, _i]),
        "ec_model_close": (None, [_vp]),
        "ec_model_info": (_i, [_vp, _vp]),
        "ec_model_set_stream": (_i, [_vp, _vp]),
        "ec_forward_device": (_i, [_vp, _vp, _vp, _vp, _i, _vp]),
        "ec_forward_argmax": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _vp]),
        "ec_forward_shard_argmax": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _vp]),
        "ec_decode_greedy": (_i, [_vp, _vp, _i, _i, _vp]),
        "ec_decode_profile": (_i, [_vp, _vp, _i, _i, _vp]),
        "ec_decode_greedy_cycle": (_i, [_vp, _vp, _i, _i, _i, _vp]),
        "ec_decode_trace": (_i, [_vp, _vp, _i, _i, _vp, _i]),
        "ec_decode_batch": (_i, [_vp, _vp, _vp, _i, _vp]),
        "ec_batch_hidden": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
        "ec_lm_shard_keys": (_i, [_vp, _vp, _i, _vp]),
        "ec_keys_advance": (_i, [_vp, _vp, _i, _vp, _vp]),
        "ec_batch_graph_kernels": (_i, [_vp, _i]),
        "ec_model_packed": (C.c_longlong, [_vp, _i, _i, _vp, C.c_size_t, _vp]),
        "ec_kv_release": (_i, [_vp, _i]),
        "ec_kv_info": (_i, [_vp, _vp]),
        "ec_model_kv": (_i, [_vp, _vp]),
        "ec_tree_attention": (_i, [_vp, _vp, _vp]),
        "ec_tree_attention_work": (C.c_size_t, [_i, _i, _i, _i, _i, _i]),
        "ec_tree_commit": (_i, [_vp, _vp, _vp]),
        "ec_kv_copy": (_i, [_vp, _i, _vp, _vp, _vp, _vp, _vp]),
        "ec_sample": (_i, [_vp, _vp, _vp, _i, C.c_longlong, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp]),
        "ec_forward_tree": (_i, [_vp, _vp, _vp, _vp, _vp, _vp]),
        "ec_kv_fork": (_i, [_vp, _i, _vp, _i, _i]),
        "ec_decode_sample": (_i, [_vp, _vp, _vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
        "ec_model_set_taps": (_i, [_vp, _i]),
        "ec_model_get_taps": (_i, [_vp, _vp, _i]),
        "ec_model_set_vocab_shard": (_i, [_vp, _i, _i]),
        "ec_argmax_key": (C.c_uint64, [_f, _i]),
        "ec_argmax_key_decode": (None, [C.c_uint64, _vp, _vp]),
        "ec_quantize_rows": (_i, [_vp, _vp, _vp, _i, _i]),
        "ec_linear_int8": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i, _i]),
        "ec_gemm_async": (_i, [_i, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _vp]),
        "ec_device_error_take": (_i, [_vp, _vp]),
        "ec_attention_force_split": (_i, [_i]),
        "ec_reference_math": (_i, [_vp, _vp, _vp, _i, _vp]),
        "gemm_fp16_fp32": (None, [_vp, _vp, _vp, _i, _i, _i]),
        "gemm_bf16_fp32": (None, [_vp, _vp, _vp, _i, _i, _i]),
        "gemm_int8": (None, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i]),
        "gpt2_forward": (None, [_vp, _vp, _vp, _vp, _i, _vp]),
        "ecm_parse": (_i, [_vp, C.c_size_t, _vp, _i, _vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args


def load_library(path: str | os.PathLike | None = None) -> C.CDLL:
    """Load (once) and return the shared library; raise if it is not built."""
    global _LIB
    if _LIB is not None:
        return _LIB
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise RuntimeError(f"{p} is not built; run `python -m edgecore_b200.build` "
                           "(there is no CPU fallback)")
    lib = C.CDLL(str(p))
    _declare(lib)
    _LIB = lib
    return lib


def last_error() -> str:
    return (load_library().ec_last_error() or b"").decode(errors="replace")


def _ptr(a: Any) -> int | None:
    """Address of a numpy array / device tensor / raw int (None stays None)."""
    if a is None:
        return None
    if isinstance(a, int):
        return a
    if hasattr(a, "data_ptr"):
        return int(a.data_ptr())
    if isinstance(a, np.ndarray):
        if not a.flags["C_CONTIGUOUS"]:
            raise ValueError("arrays passed to the C ABI must be C-contiguous")
        return a.ctypes.data
    raise TypeError(f"cannot pass {type(a)} to the C ABI")


def _np(a, dtype) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=dtype)


def _is_dev(a) -> bool:
    return hasattr(a, "data_ptr")


# ---- standalone GEMMs (reference src/kernels.c:129-168) ----------------------

def gemm_int8(A, a_scale, B, b_scale=None, bias=None, out=None):
    """C[m][n] = bias[n] + ((float)sum_k A[m][k]*B[n][k]) * a_scale[m] * b_scale[n]."""
    lib = load_library()
    if not _is_dev(A):
        A, a_scale = _np(A, np.int8), _np(a_scale, np.float32)
    if not _is_dev(B):
        B = _np(B, np.int8)
        b_scale = None if b_scale is None else _np(b_scale, np.float32)
        bias = None if bias is None else _np(bias, np.float32)
    M, K = A.shape
    N = B.shape[0]
    if out is None:
        out = np.empty((M, N), np.float32)
    lib.gemm_int8(_ptr(out), _ptr(A), _ptr(a_scale), _ptr(B), _ptr(b_scale), _ptr(bias), M, K, N)
    return out


def _gemm16(fn, A, B16, out):
    lib = load_library()
    if not _is_dev(A):
        A = _np(A, np.float32)
    if not _is_dev(B16):
        B16 = np.ascontiguousarray(B16).view(np.uint16)
    M, K = A.shape
    N = B16.shape[0]
    if out is None:
        out = np.empty((M, N), np.float32)
    getattr(lib, fn)(_ptr(out), _ptr(A), _ptr(B16), M, K, N)
    return out


def gemm_fp16_fp32(A, B16, out=None):
    """C[m][n] = sum_k A[m][k] * fp16(B[n][k]) with fp32 accumulation."""
    return _gemm16("gemm_fp16_fp32", A, B16, out)


def gemm_bf16_fp32(A, B16, out=None):
    """Same as gemm_fp16_fp32 with bfloat16 weights (uint16 bit patterns)."""
    return _gemm16("gemm_bf16_fp32", A, B16, out)


def gemm_async(wt: int, out, A, a_scale, B, b_scale=None, bias=None, stream=None) -> None:
    """gemm_int8 (wt 0) / gemm_fp16_fp32 (1) / gemm_bf16_fp32 (2) on device
    tensors, enqueued on `stream` (an int cudaStream_t or None) without a host
    synchronisation; errors inside kernels surface in device_error_take()."""
    lib = load_library()
    M, K = A.shape
    N = B.shape[0]
    if lib.ec_gemm_async(int(wt), _ptr(out), _ptr(A), _ptr(a_scale), _ptr(B), _ptr(b_scale), _ptr(bias),
                         M, K, N, stream):
        raise RuntimeError(last_error())


def reference_math(d_x, d_exp=None, d_tanh=None, stream=None) -> None:
    """The library's device expf / tanhf (restated host libm) on a device float tensor."""
    n = int(d_x.numel())
    if load_library().ec_reference_math(_ptr(d_x), _ptr(d_exp), _ptr(d_tanh), n, stream):
        raise RuntimeError(last_error())


def attention_force_split(on: bool) -> None:
    """Force (True) or release (False) the split attention kernels of the
    per-layer path, process-wide (tests and measurement)."""
    load_library().ec_attention_force_split(1 if on else 0)


def device_error_take(stream=None) -> int:
    """Synchronise `stream`, then read and clear the library's device error
    code (0 none, 1 a bounded wait gave up, 2 an out-of-range index)."""
    code = C.c_int(0)
    if load_library().ec_device_error_take(stream, C.byref(code)):
        raise RuntimeError(last_error())
    return code.value


def quantize_rows(X):
    """Per-row int8 activation quantisation (reference src/gpt2.c:446-461)."""
    lib = load_library()
    X = _np(X, np.float32)
    M, K = X.shape
    q = np.empty((M, K), np.int8)
    s = np.empty(M, np.float32)
    if lib.ec_quantize_rows(_ptr(q), _ptr(s), _ptr(X), M, K):
        raise RuntimeError(last_error())
    return q, s


def linear_int8(X, W, w_scale, bias=None, out=None):
    """The W8A8 linear of reference linear() (src/gpt2.c:437-462)."""
    lib = load_library()
    if not _is_dev(X):
        X = _np(X, np.float32)
    if not _is_dev(W):
        W, w_scale = _np(W, np.int8), _np(w_scale, np.float32)
        bias = None if bias is None else _np(bias, np.float32)
    M, K = X.shape
    N = W.shape[0]
    if out is None:
        out = np.empty((M, N), np.float32)
    if lib.ec_linear_int8(_ptr(out), _ptr(X), _ptr(W), _ptr(w_scale), _ptr(bias), M, K, N):
        raise RuntimeError(last_error())
    return out


def argmax_key(maxv: float, idx: int) -> int:
    return int(load_library().ec_argmax_key(float(maxv), int(idx)))


def argmax_key_decode(key: int) -> tuple[float, int]:
    v, i = C.c_float(), C.c_int()
    load_library().ec_argmax_key_decode(C.c_uint64(key), C.byref(v), C.byref(i))
    return v.value, i.value


# ---- serving operators on device tensors --------------------------------------
#
# `stream` is a cudaStream_t as an int.  None is the legacy default stream, not torch's current one: inside
# torch.cuda.stream(s), whose work it does not wait for, pass s.cuda_stream.

# ec_kv_pages, ec_tree_attn and ec_tree_path, field by field: packed bytes cost
# a quarter of a ctypes structure, on calls of a few microseconds
_KV_PAGES = struct.Struct("PPqqqP6i")
_TREE_ATTN = struct.Struct("PPqq9ifPPPPPN")
_TREE_PATH = struct.Struct("4i9P")


class _TreeStep(C.Structure):
    """ec_tree_step"""
    _fields_ = [("n_seq", _i), ("max_path", _i), ("slots", _vp), ("row_start", _vp), ("base", _vp), ("tokens", _vp),
                ("parents", _vp), ("u", _vp), ("temperature", _vp), ("top_p", _vp), ("min_p", _vp), ("top_k", _vp)]


_TYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2, "torch.int32": 3, "torch.int64": 4}
_TYPE_OF: dict = {}


def _new_type(d) -> int:
    code = _TYPE_OF[d] = _TYPES.get(str(d), -1)
    return code


def _type(t) -> int:
    """Code of a tensor's element type (0..2 as the C ABI's EC_T_*, 3 int32, 4 int64; -1: any other)."""
    d = t.dtype
    return _TYPE_OF[d] if d in _TYPE_OF else _new_type(d)


def _vec(t, name: str, code: int, n: int | None = None) -> int:
    """Address of a contiguous vector of the given type and, if given, length (0 for None)."""
    if t is None:
        return 0
    shape = t.shape
    if len(shape) != 1 or _type(t) != code or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D tensor of {list(_TYPES)[code]}")
    if n is not None and shape[0] != n:
        raise ValueError(f"{name} has {shape[0]} elements, {n} are needed")
    return t.data_ptr()


def _words(mask, rows: int):
    if _type(mask) != 4 or mask.dim() != 2 or not mask.is_contiguous() or mask.shape[0] < rows:
        raise ValueError(f"mask must be a contiguous int64 tensor [{rows}][words]")
    return mask.shape[1]


def _table(page_table):
    if _type(page_table) != 3 or page_table.dim() != 2 or not page_table.is_contiguous():
        raise ValueError("page_table must be a contiguous int32 tensor [slots][pages per slot]")
    return page_table.shape


def _layers(k, v, page_table) -> bytes:
    """The arena of all layers: k and v [layers][pages][64][dim] (dim contiguous, any other strides)."""
    shape, st = k.shape, k.stride()
    if len(shape) != 4 or shape[1] < 1 or shape[2] != 64 or st[3] != 1 or v.shape != shape or v.stride() != st or v.dtype != k.dtype:
        raise ValueError("k and v must be alike: [layers][pages][64][dim] with contiguous positions")
    slots, per_slot = _table(page_table)
    return _KV_PAGES.pack(k.data_ptr(), v.data_ptr(), st[0], st[1], st[2], page_table.data_ptr(), _type(k), shape[0], shape[1], slots,
                          per_slot, shape[3])


def tree_mask(parents) -> np.ndarray:
    """Mask rows (int64 [nodes][ceil(nodes / 64)]) of a drafted tree: parents[i] < i is the parent of node i, -1 for a
    root; bit j of row i is set when j is i or an ancestor of it."""
    parents = np.asarray(parents)
    n = len(parents)
    out = np.zeros((n, max(1, (n + 63) // 64)), np.uint64)
    for i in range(n):
        p = int(parents[i])
        if p >= i or p < -1:
            raise ValueError(f"parents[{i}] = {p}: a parent comes before its node (-1: a root)")
        if p >= 0:
            out[i] = out[p]
        out[i, i // 64] |= np.uint64(1 << (i % 64))
    return out.view(np.int64)


def tree_attention_work(n_seq: int, rows: int, n_head: int, n_kv_head: int, head_dim: int, max_len: int) -> int:
    """Bytes of workspace with which tree_attention splits long caches as far as it pays, for any type of q and window;
    max_len as in the call (0: any length)."""
    return int(load_library().ec_tree_attention_work(n_seq, rows, n_head, n_kv_head, head_dim, max_len))


def tree_attention(out, q, k, v, page_table, row_start, base, mask, *, slots=None, window: int = 0, scale: float = 0.0,
                   max_len: int = 0, workspace=None, stream=None):
    """Attention of drafted-token trees over a paged KV arena (ec_tree_attention) on device tensors, enqueued on `stream` (an int
    cudaStream_t; None: the legacy default stream, not torch's current one).

    q, out [rows][heads * head_dim] (or [rows][heads][head_dim]) fp32 or of the cache's type, any row stride; k, v
    [pages][64][KV heads][head_dim] fp16 or bf16; page_table int32 [slots][pages per slot]; row_start int32 [sequences + 1],
    base and slots int32 [sequences]; mask int64 [rows][words] (tree_mask).  workspace: a contiguous tensor, any type."""
    qs, ks, kst, qst, ost = q.shape, k.shape, k.stride(), q.stride(), out.stride()
    if len(ks) != 4 or ks[0] < 1 or ks[1] != 64 or kst[3] != 1 or (ks[2] > 1 and kst[2] != ks[3]) or v.shape != ks or v.stride() != kst:
        raise ValueError("k and v must be alike: [pages][64][KV heads][head_dim] with contiguous positions")
    if len(qs) not in (2, 3) or out.shape != qs or out.dtype != q.dtype or v.dtype != k.dtype:
        raise ValueError("q and out must be alike: [rows][heads * head_dim] or [rows][heads][head_dim]")
    hd = ks[3]
    wide = qs[1] if len(qs) == 2 else qs[1] * qs[2]
    if wide % hd or (len(qs) == 3 and qs[2] != hd):
        raise ValueError(f"rows of {wide} for heads of {hd}")
    for st in (qst, ost):
        if (wide and st[-1] != 1) or (len(qs) == 3 and qs[1] > 1 and st[1] != hd):
            raise ValueError("the rows of q and out must be contiguous")
    rows, n_seq = qs[0], base.shape[0]
    slots_n, per_slot = _table(page_table)
    kv = _KV_PAGES.pack(k.data_ptr(), v.data_ptr(), 0, kst[0], kst[1], page_table.data_ptr(), _type(k), 1, ks[0], slots_n, per_slot,
                        ks[2] * hd)
    work = nbytes = 0
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        work, nbytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    a = _TREE_ATTN.pack(q.data_ptr(), out.data_ptr(), qst[0], ost[0], _type(q), n_seq, rows, wide // hd, ks[2], hd, window, max_len,
                  _words(mask, rows), scale, _vec(slots, "slots", 3, n_seq), _vec(row_start, "row_start", 3, n_seq + 1),
                  _vec(base, "base", 3), mask.data_ptr(), work, nbytes)
    if load_library().ec_tree_attention(kv, a, stream):
        raise RuntimeError(last_error())
    return out


def tree_commit(k, v, page_table, row_start, base, mask, tokens, picked, accepted, n_accepted, new_base, *, slots=None,
                stream=None) -> None:
    """Accept the confirmed path of every drafted tree and move its K and V rows to the front (ec_tree_commit), on `stream` as
    in tree_attention.

    k, v [layers][pages][64][dim]; tokens, picked int32 [rows]; accepted int32 [sequences][most nodes of a path], n_accepted
    and new_base int32 [sequences] (new_base may be base) are written; the others as for tree_attention."""
    kv = _layers(k, v, page_table)
    n_seq = base.shape[0]
    rows = tokens.shape[0]
    if _type(accepted) != 3 or accepted.dim() != 2 or accepted.shape[0] != n_seq or not accepted.is_contiguous():
        raise ValueError(f"accepted must be a contiguous int32 tensor [{n_seq}][nodes]")
    a = _TREE_PATH.pack(n_seq, rows, _words(mask, rows), accepted.shape[1], _vec(slots, "slots", 3, n_seq),
                  _vec(row_start, "row_start", 3, n_seq + 1), _vec(base, "base", 3), mask.data_ptr(), _vec(tokens, "tokens", 3),
                  _vec(picked, "picked", 3, rows), accepted.data_ptr(), _vec(n_accepted, "n_accepted", 3, n_seq),
                  _vec(new_base, "new_base", 3, n_seq))
    if load_library().ec_tree_commit(kv, a, stream):
        raise RuntimeError(last_error())


def kv_copy(k, v, page_table, src, dst, start, end, *, stream=None) -> None:
    """Copy positions [start[j], end[j]) of slot src[j] to slot dst[j] in every layer (ec_kv_copy), on `stream` as in
    tree_attention; k, v
    [layers][pages][64][dim], the others int32 vectors of one length.  Jobs of which one writes what the other writes or reads
    are both skipped and reported (device_error_take), as is one with a bad slot or range."""
    kv = _layers(k, v, page_table)
    n = src.shape[0]
    if load_library().ec_kv_copy(kv, n, _vec(src, "src", 3), _vec(dst, "dst", 3, n), _vec(start, "start", 3, n),
                                 _vec(end, "end", 3, n), stream):
        raise RuntimeError(last_error())


def sample(ids, logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None, prob=None, stream=None):
    """Draw one token per row of logits [rows][vocab] (fp32, fp16 or bf16, any row stride) with the uniform numbers u[rows]
    (ec_sample): temperature, top-k, top-p and min-p per row, each a vector or None for off.  Writes ids int32 [rows] and, if
    given, prob fp32 [rows]; returns ids.  `stream` as in tree_attention."""
    shape, st = logits.shape, logits.stride()
    if len(shape) != 2 or (shape[1] > 1 and st[1] != 1):
        raise ValueError("logits must be [rows][vocab] with contiguous rows")
    rows = shape[0]
    if load_library().ec_sample(_vec(ids, "ids", 3, rows), _vec(prob, "prob", 0, rows), logits.data_ptr(), _type(logits), st[0], rows,
                                shape[1], _vec(temperature, "temperature", 0, rows), _vec(top_k, "top_k", 3, rows),
                                _vec(top_p, "top_p", 0, rows), _vec(min_p, "min_p", 0, rows), _vec(u, "u", 0, rows), stream):
        raise RuntimeError(last_error())
    return ids


# ---- model -------------------------------------------------------------------

class Model:
    """A model loaded on the current CUDA device (gpt2_load on a heap GPT2)."""

    INFO = ("arch", "precision", "n_layer", "n_head", "n_kv_head", "n_embd", "head_dim",
            "intermediate", "vocab", "n_ctx", "eff_ctx", "batch_cap", "n_kv_embd", "tie", "device")

    def __init__(self, path: str | os.PathLike, batch_cap: int = 1, max_ctx: int = 0):
        self.lib = load_library()
        self.h = self.lib.ec_model_open(str(path).encode(), int(batch_cap), int(max_ctx))
        if not self.h:
            raise RuntimeError(f"gpt2_load({path}) failed: {last_error()}")
        info = np.zeros(16, np.int32)
        self._check(self.lib.ec_model_info(self.h, info.ctypes.data))
        for k, v in zip(self.INFO, info):
            setattr(self, k, int(v))

    def _check(self, rc: int) -> None:
        if rc:
            raise RuntimeError(last_error())

    def close(self) -> None:
        if getattr(self, "h", None):
            self.lib.ec_model_close(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward(self, tokens, positions, seqs=None, out=None) -> np.ndarray:
        """gpt2_forward with host arrays: logits [M][vocab] fp32, written into
        `out` when given (a C-contiguous float32 [M][vocab] array, reused the
        way the reference runtime reuses its one logits buffer)."""
        t, p = _np(tokens, np.int32), _np(positions, np.int32)
        s = None if seqs is None else _np(seqs, np.int32)
        M = len(t)
        if out is None:
            out = np.empty((M, self.vocab), np.float32)
        elif out.dtype != np.float32 or not out.flags.c_contiguous or out.shape != (M, self.vocab):
            raise ValueError(f"out must be a C-contiguous float32 array of shape ({M}, {self.vocab})")
        self.lib.gpt2_forward(self.h, _ptr(t), _ptr(p), _ptr(s), M, _ptr(out))
        return out

    def forward_argmax(self, tokens, positions, seqs=None, shard: bool = False):
        t, p = _np(tokens, np.int32), _np(positions, np.int32)
        s = None if seqs is None else _np(seqs, np.int32)
        M = len(t)
        ids = np.empty(M, np.int32)
        mx = np.empty(M, np.float32)
        fn = self.lib.ec_forward_shard_argmax if shard else self.lib.ec_forward_argmax
        self._check(fn(self.h, _ptr(t), _ptr(p), _ptr(s), M, _ptr(ids), _ptr(mx)))
        return ids, mx

    def forward_taps(self, tokens, positions, seqs=None):
        """Logits plus residual taps [n_layer+1][M][n_embd]."""
        M = len(tokens)
        self._check(self.lib.ec_model_set_taps(self.h, M))
        try:
            logits = self.forward(tokens, positions, seqs)
            taps = np.empty((self.n_layer + 1, M, self.n_embd), np.float32)
            self._check(self.lib.ec_model_get_taps(self.h, _ptr(taps), M))
        finally:
            self.lib.ec_model_set_taps(self.h, 0)
        return logits, taps

    def forward_device(self, d_tokens, d_positions, d_seqs, M: int, d_logits) -> None:
        self._check(self.lib.ec_forward_device(self.h, _ptr(d_tokens), _ptr(d_positions), _ptr(d_seqs),
                                               int(M), _ptr(d_logits)))

    def decode_greedy(self, d_tokens, start_pos: int, n_steps: int, d_out_ids=None) -> None:
        self._check(self.lib.ec_decode_greedy(self.h, _ptr(d_tokens), int(start_pos), int(n_steps),
                                              _ptr(d_out_ids)))

    def decode_greedy_cycle(self, d_tokens, start_pos: int, period: int, n_steps: int, d_out_ids=None) -> None:
        self._check(self.lib.ec_decode_greedy_cycle(self.h, _ptr(d_tokens), int(start_pos), int(period),
                                                    int(n_steps), _ptr(d_out_ids)))

    def decode_batch(self, d_tokens, d_positions, n_steps: int, d_out_ids=None) -> None:
        """Greedy decode of n_steps tokens for all batch_cap slots (device
        int32 tokens / positions [batch_cap], updated in place; ids into
        d_out_ids [n_steps][batch_cap] when given), one captured CUDA graph
        per step on the model stream."""
        self._check(self.lib.ec_decode_batch(self.h, _ptr(d_tokens), _ptr(d_positions), int(n_steps),
                                             _ptr(d_out_ids)))

    def decode_sample(self, d_tokens, d_positions, n_steps: int, d_u, temperature=None, top_k=None, top_p=None, min_p=None,
                      d_out_ids=None, d_out_prob=None) -> None:
        """decode_batch with every token drawn by sample(): step s of slot m uses d_u[s][m] (device fp32
        [n_steps][batch_cap]) and the slot's settings (device arrays [batch_cap]; top_k int32, the others fp32; None: off);
        ids and, fp32, their probabilities into d_out_ids and d_out_prob [n_steps][batch_cap] when given."""
        self._check(self.lib.ec_decode_sample(self.h, _ptr(d_tokens), _ptr(d_positions), int(n_steps), _ptr(d_u), _ptr(temperature),
                                              _ptr(top_k), _ptr(top_p), _ptr(min_p), _ptr(d_out_ids), _ptr(d_out_prob)))

    def forward_tree(self, trees, base, slots=None, max_path: int | None = None, u=None, temperature=None, top_k=None, top_p=None,
                     min_p=None) -> dict:
        """One step of drafted trees (ec_forward_tree).  trees: (tokens, parents) of each sequence, the root first with parent
        -1: the last token that is not in the cache yet.  base: committed positions of each.  With u (one number in [0, 1) per
        node of all trees in order) the choices are drawn as by sample(), with settings per node (or one number for all);
        without, they are the argmax.  The accepted rows are committed.  Returns accepted (a list of tokens per sequence, the
        last of them the next root), picked (the choice after every node) and, with u, prob."""
        trees = [(_np(t, np.int32).reshape(-1), _np(p, np.int32).reshape(-1)) for t, p in trees]
        n = len(trees)
        for t, p in trees:
            if len(t) != len(p):
                raise ValueError(f"a tree has {len(t)} tokens and {len(p)} parents")
        base = _np(base, np.int32).reshape(-1)
        slots = None if slots is None else _np(slots, np.int32).reshape(-1)
        if len(base) != n or (slots is not None and len(slots) != n):
            raise ValueError(f"{n} trees need {n} bases and slots")
        start = np.zeros(n + 1, np.int32)
        start[1:] = np.cumsum([len(t) for t, _ in trees])
        rows = int(start[n])
        tokens, parents = (np.concatenate([t[i] for t in trees] + [np.zeros(0, np.int32)]) for i in range(2))
        if max_path is None:
            max_path = max([1] + [len(t) for t, _ in trees])

        def each(v, dtype, name):
            if v is None:
                return None
            v = np.ascontiguousarray(np.broadcast_to(np.asarray(v, dtype), (rows,)) if np.ndim(v) == 0 else np.asarray(v, dtype))
            if v.shape != (rows,):
                raise ValueError(f"{name} must be one number or {rows}, one for each node")
            return v

        if u is not None and np.ndim(u) == 0 and rows != 1:
            raise ValueError("u must have one number for each node")
        vals = [each(v, t, k) for v, t, k in ((u, np.float32, "u"), (temperature, np.float32, "temperature"), (top_p, np.float32, "top_p"),
                                              (min_p, np.float32, "min_p"), (top_k, np.int32, "top_k"))]
        step = _TreeStep(n, int(max_path), _ptr(slots), _ptr(start), _ptr(base), _ptr(tokens), _ptr(parents), *(_ptr(v) for v in vals))
        picked, prob = np.empty(rows, np.int32), np.empty(rows, np.float32)
        accepted, count = np.empty((n, max(1, int(max_path))), np.int32), np.empty(n, np.int32)
        self._check(self.lib.ec_forward_tree(self.h, C.addressof(step), _ptr(picked), _ptr(prob) if u is not None else None, _ptr(accepted),
                                             _ptr(count)))
        out = {"accepted": [accepted[b, :count[b]].tolist() for b in range(n)], "picked": picked}
        return out | {"prob": prob} if u is not None else out

    def kv_fork(self, src: int, dst, length: int) -> None:
        """Slots dst take over positions [0, length) of slot src, copied into pages of their own (ec_kv_fork)."""
        dst = _np(dst, np.int32).reshape(-1)
        self._check(self.lib.ec_kv_fork(self.h, int(src), _ptr(dst), len(dst), int(length)))

    def batch_hidden(self, d_tokens, d_positions, M: int, max_pos_end: int, d_hidden) -> None:
        """Rows m < M (slot m) through every layer and the final norm into
        d_hidden [M][n_embd] fp32 (device); every position < max_pos_end."""
        self._check(self.lib.ec_batch_hidden(self.h, _ptr(d_tokens), _ptr(d_positions), int(M), int(max_pos_end),
                                             _ptr(d_hidden)))

    def lm_shard_keys(self, d_hidden, rows: int, d_keys) -> None:
        """lm_head of the vocab shard over `rows` hidden rows, per-row argmax
        as signed int64 keys (signed max across shards = the global greedy id)."""
        self._check(self.lib.ec_lm_shard_keys(self.h, _ptr(d_hidden), int(rows), _ptr(d_keys)))

    def keys_advance(self, d_keys, M: int, d_tokens, d_positions) -> None:
        """tokens[m] = index in keys[m], positions[m] += 1 (device arrays)."""
        self._check(self.lib.ec_keys_advance(self.h, _ptr(d_keys), int(M), _ptr(d_tokens), _ptr(d_positions)))

    def kv_release(self, slot: int = -1) -> None:
        """Return the KV pages of `slot` (all slots when < 0) to the arena."""
        self._check(self.lib.ec_kv_release(self.h, int(slot)))

    def kv_info(self) -> dict:
        """{pages, free, page_positions, pages_per_slot} of the paged KV arena."""
        info = np.zeros(4, np.int32)
        self._check(self.lib.ec_kv_info(self.h, _ptr(info)))
        return dict(zip(("pages", "free", "page_positions", "pages_per_slot"), (int(v) for v in info)))

    PACKED = {"qkv": 0, "o": 1, "up": 2, "down": 3, "lm_head": 4}

    def packed(self, layer: int, which: str) -> tuple[np.ndarray, dict]:
        """The device-packed rows of one linear (ec_model_packed): uint8
        [N][ldw * element bytes] and {N, K, Kp, ldw, elt}."""
        info = np.zeros(5, np.int32)
        w = self.PACKED[which]
        n = self.lib.ec_model_packed(self.h, int(layer), w, None, 0, _ptr(info))
        if n < 0:
            raise RuntimeError(last_error())
        out = np.empty(int(n), np.uint8)
        if self.lib.ec_model_packed(self.h, int(layer), w, _ptr(out), out.size, _ptr(info)) < 0:
            raise RuntimeError(last_error())
        N, K, Kp, ldw, elt = (int(v) for v in info)
        return out.reshape(N, ldw * elt), {"N": N, "K": K, "Kp": Kp, "ldw": ldw, "elt": elt}

    def batch_graph_kernels(self, kind: int) -> int:
        """Kernel launches in the captured step graph (0: decode_batch, 1: batch_hidden, 2: decode_sample)."""
        n = self.lib.ec_batch_graph_kernels(self.h, int(kind))
        if n < 0:
            raise RuntimeError(last_error())
        return n

    TRACE_CODES = {1: "barrier", 2: "operand", 3: "tiles", 4: "attention", 5: "lm_head", 6: "argmax",
                   7: "tile_in", 8: "tile_free", 9: "tile_done", 10: "issue", 11: "staged", 12: "stats",
                   13: "scores", 14: "softmax", 15: "phase_in"}

    def decode_trace(self, d_tokens, start_pos: int, n_steps: int, cap: int = 1 << 16):
        """Timeline of CTA 0 of the persistent decode kernel: list of (event, ns)
        sorted by time (consumer and producer events interleaved)."""
        buf = np.zeros(cap, np.uint64)
        n = self.lib.ec_decode_trace(self.h, _ptr(d_tokens), int(start_pos), int(n_steps), _ptr(buf), cap)
        if n < 0:
            raise RuntimeError(last_error())
        ev = [(self.TRACE_CODES.get(int(v) >> 56, "?"), int(v) & ((1 << 56) - 1)) for v in buf[:n]]
        return sorted(ev, key=lambda e: e[1])

    def decode_profile(self, d_tokens, start_pos: int, n_steps: int) -> dict:
        """Per-kernel-class event timings of an instrumented decode."""
        out = np.zeros(16, np.float64)
        self._check(self.lib.ec_decode_profile(self.h, _ptr(d_tokens), int(start_pos), int(n_steps), _ptr(out)))
        names = ("decode_step", "gemm", "attention", "norm", "other")
        return {n: {"ms": out[3 * i], "bytes": out[3 * i + 1], "launches": int(out[3 * i + 2])}
                for i, n in enumerate(names)} | {"steps": int(out[15])}

    def set_stream(self, stream_ptr: int | None) -> None:
        self._check(self.lib.ec_model_set_stream(self.h, stream_ptr))

    def set_vocab_shard(self, v0: int, v1: int) -> None:
        self._check(self.lib.ec_model_set_vocab_shard(self.h, int(v0), int(v1)))
