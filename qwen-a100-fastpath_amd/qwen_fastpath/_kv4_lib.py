"""ctypes binding of libqf_kv4.so, the C ABI declared in include/qf_kv4.h, and the extension module through which the
package calls it (csrc/qf_kv4_call.cpp).

Both are built in-tree by qwen-a100-fastpath_amd/csrc/Makefile next to this file.  There is no fallback implementation: if
one is missing, every GPU entry point raises.
"""
from __future__ import annotations

import ctypes
import os

import torch

from ._lib import QFError

LIB_NAME = "libqf_kv4.so"
LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), LIB_NAME)
ABI_VERSION = 1

TILE = 16                # QF_KV4_TILE
MAX_REQS = 4096          # QF_STEP_MAX_REQS
MAX_TOKENS = 1 << 29     # QF_STEP_MAX_TOKENS
HEAD_SIZES = (64, 128, 256)
CACHE_NONE, CACHE_PAGES, CACHE_KV4 = 0, 1, 2

# Every symbol include/qf_kv4.h declares.
EXPORTS = (
    "qf_kv4_abi_version",
    "qf_step_tables",
    "qf_qk_norm_rope",
    "qf_kv4_load",
    "qf_kv4_attention",
    "qf_kv4_attention_workspace_bytes",
)

_p, _i64, _i32, _f32, _f64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_double


class Heads(ctypes.Structure):
    _fields_ = [("data", _p), ("stride_tok", _i64), ("stride_head", _i64)]


class Pages(ctypes.Structure):
    _fields_ = [("data", _p), ("stride_block", _i64), ("stride_tok", _i64), ("stride_head", _i64)]


class RopeArgs(ctypes.Structure):
    _fields_ = ([(n, Heads) for n in ("query", "key", "value", "query_out", "key_out")]
                + [(n, _p) for n in ("q_weight", "k_weight", "positions", "cos_sin", "slots", "cache")]
                + [("cache_stride", _i64), ("key_pages", Pages), ("value_pages", Pages), ("num_positions", _i64),
                   ("num_blocks", _i64), ("eps", _f64), ("weight_offset", _f64)]
                + [(n, _i32) for n in ("cos_sin_f32", "rot", "interleaved", "cache_kind", "page_size", "num_tokens", "num_heads",
                                       "num_kv_heads", "head_size")])


class AttentionArgs(ctypes.Structure):
    _fields_ = [("query", Heads), ("out", Heads), ("cache", _p), ("cache_stride", _i64), ("num_blocks", _i64),
                ("block_table", _p), ("bt_stride", _i64), ("seq_lens", _p), ("cu_q", _p), ("scale", _f32)] + [
        (n, _i32) for n in ("max_blocks", "num_tokens", "num_reqs", "q_len", "num_heads", "num_kv_heads", "head_size", "page_size")]


_lib: ctypes.CDLL | None = None
_module = None


def load() -> ctypes.CDLL:
    """Load the library once.  Raises ImportError (never falls back) when it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `make -C qwen-a100-fastpath_amd/csrc` "
            "(or __graft_entry__.build()); its operators have no non-HIP implementation")
    L = ctypes.CDLL(LIB_PATH)
    for name, res, args in (
            ("qf_kv4_abi_version", _i32, []),
            ("qf_step_tables", _i32, [_p, _p, _p, _p, _i64, _i32, _p, _p, _i32, _i32, _i32, _i32] + [_p] * 8),
            ("qf_qk_norm_rope", _i32, [ctypes.POINTER(RopeArgs), _p]),
            ("qf_kv4_load", _i32, [_p, _i64, _i64, _i32, _i32, _i32, _p, _i32, _p, _p, _p]),
            ("qf_kv4_attention", _i32, [ctypes.POINTER(AttentionArgs), _p, ctypes.c_size_t, _p]),
            ("qf_kv4_attention_workspace_bytes", ctypes.c_size_t, [ctypes.POINTER(AttentionArgs)])):
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    v = L.qf_kv4_abi_version()
    if v != ABI_VERSION:
        raise ImportError(f"{LIB_PATH}: ABI version {v}, expected {ABI_VERSION}")
    _lib = L
    return L


def module():
    """The extension, whose functions return None where a call is not as the kernels take it."""
    global _module
    if _module is None:
        load()
        try:
            from . import _qf_kv4_call
        except ImportError as e:
            raise ImportError("qwen_fastpath._qf_kv4_call cannot be loaded: build it with `make -C "
                              f"qwen-a100-fastpath_amd/csrc` (or __graft_entry__.build()): {e}") from e
        _module = _qf_kv4_call
    return _module


def try_call(name: str, *args):
    """A call on torch's current stream of the current device: its result, or None where the arguments are not as the kernels
    take them.  Raises QFError where the library refuses it."""
    device = torch._C._cuda_getDevice()
    r = getattr(_module or module(), name)(*args, device, torch._C._cuda_getCurrentRawStream(device))
    if type(r) is int:
        raise QFError(r, name)
    return r


def call(name: str, index: int, *args):
    """A checked call on torch's current stream of GPU `index`, whatever the current device is."""
    with torch.cuda.device(index):
        r = try_call(name, *args)
    if r is None:
        raise ValueError(f"{name}: the arguments are not as the kernels take them")
    return r


def plain(t):
    """A tensor of a subclass as the tensor it is."""
    return t if t is None or type(t) in (torch.Tensor, torch.nn.Parameter) else t.as_subclass(torch.Tensor)


def gpu(first: torch.Tensor, *others) -> int:
    """Index of the GPU that every tensor handed to the library lives on."""
    if not first.is_cuda:
        raise TypeError(f"expected a GPU tensor, got one on {first.device}")
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on {first.device} and {t.device}: all must be on one GPU")
    return index


def vector(t: torch.Tensor, dtype: torch.dtype, n: int, name: str, align: int = 1) -> torch.Tensor:
    """t, contiguous; an error where it is not dtype [n]."""
    if t.dtype is not dtype or tuple(t.shape) != (n,):
        raise TypeError(f"{name} must be {dtype} [{n}], got {t.dtype} {list(t.shape)}")
    if not t.is_contiguous() or t.data_ptr() % align:
        t = t.clone(memory_format=torch.contiguous_format)
    return plain(t)


def _fit(t: torch.Tensor) -> bool:
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1))


def heads(t: torch.Tensor, shape: tuple, name: str) -> torch.Tensor:
    """t as the kernels read it; an error where it is not bf16 of that shape."""
    if t.dtype is not torch.bfloat16 or tuple(t.shape) != shape:
        raise TypeError(f"{name} must be bf16 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return plain(t if _fit(t) else t.clone(memory_format=torch.contiguous_format))


def head_size(t: torch.Tensor, name: str) -> int:
    if t.dim() != 3 or t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bf16 [tokens, heads, head size], got {t.dtype} {list(t.shape)}")
    if t.shape[2] not in HEAD_SIZES or t.shape[1] < 1:
        raise ValueError(f"{name}: head sizes are {HEAD_SIZES}, got {list(t.shape)}")
    return t.shape[2]


def output(t: torch.Tensor | None, shape: tuple, name: str) -> torch.Tensor | None:
    """A tensor that is written: no copy can stand for it."""
    if t is None:
        return None
    if t.dtype is not torch.bfloat16 or tuple(t.shape) != shape or not _fit(t) or overlaps(t):
        raise ValueError(f"{name} must be bf16 {list(shape)} with 16-byte aligned heads that do not overlap, the last dimension "
                         f"contiguous and strides of multiples of 8, got {t.dtype} {list(t.shape)} with strides {t.stride()}")
    return plain(t)


def overlaps(t: torch.Tensor) -> bool:
    room = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < room:
            return True
        room = s * (n - 1) + room
    return False


def cache_sizes(cache: torch.Tensor) -> tuple[int, int, int]:
    """(kv heads, head size, page size) of a 4-bit cache; an error where it is none."""
    if cache.dim() != 4 or cache.dtype is not torch.uint8 or cache.shape[3] not in [17 * d for d in HEAD_SIZES] or 0 in cache.shape:
        raise TypeError("a 4-bit cache is uint8 [blocks, kv heads, page size / 16, 17 * head size] (kv4_cache), got "
                        f"{cache.dtype} {list(cache.shape)}")
    n, h, tiles, record = cache.shape
    strides = [(cache.stride(3), 1)] + ([(cache.stride(2), record)] if tiles > 1 else []) + (
        [(cache.stride(1), tiles * record)] if h > 1 else [])
    if any(a != b for a, b in strides) or cache.data_ptr() % 16 or (n > 1 and (
            cache.stride(0) % 16 or cache.stride(0) < h * tiles * record)):
        raise ValueError(f"a 4-bit cache's blocks are contiguous, 16-byte aligned and apart, got strides {cache.stride()}")
    return h, record // 17, tiles * TILE
