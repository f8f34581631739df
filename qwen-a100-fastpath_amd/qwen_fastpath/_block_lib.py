"""ctypes binding of libqf_block.so, the C ABI declared in include/qf_block.h, and the extension module that makes a
call in its plain form without the steps in Python (csrc/qf_block_call.cpp).

Both are built in-tree by qwen-a100-fastpath_amd/csrc/Makefile next to this file.  There is no fallback implementation: if
one is missing, every GPU entry point raises.
"""
from __future__ import annotations

import ctypes
import functools
import os

import torch

from ._lib import QFError

LIB_NAME = "libqf_block.so"
LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), LIB_NAME)
ABI_VERSION = 1

BLOCK = 128              # QF_FP8_BLOCK
MAX_DECODE_M = 16        # QF_FP8_MAX_DECODE_M
NORM_MAX_N = 32768       # QF_BLOCK_NORM_MAX_N
MOE_MAX_EXPERTS = 512    # QF_MOE_MAX_EXPERTS
MOE_MAX_TOP_K = 16       # QF_MOE_MAX_TOP_K
GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_FULL = 0, 1, 2, 3
ACTS = {"none": 0, "sigmoid": 1}

# Every symbol include/qf_block.h declares.
EXPORTS = (
    "qf_block_abi_version",
    "qf_fp8_w8a16_gemm",
    "qf_fp8_w8a16_workspace_bytes",
    "qf_quantize_tokens_fp8",
    "qf_fp8_w8a8_workspace_bytes",
    "qf_fp8_w8a8_linear",
    "qf_block_norm_rows",
    "qf_moe_few_workspace_bytes",
    "qf_moe_few_tokens",
)

_lib: ctypes.CDLL | None = None
_plain = None


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
    p, i64, i32, sz, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_float
    product = [p, i64, p, i64, i32, p, p, p, i64, i32, i32, i32, i32]
    for name, res, args in (
            ("qf_block_abi_version", i32, []),
            ("qf_fp8_w8a16_workspace_bytes", sz, [i32] * 4),
            ("qf_fp8_w8a16_gemm", i32, product + [p, sz, p]),
            ("qf_quantize_tokens_fp8", i32, [p, i64, i32, i32, p, i64, p, p]),
            ("qf_fp8_w8a8_workspace_bytes", sz, [i32] * 3),
            ("qf_fp8_w8a8_linear", i32, product + [p, sz, p]),
            ("qf_block_norm_rows", i32, [p, i64, p, i64, i32, p, p, f32, p, i64, i32, i32, f32, f32, i32, i32, p, i64, p,
                                         i64, p]),
            ("qf_moe_few_workspace_bytes", sz, [i32] * 5),
            ("qf_moe_few_tokens", i32, [p, i64, p, i64, i32, p, p, p, p, p, i64, i32, i32, i32, i32, i32, i32, p, sz, p])):
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    v = L.qf_block_abi_version()
    if v != ABI_VERSION:
        raise ImportError(f"{LIB_PATH}: ABI version {v}, expected {ABI_VERSION}")
    _lib = L
    return L


def plain():
    """(module, device, stream): the extension, whose functions return None where a call is not in the plain form, and what
    they take, the current device with torch's current stream on it."""
    global _plain
    if _plain is None:
        load()
        try:
            from . import _qf_block_call
        except ImportError as e:
            raise ImportError("qwen_fastpath._qf_block_call cannot be loaded: build it with `make -C "
                              f"qwen-a100-fastpath_amd/csrc` (or __graft_entry__.build()): {e}") from e
        _plain = _qf_block_call
    device = torch._C._cuda_getDevice()
    return _plain, device, torch._C._cuda_getCurrentRawStream(device)


@functools.lru_cache(maxsize=4096)
def workspace_bytes(name: str, *sizes: int) -> int:
    """A call's workspace by its sizes (which settle it): asked of the library once."""
    return getattr(load(), name)(*sizes)


def same_gpu(first: torch.Tensor, *others) -> int:
    """Index of the GPU that every tensor handed to the library lives on: a host pointer, or another device's, reaching a
    kernel faults the device."""
    if not first.is_cuda:
        raise TypeError(f"expected a GPU tensor, got one on {first.device}")
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on {first.device} and {t.device}: all must be on one GPU")
    return index


def call(name: str, index: int, *args) -> None:
    """Run an entry point on torch's current stream of GPU `index` (its last argument), whatever the current device is."""
    fn = getattr(_lib or load(), name)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        raise QFError(rc, name)
