"""What the operators of the 4-bit cache launch over their ranges, without a GPU (launches.py's recorder): every launch within the
device's limits, its LDS asked for where it is past the 64 KiB that a launch may have by default, every kernel of the library
reached by some call, and workspaces that hold what the launches' sizes say."""
import os
import random
import re
import shutil
import subprocess
import sys

import pytest

import launches
from qwen_fastpath import _kv4_lib as K

LDS, DEFAULT_LDS = 160 * 1024, 64 * 1024
LLVM = "/opt/rocm/llvm/bin"

_CHILD = """
import ctypes, sys, types
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
for n in ("torch", "binding", "binding._lib"):  # the binding alone: torch would register its own kernels with the recorder
    sys.modules[n] = types.ModuleType(n)
sys.modules["binding"].__path__ = [sys.argv[2]]
sys.modules["binding._lib"].QFError = RuntimeError
import binding._kv4_lib as K
L, P = K.load(), %d
H = K.Heads(P, 1 << 20, 256)

def tables(B, T):
    return L.qf_step_tables(P, P, P, P, 64, 64, P, P, 100, B, 16, T, P, P, P, P, P, P, P, None), 0

def rope(T, heads, kv, D, inter, f32, kind):
    none = K.Heads(None, 0, 0)
    pages = K.Pages(P, 1 << 20, 1 << 10, 256)
    a = K.RopeArgs(query=H if heads else none, key=H, value=H if kind else none, query_out=H if heads else none, key_out=H, q_weight=P,
                   k_weight=P, positions=P, cos_sin=P, slots=P, cache=P, cache_stride=kv * 17 * D, key_pages=pages, value_pages=pages,
                   num_positions=9, num_blocks=9, eps=1e-6, weight_offset=0.0, cos_sin_f32=f32, rot=32, interleaved=inter,
                   cache_kind=kind, page_size=16, num_tokens=T, num_heads=heads, num_kv_heads=kv, head_size=D)
    return L.qf_qk_norm_rope(ctypes.byref(a), None), 0

def load(T, kv, D):
    return L.qf_kv4_load(P, kv * 17 * D, 9, 16, kv, D, P, T, P, P, None), 0

def attention(B, q, heads, kv, D, ragged, most):
    a = K.AttentionArgs(query=H, out=H, cache=P, cache_stride=kv * 17 * D, num_blocks=9, block_table=P, bt_stride=most, seq_lens=P,
                        cu_q=P if ragged else None, scale=0.1, max_blocks=most, num_tokens=B * q, num_reqs=B, q_len=q, num_heads=heads,
                        num_kv_heads=kv, head_size=D, page_size=16)
    n = L.qf_kv4_attention_workspace_bytes(ctypes.byref(a))
    return L.qf_kv4_attention(ctypes.byref(a), P, n, None), n

for line in sys.stdin:
    name, *args = line.split()
    print("call", *globals()[name](*map(int, args)), flush=True)
""" % launches.P


def _record(calls):
    """[(status, workspace bytes, [(symbol, grid, threads, dynamic LDS, LDS asked for), ...])]"""
    text = "\n".join(" ".join(map(str, c)) for c in calls) + "\n"
    out = subprocess.run([sys.executable, "-c", _CHILD, launches._recorder(), os.path.dirname(K.LIB_PATH)], input=text,
                         check=True, capture_output=True, text=True, timeout=300).stdout
    got, pending, raised = [], [], {}
    for line in out.splitlines():
        what, *v = line.split()
        if what == "raise":
            raised[v[0]] = int(v[1])
        elif what == "launch":
            n = list(map(int, v[1:]))
            pending.append((v[0], tuple(n[:3]), n[3] * n[4] * n[5], n[6], raised.get(v[0], 0)))
        elif what == "call":
            got.append((int(v[0]), int(v[1]), pending))
            pending = []
    assert len(got) == len(calls)
    return got


@pytest.fixture(scope="module")
def static_lds(tmp_path_factory):
    """{kernel symbol: bytes of static LDS} of the built library."""
    if not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("ROCm LLVM tools absent")
    d = tmp_path_factory.mktemp("lib")
    shutil.copy(K.LIB_PATH, d / "lib.so")
    subprocess.run([os.path.join(LLVM, "llvm-objdump"), "--offloading", str(d / "lib.so")], cwd=d, check=True, capture_output=True)
    sizes = {}
    for f in os.listdir(d):
        if "gfx950" in f:
            notes = subprocess.run([os.path.join(LLVM, "llvm-readelf"), "--notes", str(d / f)], check=True, capture_output=True,
                                   text=True).stdout
            for kernel in notes.split("  - .agpr_count:")[1:]:
                sizes[re.search(r"\.name:\s+(\S+)", kernel).group(1)] = int(
                    re.search(r"\.group_segment_fixed_size:\s+(\d+)", kernel).group(1))
    return sizes


def _calls():
    rng = random.Random(1)
    size = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    calls = [("tables", B, T) for B in (1, 255, 4096) for T in (0, 1, 257, 1 << 20)]
    calls += [("rope", size(1, 20000), rng.choice([0, 1, 3, 16, 64]), rng.choice([1, 2, 8]), D, i, f, kind)
              for D in (64, 128, 256) for i in (0, 1) for f in (0, 1) for kind in (0, 1, 2) for _ in range(6)]
    calls += [("load", size(1, 50000), kv, D) for D in (64, 128, 256) for kv in (1, 8)]
    for D in (64, 128, 256):
        for _ in range(150):
            kv = rng.choice([1, 2, 4, 8])
            calls.append(("attention", size(1, 300), rng.choice([1, 1, 2, 5, 40, size(1, 3000)]), kv * rng.choice([1, 3, 8, 16]), kv, D,
                          rng.randint(0, 1), rng.choice([4, 4096])))
        calls += [("attention", 1, 100, 64, 8, D, r, 512) for r in (0, 1)] + [("attention", 60000, 1, 8, 2, D, 0, 8)]
    return calls


def test_launches(static_lds):
    seen = set()
    calls = _calls()
    for call, (rc, _, made) in zip(calls, _record(calls)):
        assert rc == 0 and made, call
        for symbol, grid, threads, lds, raised in made:
            total = static_lds[symbol] + lds
            assert total <= LDS, (call, symbol)
            assert total <= DEFAULT_LDS or raised >= lds, f"{call}: {symbol} takes {total} bytes of LDS unasked"
            assert threads <= 1024 and 0 < grid[0] * threads < 2 ** 32 and 0 < grid[1] < 65536 and 0 < grid[2] < 65536, (call, symbol, grid)
            seen.add(symbol)
    assert seen == set(static_lds), set(static_lds) - seen  # nothing stays that no call reaches


def test_a_grid_past_32_bits_is_refused():
    for call, (rc, _, made) in zip(*(lambda c: (c, _record(c)))([
            ("attention", 1, 1 << 27, 512, 64, 128, 0, 8), ("rope", 1 << 30, 64, 8, 128, 0, 0, 2), ("load", 1 << 30, 1, 256)])):
        assert rc == 2 and not made, (call, rc, made)


def test_workspaces_hold_what_the_launches_write():
    """The partial results that the launched grids have places for, in the bytes that the call asks for: a tile of fp32 sums with a
    maximum and a sum a row for each workgroup of the split kernel, and for each compute unit where row tiles may be split."""
    cus, seen = 256, set()  # what the library takes without a device
    calls = [c for c in _calls() if c[0] == "attention"]
    for call, (_, given, made) in zip(calls, _record(calls)):
        _, B, q, heads, kv, D, _, _ = call
        need, kinds = 0, tuple(re.search(r"attn_\w+?_kernel", m[0]).group(0) for m in made)
        for symbol, grid, *_ in made:
            if "attn_split_kernel" in symbol:
                _, rt, rg = map(int, re.search(r"attn_split_kernelILi(\d+)ELi(\d+)ELi(\d+)E", symbol).groups())
                assert 16 * rt * rg >= min(q * heads // kv, 64) and grid[1] == kv, call
                need += grid[0] * kv * (16 * rt * rg * D * 4 + min(q * heads // kv, 64) * 8) + B * 8
            if "attn_tile_combine_kernel" in symbol:
                need += cus * (128 if D == 256 else 256) * (4 * D + 8)
        assert given >= need, (call, kinds, given, need)
        assert (given == 0) == (need == 0), (call, kinds)
        seen.add(kinds)
    assert len(seen) == 4, seen  # few rows; tiles; tiles that may be split; tiles beside few rows
