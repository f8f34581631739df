"""What the entry points of libqf_block.so would launch, without a GPU: their host code runs in a process of its own with
the HIP runtime's launch calls stood in for (launch_record.c), on addresses that are never read."""
import functools
import os
import re
import subprocess
import sys
import tempfile
from dataclasses import dataclass

HERE = os.path.dirname(os.path.abspath(__file__))
P = 1 << 20  # an aligned address that is never read

_CHILD = """
import ctypes, sys
ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
L = ctypes.CDLL(sys.argv[2])
p, i64, i32, f32, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
for n in ("qf_fp8_w8a16_workspace_bytes", "qf_fp8_w8a8_workspace_bytes", "qf_moe_few_workspace_bytes"):
    getattr(L, n).restype = sz
P, ROOM = %d, sz(1 << 60)

def decode(layout, M, N, K):
    rc = L.qf_fp8_w8a16_gemm(p(P), i64(K), p(P), i64(K), layout, p(P), None, p(P), i64(N), 0, M, N, K, p(P), ROOM, None)
    return rc, L.qf_fp8_w8a16_workspace_bytes(M, N, K, layout)

def w8a8(layout, M, N, K):
    rc = L.qf_fp8_w8a8_linear(p(P), i64(K), p(P), i64(K), layout, p(P), None, p(P), i64(N), 0, M, N, K, p(P), ROOM, None)
    return rc, L.qf_fp8_w8a8_workspace_bytes(M, N, K)

def quantize(M, K):
    return L.qf_quantize_tokens_fp8(p(P), i64(K), M, K, p(P), i64(K), p(P), None), 0

def norm(M, N, wide):
    return L.qf_block_norm_rows(p(P), i64(N), p(P), i64(N), wide, None, None, f32(0), None, i64(0), 0, 0, f32(1), f32(0), M, N,
                                p(P), i64(N), p(P), i64(N), None), 0

def moe(T, E, k, H, I):
    rc = L.qf_moe_few_tokens(p(P), i64(H), p(P), i64(E), 1, p(P), p(P), p(P), p(P), p(P), i64(H), T, E, k, H, I, 1, p(P), ROOM, None)
    return rc, L.qf_moe_few_workspace_bytes(T, E, k, H, I)

for line in sys.stdin:
    name, *args = line.split()
    print("call", *globals()[name](*map(int, args)), flush=True)
""" % P


@dataclass(frozen=True)
class Launch:
    kernel: str      # the kernel's name without its namespace and argument types
    params: tuple    # its template parameters: whole numbers, or a tile's as a tuple
    grid: tuple
    threads: int
    lds: int         # dynamic
    raised: int      # the dynamic LDS it was allowed before, 0 where nothing was asked for
    symbol: str


def _parse(symbol):
    """(name, template parameters) of a mangled kernel of namespace qfb: numbers, booleans and Tile<...> types."""
    m = re.match(r"_ZN3qfb(\d+)(\w+)$", symbol)
    name, rest = m.group(2)[:int(m.group(1))], m.group(2)[int(m.group(1)):]
    params = []
    if rest.startswith("I"):
        rest = rest[1:]
        while not rest.startswith("E"):
            if t := re.match(r"NS_4TileI((?:Li\d+E)+)EE", rest):
                params.append(tuple(map(int, re.findall(r"Li(\d+)E", t.group(1)))))
            else:
                t = re.match(r"L[ib](\d+)E", rest)
                params.append(int(t.group(1)))
            rest = rest[t.end():]
    return name, tuple(params)


@functools.lru_cache(maxsize=None)
def _recorder():
    d = tempfile.mkdtemp(prefix="launch_record_")
    so = os.path.join(d, "launch_record.so")
    subprocess.run(["gcc", "-O1", "-Wall", "-fPIC", "-shared", "-o", so, os.path.join(HERE, "launch_record.c")], check=True)
    return so


def record(calls):
    """[(status, workspace bytes, [Launch, ...])] of calls ("decode", layout, M, N, K), ("w8a8", layout, M, N, K),
    ("quantize", M, K), ("norm", M, N, wide) and ("moe", T, E, k, H, I)."""
    from qwen_fastpath import _block_lib as B
    text = "\n".join(" ".join(map(str, c)) for c in calls) + "\n"
    out = subprocess.run([sys.executable, "-c", _CHILD, _recorder(), B.LIB_PATH], input=text, check=True,
                         capture_output=True, text=True, timeout=300).stdout
    got, pending, raised = [], [], {}
    for line in out.splitlines():
        what, *v = line.split()
        if what == "raise":
            raised[v[0]] = int(v[1])
        elif what == "launch":
            n = list(map(int, v[1:]))
            pending.append(Launch(*_parse(v[0]), tuple(n[:3]), n[3] * n[4] * n[5], n[6], raised.get(v[0], 0), v[0]))
        elif what == "call":
            got.append((int(v[0]), int(v[1]), pending))
            pending = []
    assert len(got) == len(calls)
    return got


def decode_form(call, recorded):
    """(layout, blocks a wavefront, KiB of x in LDS a block or 0, K split) of a ("decode", ...) call."""
    _, bytes_, made = recorded
    return (*made[-1].params, bytes_ > 0)


def w8a8_splits(call, recorded):
    """(channels and tokens of the last launch's tile, its K splits, whether a launch of whole rounds goes before it)."""
    _, _, M, N, _ = call
    tiles = [l for l in recorded[2] if l.kernel == "fp8_tile_kernel"]
    shape = lambda l: (16 * l.params[1][0] * l.params[1][2], 16 * l.params[1][1] * l.params[1][3])  # noqa: E731
    if len(tiles) == 2:
        channels, tokens = shape(tiles[0])
        N -= tiles[0].grid[0] // -(-M // tokens) * channels
    channels, tokens = shape(tiles[-1])
    n = -(-N // channels) * -(-M // tokens)
    assert tiles[-1].grid[0] % n == 0
    return channels, tokens, tiles[-1].grid[0] // n, len(tiles) == 2


def w8a8_form(call, recorded):
    """(layout, channels, tokens, K split, behind a first launch) of a ("w8a8", ...) call."""
    channels, tokens, splits, behind = w8a8_splits(call, recorded)
    return call[1], channels, tokens, splits > 1, behind


def decode_splits(call, recorded):
    """K splits of a ("decode", ...) call: its workspace is the counters and a KiB for each split and tile."""
    _, bytes_, _ = recorded
    counters = 64 * 1024
    return 1 if bytes_ == 0 else (bytes_ - counters) // (1024 * -(-call[3] // 16))
