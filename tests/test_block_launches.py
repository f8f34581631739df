"""What the block-scaled operators launch over their ranges, without a GPU (launches.py): every launch within the device's
limits, its LDS asked for where it is past the 64 KiB that a launch may have by default."""
import os
import random
import re
import shutil
import subprocess

import pytest

import launches
from qwen_fastpath import _block_lib as B

LDS, DEFAULT_LDS = 160 * 1024, 64 * 1024
LLVM = "/opt/rocm/llvm/bin"


@pytest.fixture(scope="module")
def static_lds(tmp_path_factory):
    """{kernel symbol: bytes of static LDS} of the built library."""
    if not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("ROCm LLVM tools absent")
    d = tmp_path_factory.mktemp("lib")
    shutil.copy(B.LIB_PATH, d / "lib.so")
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


def _check(calls, static_lds):
    seen = set()
    for call, (rc, _, made) in zip(calls, launches.record(calls)):
        assert rc == 0 and made, call
        for l in made:
            total = static_lds[l.symbol] + l.lds
            assert total <= LDS, (call, l)
            assert total <= DEFAULT_LDS or l.raised >= l.lds, f"{call}: {l.kernel}{l.params} takes {total} bytes of LDS unasked"
            assert l.threads <= 1024 and l.grid[0] * l.threads < 2 ** 32 and l.grid[1] < 65536 and l.grid[2] == 1, (call, l)
            seen.add((l.kernel, l.params))
    return seen


def test_experts_layer(static_lds):
    calls = [("moe", T, E, min(8, E), H, 64) for T in (1, 9, 16) for E in (8, 60, 100, 200, 512)
             for H in (64, 512, 1024, 2048, 2560, 4032, 4096, 4160, 7168, 8192, 1 << 20)]
    seen = _check(calls, static_lds)
    assert {p for k, p in seen if k == "moe_up_kernel"} == {(16, 4), (16, 8), (64, 1), (64, 2), (64, 4), (64, 8)}


def test_products_and_norms(static_lds):
    rng = random.Random(1)
    size = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    calls = [("decode", rng.randint(0, 1), rng.randint(1, 16), size(1, 300000), 64 * size(1, 1000)) for _ in range(600)]
    calls += [("w8a8", rng.randint(0, 1), size(1, 20000), size(1, 300000), 64 * size(1, 4096)) for _ in range(400)]
    calls += [("quantize", size(1, 100000), 64 * size(1, 1000)) for _ in range(20)]
    calls += [("norm", size(1, 100000), 8 * size(1, 4096), w) for _ in range(40) for w in (0, 1)]
    _check(calls, static_lds)
