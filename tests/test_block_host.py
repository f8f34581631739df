"""libqf_block.so without a GPU: its exports, its argument checks (every call here is refused before any HIP call) and the
refusals of the Python entry points."""
import ctypes
import os
import re

import pytest
import torch

import block_helpers as H
import qwen_fastpath as qf
from qwen_fastpath import _block_lib as B

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "qf_block.h")
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
P = 1 << 20  # an aligned address that is never read


def _define(name):
    return int(re.search(rf"#define {name} (\d+)", open(HEADER).read()).group(1))


def test_header_and_binding_agree():
    text = open(HEADER).read()
    assert sorted(set(re.findall(r"^\s*\w+\**\s+\**(qf_\w+)\(", text, flags=re.M))) == sorted(B.EXPORTS)
    lib = B.load()
    assert all(hasattr(lib, n) for n in B.EXPORTS)
    assert lib.qf_block_abi_version() == _define("QF_BLOCK_ABI_VERSION") == B.ABI_VERSION
    assert (_define("QF_FP8_BLOCK"), _define("QF_FP8_MAX_DECODE_M"), _define("QF_BLOCK_NORM_MAX_N"),
            _define("QF_MOE_MAX_EXPERTS"), _define("QF_MOE_MAX_TOP_K")) == (
        B.BLOCK, B.MAX_DECODE_M, B.NORM_MAX_N, B.MOE_MAX_EXPERTS, B.MOE_MAX_TOP_K)


def _product(a8=False, **kw):
    v = dict(x=P, ldx=256, w=P, ldw=256, layout=0, scale=P, bias=None, y=P, ldy=64, out=0, M=4, N=64, K=256, ws=P,
             nbytes=1 << 30)
    v.update(kw)
    args = [v[n] for n in ("x", "ldx", "w", "ldw", "layout", "scale", "bias", "y", "ldy", "out", "M", "N", "K")]
    if a8:
        return B.load().qf_fp8_w8a8_linear(*args, v["ws"], v["nbytes"], None)
    return B.load().qf_fp8_w8a16_gemm(*args, v["ws"], v["nbytes"], None)


@pytest.mark.parametrize("a8", [False, True])
@pytest.mark.parametrize("kw,want", [
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(scale=None), INVALID), (dict(y=None), INVALID),
    (dict(M=0), INVALID), (dict(N=0), INVALID), (dict(K=0), INVALID), (dict(out=2), INVALID), (dict(layout=2), INVALID),
    (dict(ldx=248), INVALID), (dict(ldy=63), INVALID), (dict(ldw=240), INVALID), (dict(K=100), UNSUPPORTED),
    (dict(ldx=260), UNSUPPORTED), (dict(ldw=264), UNSUPPORTED), (dict(x=P + 8), UNSUPPORTED), (dict(w=P + 4), UNSUPPORTED)])
def test_product_refusals(a8, kw, want):
    assert _product(a8, **kw) == want


def test_product_limits():
    assert _product(M=17) == UNSUPPORTED
    need = B.load().qf_fp8_w8a8_workspace_bytes(4, 64, 256)
    assert need > 0
    assert _product(True, nbytes=need - 1) == WORKSPACE and _product(True, ws=None) == WORKSPACE
    assert _product(True, ws=P + 8) == WORKSPACE
    for M, N, K in ((0, 64, 64), (4, 0, 64), (4, 64, 0), (4, 64, 100)):
        assert B.load().qf_fp8_w8a8_workspace_bytes(M, N, K) == 0


def test_sizes_past_a_launch():
    """Grids of 2^32 threads and more, and rows of activations whose scales outgrow a workgroup, are refused."""
    w8a8 = B.load().qf_fp8_w8a8_workspace_bytes
    assert w8a8(2 ** 28 - 16, 16, 64) > 0 and w8a8(2 ** 28, 16, 64) == 0
    assert w8a8(32, 16, 2 ** 18) > 0 and w8a8(32, 16, 2 ** 18 + 64) == 0
    assert _product(True, M=2 ** 28, nbytes=1 << 62) == UNSUPPORTED
    assert _product(True, K=2 ** 18 + 64, ldx=2 ** 18 + 64, ldw=2 ** 18 + 64, nbytes=1 << 62) == UNSUPPORTED
    assert B.load().qf_quantize_tokens_fp8(P, 64, 2 ** 28, 64, P, 64, P, None) == UNSUPPORTED
    for M, N in ((2 ** 22, 8192), (2 ** 26, 512), (2 ** 28, 128), (2 ** 31 - 1, 8)):
        assert B.load().qf_block_norm_rows(P, N, P, N, 0, None, None, 0.0, None, 0, 0, 0, 1.0, 1e-6, M, N, P, N, P, N,
                                           None) == UNSUPPORTED


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), INVALID), (dict(xq=None), INVALID), (dict(s=None), INVALID), (dict(M=0), INVALID),
    (dict(ldx=64), INVALID), (dict(ldq=64), INVALID), (dict(K=72), UNSUPPORTED), (dict(ldx=132), UNSUPPORTED),
    (dict(xq=P + 4), UNSUPPORTED), (dict(x=P + 2), UNSUPPORTED)])
def test_quantiser_refusals(kw, want):
    v = dict(x=P, ldx=128, M=4, K=128, xq=P, ldq=128, s=P)
    v.update(kw)
    assert B.load().qf_quantize_tokens_fp8(*(v[n] for n in ("x", "ldx", "M", "K", "xq", "ldq", "s")), None) == want


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), INVALID), (dict(residual=None), INVALID), (dict(y=None), INVALID), (dict(h=None), INVALID),
    (dict(M=0), INVALID), (dict(N=0), INVALID), (dict(kind=4, gate=P), INVALID), (dict(kind=1), INVALID),
    (dict(gate=P), INVALID), (dict(act=2), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID),
    (dict(ldy=56), INVALID), (dict(ldh=56), INVALID), (dict(ldx=-64), INVALID), (dict(N=60), UNSUPPORTED),
    (dict(N=32776, ldx=32776, ldr=32776, ldy=32776, ldh=32776), UNSUPPORTED), (dict(ldx=68), UNSUPPORTED),
    (dict(ldr=68), UNSUPPORTED), (dict(ldy=68), UNSUPPORTED), (dict(ldh=68), UNSUPPORTED), (dict(x=P + 8), UNSUPPORTED),
    (dict(post=P + 8), UNSUPPORTED), (dict(pre=P + 8), UNSUPPORTED), (dict(gate=P + 8, kind=3, ldg=64), UNSUPPORTED),
    (dict(gate=P, kind=3, ldg=60), UNSUPPORTED), (dict(residual=P + 8, f32=1), UNSUPPORTED)])
def test_norm_refusals(kw, want):
    v = dict(x=P, ldx=64, residual=P, ldr=64, f32=0, post=None, pre=None, off=0.0, gate=None, ldg=0, kind=0, act=0,
             alpha=1.0, eps=1e-6, M=4, N=64, y=P, ldy=64, h=P, ldh=64)
    v.update(kw)
    names = "x ldx residual ldr f32 post pre off gate ldg kind act alpha eps M N y ldy h ldh".split()
    assert B.load().qf_block_norm_rows(*(v[n] for n in names), None) == want


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), INVALID), (dict(logits=None), INVALID), (dict(w13=None), INVALID), (dict(s13=None), INVALID),
    (dict(w2=None), INVALID), (dict(s2=None), INVALID), (dict(y=None), INVALID), (dict(T=0), INVALID), (dict(E=0), INVALID),
    (dict(k=0), INVALID), (dict(ldx=120), INVALID), (dict(ldl=7), INVALID), (dict(ldy=120), INVALID),
    (dict(T=17), UNSUPPORTED), (dict(E=513, ldl=513), UNSUPPORTED), (dict(k=9), UNSUPPORTED),
    (dict(k=17, E=32, ldl=32), UNSUPPORTED), (dict(H=100), UNSUPPORTED), (dict(I=96), UNSUPPORTED),
    (dict(ldx=132), UNSUPPORTED), (dict(ldy=130), UNSUPPORTED), (dict(x=P + 8), UNSUPPORTED), (dict(w13=P + 8), UNSUPPORTED),
    (dict(w2=P + 8), UNSUPPORTED), (dict(y=P + 4), UNSUPPORTED), (dict(nbytes=100), WORKSPACE), (dict(ws=None), WORKSPACE),
    (dict(ws=P + 8), WORKSPACE)])
def test_moe_refusals(kw, want):
    v = dict(x=P, ldx=128, logits=P, ldl=8, f32=1, w13=P, s13=P, w2=P, s2=P, y=P, ldy=128, T=4, E=8, k=2, H=128, I=64, re=1,
             ws=P, nbytes=1 << 30)
    v.update(kw)
    names = "x ldx logits ldl f32 w13 s13 w2 s2 y ldy T E k H I re ws nbytes".split()
    assert B.load().qf_moe_few_tokens(*(v[n] for n in names), None) == want


def test_moe_workspace():
    f = B.load().qf_moe_few_workspace_bytes
    assert f(16, 128, 8, 2048, 768) >= 16 * 8 * 768 * 2
    for bad in ((0, 8, 2, 64, 64), (17, 8, 2, 64, 64), (1, 8, 9, 64, 64), (1, 8, 2, 100, 64), (1, 8, 2, 64, 32), (1, 513, 2, 64, 64)):
        assert f(*bad) == 0


BF16 = torch.bfloat16


def test_host_tensors_are_refused():
    x = torch.zeros(4, 128, dtype=BF16)
    q, s = H.weight(H.gen(0), 64, 128)
    for f in (qf.fp8_linear, qf.fp8_w8a16_mm, qf.fp8_w8a8_mm):
        with pytest.raises(TypeError):
            f(x, q.t(), s)
    for f in (lambda: qf.quantize_tokens_fp8(x), lambda: qf.fp8_to_tiled(q.t()), lambda: qf.block_norm_rows(x, x),
              lambda: qf.moe_few_tokens(x, torch.zeros(4, 2), q.view(-1), s, q.view(-1), s, 1)):
        with pytest.raises(TypeError):
            f()


@pytest.mark.parametrize("call", [
    lambda x, q, s: qf.fp8_linear(x.float(), q.t(), s),
    lambda x, q, s: qf.fp8_linear(x, q.float().t(), s),
    lambda x, q, s: qf.fp8_linear(x, q.t(), s.double()),
    lambda x, q, s: qf.fp8_w8a8_mm(x, q.t(), s, torch.float16),
    lambda x, q, s: qf.fp8_w8a16_mm(x.view(-1), q.t(), s),
    lambda x, q, s: qf.fp8_to_tiled(q.view(torch.int8).t()),
    lambda x, q, s: qf.fp8_from_tiled(q.view(torch.int8).view(-1), 64, 128),
    lambda x, q, s: qf.quantize_tokens_fp8(x.float()),
    lambda x, q, s: qf.block_norm_rows(x.float(), x),
    lambda x, q, s: qf.block_norm_rows(x, x.half()),
    lambda x, q, s: qf.moe_few_tokens(x.float(), s, q, s, q, s, 1),
    lambda x, q, s: qf.moe_few_tokens(x, s.half(), q, s, q, s, 1),
    lambda x, q, s: qf.moe_few_tokens(x, s, q.float(), s, q, s, 1)])
def test_types_are_refused(call):
    x = torch.zeros(4, 128, dtype=BF16)
    with pytest.raises(TypeError):
        call(x, *H.weight(H.gen(0), 64, 128))


@pytest.mark.parametrize("call", [
    lambda x, q, s: qf.fp8_w8a16_mm(torch.zeros(17, 128, dtype=BF16), q.t(), s),
    lambda x, q, s: qf.fp8_from_tiled(q.view(-1)[:64], 64, 128),
    lambda x, q, s: qf.block_norm_rows(x, x[:2]),
    lambda x, q, s: qf.block_norm_rows(x[:, :60], x[:, :60]),
    lambda x, q, s: qf.block_norm_rows(x, x, gate_act="tanh"),
    lambda x, q, s: qf.block_norm_rows(x, x, eps=-1.0)])
def test_values_are_refused(call):
    x = torch.zeros(4, 128, dtype=BF16)
    with pytest.raises(ValueError):
        call(x, *H.weight(H.gen(0), 64, 128))


def test_sizes_are_checked_before_any_launch(monkeypatch):
    """The shape checks behind the device check, with the device check stood in for: nothing may reach the library."""
    monkeypatch.setattr(B, "same_gpu", lambda *t: t[0].device)
    monkeypatch.setattr(B, "call", lambda name, *a: pytest.fail(f"{name} was called"))
    x = torch.zeros(4, 128, dtype=BF16)
    q, s = H.weight(H.gen(0), 64, 128)
    bad_bias = torch.zeros(63, dtype=BF16)
    for args, kw in (((x, q, s), {}), ((x[:, :96], q[:, :96].t(), s), {}), ((x, q.t(), s[:, :0]), {}),
                     ((x, q.t(), torch.zeros(2, 1)), {}), ((x, q.view(-1)[:-16], s), {}),
                     ((x, q.view(-1), s), dict(out_features=80)), ((x, q.view(-1), s), dict(out_features=48)),
                     ((x, q.t(), s), dict(out_features=63)), ((x, q[:, :120].t(), s), {})):
        with pytest.raises(ValueError):
            qf.fp8_linear(*args, **kw)
    with pytest.raises(TypeError):
        qf.fp8_linear(x, q.t(), s, bad_bias)
    with pytest.raises(ValueError):
        qf.quantize_tokens_fp8(x[:, :96])
    for kw in (dict(gate=torch.zeros(3, dtype=BF16)), dict(gate=torch.zeros(3, 1, dtype=BF16)),
               dict(y=torch.zeros(4, 128)), dict(h=torch.zeros(4, 120, dtype=BF16)),
               dict(y=torch.zeros(128, dtype=BF16).expand(4, 128))):
        with pytest.raises(ValueError):
            qf.block_norm_rows(x, x, **kw)
    for kw in (dict(post_weight=torch.zeros(64, dtype=BF16)), dict(pre_weight=torch.zeros(128)),
               dict(gate=torch.zeros(128))):
        with pytest.raises(TypeError):
            qf.block_norm_rows(x, x, **kw)
    E, I = 3, 64
    w13 = torch.zeros(E * 2 * I * 128, dtype=torch.uint8).view(H.FP8)
    w2 = torch.zeros(E * 128 * I, dtype=torch.uint8).view(H.FP8)
    good = dict(x=x, router_logits=torch.zeros(4, E), w13=w13, s13=torch.zeros(E, 2, 1), w2=w2, s2=torch.zeros(E, 1, 1), top_k=2)
    for kw in (dict(x=torch.zeros(17, 128, dtype=BF16), router_logits=torch.zeros(17, E)), dict(router_logits=torch.zeros(5, E)),
               dict(top_k=4), dict(top_k=0), dict(w13=w13[:-16]), dict(w2=w2[:-16]), dict(s13=torch.zeros(E, 1, 1)),
               dict(s2=torch.zeros(E, 1, 2)), dict(w13=w13.view(-1, 128)), dict(x=x[:, :120])):
        with pytest.raises(ValueError):
            qf.moe_few_tokens(**{**good, **kw})


def test_op_has_a_fake():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(2, 3, 128, dtype=BF16, device="cuda")
        s = torch.empty(1, 1, device="cuda")
        w = torch.empty(64, 128, dtype=H.FP8, device="cuda")
        assert torch.ops.qwen_fastpath.qf_fp8_linear(x, w.t(), s).shape == (2, 3, 64)
        assert torch.ops.qwen_fastpath.qf_fp8_linear(x, w.view(-1), s, None, 60).shape == (2, 3, 60)


def test_kernels_use_no_scratch(tmp_path):
    """Every kernel of the library's code objects (one a source file) keeps its working set in registers and LDS."""
    import shutil
    import subprocess
    llvm = "/opt/rocm/llvm/bin"
    if not (os.path.exists(B.LIB_PATH) and os.path.exists(os.path.join(llvm, "llvm-objdump"))):
        pytest.skip("built library or ROCm LLVM tools absent")
    copy = tmp_path / "lib.so"
    shutil.copy(B.LIB_PATH, copy)
    subprocess.run([os.path.join(llvm, "llvm-objdump"), "--offloading", str(copy)], cwd=tmp_path, check=True,
                   capture_output=True)
    kernels = {}
    for f in os.listdir(tmp_path):
        if "gfx950" in f:
            notes = subprocess.run([os.path.join(llvm, "llvm-readelf"), "--notes", str(tmp_path / f)], check=True,
                                   capture_output=True, text=True).stdout
            kernels.update(zip(re.findall(r"\.name:\s+(\S+)", notes),
                               map(int, re.findall(r"\.private_segment_fixed_size:\s+(\d+)", notes))))
    assert not {n: s for n, s in kernels.items() if s}
    for name in ("fp8_tile_kernel", "fp8_decode_kernel", "block_norm_kernel", "moe_up_kernel", "moe_down_kernel"):
        assert any(name in n for n in kernels), name
