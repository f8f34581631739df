"""libqf_kv4.so without a GPU: its exports, its argument checks (every call here is refused before any HIP call), the refusals
of the Python entry points, and the references of the GPU tests against themselves."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import kv4_helpers as H
import qwen_fastpath as qf
from qwen_fastpath import _kv4_lib as K

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "qf_kv4.h")
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
P = 1 << 20  # an aligned address that is never read
BF16, I32, I64, U8 = torch.bfloat16, torch.int32, torch.int64, torch.uint8


def _define(name):
    return eval(re.search(rf"#define {name} (.+)", open(HEADER).read()).group(1))


def test_header_and_binding_agree():
    text = open(HEADER).read()
    assert sorted(set(re.findall(r"^\s*\w+\**\s+\**(qf_\w+)\(", text, flags=re.M))) == sorted(K.EXPORTS)
    lib = K.load()
    assert all(hasattr(lib, n) for n in K.EXPORTS)
    assert lib.qf_kv4_abi_version() == _define("QF_KV4_ABI_VERSION") == K.ABI_VERSION
    assert (_define("QF_KV4_TILE"), _define("QF_STEP_MAX_REQS"), _define("QF_STEP_MAX_TOKENS")) == (K.TILE, K.MAX_REQS, K.MAX_TOKENS)
    assert K.module() is not None


def test_structures_match_the_header(tmp_path):
    fields = {"qf_qk_norm_rope_args": K.RopeArgs, "qf_kv4_attention_args": K.AttentionArgs}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "qf_kv4.h"\nint main() {\n'
    for c, t in fields.items():
        src += "".join(f'  printf("%zu ", offsetof({c}, {n}));\n' for n, _ in t._fields_) + f'  printf("%zu\\n", sizeof({c}));\n'
    (tmp_path / "s.c").write_text(src + "  return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), "-o", tmp_path / "s", tmp_path / "s.c"], check=True)
    lines = subprocess.run([tmp_path / "s"], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, t in zip(lines, fields.values()):
        assert list(map(int, line.split())) == [getattr(t, n).offset for n, _ in t._fields_] + [ctypes.sizeof(t)]


@pytest.mark.parametrize("kw,want", [
    (dict(context=None), INVALID), (dict(q=None), INVALID), (dict(held=None), INVALID), (dict(table=None), INVALID),
    (dict(stack=None), INVALID), (dict(count=None), INVALID), (dict(cu=None), INVALID), (dict(seq=None), INVALID),
    (dict(pos=None), INVALID), (dict(slots=None), INVALID), (dict(held_out=None), INVALID), (dict(count_out=None), INVALID),
    (dict(fits=None), INVALID), (dict(B=0), INVALID), (dict(page=0), INVALID), (dict(T=-1), INVALID), (dict(width=0), INVALID),
    (dict(stride=7), INVALID), (dict(free=-1), INVALID), (dict(B=4097), UNSUPPORTED), (dict(T=(1 << 29) + 1), UNSUPPORTED),
    (dict(free=(1 << 29) + 1), UNSUPPORTED), (dict(width=(1 << 29) + 1, stride=1 << 30), UNSUPPORTED)])
def test_tables_refusals(kw, want):
    v = dict(context=P, q=P, held=P, table=P, stride=8, width=8, stack=P, count=P, free=64, B=4, page=16, T=20, cu=P, seq=P, pos=P,
             slots=P, held_out=P, count_out=P, fits=P)
    v.update(kw)
    names = "context q held table stride width stack count free B page T cu seq pos slots held_out count_out fits".split()
    assert K.load().qf_step_tables(*(v[n] for n in names), None) == want


def _rope(**kw):
    h, pages = K.Heads(P, 1024, 128), K.Pages(P, 4096, 256, 128)
    v = dict(query=h, key=h, value=h, query_out=h, key_out=K.Heads(), q_weight=P, k_weight=P, positions=P, cos_sin=P, slots=P,
             cache=P, cache_stride=2 * 17 * 128, key_pages=pages, value_pages=pages, num_positions=100, num_blocks=4, eps=1e-6,
             weight_offset=0.0, cos_sin_f32=0, rot=64, interleaved=0, cache_kind=K.CACHE_KV4, page_size=16, num_tokens=5,
             num_heads=8, num_kv_heads=2, head_size=128)
    v.update(kw)
    return K.load().qf_qk_norm_rope(ctypes.byref(K.RopeArgs(**v)), None)


NONE = K.Heads()


@pytest.mark.parametrize("kw,want", [
    (dict(key=NONE), INVALID), (dict(query_out=NONE), INVALID), (dict(query=NONE), INVALID), (dict(value=NONE), INVALID),
    (dict(num_tokens=0), INVALID), (dict(num_heads=0), INVALID), (dict(num_kv_heads=0), INVALID), (dict(cache_kind=3), INVALID),
    (dict(cache_kind=-1), INVALID), (dict(cache=None), INVALID), (dict(slots=None), INVALID), (dict(num_blocks=0), INVALID),
    (dict(page_size=0), INVALID), (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(rot=-16), INVALID),
    (dict(rot=144), INVALID), (dict(positions=None), INVALID), (dict(cos_sin=None), INVALID), (dict(num_positions=0), INVALID),
    (dict(cache_kind=0), INVALID), (dict(cache_kind=0, value=NONE, key_out=NONE), INVALID),
    (dict(cache_kind=1, key_pages=K.Pages()), INVALID), (dict(cache_kind=1, value_pages=K.Pages()), INVALID),
    (dict(head_size=96), UNSUPPORTED), (dict(rot=40), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
    (dict(cache=P + 8), UNSUPPORTED), (dict(cache_stride=2 * 17 * 128 + 8), UNSUPPORTED), (dict(cache_stride=17 * 128), UNSUPPORTED),
    (dict(query=K.Heads(P + 8, 1024, 128)), UNSUPPORTED), (dict(key=K.Heads(P, 1020, 128)), UNSUPPORTED),
    (dict(value=K.Heads(P, 1024, 132)), UNSUPPORTED), (dict(query_out=K.Heads(P, -1024, 128)), UNSUPPORTED),
    (dict(key_out=K.Heads(P, 1024, 4)), UNSUPPORTED), (dict(q_weight=P + 2), UNSUPPORTED), (dict(k_weight=P + 8), UNSUPPORTED),
    (dict(cos_sin=P + 4), UNSUPPORTED), (dict(cache_kind=1, key_pages=K.Pages(P, 4096, 256, 4)), UNSUPPORTED),
    (dict(cache_kind=1, value_pages=K.Pages(P + 8, 4096, 256, 128)), UNSUPPORTED),
    (dict(cache_kind=1, key_pages=K.Pages(P, 4100, 256, 128)), UNSUPPORTED),
    (dict(num_tokens=2 ** 31 - 1), UNSUPPORTED), (dict(num_blocks=2 ** 41), UNSUPPORTED), (dict(num_heads=2 ** 31 - 1), UNSUPPORTED)])
def test_rope_refusals(kw, want):
    assert _rope(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(cache=None), INVALID), (dict(slots=None), INVALID), (dict(key=None), INVALID), (dict(value=None), INVALID),
    (dict(blocks=0), INVALID), (dict(page=0), INVALID), (dict(heads=0), INVALID), (dict(T=0), INVALID), (dict(D=80), UNSUPPORTED),
    (dict(page=40), UNSUPPORTED), (dict(stride=17 * 64), UNSUPPORTED), (dict(cache=P + 8), UNSUPPORTED),
    (dict(key=P + 8), UNSUPPORTED), (dict(value=P + 2), UNSUPPORTED), (dict(T=2 ** 31 - 1, heads=2, stride=4 * 17 * 64), UNSUPPORTED)])
def test_load_refusals(kw, want):
    v = dict(cache=P, stride=2 * 17 * 64, blocks=4, page=32, heads=1, D=64, slots=P, T=5, key=P, value=P)
    v.update(kw)
    assert K.load().qf_kv4_load(*(v[n] for n in "cache stride blocks page heads D slots T key value".split()), None) == want


def test_a_load_whose_threads_pass_64_bits_is_refused():
    """(2^31 - 1)^2 heads of 8 lanes are more than 2^64 threads: their number must not wrap to a small one."""
    n = 2 ** 31 - 1
    assert K.load().qf_kv4_load(P, 2 * 17 * 64 * n, 4, 32, n, 64, P, n, P, P, None) == UNSUPPORTED



def _attention(ws=P, nbytes=1 << 40, **kw):
    v = dict(query=K.Heads(P, 1024, 128), out=K.Heads(P, 1024, 128), cache=P, cache_stride=2 * 17 * 128, num_blocks=9, block_table=P,
             bt_stride=8, seq_lens=P, cu_q=None, scale=0.1, max_blocks=8, num_tokens=8, num_reqs=4, q_len=2, num_heads=8,
             num_kv_heads=2, head_size=128, page_size=16)
    v.update(kw)
    args = K.AttentionArgs(**v)
    return K.load().qf_kv4_attention(ctypes.byref(args), ws, nbytes, None), K.load().qf_kv4_attention_workspace_bytes(ctypes.byref(args))


@pytest.mark.parametrize("kw,want", [
    (dict(query=NONE), INVALID), (dict(out=NONE), INVALID), (dict(cache=None), INVALID), (dict(block_table=None), INVALID),
    (dict(seq_lens=None), INVALID), (dict(num_blocks=0), INVALID), (dict(max_blocks=0), INVALID), (dict(bt_stride=-1), INVALID),
    (dict(num_tokens=0), INVALID), (dict(num_tokens=7), INVALID), (dict(num_reqs=0), INVALID), (dict(q_len=0), INVALID),
    (dict(num_heads=0), INVALID), (dict(num_kv_heads=0), INVALID), (dict(page_size=0), INVALID), (dict(scale=float("nan")), INVALID),
    (dict(num_heads=9), UNSUPPORTED), (dict(head_size=96), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
    (dict(cache_stride=2 * 17 * 128 + 4), UNSUPPORTED), (dict(cache_stride=17 * 128), UNSUPPORTED), (dict(cache=P + 8), UNSUPPORTED),
    (dict(query=K.Heads(P + 8, 1024, 128)), UNSUPPORTED), (dict(out=K.Heads(P, 1028, 128)), UNSUPPORTED),
    (dict(query=K.Heads(P, 1024, -128)), UNSUPPORTED), (dict(num_reqs=65536, num_tokens=1 << 20), UNSUPPORTED),
    (dict(q_len=1 << 30, num_tokens=1 << 30, cu_q=P), UNSUPPORTED), (dict(max_blocks=1 << 27), UNSUPPORTED)])
def test_attention_refusals(kw, want):
    assert _attention(**kw)[0] == want


def test_attention_workspace():
    need = _attention(ws=None)[1]
    assert need > 0 and _attention(ws=None)[0] == WORKSPACE
    assert _attention(nbytes=need - 1)[0] == WORKSPACE and _attention(ws=P + 8)[0] == WORKSPACE
    assert _attention(num_heads=9)[1] == 0 and _attention(head_size=96)[1] == 0 and _attention(q_len=0)[1] == 0


# ---- the Python entry points ----

def _good():
    x = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)  # noqa: E731
    return dict(
        tables=dict(context_lens=x(3, dtype=I32), query_lens=x(3, dtype=I32), held=x(3, dtype=I32), block_table=x(3, 4, dtype=I32),
                    free_blocks=x(9, dtype=I32), free_count=x(1, dtype=I32), page_size=16, num_tokens=7),
        rope=dict(query=x(5, 4, 128), key=x(5, 2, 128), positions=x(5, dtype=I64), cos_sin=x(9, 64), q_weight=x(128), k_weight=x(128),
                  value=x(5, 2, 128), cache=x(3, 2, 1, 17 * 128, dtype=U8), slots=x(5, dtype=I64)),
        store=dict(key=x(5, 2, 64), value=x(5, 2, 64), cache=x(3, 2, 2, 17 * 64, dtype=U8), slots=x(5, dtype=I64)),
        load=dict(cache=x(3, 2, 2, 17 * 64, dtype=U8), slots=x(5, dtype=I64)),
        attention=dict(query=x(6, 4, 128), cache=x(3, 2, 1, 17 * 128, dtype=U8), seq_lens=x(3, dtype=I32), block_table=x(3, 2, dtype=I32),
                       scale=0.1, q_len=2))


CALLS = dict(tables=qf.step_tables, rope=qf.qk_norm_rope, store=qf.kv4_store, load=qf.kv4_load, attention=qf.kv4_attention)


@pytest.mark.parametrize("name", CALLS)
def test_host_tensors_are_refused(name):
    with pytest.raises(TypeError, match="GPU tensor"):
        CALLS[name](**_good()[name])


z = torch.zeros
WRONG = [
    ("tables", dict(context_lens=z(3, 1, dtype=I32))), ("tables", dict(context_lens=z(0, dtype=I32))),
    ("tables", dict(context_lens=z(4097, dtype=I32))), ("tables", dict(query_lens=z(4, dtype=I32))),
    ("tables", dict(query_lens=z(3, dtype=I64))), ("tables", dict(held=z(2, dtype=I32))), ("tables", dict(free_count=z(2, dtype=I32))),
    ("tables", dict(free_blocks=z(3, 3, dtype=I32))), ("tables", dict(free_blocks=z(3, dtype=I64))),
    ("tables", dict(block_table=z(2, 4, dtype=I32))), ("tables", dict(block_table=z(3, 4, dtype=I64))),
    ("tables", dict(block_table=z(4, 3, dtype=I32).t())), ("tables", dict(block_table=z(4, dtype=I32).expand(3, 4))),
    ("tables", dict(page_size=0)), ("tables", dict(num_tokens=-1)), ("tables", dict(num_tokens=1 << 30)),
    ("rope", dict(query=z(5, 4, 128))), ("rope", dict(query=z(5, 4, 96, dtype=BF16))), ("rope", dict(query=z(5, 512, dtype=BF16))),
    ("rope", dict(key=z(4, 2, 128, dtype=BF16))), ("rope", dict(key=z(5, 2, 64, dtype=BF16))), ("rope", dict(key=z(5, 2, 128))),
    ("rope", dict(value=z(5, 1, 128, dtype=BF16))), ("rope", dict(value=None)), ("rope", dict(slots=None)),
    ("rope", dict(slots=z(5, dtype=I32))), ("rope", dict(positions=z(5, dtype=I32))), ("rope", dict(positions=None)),
    ("rope", dict(cos_sin=None)), ("rope", dict(cos_sin=z(9, 72, dtype=BF16))), ("rope", dict(cos_sin=z(9, 144, dtype=BF16))),
    ("rope", dict(cos_sin=z(9, 64, dtype=torch.float16))), ("rope", dict(cos_sin=z(0, 64, dtype=BF16))),
    ("rope", dict(cos_sin=z(9, 0, dtype=BF16))), ("rope", dict(q_weight=z(64, dtype=BF16))), ("rope", dict(k_weight=z(128))),
    ("rope", dict(eps=-1.0)), ("rope", dict(eps=float("nan"))), ("rope", dict(cache=z(3, 4, 1, 17 * 128, dtype=U8))),
    ("rope", dict(cache=z(3, 2, 1, 17 * 64, dtype=U8))), ("rope", dict(cache=z(3, 2, 1, 16 * 128, dtype=U8))),
    ("rope", dict(cache=z(3, 2, 1, 17 * 128))), ("rope", dict(cache=(z(3, 16, 2, 128, dtype=BF16),))),
    ("rope", dict(cache=(z(3, 16, 2, 128, dtype=BF16), z(3, 16, 2, 128)))),
    ("rope", dict(cache=(z(3, 16, 2, 128, dtype=BF16), z(3, 8, 2, 128, dtype=BF16)))),
    ("rope", dict(cache=(z(3, 16, 4, 128, dtype=BF16),) * 2)), ("rope", dict(cache=(z(3, 16, 2, 132, dtype=BF16)[..., :128],) * 2)),
    ("rope", dict(cache=None)), ("rope", dict(query_out=z(5, 4, 128))), ("rope", dict(query_out=z(4, 4, 128, dtype=BF16))),
    ("rope", dict(query_out=z(1, 4, 128, dtype=BF16).expand(5, 4, 128))), ("rope", dict(key_out=z(5, 2, 132, dtype=BF16)[..., :128])),
    ("store", dict(key=z(5, 2, 96, dtype=BF16))), ("store", dict(value=z(4, 2, 64, dtype=BF16))), ("store", dict(slots=z(4, dtype=I64))),
    ("store", dict(cache=z(3, 2, 2, 17 * 128, dtype=U8))), ("store", dict(cache=z(3, 2, 2, 2 * 17 * 64, dtype=U8)[..., ::2])),
    ("store", dict(cache=z(1, 2, 2, 17 * 64, dtype=U8).expand(3, 2, 2, 17 * 64))),
    ("load", dict(slots=z(5, dtype=I32))), ("load", dict(slots=z(5, 1, dtype=I64))), ("load", dict(cache=z(3, 2, 17 * 64, dtype=U8))),
    ("attention", dict(q_len=None)), ("attention", dict(cu_q=z(4, dtype=I32))), ("attention", dict(q_len=None, cu_q=z(4, dtype=I32))),
    ("attention", dict(q_len=None, max_q=2)), ("attention", dict(q_len=0)), ("attention", dict(q_len=3)),
    ("attention", dict(q_len=None, cu_q=z(3, dtype=I32), max_q=2)), ("attention", dict(q_len=None, cu_q=z(4, dtype=I64), max_q=2)),
    ("attention", dict(query=z(6, 4, 128))), ("attention", dict(query=z(6, 3, 128, dtype=BF16))),
    ("attention", dict(query=z(6, 4, 64, dtype=BF16))), ("attention", dict(seq_lens=z(3, dtype=I64))),
    ("attention", dict(seq_lens=z(3, 1, dtype=I32))), ("attention", dict(block_table=z(2, 2, dtype=I32))),
    ("attention", dict(block_table=z(3, 2, dtype=I64))), ("attention", dict(block_table=z(3, 0, dtype=I32))),
    ("attention", dict(block_table=z(1, dtype=I32).expand(3, 1 << 27))),
    ("attention", dict(scale=float("nan"))), ("attention", dict(out=z(5, 4, 128, dtype=BF16))), ("attention", dict(out=z(6, 4, 128))),
]


@pytest.mark.parametrize("i", range(len(WRONG)))
def test_arguments_are_checked_before_any_launch(i, monkeypatch):
    """The checks behind the device check, with the device check stood in for: nothing may reach the library."""
    name, change = WRONG[i]
    monkeypatch.setattr(K, "gpu", lambda *t: 0)
    monkeypatch.setattr(K, "call", lambda name, *a: pytest.fail(f"{name} was called"))
    with pytest.raises((TypeError, ValueError)):
        CALLS[name](**{**_good()[name], **change})


@pytest.mark.parametrize("name", CALLS)
def test_good_arguments_reach_the_library(name, monkeypatch):
    called = []
    monkeypatch.setattr(K, "gpu", lambda *t: 0)
    monkeypatch.setattr(K, "call", lambda name, *a: called.append(name) or (None,) * 7)
    CALLS[name](**_good()[name])
    assert len(called) == 1


def test_copies_for_the_kernels(monkeypatch):
    """What the kernels cannot address is copied: odd strides, unaligned views, subclasses; outputs never."""
    class Sub(torch.Tensor):
        pass
    args = []
    monkeypatch.setattr(K, "gpu", lambda *t: 0)
    monkeypatch.setattr(K, "call", lambda name, index, *a: args.extend(a) or (None, None))
    good = _good()["rope"]
    q = torch.arange(5 * 4 * 129, dtype=torch.float32).to(BF16).view(5, 4, 129)[..., 1:]
    w = torch.arange(129, dtype=torch.float32).to(BF16)[1:]
    qf.qk_norm_rope(**{**good, "query": q, "q_weight": w, "value": good["value"].as_subclass(Sub),
                       "slots": torch.arange(10)[::2], "cos_sin": z(9, 128, dtype=BF16)[:, ::2]})
    query, _, value, _, cos_sin, q_weight = args[:6]
    slots = args[8]
    assert torch.equal(query, q) and query.is_contiguous() and torch.equal(q_weight, w) and q_weight.data_ptr() % 16 == 0
    assert type(value) is torch.Tensor and slots.tolist() == [0, 2, 4, 6, 8] and slots.is_contiguous() and cos_sin.is_contiguous()


def test_empty_batches(monkeypatch):
    monkeypatch.setattr(K, "gpu", lambda *t: 0)
    monkeypatch.setattr(K, "call", lambda name, *a: pytest.fail(f"{name} was called"))
    g = _good()
    none = {n: t[:0] for n, t in g["rope"].items() if n in ("query", "key", "value", "positions", "slots")}
    q, k = qf.qk_norm_rope(**{**g["rope"], **none})
    assert q.shape == (0, 4, 128) and k is None
    assert qf.qk_norm_rope(none["query"], none["key"], None, None)[1].shape == (0, 2, 128)
    qf.kv4_store(g["store"]["key"][:0], g["store"]["value"][:0], g["store"]["cache"], g["store"]["slots"][:0])
    assert [t.shape for t in qf.kv4_load(g["load"]["cache"], g["load"]["slots"][:0])] == [(0, 2, 64)] * 2
    a = {**g["attention"], "query": g["attention"]["query"][:0], "seq_lens": z(0, dtype=I32), "block_table": z(1, 1, dtype=I32)}
    assert qf.kv4_attention(**a).shape == (0, 4, 128)


def test_cache_shape():
    c = qf.kv4_cache(3, 48, 2, 64, device="cpu")
    assert c.shape == (3, 2, 3, 17 * 64) and c.dtype is U8 and not c.any()
    assert K.cache_sizes(c) == (2, 64, 48) and K.cache_sizes(torch.zeros(3, 5, 2, 3, 17 * 64, dtype=U8)[:, 1]) == (2, 64, 48)
    for bad in ((3, 24, 2, 64), (3, 0, 2, 64), (0, 16, 2, 64), (3, 16, 0, 64), (3, 16, 2, 96)):
        with pytest.raises(ValueError):
            qf.kv4_cache(*bad, device="cpu")


# ---- the references ----

def test_quantiser_reference():
    """Values by hand (the first largest magnitude, 7, takes the scale 2), and the definition's inequalities."""
    x = torch.tensor([[7.0, 6.9, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.26, -5.1, 0.0] + [0.0] * 20]).to(BF16)
    assert H.rounded(x)[0, :12].tolist() == [8.0, 6.0, 4.0, 4.0, 2.0, 2.0, 1.0, 1.0, 0.0, 0.0, -6.0, 0.0]
    x = torch.tensor([[6.9, 6.5, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.26, -5.1, 0.0] + [0.0] * 20]).to(BF16)
    assert H.rounded(x)[0, :12].tolist() == [6.0, 6.0, 4.0, 4.0, 2.0, 2.0, 1.0, 1.0, 0.0, -0.5, -6.0, 0.0]
    x[0, 5] = float("inf")
    assert H.rounded(x).isnan().all() and int(H.quantise(x)[1]) == 255
    x = (torch.randn(40, 96, generator=H.gen(0)) * torch.exp(3 * torch.randn(40, 1, generator=H.gen(1)))).to(BF16)
    y = H.rounded(x)
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    scale = torch.exp2(H.quantise(x)[1].double() - 127)[..., None]
    assert bool((top < 7 * scale).all()) and bool((top >= 3.5 * scale).all())
    assert bool(((x.double() - y).unflatten(-1, (-1, 32)).abs() <= scale).all())
    tiny = torch.full((1, 32), 2.0 ** -126).to(BF16)
    assert int(H.quantise(tiny)[1]) == 2 and H.rounded(tiny)[0, 0] == 2.0 ** -126


def test_writer_reference_covers_each_byte_once():
    for D in (64, 128, 256):
        c = torch.zeros(1, 1, 1, 17 * D, dtype=U8)
        x = torch.full((16, 1, D), 6.0).to(BF16)  # codes 7, scales 127
        H.write(c, torch.arange(16), x, -x)
        assert torch.equal(c[0, 0, 0, :8 * D], torch.full((8 * D,), 0x77, dtype=U8))
        assert torch.equal(c[0, 0, 0, 8 * D:16 * D], torch.full((8 * D,), 0xFF, dtype=U8))
        assert torch.equal(c[0, 0, 0, 16 * D:], torch.full((D,), 127, dtype=U8))


def test_attention_reference():
    """Against torch's own attention in 64 bits; a NaN that no row sees, or some rows, changes those that see it only."""
    g = H.gen(3)
    q, k, v = (torch.randn(n, h, 64, generator=g, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    got, slack = H.attention(q, [k[:6], k], [v[:6], v], [0, 2, 5], [6, 9], 0.2)
    for lo, hi, L in ((0, 2, 6), (2, 5, 9)):
        mask = torch.arange(L) <= (L - (hi - lo) + torch.arange(hi - lo))[:, None]
        want = torch.nn.functional.scaled_dot_product_attention(
            q[lo:hi].transpose(0, 1), k[:L].repeat_interleave(2, 1).transpose(0, 1), v[:L].repeat_interleave(2, 1).transpose(0, 1),
            attn_mask=mask, scale=0.2).transpose(0, 1)
        assert torch.allclose(got[lo:hi], want, atol=1e-12)
    v[8, 1, 3] = float("nan")
    bad, _ = H.attention(q, [k[:6], k], [v[:6], v], [0, 2, 5], [6, 9], 0.2)
    assert bad.isnan().nonzero().tolist() == [[4, 2, 3], [4, 3, 3]] and torch.equal(bad[:4], got[:4])
    none, _ = H.attention(q[:3], [k[:1]], [v[:1]], [0, 3], [1], 0.2)
    assert not none[:2].any() and none[2].any()


def test_table_reference():
    table = torch.tensor([[5, 0, 0], [6, 7, 0]], dtype=I32)
    r = H.tables(torch.tensor([3, 7]), torch.tensor([3, 2]), torch.tensor([1, 2]), table, [11, 12, 13, 14], 3, 4, 7)
    assert table.tolist() == [[5, 13, 0], [6, 7, 12]]
    assert r["slots"] == [23, 52, 53, 31, 48, -1, -1] and r["positions"] == [3, 4, 5, 7, 8, 0, 0]
    assert (r["held"], r["free_count"], r["cu_q"], r["seq_lens"]) == ([2, 3], [1], [0, 3, 5], [6, 9])


def test_kernels_use_no_scratch(tmp_path):
    """Every kernel of the library's code objects (one a source file) keeps its working set in registers and LDS."""
    llvm = "/opt/rocm/llvm/bin"
    if not (os.path.exists(K.LIB_PATH) and os.path.exists(os.path.join(llvm, "llvm-objdump"))):
        pytest.skip("built library or ROCm LLVM tools absent")
    copy = tmp_path / "lib.so"
    shutil.copy(K.LIB_PATH, copy)
    subprocess.run([os.path.join(llvm, "llvm-objdump"), "--offloading", str(copy)], cwd=tmp_path, check=True, capture_output=True)
    kernels = {}
    for f in os.listdir(tmp_path):
        if "gfx950" in f:
            notes = subprocess.run([os.path.join(llvm, "llvm-readelf"), "--notes", str(tmp_path / f)], check=True,
                                   capture_output=True, text=True).stdout
            kernels.update(zip(re.findall(r"\.name:\s+(\S+)", notes),
                               map(int, re.findall(r"\.private_segment_fixed_size:\s+(\d+)", notes))))
    assert not {n: s for n, s in kernels.items() if s}
    for name in ("step_tables_kernel", "qk_norm_rope_kernel", "kv4_load_kernel", "attn_split_kernel", "attn_tile_kernel"):
        assert any(name in n for n in kernels), name
