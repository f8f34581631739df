"""bf16 pages that qk_norm_rope writes: heads that share memory are refused, whatever order the dimensions stand in."""
import pytest
import torch

import qwen_fastpath as qf
from qwen_fastpath import _kv4_lib as K

BF16, D = torch.bfloat16, 128


def _arguments(pages, device="cpu"):
    x = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device=device)  # noqa: E731
    return dict(query=x(5, 4, D), key=x(5, 2, D), positions=None, cos_sin=None, value=x(5, 2, D), slots=torch.arange(5, device=device),
                cache=pages)


def _shared(device="cpu"):
    z = lambda *s: torch.zeros(*s, dtype=BF16, device=device)  # noqa: E731
    good = z(3, 16, 2, D)
    for bad in (z(1, 16, 2, D).expand(3, 16, 2, D), z(3, 1, 2, D).expand(3, 16, 2, D), z(3, 16, 1, D).expand(3, 16, 2, D),
                z(64 * 256).as_strided((3, 16, 2, D), (4096, 256, 64, 1)), z(80 * 256).as_strided((3, 16, 2, D), (3840, 256, 128, 1))):
        yield good, bad
        yield bad, good


def _apart(device="cpu"):
    z = lambda *s: torch.zeros(*s, dtype=BF16, device=device)  # noqa: E731
    both = z(3, 2, 16, 2, D)
    yield both[:, 0], both[:, 1]
    yield tuple(z(2, 3, 2, 16, D).transpose(2, 3))  # heads before positions
    yield tuple(z(3, 16, 2, 2 * D)[..., i * D:(i + 1) * D] for i in (0, 1))
    yield tuple(z(2, 16, 3, 2, D).transpose(1, 2))  # blocks side by side
    yield tuple(z(1, 16, 2, D).as_strided((1, 16, 2, D), (0, 256, 128, 1)) for _ in range(2))  # one block


def test_on_the_host(monkeypatch):
    monkeypatch.setattr(K, "gpu", lambda *t: 0)
    called = []
    monkeypatch.setattr(K, "call", lambda name, *a: called.append(name) or (None, None))
    for pages in _shared():
        with pytest.raises(ValueError, match="share memory"):
            qf.qk_norm_rope(**_arguments(pages))
    assert not called
    for n, pages in enumerate(_apart(), 1):
        qf.qk_norm_rope(**_arguments(pages))
        assert len(called) == n


@pytest.mark.gpu
def test_on_the_gpu():
    for pages in _shared("cuda"):
        with pytest.raises(ValueError, match="share memory"):
            qf.qk_norm_rope(**_arguments(pages, "cuda"))
    for pages in _apart("cuda"):
        a = _arguments(pages, "cuda")
        a["key"] = torch.randn(5, 2, D, device="cuda").to(BF16)
        a["value"] = torch.randn(5, 2, D, device="cuda").to(BF16)
        qf.qk_norm_rope(**a)
        for page, want in zip(pages, (a["key"], a["value"])):
            assert torch.equal(page[0, :5], want) and not page[0, 5:].any() and not page[1:].any()
