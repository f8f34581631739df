"""The limits that include/qf_kv4.h states for the attention, met and passed by one, without a GPU."""
import re

import pytest

import test_kv4_host as host
from test_kv4_launches import _record

MOST = int(re.search(r"#define QF_KV4_MAX_REQS (\d+)", open(host.HEADER).read()).group(1))


@pytest.mark.parametrize("kw", [
    dict(num_reqs=MOST + 1, num_tokens=1 << 20), dict(num_kv_heads=MOST + 1, num_heads=MOST + 1, cache_stride=(MOST + 1) * 17 * 128),
    dict(q_len=1 << 28, num_tokens=1 << 28, cu_q=host.P), dict(max_blocks=(2 ** 31 - 64) // 16 + 1)])
def test_past_a_limit(kw):
    assert host._attention(**kw)[0] == host.UNSUPPORTED


def test_at_a_limit():
    """Everything a call launches, recorded: the largest counts of requests, of kv heads and of positions."""
    most = (2 ** 31 - 64) // 16
    for rc, _, made in _record([("attention", MOST, 1, 2, 1, 64, 0, 8), ("attention", 1, 1, MOST, MOST, 64, 0, 8),
                                ("attention", 1, 2, 8, 1, 64, 0, most), ("attention", 1, 70, 8, 1, 64, 1, most)]):
        assert rc == host.OK and made
