"""Sizes whose launches would not fit 32 bits are refused before any device work."""
import pytest

from test_attention_refusals import GOOD, _rc

T, N, Q, K = "tokens", "sequences", "query heads", "key heads"
AT = {"stade_hip_attention": {Q: 14, K: 15, T: 16, "keys": 17, N: 18}, "stade_hip_attention_b": {Q: 22, K: 23, T: 24, "keys": 25, N: 26}}


def _call(name, window=-1, sinks=0, **sizes):
    args, at = list(GOOD[name]), AT[name]
    named = dict(zip(("q", "k", "t", "tk", "n"), at.values()))
    for k, v in sizes.items():
        args[named[k]] = v
    args[named["n"] + 1], args[named["n"] + 2] = window, sinks
    width = 8 * args[named["q"]], 8 * args[named["k"]]
    for i, w in {"stade_hip_attention": ((2, 0), (5, 0), (7, 1), (9, 1)),
                 "stade_hip_attention_b": ((2, 0), (4, 0), (7, 0), (9, 0), (11, 1), (13, 1), (15, 1), (17, 1))}[name]:
        args[i] = width[w]
    return _rc(name, *args)


@pytest.mark.parametrize("name", AT)
def test_many_blocks(name):
    # 2^20 sequences and 8 key heads; 2^24 rows of 128 key heads
    for sizes in (dict(q=8, k=8, n=1 << 20, t=1 << 20, tk=1 << 20), dict(q=128, k=128, t=1 << 24, tk=1 << 24)):
        rc, msg = _call(name, **sizes)
        assert rc == -3 and "blocks of 128" in msg and name in msg, (rc, msg)


def test_many_keys():
    rc, msg = _call("stade_hip_attention_b", q=128, k=128, t=4, tk=1 << 24)
    assert rc == -3 and "blocks of 128 keys" in msg, (rc, msg)


def test_many_sequences_with_sinks():
    # (64 sinks of 8 values: four blocks a sequence and head)
    rc, msg = _call("stade_hip_attention_b", q=3, k=3, n=1 << 20, t=1 << 20, tk=1 << 20, window=10, sinks=64)
    assert rc == -3 and "with sinks" in msg, (rc, msg)


def test_no_query_heads():
    rc, msg = _call("stade_hip_attention_b", q=0, k=1)
    assert rc == -1 and "i_q is zero" in msg, (rc, msg)
    assert _call("stade_hip_attention_b", q=0, k=0)[0] == 0 and _call("stade_hip_attention", q=0, k=1)[0] == 0
