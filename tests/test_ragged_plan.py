"""Which kernels a ragged attention launches (b200q_attention_paged_plan), on
the host: the query's refusals, and that batches meant for the many-row kernel
reach it."""

from __future__ import annotations

import ctypes
import itertools

import pytest

from cybel_b200 import _native

SMS = 148


def plan(dtype, q_lens, kv_lens, heads, kv, window=0, prefix=0, q8=False, sms=SMS):
    """(most rows of a sequence that the few-row kernel takes, its CTAs per
    block, blocks of the many-row kernel, its CTAs per block)"""
    out = (ctypes.c_longlong * 4)()
    rc = _native.lib().b200q_attention_paged_plan(
        _native.F32 if dtype == "fp32" else _native.F16, sum(q_lens), len(q_lens), max(q_lens), max(kv_lens), heads, kv,
        window, prefix, _native.KV_Q8 if q8 else _native.KV_F16, sms, out, 4)
    assert rc == 0
    return tuple(out)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("heads,kv", [(8, 8), (8, 2), (32, 8), (40, 1)])
def test_plan(heads, kv, q8, dtype):
    g = heads // kv
    for q, n, batch in itertools.product((1, 8, 33, 500, 5000), (5000, 120_000), (1, 7, 64)):
        few, c, blocks, ct = plan(dtype, [q] * batch, [n] * batch, heads, kv, q8=q8)
        assert few >= 32 and 1 <= c <= 16
        assert (blocks > 0) == (q * g > few) and (1 <= ct <= 8 if blocks else ct == 0)
        # every sequence's rows fit in the blocks that are launched for them
        assert not blocks or blocks >= batch * kv * ((q * g + 255) // 256)
    assert plan(dtype, [1], [1], heads, kv, q8=q8)[1] == 1  # one position is not split


def test_plan_refusals():
    L = _native.lib()
    out = (ctypes.c_longlong * 4)()
    good = dict(dtype=1, n=5, batch=2, mq=3, mk=50, h=4, kv=2, w=0, pre=0, mode=0, sms=SMS, out=out, len=4)
    assert L.b200q_attention_paged_plan(*good.values()) == 0
    for kw, want in ((dict(dtype=2), -1), (dict(n=0), -1), (dict(batch=0), -1), (dict(mq=0), -1), (dict(mk=-1), -1),
                     (dict(h=0), -1), (dict(kv=0), -1), (dict(w=-1), -1), (dict(mode=2), -1), (dict(sms=0), -1),
                     (dict(out=None), -1), (dict(len=3), -1), (dict(h=5), -3), (dict(n=2 ** 30, h=8), -3)):
        assert L.b200q_attention_paged_plan(*(good | kw).values()) == want, kw


def test_the_smoke_run_reaches_both_attention_kernels():
    import __graft_entry__ as entry

    few, _, blocks, _ = entry.ragged_plan(SMS)
    g = entry.RAGGED["heads"] // entry.RAGGED["kv"]
    assert blocks > 0 and g * min(entry.RAGGED["q_lens"]) <= few < g * max(entry.RAGGED["q_lens"])
