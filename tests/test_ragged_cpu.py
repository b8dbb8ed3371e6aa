"""The ragged operators' host side without a GPU: the rotary table against
the oracle's frequencies, page bookkeeping, and every refused argument of the
Python layer and the C entry points."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from cybel_b200 import _native
from cybel_b200.kv_cache import PagedKVCache
from cybel_b200.paged_attention import RaggedBatch, RopeTable, _row_stride
from oracle.ragged_ref import frequencies


@pytest.mark.parametrize("rot", [2, 20, 64, 128, 256])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
@pytest.mark.parametrize("scaling,kw", [("none", {}), ("linear", dict(factor=3.0)),
                                        ("llama3", dict(factor=8.0, original_context=8192)),
                                        ("yarn", dict(factor=32.0, original_context=4096)),
                                        ("yarn", dict(factor=2.0, original_context=100, low=0.5, high=7.0))])
def test_rope_table(rot, theta, scaling, kw):
    t = RopeTable(rot, theta, "half", scaling, device="cpu", **kw)
    f, mag = frequencies(rot, theta, scaling, kw.get("factor", 1.0), kw.get("original_context", 0), kw.get("low"),
                         kw.get("high"))
    # a few double roundings of theta^x, the blend and the division by 2 pi; the table's step is 2^-64 turns
    assert np.allclose(t.turns_host.astype(np.float64) / 2.0 ** 64, f / (2 * math.pi), rtol=2.0 ** -48, atol=2.0 ** -64)
    assert abs(t.mag - mag) <= 2.0 ** -51 * mag


def test_rope_table_refusals():
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=258), dict(rot_dim=8, layout="rows"),
                dict(rot_dim=8, scaling="ntk")):
        with pytest.raises(ValueError):
            RopeTable(**bad, device="cpu")
    for bad in (dict(theta=1.0), dict(theta=float("inf")), dict(scaling="linear", factor=0.5),
                dict(scaling="linear", factor=float("nan")), dict(scaling="llama3", factor=8.0),
                dict(scaling="yarn", factor=8.0, original_context=4096, low=4.0, high=4.0),
                dict(scaling="yarn", factor=8.0, original_context=4096, low=0.0)):
        with pytest.raises(_native.NativeError):
            RopeTable(8, **bad, device="cpu")
    L = _native.lib()
    m = ctypes.c_double()
    assert L.b200q_rope_table(8, 1e4, 0, 1.0, 1.0, 4.0, 0, None, ctypes.byref(m)) == -1


def test_batch_lengths():
    b = RaggedBatch([2, 0, 1], [5, 0, 9], device="cpu", max_kv=20)
    assert b.n_tokens == 3 and b.cu_q.tolist() == [0, 2, 2, 3] and b.kv_len.tolist() == [5, 0, 9]
    b.update([1, 1, 1], [6, 1, 20])
    assert b.cu_q.tolist() == [0, 1, 2, 3]
    for q, kv in (([1, 1], [6, 1]), ([3, 0, 0], [6, 1, 1]), ([2, 2, 0], [6, 2, 1]), ([1, 1, 1], [6, 1, 21])):
        with pytest.raises(ValueError):
            b.update(q, kv)
    assert b.kv_lens == [6, 1, 20] and b.kv_len.tolist() == [6, 1, 20]  # a refused update changes nothing
    for q, kv in (([], []), ([1], [0]), ([-1], [3]), ([1], [2 ** 30])):
        with pytest.raises(ValueError):
            RaggedBatch(q, kv, device="cpu")


def test_ensure_batch():
    c = PagedKVCache(2, 1, 64, batch=2, page_size=16, q8=False, n_slots=6, device="cpu", head_dim=64)
    c.ensure_batch(RaggedBatch([20, 0], [20, 30], device="cpu"))
    assert (c.table_host[:, 0, :2] >= 0).all() and (c.table_host[:, 1] == -1).all() and c.pages_in_use == 4
    c.ensure_batch(RaggedBatch([1, 1], [21, 31], device="cpu"))  # only the page of position 30
    assert (c.table_host[:, 1] >= 0).sum(axis=1).tolist() == [1, 1] and (c.table_host[:, 1, 1] >= 0).all()
    assert np.array_equal(c.table.numpy(), c.table_host)
    before = c.table_host.copy()
    with pytest.raises(MemoryError):
        c.ensure_batch(RaggedBatch([1, 1], [33, 32], device="cpu"))
    assert np.array_equal(c.table_host, before)
    with pytest.raises(ValueError):
        c.ensure_batch(RaggedBatch([1], [1], device="cpu"))
    with pytest.raises(ValueError):
        c.ensure_batch(RaggedBatch([1, 1], [1, 65], device="cpu"))


def test_head_sizes():
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 64, head_dim=96, device="cpu", q8=False)


def _calls():
    """(cache, batch, rope, q, k) on the CPU: every refusal comes before the
    device is asked for."""
    c = PagedKVCache(1, 2, 64, batch=2, page_size=16, q8=False, device="cpu")
    b = RaggedBatch([3, 1], [9, 4], device="cpu")
    return c, b, RopeTable(128, device="cpu"), torch.zeros(4, 4, 128), torch.zeros(4, 2, 128)


def test_attend_refusals():
    c, b, rope, q, k = _calls()
    bad = [
        dict(q=q.double()), dict(q=q[:3]), dict(q=q[..., :64]), dict(q=q[:, :3]), dict(q=q[0]),
        dict(q=q.transpose(0, 1)), dict(q=q[:, ::2]), dict(out=q.half()), dict(out=torch.zeros(4, 4, 64)),
        dict(slopes=torch.zeros(3)), dict(slopes=torch.zeros(4, dtype=torch.float16)),
        dict(prefix=torch.zeros(2)), dict(prefix=torch.zeros(3, dtype=torch.int32)),
        dict(batch=RaggedBatch([4], [4], device="cpu")), dict(batch=RaggedBatch([3, 1], [9, 65], device="cpu")),
    ]
    for kw in bad:
        kw = dict(q=q, batch=b) | kw
        with pytest.raises(ValueError):
            c.attend(0, kw.pop("q"), kw.pop("batch"), **kw)
    with pytest.raises(RuntimeError):  # well-formed, but on the host
        c.attend(0, q, b)


def test_append_refusals():
    c, b, rope, q, k = _calls()
    bad = [
        dict(k=k.double(), v=k.double()), dict(v=k.half()), dict(k=k[:3], v=k[:3]), dict(k=q, v=q),
        dict(v=torch.zeros(4, 6, 128)[:, :2]), dict(q=q.half()), dict(q=q[:3]), dict(q=q, q_out=q.half()),
        dict(q_out=q), dict(rope=RopeTable(256, device="cpu")), dict(batch=RaggedBatch([4], [4], device="cpu")),
    ]
    for kw in bad:
        kw = dict(k=k, v=k, batch=b, rope=rope) | kw
        with pytest.raises(ValueError):
            c.append(0, kw.pop("k"), kw.pop("v"), kw.pop("batch"), **kw)
    with pytest.raises(RuntimeError):
        c.append(0, k, k, b, rope=rope, q=q)
    with pytest.raises(ValueError):
        rope.rotate(torch.zeros(2, 1, 64), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        rope.rotate(q, torch.zeros(4))


def test_row_strides():
    assert _row_stride(torch.zeros(4, 6, 128)[:, :2], "x") == 768
    assert _row_stride(torch.zeros(1, 3, 64), "x") == 192
    assert _row_stride(torch.zeros(0, 3, 64), "x") == 192
    with pytest.raises(ValueError):
        _row_stride(torch.zeros(1, 3, 64).expand(4, 3, 64), "x")


def test_over_contiguous():
    k = torch.zeros(3, 2, 50, 64, dtype=torch.float16)
    c = PagedKVCache.over_contiguous(k, torch.zeros_like(k))
    assert c.table.tolist() == [[[0]], [[1]], [[2]]] and c.page_size == 50 and c.kv_mode == _native.KV_F16
    for a, b in ((k, k[:2]), (k.float(), k.float()), (k.transpose(1, 2), k.transpose(1, 2)), (k[..., :32], k[..., :32])):
        with pytest.raises(ValueError):
            PagedKVCache.over_contiguous(a, b)
