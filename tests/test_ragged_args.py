"""What the Python layer of the ragged operators hands to the C entry points,
without a GPU: numbers past 32 bits, which ctypes would cut off silently."""

from __future__ import annotations

import pytest
import torch

from cybel_b200 import _native, paged_attention
from cybel_b200.kv_cache import PagedKVCache
from cybel_b200.paged_attention import RaggedBatch, RopeTable


@pytest.fixture
def calls(monkeypatch):
    """(function name, arguments as ctypes would pass them) of each call."""
    got = []

    def call(index, fn, what, *args):
        got.append([t(a).value if t.__name__.startswith(("c_int", "c_long")) else a
                    for t, a in zip(fn.argtypes, args)])

    monkeypatch.setattr(paged_attention, "_call", call)
    return got


def _cache():
    return PagedKVCache(1, 2, 64, batch=2, page_size=16, q8=False, device="cpu")


@pytest.mark.parametrize("window,want", [(0, 0), (5, 5), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1),
                                         (2 ** 32, 2 ** 31 - 1), (2 ** 32 + 5, 2 ** 31 - 1), (2 ** 63 - 1, 2 ** 31 - 1)])
def test_a_window_past_32_bits_stays_one(calls, window, want):
    _cache().attend(0, torch.zeros(4, 4, 128), RaggedBatch([3, 1], [9, 4], device="cpu"), window=window)
    assert calls[0][17] == want


def test_a_negative_window_is_refused():
    with pytest.raises(ValueError):
        _cache().attend(0, torch.zeros(4, 4, 128), RaggedBatch([3, 1], [9, 4], device="cpu"), window=-2 ** 32)


def test_a_bound_past_the_batch_is_the_batch(calls):
    """max_q beyond the rows the batch holds says no more than they do."""
    b = RaggedBatch([3, 1], [9, 4], device="cpu", max_q=2 ** 32 + 1)
    assert b.max_q == 4
    b.update([0, 4], [0, 9 - 1])
    _cache().attend(0, torch.zeros(4, 4, 128), b)
    assert calls[0][6] == 4


def test_rope_context_past_32_bits_is_refused():
    with pytest.raises((ValueError, _native.NativeError)):
        RopeTable(128, scaling="llama3", factor=8.0, original_context=2 ** 32 + 8192, device="cpu")
    with pytest.raises((ValueError, _native.NativeError)):
        RopeTable(2 ** 32 + 128, device="cpu")


def test_a_view_of_caches_on_two_devices_is_refused():
    k = torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        PagedKVCache.over_contiguous(k, torch.zeros_like(k, device="meta"))
    with pytest.raises(ValueError):  # no position to hold
        PagedKVCache.over_contiguous(k[:, :, :0], k[:, :, :0])
