"""The device status keeps a bit per kind, whichever kernel sets its own last:
a wait that ran out (a peer's flag that nothing sets, 1 ms limit) and page
table entries that name no page, one after the other in both orders."""

from __future__ import annotations

import ctypes

import pytest

pytestmark = pytest.mark.gpu

TIMEOUT, BAD_PAGE = 1, 2


def _time_out():
    import torch

    from cybel_b200 import _native

    L = _native.lib()
    rows, n_local, world = 2, 256, 2
    data = rows * world * n_local * 4
    own, peer = (torch.zeros(data + 256, dtype=torch.uint8, device="cuda") for _ in range(2))
    counters = torch.zeros(16, dtype=torch.int32, device="cuda")
    local = torch.ones(rows * n_local, device="cuda")
    bases = (ctypes.c_void_p * 2)(own.data_ptr(), peer.data_ptr())
    prev = L.b200q_set_peer_wait_ns(1_000_000)
    try:
        assert L.b200q_allgather_peer(local.data_ptr(), rows, n_local, bases, 0, data, 0, world, counters.data_ptr(), 0, None,
                                      0, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
    finally:
        L.b200q_set_peer_wait_ns(prev)


def _cache():
    from cybel_b200.kv_cache import PagedKVCache

    return PagedKVCache(1, 1, 32, batch=1, page_size=16, q8=False)  # no page assigned


def _decode():
    import torch

    c = _cache()
    x = torch.ones(1, 1, 128, device="cuda")
    out = torch.empty_like(x)
    c.attention(0, x.data_ptr(), x.data_ptr(), x.data_ptr(), 3, 1, 10000.0, out.data_ptr(), None, 0,
                torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()


def _append():
    import torch

    from cybel_b200.paged_attention import RaggedBatch

    x = torch.ones(1, 1, 128, device="cuda")
    _cache().append(0, x, x, RaggedBatch([1], [4]))
    torch.cuda.synchronize()


@pytest.mark.parametrize("pages", [_decode, _append])
@pytest.mark.parametrize("timeout_first", [True, False])
def test_one_kind_does_not_hide_the_other(timeout_first, pages):
    import torch

    from cybel_b200 import _native

    L = _native.lib()
    dev = torch.cuda.current_device()
    torch.cuda.synchronize()
    _native.check_device(dev)
    for f in (_time_out, pages) if timeout_first else (pages, _time_out):
        f()
    assert L.b200q_device_status(dev) == TIMEOUT | BAD_PAGE
    assert L.b200q_device_status(dev) == 0  # cleared by the read
    pages()
    _time_out()
    with pytest.raises(_native.NativeError, match="page"):  # a timeout's error that names the page, too
        _native.check_device(dev)
    _native.check_device(dev)
    pages()
    assert L.b200q_device_status(dev) == BAD_PAGE
    _time_out()
    assert L.b200q_device_status(dev) == TIMEOUT
