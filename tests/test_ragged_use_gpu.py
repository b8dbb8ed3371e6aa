"""The ragged operators as a program mixes them with the rest of the
framework: the order of their launches, the calls at the ends of their ranges,
and both attention kernels on the inputs that can tell them apart.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _clean():
    import torch

    from cybel_b200 import _native

    torch.cuda.synchronize()
    _native.check_device(0)


@pytest.mark.parametrize("between", [False, True])
@pytest.mark.parametrize("q8", [False, True])
def test_one_position_attention_right_behind_an_append(q8, between):
    """PagedKVCache.attention, which loads cached rows before it waits for
    the kernel ahead, sees every row of an append queued just before it, with
    and without an attend in between: a captured graph's outputs are those of
    the same calls with the host waiting after each. (A row read too early
    shows: the pages hold NaN until the append.)"""
    import torch

    from cybel_b200.kv_cache import PagedKVCache
    from cybel_b200.paged_attention import RaggedBatch, RopeTable

    heads, kv, hd, seqs, n = 8, 2, 128, 4, 2000
    c = PagedKVCache(1, kv, n + 1, batch=seqs, page_size=64, q8=q8)
    c.ensure(0, n)
    batch = RaggedBatch([n] * seqs, [n] * seqs)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    rand = (lambda *s: torch.randn(*s, hd, generator=g, device="cuda"))
    k, v, q = rand(seqs * n, kv), rand(seqs * n, kv), rand(seqs * n, heads)
    q1, k1, v1 = rand(seqs, heads), rand(seqs, kv), rand(seqs, kv)
    out, seen = torch.empty_like(q1), torch.empty_like(q)
    rope = RopeTable(hd)

    def wipe():
        for t in (c.ks, c.vs) if q8 else (c.k, c.v):
            t.fill_(float("nan"))
        out.zero_()

    def body(wait=(lambda: None)):
        c.append(0, k, v, batch, rope=rope)
        wait()
        if between:
            c.attend(0, q, batch, out=seen)
            wait()
        c.attention(0, q1.data_ptr(), k1.data_ptr(), v1.data_ptr(), n, heads, 10000.0, out.data_ptr(), None, 0,
                    torch.cuda.current_stream().cuda_stream)

    wipe()
    side = torch.cuda.Stream()  # (the attention's scratch belongs to its stream and has to exist before a capture)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(torch.cuda.synchronize)
    _clean()
    want = out.clone()
    assert torch.isfinite(want).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        body()
    for _ in range(5):
        wipe()
        graph.replay()
        _clean()
        assert torch.equal(out, want)
