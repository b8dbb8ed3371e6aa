"""``DecodeStack.prefill`` (the prompt in passes of several rows over the paged
append and the paged attention) against the float64 restatement stepping the
same tokens one at a time (oracle/decode_ref.py): the last row's logits and
those of the decode step after it within max |d| / max |ref| <= 2e-3, the
bound that the stack's other multi-row pass (verify) is held to, for every
cache, for one pass and for passes that end inside a page and a tile, and
for a prompt continued where another ended.
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return float(np.max(np.abs(np.asarray(a, np.float64) - b)) / max(np.max(np.abs(b)), 1e-30))


def _model(heads, kv_heads, seed=4):
    from cybel_b200.decode import StackShape, random_layer, random_rows
    from cybel_b200.formats import Q4_K, Q6_K

    shape = StackShape(layers=2, hidden=128 * heads, heads=heads, kv_heads=kv_heads, ffn=768, vocab=512)
    rng = np.random.default_rng(seed)
    layers = [random_layer(shape, rng) for _ in range(shape.layers)]
    embed = random_rows(Q4_K, shape.vocab, shape.hidden, rng, std=1.0)
    head = random_rows(Q6_K, shape.vocab, shape.hidden, rng)
    out_norm = (1 + 0.1 * rng.standard_normal(shape.hidden)).astype(np.float32)
    return shape, layers, embed, head, out_norm


@pytest.mark.parametrize("kv", ["contiguous", "paged", "q8"])
@pytest.mark.parametrize("heads,kv_heads,n,chunk", [(4, 2, 1, 512), (4, 2, 83, 512), (4, 4, 83, 32), (4, 1, 60, 7)])
def test_prompt_then_step(heads, kv_heads, n, chunk, kv):
    import torch

    from cybel_b200 import _native
    from cybel_b200.decode import DecodeStack
    from cybel_b200.repack_policy import RepackPolicy
    from oracle.decode_ref import DecodeRef

    shape, layers, embed, head, out_norm = _model(heads, kv_heads)
    dev = DecodeStack(shape, 100, layers, embed, head, out_norm, repack=RepackPolicy.canonical(), kv=kv, page_size=12)
    ref = DecodeRef(shape, layers, embed, head, out_norm, 100, kv_q8=kv == "q8")
    toks = [int(t) for t in np.random.default_rng(n).integers(0, shape.vocab, n + 1)]
    got = dev.prefill(toks[:n], chunk=chunk).cpu().numpy()
    for pos, t in enumerate(toks[:n]):
        want = ref.step(t, pos)
    assert _rel(got, want) <= 2e-3
    dev.set_token(toks[n])
    dev.step(n)
    assert _rel(dev.logits.cpu().numpy(), ref.step(toks[n], n)) <= 2e-3
    more = toks[:9]  # a second prompt, already on the device, behind the first
    got = dev.prefill(torch.tensor(more, device="cuda"), pos0=n + 1, chunk=4).cpu().numpy()
    for i, t in enumerate(more):
        want = ref.step(t, n + 1 + i)
    assert _rel(got, want) <= 2e-3
    _native.check_device(0)
    for bad in (dict(tokens=[]), dict(tokens=[1] * 101), dict(tokens=[1], pos0=-1), dict(tokens=[1], chunk=0)):
        with pytest.raises(ValueError):
            dev.prefill(**bad)
