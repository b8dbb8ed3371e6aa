"""``DecodeStack.prefill`` of a prompt longer than its default pass, under the
canonical and the default weight layouts: the first pass's attention is the
many-row kernel's, the rest's the few-row kernel's. Bounds and reference are
those of test_prefill_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_prefill_gpu import _model, _rel

pytestmark = pytest.mark.gpu

N = 700


@pytest.fixture(scope="module", params=["contiguous", "paged", "q8"])
def reference(request):
    from oracle.decode_ref import DecodeRef

    model = _model(8, 2)
    ref = DecodeRef(*model, N + 8, kv_q8=request.param == "q8")
    toks = [int(t) for t in np.random.default_rng(5).integers(0, model[0].vocab, N + 1)]
    for pos, t in enumerate(toks[:N]):
        want = ref.step(t, pos)
    return request.param, model, toks, want, ref.step(toks[N], N)


@pytest.mark.parametrize("canonical", [True, False])
def test_a_prompt_of_two_default_passes(reference, canonical):
    import torch

    from cybel_b200 import _native
    from cybel_b200.decode import DecodeStack
    from cybel_b200.repack_policy import RepackPolicy
    from tests.test_ragged_plan import plan

    kv, model, toks, want, after = reference
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert plan("fp32", [512], [512], 8, 2, q8=kv == "q8", sms=sms)[2]
    assert not plan("fp32", [N - 512], [N], 8, 2, q8=kv == "q8", sms=sms)[2]
    dev = DecodeStack(model[0], N + 8, *model[1:], repack=RepackPolicy.canonical() if canonical else None, kv=kv, page_size=48)
    got = dev.prefill(toks[:N]).cpu().numpy()
    assert _rel(got, want) <= 2e-3
    dev.set_token(toks[N])
    dev.step(N)
    assert _rel(dev.logits.cpu().numpy(), after) <= 2e-3
    _native.check_device(0)
