"""The tokens of a prompt, checked on the host before a kernel reads rows of
the embedding by them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cybel_b200.decode import prompt_ids


@pytest.mark.parametrize("tokens", [[3, 0, 511], (3, 0, 511), np.array([3, 0, 511]), torch.tensor([3, 0, 511]),
                                    torch.tensor([3, 0, 0, 0, 511, 0], dtype=torch.int32)[::2].clone()])
def test_rows_of_integers(tokens):
    ids = prompt_ids(tokens, 512)
    assert ids.dtype == torch.int32 and ids.tolist()[0] == 3 and ids.numel() == 3


@pytest.mark.parametrize("tokens", [[], torch.zeros(0, dtype=torch.int64), [512], [-1], [0, 2 ** 32], [2 ** 31],
                                    torch.tensor([2 ** 32]), torch.tensor([[1, 2, 3]]), torch.tensor(5),
                                    torch.tensor([1.0]), torch.tensor([True])])
def test_refusals(tokens):
    with pytest.raises(ValueError):
        prompt_ids(tokens, 512)


@pytest.mark.gpu
@pytest.mark.parametrize("qt", [12, 14, 8])
def test_a_row_outside_the_matrix_is_nan_and_reads_nothing(qt):
    from cybel_b200 import _native
    from cybel_b200 import quantize as Q
    from cybel_b200.quantized_matmul import DeviceMatrix

    n, k = 6, 512
    m = DeviceMatrix(qt, k, n, Q.quantize(np.random.default_rng(qt).standard_normal((n, k)).astype(np.float32), qt))
    rows = torch.tensor([5, 6, -1, 2 ** 31 - 1, -2 ** 31, 0], dtype=torch.int32, device="cuda")
    out = torch.zeros(6, k, device="cuda")
    assert _native.lib().b200q_dequantize_rows(qt, m.ptr, rows.data_ptr(), 6, out.data_ptr(), k, n,
                                               torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.isnan(out[1:5]).all() and torch.isfinite(out[[0, 5]]).all() and (out[[0, 5]] != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [[600], [-1], torch.tensor([[1, 2, 3]]), torch.tensor([1.0])])
def test_prefill_refuses_them(tokens):
    from cybel_b200.decode import DecodeStack
    from tests.test_prefill_gpu import _model

    stack = DecodeStack(_model(4, 2)[0], 64, *_model(4, 2)[1:])
    for t in (tokens, tokens.cuda()) if isinstance(tokens, torch.Tensor) else (tokens,):
        with pytest.raises(ValueError):
            stack.prefill(t)
    want = stack.prefill([3, 1, 4]).clone()
    wide = torch.tensor([3, 9, 1, 9, 4, 9], dtype=torch.int32, device="cuda")  # every other one, as it lies
    assert torch.equal(stack.prefill(wide[::2]), want)
