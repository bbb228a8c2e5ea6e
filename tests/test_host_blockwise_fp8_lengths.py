"""The longest reductions of products of 8-bit operands, without a GPU: 2^22 - 16 codes a row, also where the quantizer's pitch (multiples of 128) is 2^22, which a product does not read."""
import pytest
import torch

import alto_amd.mxfp4 as mx
from alto_amd.mxfp4 import _runtime as rt
from alto_amd.mxfp4 import blockwise_fp8 as F

LONGEST = 2 ** 22 - 16


@pytest.mark.parametrize("K", [2 ** 22 - 128, 2 ** 22 - 127, 2 ** 22 - 100, LONGEST])
@pytest.mark.parametrize("rows", [(2,), (2, 3)])
def test_codes_at_a_pitch_of_2_22_are_copied_to_one_that_is_read(K, rows):
    pitch = -(-K // 128) * 128   # the quantizer's
    t = torch.zeros((*rows, pitch), dtype=torch.uint8)[..., :K]
    t[..., 0], t[..., K - 1] = 1, torch.arange(2, 2 + t[..., 0].numel()).view(rows)
    got = F._operand(t.view(torch.float8_e4m3fn))
    assert got.shape == t.shape and torch.equal(got.view(torch.uint8), t)
    assert got.stride(-1) == 1 and got.stride(-2) % 16 == 0 and K <= got.stride(-2) < 2 ** 22
    assert got.untyped_storage().nbytes() >= (got.numel() // K - 1) * got.stride(-2) + -(-K // 16) * 16
    assert (got.data_ptr() == t.data_ptr()) == (pitch < 2 ** 22)


@pytest.fixture
def stand_in(monkeypatch):
    """The layers on the CPU: nothing is launched, quantizers and products leave what is allocated."""
    class Host:
        def __getattr__(self, name):
            return lambda *args: None

    class Lib:
        alto_mxfp4_fp8_token_blocks = staticmethod(lambda M, groups: (M + 127 * (groups + 2)) // 128)

        def __getattr__(self, name):
            return lambda *args: 0
    monkeypatch.setattr(rt, "require_gpu", lambda *tensors: None)
    monkeypatch.setattr(rt, "host", Host)
    monkeypatch.setattr(rt, "lib", Lib)
    monkeypatch.setattr(rt, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)


def test_steps_of_more_rows_are_refused_ahead_of_the_forward(stand_in):
    """(they ran their forward and failed in a product of the backward)"""
    w, wide = torch.zeros(1, 1).bfloat16().requires_grad_(), torch.zeros(LONGEST + 1, 1).bfloat16()
    rows = lambda n: torch.zeros(1, 1).bfloat16().expand(n, 1)  # noqa: E731
    assert mx.blockwise_fp8_linear(rows(LONGEST), w).requires_grad
    with pytest.raises(AssertionError, match="4194289 rows"):
        mx.blockwise_fp8_linear(rows(LONGEST + 1), w)
    with torch.no_grad():
        assert mx.blockwise_fp8_linear(rows(LONGEST + 1), w).shape == (LONGEST + 1, 1)
    x = rows(3).clone().requires_grad_()   # the input's gradient sums over the columns
    with pytest.raises(AssertionError, match="4194289 columns"):
        mx.blockwise_fp8_linear(x, wide)
    assert mx.blockwise_fp8_linear(x, wide[:LONGEST]).requires_grad
    assert mx.blockwise_fp8_linear(rows(LONGEST + 1), w.detach().clone()).shape == (LONGEST + 1, 1)   # (no gradient of either is asked for)


@pytest.mark.parametrize("E,most", [(1, 2 ** 22 - 1 - 127 * 3), (30, 2 ** 22 - 1 - 127 * 32)])
def test_grouped_steps_of_more_rows_are_refused_ahead_of_the_forward(stand_in, E, most):
    w, offsets = torch.zeros(E, 1, 1).bfloat16().requires_grad_(), torch.zeros(E + 1, dtype=torch.int32)
    rows = lambda n: torch.zeros(1, 1).bfloat16().expand(n, 1)  # noqa: E731
    assert mx.blockwise_fp8_grouped_linear(rows(most), w, offsets).requires_grad
    with pytest.raises(AssertionError, match=f"{most + 1} rows"):
        mx.blockwise_fp8_grouped_linear(rows(most + 1), w, offsets)
    assert mx.blockwise_fp8_grouped_linear(rows(most + 1).requires_grad_(), w.detach(), offsets).requires_grad   # (no weight gradient)
    with torch.no_grad():
        assert mx.blockwise_fp8_grouped_linear(rows(most + 1), w, offsets).shape == (most + 1, 1)
    x = rows(3).clone().requires_grad_()
    with pytest.raises(AssertionError, match="4194289 columns"):
        mx.blockwise_fp8_grouped_linear(x, torch.zeros(E, 1, 1).bfloat16().expand(E, LONGEST + 1, 1), offsets)


def test_many_groups_have_no_weight_gradients(stand_in):
    w, offsets, x = torch.zeros(1, 1, 1).bfloat16().expand(33024, 1, 1).requires_grad_(), torch.zeros(33025, dtype=torch.int32), torch.zeros(2, 1).bfloat16()
    with pytest.raises(AssertionError, match="33024 groups"):
        mx.blockwise_fp8_grouped_linear(x, w, offsets)
    with torch.no_grad():
        assert mx.blockwise_fp8_grouped_linear(x, w, offsets).shape == (2, 1)


def test_empty_gradients_of_long_reductions(stand_in):
    x, w = torch.zeros(LONGEST + 1, 0).bfloat16(), torch.zeros(2, 0).bfloat16().requires_grad_()
    assert torch.autograd.grad(mx.blockwise_fp8_linear(x, w).sum(), w)[0].shape == (2, 0)
    x, w = torch.zeros(0, 1).bfloat16().requires_grad_(), torch.zeros(1, 1).bfloat16().expand(LONGEST + 1, 1)
    assert torch.autograd.grad(mx.blockwise_fp8_linear(x, w).sum(), x)[0].shape == (0, 1)
