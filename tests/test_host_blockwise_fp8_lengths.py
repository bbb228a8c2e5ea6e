"""The longest reductions of products of 8-bit operands, without a GPU: 2^22 - 16 codes a row, also where the quantizer's pitch (multiples of 128) is 2^22, which a product does not read."""
import pytest
import torch

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
