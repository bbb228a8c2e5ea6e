"""The inverse of the 8-bit quantizer on more matrices than one launch takes."""
import pytest
import torch

import alto_amd.mxfp4 as mx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("axis,is_2d", [(-1, False), (-2, False), (-1, True), (-2, True)])
def test_many_matrices(axis, is_2d):
    B = 140000
    x = torch.randint(-7, 8, (B, 3, 5), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    x[:, 0, :] = x[:, :, 0] = 7   # (whole numbers on a scale that is a power of two: they come back as they are)
    x *= torch.exp2((torch.arange(B, device="cuda") % 11).float()).to(torch.bfloat16)[:, None, None]
    q, s = mx.convert_to_blockwise_fp8(x, axis=axis, is_2d_block=is_2d)
    for out in (torch.bfloat16, torch.float32):
        got = mx.convert_from_blockwise_fp8(q, s, axis=axis, is_2d_block=is_2d, output_dtype=out)
        assert got.dtype == out and torch.equal(got, x.to(out))
