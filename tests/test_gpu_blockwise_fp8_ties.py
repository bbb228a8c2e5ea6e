"""Codes of bf16 quotients: each of the 128 significands over each of the 128, at eight distances, where ties between two codes abound."""
import pytest
import torch

import alto_amd.mxfp4 as mx
from oracle import blockwise_fp8 as O

pytestmark = pytest.mark.gpu


def pairs():
    """[8 * 128, 256]: row 128 e + i has blocks with the largest magnitude 128 + i, and in its two blocks all of 128 .. 255 times 2^-(e+1), every other one negative."""
    sig = torch.arange(128, 256).double()
    x = torch.empty(8, 128, 2, 128, dtype=torch.float64)
    sign = torch.where(torch.arange(128) % 2 == 0, 1.0, -1.0).double()
    x[...] = (sig * sign) * torch.exp2(-torch.arange(1, 9).double()).view(8, 1, 1, 1)
    x[:, :, 0, 0], x[:, :, 1, 127] = sig, sig   # (what the first block leaves out the second one holds)
    return x.view(8 * 128, 256)


def ties(quotient, dtype):
    """How many quotients lie halfway between two codes."""
    bits, low = O._GRID[dtype]
    step = torch.exp2(((torch.frexp(quotient)[1].long() - 1).clamp(min=low) - bits).double())
    return int(((quotient / step) % 1 == 0.5).sum())


@pytest.mark.parametrize("code", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_every_significand_over_every_block_maximum(code):
    x = pairs().to(torch.bfloat16)
    assert torch.equal(x.double(), pairs())
    exp, scales, quotient = O.quantize(x, (1,), code)
    assert ties(quotient, code) == {torch.float8_e4m3fn: 1296, torch.float8_e5m2: 712}[code]   # (of the data, counted in 64 bits)
    q, s = mx.convert_to_blockwise_fp8(x.cuda(), dtype=code)
    assert torch.equal(q.cpu().double(), exp) and torch.equal(s.cpu(), scales)
    turned, scales_t = mx.convert_to_blockwise_fp8(x.t().contiguous().cuda(), axis=-2, dtype=code)
    assert torch.equal(turned.t().cpu().double(), exp) and torch.equal(scales_t.t().cpu(), scales)
    wide = x.float().cuda()   # the same numbers in fp32
    q, s = mx.convert_to_blockwise_fp8(wide, dtype=code)
    assert torch.equal(q.cpu().double(), exp) and torch.equal(s.cpu(), scales)
    # blocks of 128 x 128 of one maximum each
    tall = x.view(8, 128, 256).transpose(0, 1).reshape(128, 8, 256).repeat_interleave(16, dim=1).flatten(0, 1)   # [128 * 128, 256]
    exp, scales, _ = O.quantize(tall, (0, 1), code)
    q, s, qt, _ = mx.quantize_blockwise_fp8_rowcol(tall.cuda(), is_2d_block=True, dtype=code)
    assert torch.equal(q.cpu().double(), exp) and torch.equal(qt.cpu().double(), exp) and torch.equal(s.cpu(), scales)
