"""Wrapped weights of the 8-bit layers, their arguments by position and by name."""
import pytest
import torch

import alto_amd.mxfp4 as mx
from tests.test_gpu_blockwise_fp8_modules import CONFIG, data

pytestmark = pytest.mark.gpu


def test_arguments_by_position_and_by_name():
    w, x, b, e = data((256, 136), 1, 0.05), data((96, 256), 2), data((136,), 3), data((3, 256, 136), 4, 0.05)
    offs = torch.tensor([30, 30, 90], dtype=torch.int32, device="cuda")
    wrap = lambda t: mx.BlockwiseFP8TrainingWeightWrapperTensor(t, CONFIG)  # noqa: E731
    exp = mx.blockwise_fp8_linear(x, w.t())
    for y in (torch.mm(x, mat2=wrap(w)), torch.matmul(x, other=wrap(w)), torch.nn.functional.linear(input=x, weight=wrap(w.t().contiguous())), torch.mm(x, wrap(w), out_dtype=torch.bfloat16)):
        assert torch.equal(y, exp)
    for y in (torch.addmm(b, x, mat2=wrap(w)), torch.addmm(input=b, mat1=x, mat2=wrap(w), beta=1), torch.nn.functional.linear(x, weight=wrap(w.t().contiguous()), bias=b)):
        assert torch.equal(y, exp + b)
    exp = mx.blockwise_fp8_grouped_linear(x, e, torch.tensor([0, 30, 30, 90], dtype=torch.int32, device="cuda"), trans_weights=False)
    for y in (torch._grouped_mm(x, wrap(e), offs), torch._grouped_mm(x, mat2=wrap(e), offs=offs), torch._grouped_mm(x, wrap(e), offs, None, torch.bfloat16), torch.nn.functional.grouped_mm(x, wrap(e), offs=offs)):
        assert torch.equal(y, exp)
    with pytest.raises(AssertionError, match="out_dtype"):
        torch._grouped_mm(x, wrap(e), offs=offs, out_dtype=torch.float32)
    out = torch.zeros_like(y)
    with pytest.raises(AssertionError, match="out of mm"):
        torch.mm(x, wrap(w), out=out)
