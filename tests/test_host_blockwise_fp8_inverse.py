"""The inverse of the 8-bit quantizer on more matrices than one launch takes (65535), as the quantizer takes them."""
import pytest
import torch

import alto_amd.mxfp4 as mx
from alto_amd.mxfp4 import _runtime as rt


@pytest.mark.parametrize("axis", [-1, -2])
@pytest.mark.parametrize("B", [1, 65535, 65536, 140000])
def test_matrices_of_a_launch(monkeypatch, B, axis):
    launches = []

    class Lib:
        @staticmethod
        def alto_mxfp4_fp8_dequantize(args, stream):
            a = args._obj
            launches.append((a.B, a.codes - codes.data_ptr(), a.scales - scales.data_ptr(), a.out, a.out_sb))
            assert 1 <= a.B < 65536
            return 0
    monkeypatch.setattr(rt, "require_gpu", lambda *tensors: None)
    monkeypatch.setattr(rt, "lib", Lib)
    monkeypatch.setattr(rt, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    codes = torch.zeros((B, 2, 32), dtype=torch.uint8).view(torch.float8_e4m3fn)[..., :3]
    scales = torch.ones((B, 2, 1) if axis == -1 else (B, 1, 3))
    out = mx.convert_from_blockwise_fp8(codes, scales, axis=axis)
    assert out.shape == (B, 2, 3)
    at = 0
    for n, code, scale, to, out_sb in launches:
        assert axis == -2 or code == 64 * at   # (codes that do not lie along the axis are copied)
        assert scale == 4 * scales.stride(0) * at and to == out.data_ptr() + 2 * 6 * at and out_sb == 6
        at += n
    assert at == B
