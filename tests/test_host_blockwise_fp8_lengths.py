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


PART = 2 ** 22 - 128


def test_longer_reductions_are_taken_in_parts(stand_in, monkeypatch):
    """Each part ends with a whole block, the last one with the reduction; what a native product would be handed is recorded."""
    made, whole = [], F._gemm

    def gemm(a, a_s, b, b_s, a_2d, b_2d, trans_a, trans_b, out):
        if (a.shape[0] if trans_a else a.shape[1]) > LONGEST:
            return whole(a, a_s, b, b_s, a_2d, b_2d, trans_a, trans_b, out)
        made.append((a.shape, a_s.shape, b.shape, b_s.shape, float(a_s[0, 0]), out))
        return torch.full((a.shape[0], b.shape[0]), 2.0 ** (8 * len(made)), dtype=out)
    monkeypatch.setattr(F, "_gemm", gemm)
    K = 2 * PART + 300
    a, b, KB = torch.zeros(1, K, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(K, 2, dtype=torch.uint8).view(torch.float8_e4m3fn), -(-K // 128)
    scales = torch.arange(float(KB))
    got = mx.blockwise_fp8_gemm(a, scales.view(1, KB), b, scales.view(KB, 1), use_2dblock_b=True)
    n = PART // 128
    assert made == [((1, w), (1, s), (2, w), (1, s), at, torch.float32) for w, s, at in ((PART, n, 0), (PART, n, n), (300, 3, 2 * n))]
    assert got.dtype == torch.bfloat16 and bool((got == torch.tensor(2.0 ** 8 + 2.0 ** 16 + 2.0 ** 24).bfloat16()).all())


@pytest.mark.parametrize("offsets", [[0, 5, 5, 700], [3, 2, 1000, 900], [-7, 0, 128, 256], [0, 2 ** 31 - 1, 5, 6], [0, PART, PART, PART + 129], [0, 100, PART, 2 * PART + 1], [PART + 1, 2 * PART, 2 * PART, 2 * PART + 50]])
def test_boundaries_of_the_parts_of_weight_gradients(stand_in, monkeypatch, offsets):
    """Every block of tokens of every group is in one part and in that group there, and no other is."""
    made, whole = [], F._grouped_weights

    def weights(go, go_s, x, x_s, offs, out):
        if go.shape[0] > PART:
            return whole(go, go_s, x, x_s, offs, out)
        assert go.shape[0] == x.shape[0] == 128 * go_s.shape[0] == 128 * x_s.shape[0] and offs.dtype == torch.int32
        made.append((int(go_s[0, 0]), go.shape[0] // 128, offs.tolist()))
        return torch.ones(3, 1, 1, dtype=out)
    monkeypatch.setattr(F, "_grouped_weights", weights)
    P = 2 * PART + 128 * 9
    codes, scales = torch.zeros(1, P, dtype=torch.uint8).t().view(torch.float8_e4m3fn), torch.arange(float(P // 128)).view(-1, 1)
    got = mx.blockwise_fp8_grouped_gemm_weights(codes, scales, codes, scales, torch.tensor(offsets, dtype=torch.int32))
    assert got.shape == (3, 1, 1) and bool((got == 3).all()) and [m[:2] for m in made] == [(0, PART // 128), (PART // 128, PART // 128), (2 * PART // 128, 9)]
    last, at, want = 0, 0, []
    for o in offsets:   # the segments in whole blocks, as the quantizer lays them out
        size = max(last, o) - last
        last += size
        at += -(-size // 128)
        want.append(min(at, P // 128))
    for first, n, offs in made:
        assert all(o % 128 == 0 for o in offs)
        assert [o // 128 for o in offs] == [min(max(w - first, 0), n) for w in want]
