"""The longest reductions of products of 8-bit operands.  Codes of -1, 0 and 1: every sum is a whole number below 2^24, which fp32 holds exactly."""
import pytest
import torch

import alto_amd.mxfp4 as mx

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
LONGEST = 2 ** 22 - 16


def signs(shape, seed):
    return torch.randint(-1, 2, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").float()


def stored(t, K):
    """Codes of t [.., K] at the quantizer's pitch."""
    out = torch.zeros((*t.shape[:-1], -(-K // 128) * 128), dtype=E4M3, device="cuda")
    out.view(torch.uint8)[..., :K] = t.to(E4M3).view(torch.uint8)
    return out[..., :K]


@pytest.mark.parametrize("K", [2 ** 22 - 128, 2 ** 22 - 127, LONGEST])
def test_products(K):
    M, N, KB = 3, 5, -(-K // 128)
    a, b = signs((M, K), 1), signs((2, N, K), 2)
    ones = lambda *shape: torch.ones(shape, device="cuda")  # noqa: E731
    exp = a.double() @ b[0].double().t()
    assert exp.abs().max() > 1000
    got = mx.blockwise_fp8_gemm(stored(a, K), ones(M, KB), stored(b[0], K), ones(1, KB), use_2dblock_b=True, trans_b=True, output_dtype=torch.float32)
    assert torch.equal(got.double(), exp)
    offsets = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    got = mx.blockwise_fp8_grouped_gemm(stored(a, K), ones(M, KB), stored(b, K), ones(2, 1, KB), offsets, output_dtype=torch.float32)
    assert torch.equal(got[:1].double(), exp[:1]) and torch.equal(got[1:].double(), a[1:].double() @ b[1].double().t())


def test_more_than_the_longest_is_refused():
    K = LONGEST + 16
    ones = torch.ones((2, K // 128), device="cuda")
    t = stored(signs((2, K), 1), K)
    with pytest.raises(Exception, match="out of range"):
        mx.blockwise_fp8_gemm(t, ones, t, ones, trans_b=True)


def test_a_weight_gradient_over_as_many_rows():
    """What the quantizer makes of them along the tokens; 7 in every 128th row makes the scales powers of two."""
    M, N, K = LONGEST, 24, 16
    x, dy, w = signs((M, K), 1), signs((M, N), 2), signs((N, K), 3)
    x[::128] = dy[::128] = 7
    wg = w.clone().requires_grad_()
    dw, = torch.autograd.grad(mx.blockwise_fp8_linear(x, wg), wg, dy)
    assert torch.equal(dw.double(), dy.double().t() @ x.double())
