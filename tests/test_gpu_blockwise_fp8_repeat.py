"""Products of 8-bit operands repeat themselves bit for bit, alone and beside another stream's work: on each tile, with K in parts, by group, and the steps of the layers."""
import pytest
import torch

import alto_amd.mxfp4 as mx

pytestmark = pytest.mark.gpu


def data(*shape):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(sum(shape))).to(torch.bfloat16)


def repeats(call):
    first = call()
    side, busy = torch.cuda.Stream(), data(2048, 2048)
    torch.cuda.synchronize()
    for _ in range(6):
        with torch.cuda.stream(side):
            busy @ busy
        for a, b in zip(call(), first):
            assert torch.equal(a, b)
    torch.cuda.synchronize()


@pytest.mark.parametrize("b_2d", [True, False])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (64, 2048, 4000), (333, 4104, 2000), (256, 1024, 8192), (1500, 2048, 1024), (4352, 4096, 520)])
def test_products(M, N, K, out, b_2d):
    a, b = mx.convert_to_blockwise_fp8(data(M, K), dtype=torch.float8_e5m2), mx.convert_to_blockwise_fp8(data(N, K), is_2d_block=b_2d)
    repeats(lambda: (mx.blockwise_fp8_gemm(*a, *b, use_2dblock_b=b_2d, trans_b=True, output_dtype=out),))


@pytest.mark.parametrize("M", [8, 300, 5000])
def test_steps(M):
    x, w, e, dy = data(M, 520).requires_grad_(), data(264, 520).requires_grad_(), data(4, 264, 520).requires_grad_(), data(M, 264)
    offsets = torch.tensor([0, M // 8, M // 8, M // 2, M - 3], dtype=torch.int32, device="cuda")

    def step(y, p):
        return (y.detach(), *torch.autograd.grad(y, (x, p), dy))
    repeats(lambda: step(mx.blockwise_fp8_linear(x, w), w))
    repeats(lambda: step(mx.blockwise_fp8_grouped_linear(x, e, offsets), e))
