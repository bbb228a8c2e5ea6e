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


@pytest.mark.parametrize("K", [LONGEST + 1, 2 ** 22, 2 ** 23 - 128 + 77])
def test_products_in_parts(K):
    test_products(K)


@pytest.mark.parametrize("M,N", [(1, 1), (1, 3), (2, 1)])
def test_a_row_or_a_column_in_parts(M, N):
    """(one row has no distance to a next one that would give its length away)"""
    K = 2 ** 22 + 200
    a, b, ones = signs((M, K), 1), signs((N, K), 2), torch.ones((1, -(-K // 128)), device="cuda")
    exp = a.double() @ b.double().t()
    got = mx.blockwise_fp8_gemm(stored(a, K), ones.expand(M, -1), stored(b, K), ones, use_2dblock_b=True, trans_b=True, output_dtype=torch.float32)
    assert torch.equal(got.double(), exp)
    got = mx.blockwise_fp8_grouped_gemm(stored(a, K), ones.expand(M, -1), stored(b[None], K), ones[None], torch.tensor([0, M], dtype=torch.int32, device="cuda"), output_dtype=torch.float32)
    assert torch.equal(got.double(), exp)


@pytest.mark.parametrize("M", [LONGEST, LONGEST + 1, 2 ** 22 + 1000])
def test_a_weight_gradient_over_as_many_rows(M):
    """What the quantizer makes of them along the tokens; 7 in every 128th row makes the scales powers of two."""
    N, K = 24, 16
    x, dy, w = signs((M, K), 1), signs((M, N), 2), signs((N, K), 3)
    x[::128] = dy[::128] = 7
    wg = w.clone().requires_grad_()
    dw, = torch.autograd.grad(mx.blockwise_fp8_linear(x, wg), wg, dy)
    assert torch.equal(dw.double(), dy.double().t() @ x.double())


def rows_by_group(M, offsets):
    """Rows of signs, a 7 in the first of each 128 of every group."""
    x, dy, last = signs((M, 16), 1), signs((M, 24), 2), 0
    for lo, hi in zip(offsets, offsets[1:]):
        x[lo:hi:128] = dy[lo:hi:128] = 7
    return x, dy


@pytest.mark.parametrize("trans", [True, False])
@pytest.mark.parametrize("M,offsets", [(2 ** 22 + 5000, [3, 1000, 1000, 2 ** 22 - 50, 2 ** 22 + 4000]), (2 ** 22, [0, 1, 2, 3, 2 ** 22]), (2 ** 23, [0, 2 ** 22 + 1, 2 ** 22 + 2, 2 ** 22 + 2, 2 ** 23])])
def test_weight_gradients_by_group_over_more_rows(M, offsets, trans):
    x, dy = rows_by_group(M, offsets)
    w = signs((4, 24, 16) if trans else (4, 16, 24), 3).requires_grad_()
    dw, = torch.autograd.grad(mx.blockwise_fp8_grouped_linear(x, w, torch.tensor(offsets, dtype=torch.int32, device="cuda"), trans_weights=trans), w, dy)
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        exp = dy[lo:hi].double().t() @ x[lo:hi].double()
        assert torch.equal(dw[e].double(), exp if trans else exp.t())


def test_weight_gradients_of_very_many_groups():
    """33024 groups pad a few rows to more than 2^22."""
    E, M = 33024, 3000
    offsets = torch.sort(torch.randint(0, M + 1, (E + 1,), generator=torch.Generator().manual_seed(1)).int()).values
    x, dy = rows_by_group(M, offsets.tolist())
    w = signs((1, 24, 16), 3).expand(E, 24, 16).clone().requires_grad_()
    dw, = torch.autograd.grad(mx.blockwise_fp8_grouped_linear(x, w, offsets.cuda()), w, dy)
    some = [e for e in range(E) if offsets[e + 1] > offsets[e]]
    assert len(some) > 2000
    for e in some[::50]:
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        assert torch.equal(dw[e].double(), dy[lo:hi].double().t() @ x[lo:hi].double())
    empty = torch.ones(E, dtype=torch.bool)
    empty[some] = False
    assert not dw[empty.cuda()].any() and dw[(~empty).cuda()].any(dim=(1, 2)).all()


def test_parts_in_a_graph():
    """Captured, replayed on other boundaries and rows with eager work between."""
    M = 2 ** 22 + 500
    bounds = [[0, 100, 2 ** 22], [7, 7, 2 ** 22 + 500], [0, 2 ** 22, 2 ** 22 + 1]]
    offsets, x, dy = torch.tensor(bounds[0], dtype=torch.int32, device="cuda"), signs((M, 16), 1), signs((M, 24), 2)

    def program():
        q, s = mx.quantize_blockwise_fp8_rowcol(x, offsets=offsets)[2:]
        g, gs = mx.quantize_blockwise_fp8_rowcol(dy, offsets=offsets)[2:]
        return mx.blockwise_fp8_grouped_gemm_weights(g, gs, q, s, offsets, output_dtype=torch.float32)
    program()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = program()
    for turn in range(4):
        offsets.copy_(torch.tensor(bounds[turn % 3], dtype=torch.int32))
        x.copy_(signs((M, 16), 10 + turn))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        assert torch.equal(got, program()) and got.any()
