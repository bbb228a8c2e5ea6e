"""The layers' gradients by differences of their own results, to the last bit.

Whole numbers of at most 7, one 7 in each block: every scale is a power of two, every operand stands for its tensor's numbers exactly (three bits, which E5M2 holds too),
and the sums of at most 49 * 300 are exact in the matrix pipe (no product of 8 lies below 2^-13 of another) and in fp32.  The layer is bilinear in such numbers, so a gradient
IS the difference of two losses, without a tolerance."""
import pytest
import torch

import alto_amd.mxfp4 as mx

pytestmark = pytest.mark.gpu
CODES = [torch.float8_e4m3fn, torch.float8_e5m2]


def whole(shape, g, dims):
    """Whole numbers with a 7 at the start of each block along each of dims."""
    t = torch.randint(-7, 8, shape, generator=g).float()
    for d in dims:
        t.index_fill_(d, torch.arange(0, shape[d], 128), 7)
    return t


def differences(loss, t, entries):
    for at in entries:
        up, down = t.detach().clone(), t.detach().clone()
        up[at] += 1
        down[at] -= 1
        yield (loss(up) - loss(down)) / 2


def some(t, planted, g, n=24):
    """Entries that can be changed by one and stay whole numbers below 7 in magnitude, none of them planted."""
    free = ((t.abs() <= 5) & ~planted).nonzero()
    return [tuple(i) for i in free[torch.randperm(len(free), generator=g)[:n]].tolist()]


def planted(shape, dims):
    p = torch.zeros(shape, dtype=torch.bool)
    for d in dims:
        p.index_fill_(d, torch.arange(0, shape[d], 128), True)
    return p


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("M,N,K", [(40, 150, 260), (300, 130, 200), (1, 257, 129)])
def test_linear(M, N, K, code):
    g = torch.Generator().manual_seed(M)
    x, w, dy = whole((M, K), g, (0, 1)), whole((N, K), g, (0, 1)), whole((M, N), g, (0, 1))
    xg, wg, dyg = x.cuda().requires_grad_(), w.cuda().requires_grad_(), dy.cuda()
    y = mx.blockwise_fp8_linear(xg, wg, grad_dtype=code)
    dx, dw = torch.autograd.grad(y, (xg, wg), dyg)
    assert torch.equal(y.cpu().double(), x.double() @ w.double().t())
    assert torch.equal(dx.cpu().double(), dy.double() @ w.double()) and torch.equal(dw.cpu().double(), dy.double().t() @ x.double())
    loss = lambda a, b: float((mx.blockwise_fp8_linear(a, b).double() * dyg.double()).sum())  # noqa: E731
    with torch.no_grad():
        for t, grad, f in ((xg, dx, lambda v: loss(v, wg)), (wg, dw, lambda v: loss(xg, v))):
            entries = some(t.detach().cpu(), planted(t.shape, (0, 1)), g)
            got = [float(grad[at]) for at in entries]
            assert got == list(differences(f, t, entries))
            assert M == 1 or sum(v != 0 for v in got) >= len(entries) - 2


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("trans", [True, False])
def test_grouped(code, trans):
    g = torch.Generator().manual_seed(3)
    M, N, K, offsets = 300, 140, 200, [0, 129, 129, 170, 290]   # (the last ten rows belong to none)
    E = len(offsets) - 1
    x, dy, w = whole((M, K), g, (1,)), whole((M, N), g, (1,)), whole((E, N, K), g, (1, 2))
    starts = [r for lo, hi in zip(offsets, offsets[1:]) for r in range(lo, hi, 128)]   # the blocks along the rows start anew with each group
    x[starts], dy[starts] = 7, 7
    rows_planted = lambda shape: planted(shape, (1,)).index_fill_(0, torch.tensor(starts), True)  # noqa: E731
    w = w if trans else w.transpose(1, 2).contiguous()
    offs = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    xg, wg, dyg = x.cuda().requires_grad_(), w.cuda().requires_grad_(), dy.cuda()
    y = mx.blockwise_fp8_grouped_linear(xg, wg, offs, grad_dtype=code, trans_weights=trans)
    dx, dw = torch.autograd.grad(y, (xg, wg), dyg)
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        we = (w[e] if trans else w[e].t()).double()
        exp = dy[lo:hi].double().t() @ x[lo:hi].double()
        assert torch.equal(y[lo:hi].cpu().double(), x[lo:hi].double() @ we.t()) and torch.equal(dx[lo:hi].cpu().double(), dy[lo:hi].double() @ we)
        assert torch.equal(dw[e].cpu().double(), exp if trans else exp.t())
    loss = lambda a, b: float((mx.blockwise_fp8_grouped_linear(a, b, offs, trans_weights=trans).double() * dyg.double()).sum())  # noqa: E731
    with torch.no_grad():
        for t, grad, p, f in ((xg, dx, rows_planted(x.shape), lambda v: loss(v, wg)), (wg, dw, planted(w.shape, (1, 2)), lambda v: loss(xg, v))):
            entries = some(t.detach().cpu(), p, g)
            got = [float(grad[at]) for at in entries]
            assert got == list(differences(f, t, entries))
            assert sum(v != 0 for v in got) >= len(entries) // 2
