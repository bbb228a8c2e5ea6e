"""What the attention's gradients do with NaN and with a bias at the ends of its type: NaN where the formula has NaN and nowhere else, finite where it is finite."""
import pytest
import torch

from tests.test_gpu_attention_backward import Operands

pytestmark = pytest.mark.gpu
LOWEST, LARGEST = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max


@pytest.fixture(scope="module")
def m():
    import alto_amd.mxfp4 as mod
    return mod


def operands(D, seed):
    g = torch.Generator().manual_seed(seed)
    case = (2, 4, 2, 96, 160, D, 64, True)
    return Operands(*case, seed=seed, bias=torch.randn(2, 1, 96, 160, generator=g))


@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_a_nan_bias_reaches_every_gradient_it_belongs_to(m, D):
    """NaN on one pair of a row and a key that it sees: NaN in that row of dQ and that key's dK and dV, of that sequence, the others bit for bit as
    without it."""
    x = operands(D, seed=1)
    want = x.call(m)
    row, key = 40, 70   # (rows see the keys up to row + 64)
    x.more["bias"] = x.more["bias"].clone()
    x.more["bias"][1, 0, row, key] = float("nan")
    for got, clean, at in zip(x.call(m), want, (row, key, key)):
        assert bool(got[1, :, at].isnan().all())
        got[1, :, at] = clean[1, :, at]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_a_nan_log_sum_exp_reaches_every_gradient_it_belongs_to(m, D, biased):
    """NaN in one row's log-sum-exp: NaN in that row of dQ and in dK and dV of the keys that it sees, nothing of it in other rows, key heads and sequences."""
    x = operands(D, seed=2)
    if not biased:
        x.more["bias"] = None
    want = x.call(m)
    row, head = 33, 3
    x.lse[0, head, row] = float("nan")
    dq, dk, dv = x.call(m)
    assert bool(dq[0, head, row].isnan().all()) and bool(dk[0, 1, :row + 65].isnan().all()) and bool(dv[0, 1, :row + 65].isnan().all())
    dq[0, head, row] = want[0][0, head, row]
    assert torch.equal(dq, want[0])
    for got, clean in ((dk, want[1]), (dv, want[2])):
        assert torch.equal(got[0, 0], clean[0, 0]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_the_lowest_value_over_a_whole_row(m, D):
    """With the log-sum-exp that is the type's lowest value as well (a framework that keeps scores in base e gives it), which base 2 does not hold: the
    row gives nothing, as with -inf."""
    x = operands(D, seed=3)
    for fill in (float("-inf"), LOWEST):
        x.more["bias"] = x.more["bias"].clone()
        x.more["bias"][1, 0, 17] = fill
        x.lse[1, :, 17] = fill
        got = x.call(m)
        assert bool((got[0][1, :, 17] == 0).all())
        if fill == LOWEST:
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        want = got


@pytest.mark.parametrize("D", [64, 256])
def test_the_largest_value_on_a_key(m, D):
    """A score and a log-sum-exp at the type's largest value: the key has all of the row's probability, so that dV gets the row's dO once; dQ and dK stay finite."""
    x = operands(D, seed=4)
    hidden = Operands.__new__(Operands)
    hidden.__dict__.update(x.__dict__)
    hidden.more, hidden.lse = dict(x.more, bias=x.more["bias"].clone()), x.lse.clone()
    hidden.more["bias"][0, 0, 50] = float("-inf")
    hidden.lse[0, :, 50] = float("-inf")
    without = hidden.call(m)
    x.more["bias"] = x.more["bias"].clone()
    x.more["bias"][0, 0, 50, 20] = LARGEST
    x.lse[0, :, 50] = LARGEST
    got = x.call(m)
    assert all(bool(t.isfinite().all()) for t in got)
    more = got[2].cpu().double() - without[2].cpu().double()
    row = x.go[0, :, 50].double().view(2, 2, -1).sum(1)                  # of the query heads of each key head
    size = got[2][0, :, 20].cpu().double().abs() + without[2][0, :, 20].cpu().double().abs()
    # either sum is rounded to bf16 once, half a step each; the sums themselves are fp32 of 2 x 96 terms of order 1
    assert bool(((more[0, :, 20] - row).abs() <= size * 2.0 ** -8 + 192 * 2.0 ** -24 * 8).all())
    more[0, :, 20] = 0
    assert bool((more == 0).all())
