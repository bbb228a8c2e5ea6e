"""The 64-bit gradients that the attention backward is held to: against differences of a loss, and what they are in rows without keys."""
import pytest
import torch

from oracle.attention_oracle import attention_bwd_ref, attention_probabilities


def _inputs(Hq, Hk, Sq, Sk, D, Dv, seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, dtype=torch.float64)  # noqa: E731
    return rand(2, Hq, Sq, D), rand(2, Hk, Sk, D), rand(2, Hk, Sk, Dv), rand(2, Hq, Sq, Dv), g


@pytest.mark.parametrize("case", [(1, 1, 5, 5, 4, 3, True, "none"), (4, 2, 3, 6, 4, 5, True, "alibi"), (2, 1, 6, 4, 3, 4, False, "bias")], ids=str)
def test_gradients_equal_differences_of_the_loss(case):
    Hq, Hk, Sq, Sk, D, Dv, causal, extra = case
    q, k, v, go, g = _inputs(Hq, Hk, Sq, Sk, D, Dv, seed=Sq)
    more = dict(causal=causal, sm_scale=0.7)
    if extra == "alibi":
        more["alibi_slopes"] = torch.rand(Hq, generator=g)
    if extra == "bias":
        more["bias"] = torch.randn(2, 1, Sq, Sk, generator=g).masked_fill(torch.rand(2, 1, Sq, Sk, generator=g) < 0.2, float("-inf"))
    loss = lambda: float((attention_probabilities(q, k, v, **more)[1] * go).sum())  # noqa: E731
    _, out, lse = attention_probabilities(q, k, v, **more)
    grads = attention_bwd_ref(go, q, k, v, out, lse, **more)
    step = 1e-5
    for x, got in ((q, grads.dq), (k, grads.dk), (v, grads.dv)):
        for i in torch.randperm(x.numel(), generator=g)[:12].tolist():
            flat = x.view(-1)
            keep = float(flat[i])
            flat[i] = keep + step
            up = loss()
            flat[i] = keep - step
            down = loss()
            flat[i] = keep
            # second order: step^2 times third derivatives of order 10, and 1e-16 / step of the losses' rounding
            assert abs((up - down) / (2 * step) - float(got.reshape(-1)[i])) < 1e-7


def test_a_row_without_keys_has_no_part_in_any_gradient():
    q, k, v, go, _ = _inputs(2, 2, 4, 6, 4, 4, seed=3)
    bias = torch.zeros(2, 1, 4, 6)
    bias[1, :, 2] = float("-inf")
    more = dict(causal=False, sm_scale=0.5)
    _, out, lse = attention_probabilities(q, k, v, bias=bias, **more)
    assert bool((lse[1, :, 2] == float("-inf")).all()) and bool((out[1, :, 2] == 0).all())
    grads = attention_bwd_ref(go, q, k, v, out, lse, bias=bias, **more)
    assert bool((grads.dq[1, :, 2] == 0).all())
    keep = torch.tensor([0, 1, 3])
    alone = attention_bwd_ref(go[1:, :, keep], q[1:, :, keep], k[1:], v[1:], out[1:, :, keep], lse[1:, :, keep], **more)
    torch.testing.assert_close(grads.dk[1:], alone.dk)
    torch.testing.assert_close(grads.dv[1:], alone.dv)
