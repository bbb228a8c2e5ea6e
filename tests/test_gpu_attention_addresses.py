"""Dense tensors at addresses that no 16-byte access reads (a part of a flat buffer): the attention copies them, forward and backward."""
import pytest
import torch

from tests.test_gpu_attention_node import Declines, leaves

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def m():
    import alto_amd.mxfp4 as mod
    return mod


def moved(t):
    """The same values one element into a buffer."""
    odd = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)
    assert odd.is_contiguous() and odd.data_ptr() % 16 != 0
    return odd


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_inputs_and_gradients_at_odd_addresses(m, monkeypatch, native, dtype):
    from alto_amd.mxfp4 import _runtime as rt
    q, k, v, go = leaves(1, 4, 2, 64, 96, 64, 64, dtype=dtype)
    want_out, want_lse, _ = m.triton_attention_mxfp4(q, k, v, causal=True)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(m.triton_attention_mxfp4(*x, causal=True)[0], x, go)
    if not native:
        calls = rt.host()
        monkeypatch.setattr(rt, "host", lambda: Declines(calls))
    odd = [moved(t) for t in (q, k, v)]
    out, lse, _ = m.triton_attention_mxfp4(*odd, causal=True)
    assert torch.equal(out, want_out) and torch.equal(lse, want_lse)
    odd = [t.requires_grad_(True) for t in odd]
    for a, b in zip(torch.autograd.grad(m.triton_attention_mxfp4(*odd, causal=True)[0], odd, moved(go)), want):
        assert torch.equal(a, b)


def test_the_entry_point_on_codes(m):
    q, k, v, go = leaves(2, 4, 2, 64, 64, 64, 64)
    qq, qs, kq, ks, vq, vs = m.quantize_qkv(q, k, v)
    out, lse, _ = m.triton_attention_mxfp4(q, k, v, causal=True)
    call = lambda go, out: m.attention_mxfp4_backward(go, qq, kq, vq, qs, ks, vs, out, lse, 0.125, True)  # noqa: E731
    for a, b in zip(call(moved(go), moved(out)), call(go, out)):
        assert torch.equal(a, b)


def test_a_bias_at_an_odd_address(m):
    q, k, v, go = leaves(2, 4, 2, 64, 64, 64, 64)
    bias = torch.randn(2, 1, 64, 64, device=DEV)
    results = []
    for b in (bias, moved(bias)):
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = m.triton_attention_mxfp4(*x, bias=b, causal=False)[0]
        results.append((out.detach(), *torch.autograd.grad(out, x, go)))
    for a, b in zip(*results):
        assert torch.equal(a, b)
