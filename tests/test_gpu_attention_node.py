"""The attention's native autograd node: everyday calls take it, with the bits, the refusals and the saved-tensor rules of the Python function beside it."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def m():
    import alto_amd.mxfp4 as mod
    return mod


@pytest.fixture
def no_python_function(monkeypatch):
    from alto_amd.mxfp4 import attention as A
    monkeypatch.setattr(A.MXFP4AttentionFunction, "apply", None)


class Declines:
    """The native module without the attention's node."""

    def __init__(self, calls):
        self.calls = calls

    def __getattr__(self, name):
        return (lambda *args: None) if name == "attention_step" else getattr(self.calls, name)


def leaves(B, Hq, Hk, Sq, Sk, D, Dv, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g).to(dtype).to(DEV)  # noqa: E731
    return rand(B, Hq, Sq, D), rand(B, Hk, Sk, D), rand(B, Hk, Sk, Dv), rand(B, Hq, Sq, Dv).bfloat16()


def in_layout(layout, tensors):
    """[B, H, S, D] tensors as a caller of ``layout`` holds them (B = 1 for 'thd')."""
    if layout == "bhsd":
        return [t.clone() for t in tensors]
    tensors = [t.transpose(1, 2).contiguous() for t in tensors]
    return [t[0] for t in tensors] if layout == "thd" else tensors


def step(m, layout, tensors, needed, causal=True, **more):
    q, k, v, go = in_layout(layout, tensors)
    x = [t.requires_grad_(n) for t, n in zip((q, k, v), needed)]
    out, lse, _ = m.triton_attention_mxfp4(*x, causal=causal, layout=layout, **more)
    assert out.requires_grad and not lse.requires_grad
    out.backward(go)
    return out.detach(), lse, [t.grad for t in x], out.grad_fn


CASES = [
    # layout, B, Hq, Hk, Sq, Sk, D, Dv, causal
    ("bhsd", 2, 4, 2, 96, 96, 64, 64, True),
    ("bshd", 2, 4, 2, 96, 160, 128, 64, True),
    ("bshd", 1, 2, 2, 64, 32, 192, 128, False),
    ("bhsd", 1, 3, 1, 32, 288, 256, 128, True),
    ("thd", 1, 4, 2, 320, 320, 64, 128, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_the_node_and_the_python_function_are_the_same(m, monkeypatch, case, dtype):
    from alto_amd.mxfp4 import _runtime as rt
    layout, *sizes, causal = case
    tensors = leaves(*sizes, dtype=dtype)
    more = dict(cu_seqlens_q=[0, 64, 96, 320], cu_seqlens_k=[0, 64, 96, 320]) if layout == "thd" else {}
    for needed in ((True, True, True), (True, False, False), (False, False, True)):
        native = step(m, layout, tensors, needed, causal, **more)
        with monkeypatch.context() as p:
            calls = rt.host()
            p.setattr(rt, "host", lambda: Declines(calls))
            general = step(m, layout, tensors, needed, causal, **more)
        for i in range(2):
            assert torch.equal(native[i], general[i]) and native[i].stride() == general[i].stride()
        for a, b, n in zip(native[2], general[2], needed):
            assert (a is not None) == (b is not None) == n
            assert not n or (a.dtype == dtype and torch.equal(a, b) and a.stride() == b.stride())


def test_everyday_calls_take_the_node(m, no_python_function):
    for layout in ("bhsd", "bshd"):
        _, _, _, fn = step(m, layout, leaves(1, 2, 1, 64, 64, 64, 64), (True, True, True))
        assert fn is not None
    q, k, v, go = (t.transpose(1, 2) for t in leaves(1, 2, 2, 64, 64, 64, 64))
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y = m.triton_attention_mxfp4(*x, causal=True, layout="bshd")[0].transpose(1, 2)
    assert "MXFP4AttentionFunctionBackward" in [y.grad_fn.next_functions[0][0].name(), y.grad_fn.next_functions[0][0].next_functions[0][0].name()]


def test_q_k_and_v_as_slices_of_one_projection(m, no_python_function):
    """Strided views, and rows that no 16-byte access reads (copied)."""
    g = torch.Generator().manual_seed(3)
    for extra in (0, 3):
        whole = torch.randn(2, 96, 8, 64 + extra, generator=g).bfloat16().to(DEV).requires_grad_(True)
        q, k, v = whole[:, :, :4, extra:], whole[:, :, 4:6, extra:], whole[:, :, 6:, extra:]
        y = m.triton_attention_mxfp4(q, k, v, causal=True, layout="bshd")[0]
        (got,) = torch.autograd.grad(y.float().square().sum(), whole)
        x = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
        z = m.triton_attention_mxfp4(*x, causal=True, layout="bshd")[0]
        want = torch.autograd.grad(z.float().square().sum(), x)
        assert torch.equal(y, z) and torch.equal(got[..., extra:], torch.cat(want, 2)) and not got[..., :extra].any()


def test_a_second_derivative_is_an_error(m, no_python_function):
    q, k, v, go = leaves(1, 2, 2, 32, 32, 64, 64)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    u = go.clone().requires_grad_(True)
    out = m.triton_attention_mxfp4(*x, causal=True)[0]
    grads = torch.autograd.grad(out, x, u, create_graph=True)
    plain = torch.autograd.grad(m.triton_attention_mxfp4(*x, causal=True)[0], x, go)
    assert all(torch.equal(a, b) and a.requires_grad for a, b in zip(grads, plain))
    for g in grads:
        with pytest.raises(RuntimeError, match="not differentiable"):
            (g.float().square().sum() + u.float().sum()).backward(retain_graph=True)


def test_saved_tensor_hooks(m, no_python_function):
    """Kept on the host meanwhile, and the operands handed back at an address that is no multiple of 16."""
    tensors = leaves(1, 2, 1, 64, 96, 128, 64)
    want = step(m, "bshd", tensors, (True, True, True), causal=False)
    with torch.autograd.graph.save_on_cpu():
        got = step(m, "bshd", tensors, (True, True, True), causal=False)
    for a, b in zip(got[2], want[2]):
        assert torch.equal(a, b)

    def odd(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[t.dtype == torch.uint8:][:t.numel()]
        return flat.copy_(t.reshape(-1)), t.shape

    with torch.autograd.graph.saved_tensors_hooks(odd, lambda kept: kept[0].view(kept[1])):
        got = step(m, "bshd", tensors, (True, True, True), causal=False)
    for a, b in zip(got[2], want[2]):
        assert torch.equal(a, b)


def test_kept_tensors_and_refusals(m, no_python_function):
    q, k, v, go = leaves(1, 2, 2, 64, 64, 64, 64)
    y = m.triton_attention_mxfp4(q.requires_grad_(True), k, v, causal=True)[0]
    operands, out, lse = y.grad_fn.saved_tensors
    assert torch.equal(out, y) and lse.shape == (1, 2, 64) and operands.dtype == torch.uint8
    for bad in (torch.zeros(1, 2, 64, 96, dtype=torch.bfloat16, device=DEV), torch.zeros(1, 2, 64, 512, dtype=torch.bfloat16, device=DEV)):   # head dims of no kernel
        with pytest.raises(AssertionError):
            m.triton_attention_mxfp4(bad.requires_grad_(True), bad, v, causal=True)
    z = m.triton_attention_mxfp4(q, k, v, causal=True, sm_scale=-1.0)[0]
    with pytest.raises(AssertionError, match="sm_scale"):
        z.backward(go)
    y.backward(go)
    with pytest.raises(RuntimeError, match="second time"):
        y.backward(go)


def test_checkpointed(m, no_python_function):
    from torch.utils.checkpoint import checkpoint
    tensors = leaves(1, 2, 1, 64, 64, 64, 64)
    want = step(m, "bhsd", tensors, (True, True, True))
    x = [t.clone().requires_grad_(True) for t in tensors[:3]]
    y = checkpoint(lambda q, k, v: m.triton_attention_mxfp4(q, k, v, causal=True)[0] * 1, *x, use_reentrant=False)
    y.backward(tensors[3])
    for a, b in zip(x, want[2]):
        assert torch.equal(a.grad, b)


@pytest.mark.parametrize("needed", [(True, False, False), (False, True, False), (False, False, True)])
def test_a_second_derivative_of_some_of_the_gradients_is_an_error(m, no_python_function, needed):
    q, k, v, go = leaves(1, 2, 2, 32, 32, 64, 64)
    x = [t.requires_grad_(n) for t, n in zip((q, k, v), needed)]
    u = go.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(m.triton_attention_mxfp4(*x, causal=True)[0], [t for t in x if t.requires_grad], u, create_graph=True)
    assert grad.requires_grad
    with pytest.raises(RuntimeError, match="not differentiable"):
        grad.float().sum().backward()


def test_two_streams(m, no_python_function):
    """Steps in flight on two streams, each with the bits that it has alone."""
    both = [leaves(1, 8, 2, 256, 256, 128, 128, seed=s) for s in (1, 2)]
    want = [step(m, "bshd", t, (True, True, True)) for t in both]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(3):
        for t, s in zip(both, streams):
            with torch.cuda.stream(s):
                got.append(step(m, "bshd", t, (True, True, True)))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g[0], want[i % 2][0]) and all(torch.equal(a, b) for a, b in zip(g[2], want[i % 2][2]))


@pytest.mark.parametrize("q_is_k", [True, False])
def test_one_tensor_for_two_operands(m, no_python_function, q_is_k):
    """The same leaf as Q and K, or as K and V: its gradient is the sum of theirs."""
    q, k, v, go = leaves(1, 2, 2, 64, 64, 64, 64)
    a = q.clone().requires_grad_(True)
    y = m.triton_attention_mxfp4(a, a, v, causal=True)[0] if q_is_k else m.triton_attention_mxfp4(k, a, a, causal=True)[0]
    (got,) = torch.autograd.grad(y, a, go)
    x = [t.clone().requires_grad_(True) for t in ((q, q, v) if q_is_k else (k, q, q))]
    grads = torch.autograd.grad(m.triton_attention_mxfp4(*x, causal=True)[0], x, go)
    assert torch.equal(got, grads[0] + grads[1] if q_is_k else grads[1] + grads[2])
