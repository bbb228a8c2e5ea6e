"""Attention and rotary positions under torch's transforms: what they serve gives the bits of an eager call, what they do not they refuse."""
import pytest
import torch
from torch.autograd.forward_ad import dual_level, make_dual

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def m():
    import alto_amd.mxfp4 as mod
    return mod


def leaves(B, S, Hq, Hk, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, S, h, D, generator=g).bfloat16().to(DEV) for h in (Hq, Hk, Hk, Hq)]


def test_a_compiled_step_has_the_bits_of_an_eager_one(m):
    """Rotation and attention of a compiled block (the graphs around them without a code generator), forward and backward, twice."""
    q, k, v, go = leaves(2, 96, 4, 2, 64)
    freq = m.rotary_frequencies(64)[0].to(DEV)
    attention = m.LPScaledDotProductAttention(m.TrainingOpConfig())

    def block(q, k, v):
        a, b = m.apply_rotary(q * 2, k, freq, layout="bshd")
        a = m.apply_rotary(a, None, freq, layout="bshd")
        return attention(a, b, v, is_causal=True, rotary=m.Rotary(freq)) + q

    def step(fn):
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        y = fn(*x)
        return y.detach(), *torch.autograd.grad(y, x, go)

    want = step(block)
    torch._dynamo.reset()
    compiled = torch.compile(block, backend="aot_eager")
    for _ in range(2):
        for a, b in zip(step(compiled), want):
            assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(compiled(q, k, v), want[0])
    torch._dynamo.reset()


@pytest.mark.filterwarnings("ignore:`torch.jit")
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_traced_rotation_is_refused(m):
    q, k, _, _ = leaves(1, 32, 2, 2, 64)
    freq = m.rotary_frequencies(64)[0].to(DEV)
    for grad in (False, True):
        q.requires_grad_(grad)
        for fn, x in ((lambda q, k: m.apply_rotary(q, k, freq, layout="bshd"), (q, k)), (lambda q: m.apply_rotary(q, None, freq, layout="bshd"), (q,))):
            with pytest.raises(NotImplementedError, match="torch.jit.trace"):
                torch.jit.trace(fn, x, check_trace=False)
            fn(*x)
            with pytest.raises(NotImplementedError, match="functorch"):
                torch.func.jvp(lambda q: fn(q, *x[1:]), (q.detach(),), (q.detach(),))

def test_a_rotation_with_forward_mode_tangents_is_refused(m):
    q, k, _, _ = leaves(1, 32, 2, 2, 64)
    freq = m.rotary_frequencies(64)[0].to(DEV)
    want = m.apply_rotary(q, k, freq, layout="bshd")
    with dual_level():
        dual = make_dual(q, torch.ones_like(q))
        for call in (lambda: m.apply_rotary(dual, None, freq, layout="bshd"), lambda: m.apply_rotary(dual, k, freq, layout="bshd"),
                     lambda: m.apply_rotary(k, dual, freq, layout="bshd"), lambda: m.apply_rotary(q, k, make_dual(freq, torch.ones_like(freq)), layout="bshd")):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        for a, b in zip(m.apply_rotary(q, k, freq, layout="bshd"), want):
            assert torch.equal(a, b)
        for x in ((q.clone().requires_grad_(True), k), (q.clone().requires_grad_(True), None)):
            y = m.apply_rotary(*x, freq, layout="bshd")
            y = y if x[1] is None else y[0]
            with pytest.raises(NotImplementedError):
                y.backward(make_dual(torch.ones_like(y), torch.ones_like(y)))   # (nor of a gradient)


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.filterwarnings("ignore:`torch.jit")
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_attention_under_transforms_is_refused(m, requires_grad):
    x = leaves(1, 64, 2, 2, 64)[:3]
    want = m.triton_attention_mxfp4(*x, causal=True, layout="bshd")[0]
    x = [t.requires_grad_(requires_grad) for t in x]
    fn = lambda q, k, v: m.triton_attention_mxfp4(q, k, v, causal=True, layout="bshd")[0]  # noqa: E731
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(fn, tuple(x), check_trace=False)
    with pytest.raises(NotImplementedError, match="functorch"):
        torch.func.vmap(lambda q: fn(q, *x[1:]))(x[0].detach()[None])
    with dual_level():
        for i in range(3):
            y = list(x)
            y[i] = make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*y)
        y = fn(*x)
        assert torch.equal(y, want)
        if requires_grad:
            with pytest.raises(NotImplementedError):
                y.backward(make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("of_q", [True, False])
def test_the_gradient_of_an_additive_term_is_refused(m, of_q):
    """Also where nothing else requires one; the forward gives the bits that it gives without a graph."""
    q, k, v, go = leaves(1, 64, 2, 2, 64)
    for name, term in (("bias", torch.randn(1, 1, 64, 64, device=DEV)), ("alibi_slopes", torch.rand(2, device=DEV))):
        want = m.triton_attention_mxfp4(q, k, v, causal=True, layout="bshd", **{name: term})[0]
        y = m.triton_attention_mxfp4(q.detach().requires_grad_(of_q), k, v, causal=True, layout="bshd", **{name: term.clone().requires_grad_(True)})[0]
        assert torch.equal(y, want)
        with pytest.raises(NotImplementedError, match="detach"):
            y.backward(go)


@pytest.mark.parametrize("layout", ["bhsd", "bshd", "thd"])
def test_a_result_is_changed_in_place(m, layout):
    """A gate on the attention's result, where no gradient is asked for; where one is, autograd says that the backward needs the result that was."""
    q, k, v, _ = leaves(1, 64, 4, 2, 64)
    more = {}
    if layout == "bhsd":
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    if layout == "thd":
        (q, k, v), more = (t[0] for t in (q, k, v)), dict(cu_seqlens_q=[0, 32, 64], cu_seqlens_k=[0, 32, 64])
    want = m.triton_attention_mxfp4(q, k, v, causal=True, layout=layout, **more)
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    y, lse, _ = m.triton_attention_mxfp4(*x, causal=True, layout=layout, **more)
    assert torch.equal(y, want[0]) and torch.equal(lse, want[1]) and y.stride() == want[0].stride() and lse.stride() == want[1].stride()
    assert torch.equal(y.mul_(2), want[0] * 2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
