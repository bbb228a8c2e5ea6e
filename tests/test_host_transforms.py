"""Attention and rotary positions under torch's transforms, without a GPU: the native calls are stood in for by plain ones."""
import pytest
import torch
from torch.autograd.forward_ad import dual_level, make_dual, unpack_dual

import alto_amd.mxfp4 as mx
from alto_amd.mxfp4 import _runtime as rt
from alto_amd.mxfp4 import rotary as R

FREQ = torch.ones(16, dtype=torch.float64)


def declined(*tensors):
    """(what the native calls leave to the general ones)"""
    return torch.jit.is_tracing() or torch._C._are_functorch_transforms_active() or any(t is not None and unpack_dual(t).tangent is not None for t in tensors)


class Host:
    """Native calls that leave a trace of their operands: the attention's output is Q's first rows, its gradients are 2, 3 and 4."""

    def attend(self, q, k, v, sm_scale, causal, out, lse, *more):
        if declined(q, k, v):
            return False
        out.copy_(q[..., :out.shape[-1]])
        lse.zero_()
        return True

    def attention_gradients(self, go, q, qs, k, ks, v, vs, out, lse, sm_scale, causal, keys, bias, slopes, cu_q, cu_k, rows_outer, want_q, want_kv):
        if declined(go, out, lse, bias, slopes):
            return None

        def full(value, heads, rows, columns):
            return torch.full((q.shape[0], rows, heads, columns), value, dtype=torch.bfloat16).transpose(1, 2)

        return full(2.0, q.shape[1], q.shape[2], 2 * q.shape[3]), full(3.0, k.shape[1], k.shape[2], 2 * q.shape[3]), full(4.0, k.shape[1], k.shape[2], v.shape[2])

    def attention_step(self, *args):
        return None

    def rotary(self, *args):
        return None


class Lib:
    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def stand_in(monkeypatch):
    monkeypatch.setattr(rt, "require_gpu", lambda *tensors: None)
    monkeypatch.setattr(rt, "host", Host)
    monkeypatch.setattr(rt, "lib", Lib)
    monkeypatch.setattr(rt, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


@pytest.fixture
def plain_rotation(monkeypatch):
    """Twice x, or half of it back: a rotation as far as its callers can tell (a launch takes addresses, which only tensors of real memory have)."""

    def rotate(q, k, freq, positions, interleaved, factor, layout, inverse):
        return [None if t is None or t.data_ptr() == 0 else t * (0.5 if inverse else 2) for t in (q, k)]

    monkeypatch.setattr(R, "_rotate", rotate)


def tensors(requires_grad):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(1, 2, 64, 64, generator=g).bfloat16().requires_grad_(requires_grad) for _ in range(3)]


def compiled(fn):
    return torch.compile(fn, backend="aot_eager")


@pytest.mark.parametrize("layout", ["bhsd", "bshd", "thd"])
def test_a_compiled_training_step_of_the_attention(stand_in, layout):
    """The caller's graph breaks at the attention, which runs as in an eager step, its gradients too."""
    x = tensors(True)
    if layout == "thd":
        x = [t.detach()[0].transpose(0, 1).contiguous().requires_grad_(True) for t in x]
    more = dict(cu_seqlens_q=[0, 64], cu_seqlens_k=[0, 64]) if layout == "thd" else {}
    fn = compiled(lambda q, k, v: mx.triton_attention_mxfp4(q * 2, k, v, causal=True, layout=layout, **more)[0] * 3)
    for _ in range(2):
        y = fn(*x)
        grads = torch.autograd.grad(y.sum(), x)
        assert [float(t.float().amin()) for t in grads] == [4.0, 3.0, 4.0] == [float(t.float().amax()) for t in grads]
    with torch.no_grad():
        assert fn(*x).shape == y.shape


def test_a_compiled_training_step_of_the_rotation(stand_in, plain_rotation):
    q, k, _ = tensors(True)
    fn = compiled(lambda q, k: [t + 1 for t in mx.apply_rotary(q, k, FREQ)])
    for _ in range(2):
        a, b = fn(q, k)
        assert torch.equal(a, 2 * q + 1) and torch.equal(b, 2 * k + 1)
        assert all(bool((t == 0.5).all()) for t in torch.autograd.grad(a.sum() + b.sum(), (q, k)))
    alone = compiled(lambda q: mx.apply_rotary(q, None, FREQ) + 1)
    assert all(bool((t == 0.5).all()) for t in torch.autograd.grad(alone(q).sum(), (q,)))
    with torch.no_grad():
        assert torch.equal(fn(q, k)[0], 2 * q + 1)


def test_a_compiled_module_with_rotated_positions(stand_in, plain_rotation):
    x = [t.detach().transpose(1, 2).contiguous().requires_grad_(True) for t in tensors(True)]
    attention = mx.LPScaledDotProductAttention(mx.TrainingOpConfig())
    fn = compiled(lambda q, k, v: attention(q, k, v, rotary=mx.Rotary(FREQ)).float().square())
    y = fn(*x)
    grads = torch.autograd.grad(y.sum(), x)
    assert [float(t.float().amax()) for t in grads] == [1.0, 1.5, 4.0]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.filterwarnings("ignore:`torch.jit")
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_traced_rotation_is_refused(stand_in, requires_grad):
    """(its trace would hold the outputs' allocation alone)"""
    q, k, _ = tensors(requires_grad)
    for fn, x in ((lambda q, k: mx.apply_rotary(q, k, FREQ), (q, k)), (lambda q: mx.apply_rotary(q, None, FREQ), (q,))):
        with pytest.raises(NotImplementedError, match="torch.jit.trace"):
            torch.jit.trace(fn, x, check_trace=False)


def test_a_rotation_under_functorch_is_refused(stand_in):
    q, k, _ = tensors(False)
    for fn in (lambda q: mx.apply_rotary(q, None, FREQ), lambda q: mx.apply_rotary(q, k, FREQ)[0]):
        with pytest.raises(NotImplementedError, match="functorch"):
            torch.func.jvp(fn, (q,), (q,))
        with pytest.raises(NotImplementedError, match="functorch"):
            torch.func.grad(lambda q: fn(q).float().sum())(q)
    with pytest.raises(NotImplementedError, match="functorch"):
        torch.func.vmap(lambda q: mx.apply_rotary(q, None, FREQ, layout="thd"))(q)

@pytest.mark.parametrize("requires_grad", [False, True])
def test_a_rotation_with_forward_mode_tangents_is_refused(stand_in, plain_rotation, requires_grad):
    """(they would be lost: the launches see no tangent)"""
    q, k, _ = tensors(requires_grad)
    with dual_level():
        dual = make_dual(q, torch.ones_like(q))
        for call in (lambda: mx.apply_rotary(dual, None, FREQ), lambda: mx.apply_rotary(dual, k, FREQ), lambda: mx.apply_rotary(k, dual, FREQ),
                     lambda: mx.apply_rotary(q, None, make_dual(FREQ, torch.ones_like(FREQ)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert mx.apply_rotary(q, None, FREQ).shape == q.shape   # (no tangent: nothing to lose)
        y = mx.apply_rotary(q.detach().requires_grad_(True), None, FREQ)
        with pytest.raises(NotImplementedError):
            y.backward(make_dual(torch.ones_like(y), torch.ones_like(y)))   # (nor of a gradient)


ATTENTION = [dict(), dict(bias=torch.zeros(1, 1, 64, 64)), dict(alibi_slopes=torch.ones(2))]


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("more", ATTENTION, ids=["plain", "bias", "slopes"])
@pytest.mark.filterwarnings("ignore:`torch.jit")
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_attention_under_transforms_is_refused(stand_in, requires_grad, more):
    """A trace of it would hold the outputs' allocation alone, its tangents would be lost."""
    x = tensors(requires_grad)
    call = lambda q, k, v: mx.triton_attention_mxfp4(q, k, v, causal=True, **more)[0]  # noqa: E731
    packed = lambda q, k, v: mx.triton_attention_mxfp4(*(t[0].transpose(0, 1) for t in (q, k, v)), causal=True, layout="thd", cu_seqlens_q=[0, 64], cu_seqlens_k=[0, 64])[0]  # noqa: E731
    for fn in (call, packed):
        with pytest.raises(NotImplementedError, match="torch.jit.trace"):
            torch.jit.trace(fn, tuple(x), check_trace=False)
        with pytest.raises(NotImplementedError, match="functorch"):
            torch.func.grad(lambda q: fn(q, *x[1:]).float().sum())(x[0].detach())
        with dual_level():
            for i in range(3):
                y = list(x)
                y[i] = make_dual(x[i], torch.ones_like(x[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(*y)
    with dual_level():
        for name, t in more.items():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                mx.triton_attention_mxfp4(*x, causal=True, **{name: make_dual(t, torch.ones_like(t))})
        if requires_grad:
            y = call(*x)
            with pytest.raises(NotImplementedError):
                y.backward(make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.filterwarnings("ignore:`torch.jit")
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_the_entry_points_on_codes_under_transforms_are_refused(stand_in):
    codes, scales, rows = torch.zeros(1, 2, 64, 32, dtype=torch.uint8), torch.zeros(1, 2, 2, 2, dtype=torch.uint8), tensors(False)[0]
    lse, bias = torch.zeros(1, 2, 64), torch.zeros(1, 1, 64, 64)
    operands = codes, codes, codes, scales, scales, scales
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(lambda go: mx.attention_mxfp4_backward(go, *operands, rows, lse, 0.1, True), rows, check_trace=False)
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(lambda bias: mx.attention_mxfp4_forward(*operands, 0.1, True, bias=bias), bias, check_trace=False)
    with pytest.raises(NotImplementedError, match="torch.jit.trace"):
        torch.jit.trace(lambda q: mx.quantize_qkv(q, rows, rows)[:2], rows, check_trace=False)
    with dual_level():
        for go, out in ((make_dual(rows, rows), rows), (rows, make_dual(rows, rows))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                mx.attention_mxfp4_backward(go, *operands, out, lse, 0.1, True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            mx.attention_mxfp4_forward(*operands, 0.1, True, bias=make_dual(bias, bias))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            mx.quantize_qkv(rows, rows, make_dual(rows, rows))


@pytest.mark.parametrize("of_q", [True, False])
@pytest.mark.parametrize("name", ["bias", "alibi_slopes"])
def test_the_gradient_of_an_additive_term_is_refused(stand_in, name, of_q):
    """Also where nothing else requires one: no result without a graph, no gradient left out."""
    x = tensors(False)
    x[0].requires_grad_(of_q)
    term = (torch.zeros(1, 1, 64, 64) if name == "bias" else torch.ones(2)).requires_grad_(True)
    y = mx.triton_attention_mxfp4(*x, causal=True, **{name: term})[0]
    with pytest.raises(NotImplementedError, match="detach"):
        y.sum().backward()
    with torch.no_grad():
        assert not mx.triton_attention_mxfp4(*x, causal=True, **{name: term})[0].requires_grad
    if of_q:
        y = mx.triton_attention_mxfp4(*x, causal=True, **{name: term.detach()})[0]
        assert bool((torch.autograd.grad(y.sum(), x[0])[0] == 2).all())


def test_the_gradient_of_slopes_is_refused_for_packed_sequences(stand_in):
    x = [t[0].transpose(0, 1) for t in tensors(False)]
    slopes = torch.ones(2, requires_grad=True)
    y = mx.triton_attention_mxfp4(*x, causal=True, alibi_slopes=slopes, layout="thd", cu_seqlens_q=[0, 64], cu_seqlens_k=[0, 64])[0]
    with pytest.raises(NotImplementedError, match="detach"):
        y.sum().backward()


@pytest.mark.parametrize("layout", ["bhsd", "bshd", "thd"])
def test_a_result_is_changed_in_place(stand_in, layout):
    """With a graph behind it as without one; a backward, which needs the output that was, then says so."""
    for requires_grad in (False, True):
        x = tensors(requires_grad)
        if layout == "thd":
            x = [t[0].transpose(0, 1) for t in x]
        more = dict(cu_seqlens_q=[0, 64], cu_seqlens_k=[0, 64]) if layout == "thd" else {}
        y = mx.triton_attention_mxfp4(*x, causal=True, layout=layout, **more)[0]
        assert y.is_contiguous()
        y.zero_().add_(2)   # (what stands in for the launch leaves memory as it was: anything)
        assert bool((y == 2).all())
        if requires_grad:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.sum().backward()
