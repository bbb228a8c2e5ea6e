"""Rotary positions (through the C ABI) against the rotation in 64 bits.

Tolerance: half a step of the result's type, and of fp32 the roundings of cosine, sine, two products and a sum: four of 2^-24 of |c x1| + |s x2|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def m():
    import alto_amd.mxfp4 as mod
    return mod


def expected(x, inv_freq, positions, interleaved, factor, layout, inverse=False):
    """(rotated, bound) of a CPU tensor, fp64."""
    R = 2 * inv_freq.shape[0]
    angle = positions.double()[..., None] * inv_freq.double()
    c, s = torch.cos(angle) * factor, torch.sin(angle) * factor * (-1 if inverse else 1)
    c, s = (t.unsqueeze(-3 if layout == "bhsd" else -2) for t in (c, s))
    f = x.double()
    a, b = (f[..., 0:R:2], f[..., 1:R:2]) if interleaved else (f[..., :R // 2], f[..., R // 2:R])
    y, size = (c * a - s * b, s * a + c * b), ((c * a).abs() + (s * b).abs(), (s * a).abs() + (c * b).abs())
    join = (lambda t: torch.stack(t, -1).flatten(-2)) if interleaved else (lambda t: torch.cat(t, -1))
    rest = f[..., R:]
    y = torch.cat((join(y), rest), -1)
    bound = torch.cat((join(size) * 4 * 2.0 ** -24, torch.zeros_like(rest)), -1)
    step = torch.finfo(x.dtype).eps / 2
    bound[..., :R] += step * y[..., :R].abs() + 1e-30
    return y, bound


def check(got, x, *args, **kw):
    y, bound = expected(x, *args, **kw)
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.cpu().double() - y).abs()
    assert bool((off <= bound).all()), float((off - bound).max())


def shape(layout, B, S, H, D):
    return {"bhsd": (B, H, S, D), "bshd": (B, S, H, D), "thd": (S, H, D)}[layout]


def tensors(layout, B, S, Hq, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape(layout, B, S, h, D), generator=g).to(dtype) for h in (Hq, Hk)]


CASES = [
    # layout, B, S, Hq, Hk, D, R
    ("bhsd", 1, 1, 1, 1, 64, 64),
    ("bshd", 2, 17, 4, 2, 128, 128),
    ("thd", 1, 33, 8, 1, 64, 32),
    ("bshd", 3, 5, 3, 1, 80, 20),        # half of R no multiple of 8
    ("bhsd", 2, 7, 2, 2, 66, 66),        # pairs 33 apart
    ("bhsd", 1, 9, 1, 1, 7, 2),          # an odd head
    ("bshd", 1, 1030, 6, 2, 96, 48),
    ("bshd", 2, 2500, 5, 3, 192, 192),   # several tokens a workgroup, the last with fewer
    ("bshd", 16, 1, 32, 8, 128, 128),    # single tokens: their heads are dealt out
    ("bshd", 1, 1, 64, 8, 256, 64),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_rotation_and_its_gradient(m, case, dtype, interleaved):
    layout, B, S, Hq, Hk, D, R = case
    q, k = tensors(layout, B, S, Hq, Hk, D, dtype, seed=S)
    freq, _ = m.rotary_frequencies(R)
    positions = torch.arange(S)
    qd, kd = (t.to(DEV).requires_grad_(True) for t in (q, k))
    q2, k2 = m.apply_rotary(qd, kd, freq.to(DEV), interleaved=interleaved, factor=1.25, layout=layout)
    check(q2.detach(), q, freq, positions, interleaved, 1.25, layout)
    check(k2.detach(), k, freq, positions, interleaved, 1.25, layout)
    gq, gk = tensors(layout, B, S, Hq, Hk, D, dtype, seed=S + 1)
    dq, dk = torch.autograd.grad((q2, k2), (qd, kd), (gq.to(DEV), gk.to(DEV)))
    check(dq, gq, freq, positions, interleaved, 1.25, layout, inverse=True)
    check(dk, gk, freq, positions, interleaved, 1.25, layout, inverse=True)


def test_gradient_equals_differences(m):
    """The rotation is linear: <dq, x> is the difference of <g, rotated> between q + x and q, to fp32's rounding of sums of 320 terms of order 1."""
    q, k = tensors("bshd", 1, 5, 2, 1, 32, torch.float32)
    g, x = tensors("bshd", 1, 5, 2, 2, 32, torch.float32, seed=1)
    freq = m.rotary_frequencies(16)[0].to(DEV)
    qd = q.to(DEV).requires_grad_(True)
    y = m.apply_rotary(qd, None, freq, layout="bshd")
    (dq,) = torch.autograd.grad(y, qd, g.to(DEV))
    moved = m.apply_rotary((q + x).to(DEV), None, freq, layout="bshd")
    assert abs(float((dq.cpu().double() * x.double()).sum() - ((moved - y.detach()).cpu().double() * g.double()).sum())) < 320 * 8 * 2 ** -24 * 4


@pytest.mark.parametrize("kind", ["int32", "int64", "batch", "one batch", "negative", "far"])
def test_positions(m, kind):
    B, S = 3, 40
    q, k = tensors("bshd", B, S, 4, 2, 64, torch.float32, seed=2)
    g = torch.Generator().manual_seed(3)
    positions = torch.randint(0, 5000, (S,), generator=g)
    if kind == "int32":
        positions = positions.int()
    if kind == "batch":
        positions = torch.randint(0, 5000, (S, B), generator=g).t()   # rows not of unit stride
    if kind == "one batch":
        positions = positions[None]
    if kind == "negative":
        positions = -positions
    if kind == "far":
        positions = torch.tensor([2 ** 31 - 1, 2 ** 40 + 12345] * (S // 2))   # (the angle is rounded to 64 bits on either side alike)
    freq, factor = m.rotary_frequencies(64, base=500000.0, scaling=dict(type="yarn", factor=4, original_length=4096))
    got = m.apply_rotary(q.to(DEV), k.to(DEV), freq.to(DEV), positions.to(DEV), factor=factor, layout="bshd")
    for y, x in zip(got, (q, k)):
        check(y, x, freq, positions, False, factor, "bshd")


def test_inputs_of_any_layout(m):
    freq = m.rotary_frequencies(64)[0].to(DEV)
    g = torch.Generator().manual_seed(5)
    whole = torch.randn(2, 21, 10, 64, generator=g).bfloat16().to(DEV)      # heads of Q, K and V of one projection
    q, k = whole[:, :, :6], whole[:, :, 6:8]
    want = m.apply_rotary(q.contiguous(), k.contiguous(), freq, layout="bshd")
    for a, b in zip(m.apply_rotary(q, k, freq, layout="bshd"), want):
        assert torch.equal(a, b)
    for a, b in zip(m.apply_rotary(q.transpose(1, 2), k.transpose(1, 2), freq, layout="bhsd"), want):
        assert torch.equal(a.transpose(1, 2), b)
    one = k[:, :, :1].expand(2, 21, 4, 64)                                  # a head for all: stride 0
    assert torch.equal(m.apply_rotary(one, None, freq, layout="bshd"), want[1][:, :, :1].expand(2, 21, 4, 64))
    odd = torch.empty(2 * 21 * 6 * 64 + 3, dtype=torch.bfloat16, device=DEV)[3:].view(2, 21, 6, 64)   # not aligned
    odd.copy_(q)
    assert torch.equal(m.apply_rotary(odd, None, freq, layout="bshd"), want[0])
    turned = q.transpose(2, 3).contiguous().transpose(2, 3)                 # no unit stride along the head
    assert torch.equal(m.apply_rotary(turned, None, freq, layout="bshd"), want[0])
    empty = torch.empty(2, 0, 6, 64, dtype=torch.bfloat16, device=DEV)
    assert m.apply_rotary(empty, None, freq, layout="bshd").shape == (2, 0, 6, 64)


def test_gradients_of_one_of_the_two_and_of_a_sum(m):
    q, k = (t.to(DEV) for t in tensors("bhsd", 1, 6, 2, 2, 32, torch.float32))
    freq = m.rotary_frequencies(32)[0].to(DEV)
    ones = torch.ones(1, 2, 6, 32)
    for x, y in ((0, 1), (1, 0)):
        leaves = [q.clone(), k.clone()]
        leaves[x].requires_grad_(True)
        m.apply_rotary(*leaves, freq)[x].sum().backward()     # (the gradient of a sum has strides of 0)
        check(leaves[x].grad, ones, freq.cpu(), torch.arange(6), False, 1.0, "bhsd", inverse=True)
        assert leaves[y].grad is None


def test_offsets_beyond_32_bits(m):
    H, D, S = 64, 128, 2 ** 18 + 40
    q = torch.empty((1, S, H, D), dtype=torch.bfloat16, device=DEV)
    q.view(-1)[: 2 ** 20].normal_()
    q[:, -8:].normal_()
    freq = m.rotary_frequencies(D)[0].to(DEV)
    y = m.apply_rotary(q, None, freq, layout="bshd")
    last = torch.arange(S - 8, S)
    check(y[:, -8:], q[:, -8:].cpu(), freq.cpu(), last, False, 1.0, "bshd")
    check(y[:, :8], q[:, :8].cpu(), freq.cpu(), torch.arange(8), False, 1.0, "bshd")


def test_captured_and_on_another_stream(m):
    """Three replays with new contents of the captured inputs, positions among them, and eager work between them."""
    q, k = (t.to(DEV) for t in tensors("bshd", 2, 19, 4, 2, 64, torch.bfloat16))
    freq, positions = m.rotary_frequencies(64)[0].to(DEV), torch.arange(19, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = m.apply_rotary(q, k, freq, positions, layout="bshd")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.apply_rotary(q, k, freq, positions, layout="bshd")
    for i in range(3):
        q.normal_()
        k.normal_()
        positions += 1000 * i
        graph.replay()
        want = m.apply_rotary(q, k, freq, positions, layout="bshd")
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert eager[0].shape == q.shape


def test_refusals(m):
    q = torch.zeros(1, 2, 4, 8, dtype=torch.bfloat16, device=DEV)
    freq = m.rotary_frequencies(8)[0].to(DEV)
    with pytest.raises(AssertionError):
        m.apply_rotary(q.half(), None, freq)
    with pytest.raises(AssertionError):
        m.apply_rotary(q, q.float(), freq)
    with pytest.raises(AssertionError):
        m.apply_rotary(q, None, freq.float())
    with pytest.raises(AssertionError):
        m.apply_rotary(q, None, m.rotary_frequencies(10)[0].to(DEV))
    with pytest.raises(AssertionError):
        m.apply_rotary(q, q[:, :, :3], freq)
    with pytest.raises(AssertionError):
        m.apply_rotary(q, None, freq, torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(AssertionError):
        m.apply_rotary(q, None, freq, torch.zeros(4, device=DEV))
    with pytest.raises(NotImplementedError):
        m.apply_rotary(q, None, freq, layout="sbhd")
    with pytest.raises(RuntimeError):
        m.apply_rotary(q, None, freq.cpu())
    with pytest.raises(AssertionError):
        m.apply_rotary(q[:, :0], q, freq)
    with pytest.raises(NotImplementedError):
        m.apply_rotary(q, q, freq.clone().requires_grad_(True))


def test_nothing_to_rotate(m):
    """No tokens, no sequences, no heads of K: as empty as they came."""
    freq = m.rotary_frequencies(8)[0].to(DEV)
    q = torch.randn(2, 3, 5, 8, dtype=torch.bfloat16, device=DEV)
    for a, b in ((q[:0], q[:0]), (q[:, :, :0], q[:, :1, :0])):
        got = m.apply_rotary(a, b, freq)
        assert got[0].shape == a.shape and got[1].shape == b.shape
    got = m.apply_rotary(q, q[:, :0], freq)
    assert torch.equal(got[0], m.apply_rotary(q, None, freq)) and got[1].numel() == 0


def test_native_call_and_python_function_are_the_same(m, monkeypatch):
    """What the native call declines takes the Python function's way, with the same bits; the second derivative through either is the rotation."""
    from alto_amd.mxfp4 import _runtime as rt
    q, k = (t.to(DEV) for t in tensors("bshd", 2, 9, 4, 2, 64, torch.bfloat16))
    g, h = (t.to(DEV) for t in tensors("bshd", 2, 9, 4, 2, 64, torch.bfloat16, seed=1))
    freq, positions = m.rotary_frequencies(32)[0].to(DEV), torch.arange(9, 18, device=DEV)

    def everything():
        x, y = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        a, b = m.apply_rotary(x, y, freq, positions, interleaved=True, factor=0.5, layout="bshd")
        u = g.clone().requires_grad_(True)
        dx, dy = torch.autograd.grad((a, b), (x, y), (u, h), create_graph=True)
        (du,) = torch.autograd.grad(dx, u, q)
        return a.detach(), b.detach(), dx.detach(), dy, du, a.grad_fn.name()

    native = everything()
    calls = rt.host()

    class Declines:
        def __getattr__(self, name):
            return (lambda *a: None) if name == "rotary" else getattr(calls, name)

    monkeypatch.setattr(rt, "host", lambda: Declines())
    general = everything()
    assert native[-1] != general[-1]
    for a, b in zip(native[:-1], general[:-1]):
        assert torch.equal(a, b)
    assert torch.equal(native[4], native[0])   # d<R^T u, q>/du = R q
