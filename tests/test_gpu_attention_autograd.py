"""The attention's backward through its public entry points: every layout, the module with rotated positions, graphs and streams."""
import pytest
import torch

from tests.test_gpu_attention_backward import Operands, check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def m():
    import alto_amd.mxfp4 as mod
    return mod


def leaves(B, Hq, Hk, Sq, Sk, D, Dv, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g).to(dtype).to(DEV)  # noqa: E731
    return rand(B, Hq, Sq, D), rand(B, Hk, Sk, D), rand(B, Hk, Sk, Dv), rand(B, Hq, Sq, Dv).bfloat16()


def by_codes(m, q, k, v, go, causal, **kw):
    """Gradients through the entry points on codes."""
    qq, qs, kq, ks, vq, vs = m.quantize_qkv(q, k, v)
    out, lse, _ = m.triton_attention_mxfp4(q, k, v, causal=causal, **kw)
    return out, lse, m.attention_mxfp4_backward(go, qq, kq, vq, qs, ks, vs, out, lse, q.shape[-1] ** -0.5, causal, **kw)


def same(got, want):
    for a, b in zip(got, want):
        assert a.shape == b.shape and torch.equal(a, b)


CASES = [(2, 4, 2, 96, 96, 64, 64, True), (1, 2, 2, 64, 160, 128, 128, False), (1, 4, 1, 160, 160, 192, 128, True)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_autograd_gives_the_gradients_on_the_codes(m, case):
    *sizes, causal = case
    q, k, v, go = leaves(*sizes, seed=1)
    out, lse, want = by_codes(m, q, k, v, go, causal)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    y, lse2, _ = m.triton_attention_mxfp4(*x, causal=causal)
    assert torch.equal(y, out) and torch.equal(lse2, lse) and y.requires_grad and not lse2.requires_grad
    same(torch.autograd.grad(y, x, go), want)
    # the same in [B, S, H, D]
    x = [t.transpose(1, 2).contiguous().requires_grad_(True) for t in (q, k, v)]
    y, lse2, _ = m.triton_attention_mxfp4(*x, causal=causal, layout="bshd")
    assert torch.equal(y.transpose(1, 2), out) and torch.equal(lse2, lse)
    grads = torch.autograd.grad(y, x, go.transpose(1, 2))
    same([t.transpose(1, 2) for t in grads], want)
    assert all(t.is_contiguous() for t in grads)


def test_the_formula_end_to_end(m):
    """Gradients of the whole call against the 64-bit formula on the values of its codes, with the output and log-sum-exp that it left."""
    x = Operands(1, 4, 2, 128, 128, 128, 128, True, seed=3)
    q, k, v = (t.bfloat16().to(DEV).requires_grad_(True) for t in x.values)   # values on the grid: their codes are they
    out, lse, _ = m.triton_attention_mxfp4(q, k, v, causal=True)
    x.out, x.lse = out.detach().cpu(), lse.cpu()
    check(torch.autograd.grad(out, (q, k, v), x.go.to(DEV)), x.expected())


def test_packed_sequences(m):
    starts, Hq, Hk, D = [0, 64, 96, 320], 4, 2, 64
    q, k, v, go = leaves(1, Hq, Hk, 320, 320, D, D, seed=4)
    x = [t[0].transpose(0, 1).contiguous().requires_grad_(True) for t in (q, k, v)]
    out, lse, _ = m.triton_attention_mxfp4(*x, cu_seqlens_q=starts, cu_seqlens_k=starts, causal=True, layout="thd")
    with torch.no_grad():
        want, want_lse, _ = m.triton_attention_mxfp4(*x, cu_seqlens_q=starts, cu_seqlens_k=starts, causal=True, layout="thd")
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and out.stride() == want.stride() and lse.stride() == want_lse.stride()
    grads = torch.autograd.grad(out, x, go[0].transpose(0, 1))
    for a, b in zip(starts, starts[1:]):
        alone = by_codes(m, *(t[:, :, a:b].contiguous() for t in (q, k, v, go)), True)[2]
        same([t[a:b].transpose(0, 1)[None] for t in grads], alone)


def test_bias_slopes_and_a_padded_key_block(m):
    q, k, v, go = leaves(2, 4, 2, 64, 96, 64, 64, seed=5)
    bias = torch.randn(2, 1, 64, 96, device=DEV)
    bias[1, :, 3] = float("-inf")
    slopes = torch.rand(4, device=DEV)
    for kw in (dict(bias=bias), dict(alibi_slopes=slopes), dict(bias=bias, alibi_slopes=slopes)):
        out, lse, want = by_codes(m, q, k, v, go, False, **kw)
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        y, lse2, _ = m.triton_attention_mxfp4(*x, causal=False, **kw)
        assert torch.equal(y.nan_to_num(), out.nan_to_num()) and torch.equal(lse2, lse)
        grads = torch.autograd.grad(y, x, go)
        same(grads, want)
        assert all(bool(torch.isfinite(t).all()) for t in grads)
        if "bias" in kw:
            assert bool((grads[0][1, :, 3] == 0).all())
    y = m.triton_attention_mxfp4(*x, bias=bias.requires_grad_(True), causal=False)[0]   # (runs; its gradient is refused)
    with pytest.raises(NotImplementedError):
        y.backward(go)


def test_fp32_inputs_and_some_of_the_gradients(m):
    q, k, v, go = leaves(1, 2, 1, 64, 64, 64, 64, seed=6, dtype=torch.float32)
    want = by_codes(m, q, k, v, go, True)[2]
    for needed in ((True, True, True), (True, False, False), (False, True, False), (False, False, True)):
        x = [t.clone().requires_grad_(n) for t, n in zip((q, k, v), needed)]
        out, _, _ = m.triton_attention_mxfp4(*x, causal=True)
        out.backward(go)
        for t, n, w in zip(x, needed, want):
            assert (t.grad is not None) == n
            if n:
                assert t.grad.dtype == torch.float32 and torch.equal(t.grad, w.float())


def test_a_sum_and_a_second_derivative(m):
    q, k, v, go = leaves(1, 2, 2, 32, 32, 64, 64, seed=7)
    want = by_codes(m, q, k, v, torch.ones_like(go), True)[2]
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(m.triton_attention_mxfp4(*x, causal=True)[0].sum(), x, create_graph=True)
    same(grads, want)
    with pytest.raises(RuntimeError):
        grads[0].sum().backward()


def test_the_module_with_rotated_positions(m):
    """Rotation, attention and both backwards as a block runs them: bit for bit the operators one after the other."""
    B, S, Hq, Hk, D = 2, 96, 4, 2, 128
    q, k, v, go = (t.transpose(1, 2).contiguous() for t in leaves(B, Hq, Hk, S, S, D, D, seed=8))
    freq, factor = m.rotary_frequencies(D, scaling=dict(type="yarn", factor=8, original_length=4096), device=DEV)
    positions = torch.arange(5, 5 + S, device=DEV)
    attention = m.LPScaledDotProductAttention(m.TrainingOpConfig())
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = attention(*x, is_causal=True, rotary=m.Rotary(freq, positions, factor=factor))
    grads = torch.autograd.grad(out, x, go)
    q2, k2 = m.apply_rotary(q, k, freq, positions, factor=factor, layout="bshd")
    assert torch.equal(out, attention(q2, k2, v, is_causal=True))
    want = by_codes(m, *(t.transpose(1, 2) for t in (q2, k2, v, go)), True)[2]
    assert torch.equal(grads[2].transpose(1, 2), want[2])
    leaf_q, leaf_k = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    rotated = m.apply_rotary(leaf_q, leaf_k, freq, positions, factor=factor, layout="bshd")
    same(grads[:2], torch.autograd.grad(rotated, (leaf_q, leaf_k), tuple(t.transpose(1, 2) for t in want[:2])))
    with torch.no_grad():
        assert torch.equal(attention(q, k, v, is_causal=True, rotary=m.Rotary(freq, positions, factor=factor)), out)


def test_a_captured_step_is_replayed(m):
    """Forward and backward in one graph, replayed on new contents with eager steps of the same leaves between the replays."""
    q, k, v, go = leaves(1, 4, 2, 160, 160, 64, 64, seed=9)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    freq = m.rotary_frequencies(64, device=DEV)[0]

    def step():
        a, b = m.apply_rotary(x[0], x[1], freq)
        out = m.triton_attention_mxfp4(a, b, x[2], causal=True)[0]
        return out.detach(), *torch.autograd.grad(out, x, go)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            for t in x:
                t.normal_()
        go.normal_()
        graph.replay()
        torch.cuda.synchronize()
        same(got, step())


def test_two_steps_at_once(m):
    """Two streams, a call in flight on either."""
    a, b = (leaves(2, 8, 2, 256, 256, 128, 128, seed=s) for s in (10, 11))
    want = [by_codes(m, *x, True)[2] for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for x, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(by_codes(m, *x, True)[2])
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        same(g, want[i % 2])


def test_offsets_beyond_32_bits(m):
    """More than 2^31 elements in Q, dO and dQ: the last batch's gradients are those of its own call."""
    B, H, S, D = 8200, 64, 32, 128
    g = torch.Generator(device=DEV).manual_seed(0)
    codes = lambda *shape: torch.randint(0, 256, shape, dtype=torch.uint8, device=DEV, generator=g)  # noqa: E731
    q, k, v = codes(B, H, S, D // 2), codes(B, 1, S, D // 2), codes(B, 1, D, S // 2)
    scale = lambda heads: torch.full((B, heads, 1, D // 32), 125, dtype=torch.uint8, device=DEV)  # noqa: E731
    out, lse = m.attention_mxfp4_forward(q[:1], torch.cat([k[:1], k[:1]], 2), torch.cat([v[:1], v[:1]], 3), scale(H)[:1], torch.cat([scale(1)[:1]] * 2, 2),
                                         torch.cat([scale(1)[:1]] * 2, 2), D ** -0.5, True, seqlen_k=32)
    out, lse = out.expand(B, H, S, D), lse.expand(B, H, S)   # (any output will do, of all batches the same)
    go = torch.empty((B, H, S, D), dtype=torch.bfloat16, device=DEV)
    go[-1].normal_(generator=g)
    go[:-1] = 0.5
    got = m.attention_mxfp4_backward(go, q, k, v, scale(H), scale(1), scale(1), out, lse, D ** -0.5, True)
    last = slice(B - 1, B)
    want = m.attention_mxfp4_backward(go[last], q[last], k[last], v[last], scale(H)[last], scale(1)[last], scale(1)[last], out[last], lse[last], D ** -0.5, True)
    same([t[last] for t in got], want)


def test_refusals(m):
    q, k, v, go = leaves(1, 2, 2, 32, 32, 64, 64, seed=12)
    qq, qs, kq, ks, vq, vs = m.quantize_qkv(q, k, v)
    out, lse, _ = m.triton_attention_mxfp4(q, k, v, causal=True)
    args = [go, qq, kq, vq, qs, ks, vs, out, lse, 0.125, True]

    def refused(error, **at):
        changed = [at.get(f"a{i}", a) for i, a in enumerate(args)]
        with pytest.raises(error):
            m.attention_mxfp4_backward(*changed, **{n: x for n, x in at.items() if not n.startswith("a")})

    refused(AssertionError, a0=go.float())
    refused(AssertionError, a0=go[:, :, :16])
    refused(AssertionError, a1=qq[:, :1])
    refused(AssertionError, a8=lse.double())
    refused(AssertionError, a9=0.0)
    refused(AssertionError, a9=-1.0)
    refused(AssertionError, seqlen_k=16)
    refused(AssertionError, seqlen_k=0)
    refused(AssertionError, cu_seqlens_q=[0, 32])
    refused(AssertionError, cu_seqlens_q=[0, 16, 32], cu_seqlens_k=[0, 16, 32])
    refused(AssertionError, cu_seqlens_q=[0, 64], cu_seqlens_k=[0, 64])
    refused(RuntimeError, bias=torch.zeros(1, 1, 32, 33, device=DEV))
    refused(AssertionError, bias=torch.zeros(1, 1, 32, 32, device=DEV), cu_seqlens_q=[0, 32], cu_seqlens_k=[0, 32])
    refused(RuntimeError, a0=go.cpu())
    y = m.triton_attention_mxfp4(q.requires_grad_(True), k, v, sm_scale=0.0)[0]   # (the mean of the values that a row sees)
    with pytest.raises(AssertionError):
        y.backward(go)
