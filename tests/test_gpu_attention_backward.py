"""Gradients of the MXFP4 attention (through the C ABI) against the 64-bit formula on the values of the same codes.

Tolerance: element by element what the oracle derives (half steps of bf16 at P, dS and the result, fp32 arithmetic between them)."""
import pytest
import torch

from oracle import mxfp4_oracle as O
from oracle.attention_oracle import attention_bwd_ref, attention_probabilities

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def m():
    import alto_amd.mxfp4 as mod
    return mod


class Operands:
    """Quantized Q, K, V with their values, and what an exact forward leaves of them."""

    def __init__(self, B, Hq, Hk, Sq, Sk, D, Dv, causal, seed, bias=None, alibi_slopes=None, magnitude=1.0, used=None):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *shape: torch.randn(shape, generator=g)  # noqa: E731
        q, k, v = (magnitude * rand(B, Hq, Sq, D)).bfloat16(), rand(B, Hk, Sk, D).bfloat16(), rand(B, Hk, Sk, Dv).bfloat16()
        self.q, self.qs = O.quantize(q, axis=-1, is_2d_block=True)
        self.k, self.ks = O.quantize(k, axis=-1, is_2d_block=True)
        vq, self.vs = O.quantize(v, axis=-1, is_2d_block=True)
        self.v, _ = O.quantize(v.transpose(-1, -2).contiguous(), axis=-1, is_2d_block=True)
        back = lambda c, s: O.dequantize(c, s, torch.float32, axis=-1, is_2d_block=True)  # noqa: E731
        used = Sk if used is None else used
        self.values = back(self.q, self.qs), back(self.k, self.ks)[:, :, :used], back(vq, self.vs)[:, :, :used]
        self.more = dict(causal=causal, sm_scale=D ** -0.5, bias=bias, alibi_slopes=alibi_slopes)
        _, out, lse = attention_probabilities(*self.values, **self.more)
        self.out, self.lse = out.bfloat16(), lse.float()
        self.go = rand(B, Hq, Sq, Dv).bfloat16()

    def expected(self):
        return attention_bwd_ref(self.go.cpu(), *self.values, self.out.cpu(), self.lse, **self.more)

    def call(self, m, **kw):
        put = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        args = [put(t) for t in (self.go, self.q, self.k, self.v, self.qs, self.ks, self.vs, self.out, self.lse)]
        return m.attention_mxfp4_backward(*args, self.more["sm_scale"], self.more["causal"], bias=put(self.more["bias"]),
                                          alibi_slopes=put(self.more["alibi_slopes"]), **kw)


def check(got, ref, what=""):
    for name, x, exact, bound in zip(("dq", "dk", "dv"), got, ref[:3], ref[3:]):
        assert x.dtype == torch.bfloat16 and x.shape == exact.shape, (what, name, x.shape, exact.shape)
        off = (x.cpu().double() - exact).abs() / bound
        assert float(off.max()) <= 1.0, f"{what} {name}: {int((off > 1).sum())} of {off.numel()} out of bounds, worst {float(off.max()):.3g} at {tuple((off == off.max()).nonzero()[0].tolist())}"


CASES = [
    # B, Hq, Hk, Sq, Sk, D, Dv, causal
    (1, 1, 1, 32, 32, 64, 64, False),
    (1, 1, 1, 32, 32, 64, 64, True),
    (1, 2, 1, 64, 64, 128, 128, True),
    (2, 4, 4, 96, 96, 64, 128, True),
    (1, 4, 2, 128, 160, 128, 64, True),        # Sq < Sk: the mask is aligned to the bottom-right corner
    (1, 8, 1, 256, 256, 128, 128, True),
    (2, 2, 2, 224, 64, 64, 64, False),         # more rows than keys
    (1, 3, 1, 32, 544, 128, 128, True),        # one tile of rows, keys over several workgroups
    (1, 2, 2, 96, 128, 192, 128, False),
    (1, 3, 3, 160, 320, 192, 64, True),
    (1, 2, 1, 64, 192, 256, 128, False),
    (1, 5, 5, 288, 288, 256, 64, True),
    (1, 2, 1, 64, 2080, 64, 64, False),        # few rows: their lists of keys in several parts
    (2, 1, 1, 96, 1504, 128, 128, True),
    (1, 1, 1, 32, 3200, 192, 64, True),
    (1, 4, 1, 1280, 96, 64, 128, False),       # few keys: their lists of rows in several parts
    (1, 2, 1, 1312, 1344, 256, 128, True),     # both, of blocks that differ
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c)))
def test_gradients_match_the_formula(m, case):
    x = Operands(*case, seed=sum(case))
    check(x.call(m), x.expected())


@pytest.mark.parametrize("case", [(2, 4, 2, 96, 160, 128, 128, False), (2, 2, 2, 64, 64, 64, 64, True), (1, 2, 1, 64, 96, 192, 128, False), (1, 2, 1, 32, 64, 256, 64, True), (1, 1, 1, 96, 1600, 128, 64, True)],
                         ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("extra", ["bias", "alibi", "both"])
def test_additive_terms(m, case, extra):
    B, Hq, Hk, Sq, Sk, D, Dv, causal = case
    g = torch.Generator().manual_seed(5)
    bias = alibi = None
    if extra != "alibi":   # keys hidden here and there, one sequence's first row without any
        bias = torch.randn(B, 1, Sq, Sk, generator=g).masked_fill(torch.rand(B, 1, Sq, Sk, generator=g) < 0.3, float("-inf"))
        bias[-1, :, 0] = float("-inf")
        bias[0, :, :, 0] = 0.0
    if extra != "bias":
        alibi = torch.rand(B, Hq, generator=g)
    x = Operands(*case, seed=6, bias=bias, alibi_slopes=alibi)
    got = x.call(m)
    check(got, x.expected(), extra)
    if bias is not None:
        assert bool((got[0][-1, :, 0] == 0).all())


@pytest.mark.parametrize("case", [(2, 4, 2, 96, 160, 128, 64, True), (2, 2, 2, 160, 192, 192, 128, False), (1, 2, 1, 64, 1280, 64, 64, True)],
                         ids=lambda c: "x".join(map(str, c)))
def test_a_bias_of_any_layout(m, case):
    """Broadcast rows, batches and heads, a part of something larger at an odd place with rows an odd number of elements apart: the bits of its dense copy."""
    B, Hq, _, Sq, Sk, *_ = case
    g = torch.Generator().manual_seed(8)
    held = torch.randn(B, Hq, Sq, Sk + 3, generator=g).to(DEV)
    for bias in (held[:, :, :, 1:-2], held[:, :1, :, 3:], held[:1, :, :1, :-3].expand(B, Hq, Sq, Sk), held[:1, 1:2, :, 2:-1]):
        assert bias.shape[-1] == Sk
        x = Operands(*case, seed=9, bias=bias.cpu())
        x.more["bias"] = bias
        got = x.call(m)
        x.more["bias"] = bias.expand(B, Hq, Sq, Sk).contiguous()
        for a, b in zip(got, x.call(m)):
            assert torch.equal(a, b)
        x.more["bias"] = bias.cpu()
        check(got, x.expected())


@pytest.mark.parametrize("Sk,biased", [(64, True), (64, False), (96, True), (32, False)])
def test_many_workgroups_of_short_lists(m, Sk, biased):
    """Several workgroups after one another on every unit, whose waves drift apart from the first tile on."""
    g = torch.Generator().manual_seed(15)
    x = Operands(2, 16, 4, 1024, Sk, 128, 128, False, seed=14, bias=torch.randn(2, 1, 1024, Sk, generator=g) if biased else None)
    ref = x.expected()
    for _ in range(4):
        check(x.call(m), ref)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_bias_of_extreme_values(m, D):
    """Where the mask hides a key the bias may hold anything; the type's lowest value hides like -inf, in rows that see nothing too; a row that sees
    nothing but keys at -1e9, whose lse has no bits left for its scores, keeps probabilities of at most one."""
    case = (1, 2, 1, 96, 160, D, 64, True)
    Sq, Sk = case[3:5]
    g = torch.Generator().manual_seed(10)
    hidden = torch.arange(Sk)[None, :] > torch.arange(Sq)[:, None] + Sk - Sq
    bias = torch.randn(1, 2, Sq, Sk, generator=g).masked_fill(torch.rand(1, 2, Sq, Sk, generator=g) < 0.3, float("-inf"))
    bias[:, :, 5] = bias[:, 1, 40:] = float("-inf")
    bias[:, 0, :, 0] = 0.0
    bias[:, 0, 5] = float("-inf")
    x = Operands(*case, seed=12, bias=bias)
    want = x.call(m)
    check(want, x.expected())
    assert bool((want[0][:, :, 5] == 0).all()) and bool((want[0][:, 1, 40:] == 0).all())
    for fill in (float("nan"), float("inf"), torch.finfo(torch.float32).max):
        x.more["bias"] = bias.masked_fill(hidden, fill)
        for a, b in zip(x.call(m), want):
            assert torch.equal(a, b)
    x.go[:, :, 5] = x.out[:, :, 5] = float("nan")   # nor does what a row holds that sees nothing
    for a, b in zip(x.call(m), want):
        assert torch.equal(a, b)
    x.more["bias"] = bias.masked_fill(bias == float("-inf"), torch.finfo(torch.float32).min)
    for a, b in zip(x.call(m), want):
        assert torch.equal(a, b)
    bias[:, :, 7] = -1e9
    y = Operands(*case, seed=12, bias=bias)
    dq, dk, dv = y.call(m)
    assert all(bool(t.isfinite().all()) for t in (dq, dk, dv))
    limit = y.go.double().abs().sum((1, 2))   # (of the key's only head: every probability at most 1, and half a step of bf16 at it and at the result)
    assert bool((dv.cpu().double().abs().amax((1, 2)) <= limit * (1 + 2.0 ** -7)).all())


@pytest.mark.parametrize("causal", [True, False])
def test_packed_sequences_are_the_sequences_alone(m, causal):
    """Lengths of one tile, of odd numbers of tiles and of more than a workgroup's block; each sequence's gradients bit for bit those of its own call."""
    Hq, Hk, D, Dv = 4, 2, 128, 64
    lens_q, lens_k = [32, 96, 288, 160, 64], [32, 96, 288, 224, 1600] if causal else [64, 32, 96, 160, 1600]
    parts = [Operands(1, Hq, Hk, a, b, D, Dv, causal, seed=a + b) for a, b in zip(lens_q, lens_k)]
    cat = lambda name, dim: torch.cat([getattr(p, name) for p in parts], dim).contiguous()  # noqa: E731
    whole = Operands.__new__(Operands)
    whole.go, whole.out, whole.lse = cat("go", 2), cat("out", 2), cat("lse", 2)
    whole.q, whole.qs, whole.k, whole.ks, whole.v, whole.vs = cat("q", 2), cat("qs", 2), cat("k", 2), cat("ks", 2), cat("v", 3), cat("vs", 2)
    whole.more = dict(parts[0].more)
    starts = lambda lens: [0] + torch.tensor(lens).cumsum(0).tolist()  # noqa: E731
    cu_q, cu_k = starts(lens_q), starts(lens_k)
    got = whole.call(m, cu_seqlens_q=cu_q, cu_seqlens_k=torch.tensor(cu_k, dtype=torch.int32))
    for i, p in enumerate(parts):
        rows, keys = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
        mine = got[0][:, :, rows], got[1][:, :, keys], got[2][:, :, keys]
        check(mine, p.expected(), f"sequence {i}")
        if max(lens_k[i] // 32, lens_q[i] // 32 * Hq // Hk) <= 24:   # (longer lists of tiles are cut as the whole call asks for it)
            for a, b in zip(mine, p.call(m)):
                assert torch.equal(a, b)


def test_more_sequences_than_one_launch_takes(m):
    n, Hq, Hk, D = 67, 2, 1, 64
    x = Operands(n, Hq, Hk, 32, 32, D, D, True, seed=11)
    tokens = lambda t: t.transpose(0, 1).reshape(1, t.shape[1], n * t.shape[2], *t.shape[3:]).contiguous()  # noqa: E731
    y = Operands.__new__(Operands)
    y.go, y.out, y.lse, y.q, y.qs, y.k, y.ks = (tokens(t) for t in (x.go, x.out, x.lse, x.q, x.qs, x.k, x.ks))
    y.v, y.vs = x.v.permute(1, 2, 0, 3).reshape(1, Hk, D, n * 16).contiguous(), tokens(x.vs)
    y.more = x.more
    starts = list(range(0, 32 * n + 1, 32))
    got = y.call(m, cu_seqlens_q=starts, cu_seqlens_k=starts)
    for a, b in zip(got, x.call(m)):
        assert torch.equal(a, tokens(b))
    check(x.call(m), x.expected())


def test_keys_behind_the_used_ones_get_zeros(m):
    """A sequence of 96 keys among 256 that are allocated: whole workgroups of keys have nothing to sum."""
    for causal in (False, True):
        x = Operands(1, 2, 1, 64, 256, 64, 64, causal, seed=4, used=96)
        got = x.call(m, seqlen_k=96)
        check((got[0], got[1][:, :, :96], got[2][:, :, :96]), x.expected())
        assert bool((got[1][:, :, 96:] == 0).all()) and bool((got[2][:, :, 96:] == 0).all())


def test_gradients_of_the_output_in_any_layout(m):
    """grad_out and out as views: [B, S, H, D] memory, rows apart, one row for all (a sum's gradient), an odd offset (copied)."""
    x = Operands(2, 4, 2, 96, 96, 64, 64, True, seed=8)
    want = x.call(m)
    x.out = x.out.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((2, 4, 96, 80), float("nan"), dtype=torch.bfloat16, device=DEV)
    keep = x.go
    for view in (wide[..., :64], wide[..., 8:72], wide[..., 3:67]):
        view.copy_(keep)
        x.go = view
        for a, b in zip(x.call(m), want):
            assert torch.equal(a, b)
    x.go = torch.ones(1, 1, 1, 1, dtype=torch.bfloat16).expand(2, 4, 96, 64)
    check(x.call(m), x.expected())


def test_large_scores_and_probabilities_of_one(m):
    """Scores of some hundreds: a row's probability sits on one key, the others' underflow."""
    x = Operands(1, 2, 1, 128, 128, 128, 128, True, seed=21, magnitude=40.0)
    check(x.call(m), x.expected())


def test_results_do_not_change_from_run_to_run(m):
    x = Operands(2, 8, 2, 256, 256, 128, 128, True, seed=2)
    first = x.call(m)
    for _ in range(3):
        for a, b in zip(x.call(m), first):
            assert torch.equal(a, b)


def test_a_head_of_more_than_2_gb(m):
    """Keys whose rows of 512 bytes lie behind 2^31 bytes: all keys but the first and the last are zeros, which change no sum, so that the gradients
    are those of the two alone."""
    edge, Sk, D, Dv = 64, (1 << 22) + 128, 256, 64
    x = Operands(1, 1, 1, 32, 2 * edge, D, Dv, False, seed=13)
    want = x.call(m)
    y = Operands.__new__(Operands)
    y.more, y.go, y.out, y.lse, y.q, y.qs = x.more, x.go, x.out, x.lse, x.q, x.qs

    def spread(t, dim, edge):
        size = list(t.shape)
        size[dim] = size[dim] // 2 * (Sk // 64)
        big = torch.zeros(size, dtype=t.dtype, device=DEV)
        big.narrow(dim, 0, edge).copy_(t.narrow(dim, 0, edge))
        big.narrow(dim, size[dim] - edge, edge).copy_(t.narrow(dim, edge, edge))
        return big

    y.k, y.ks, y.v, y.vs = spread(x.k, 2, edge), spread(x.ks, 2, edge // 32), spread(x.v, 3, edge // 2), spread(x.vs, 2, edge // 32)
    dq, dk, dv = y.call(m)
    assert dk.shape[2] == Sk and torch.equal(dq, want[0])
    for got, exact in ((dk, want[1]), (dv, want[2])):
        assert torch.equal(got[:, :, :edge], exact[:, :, :edge]) and torch.equal(got[:, :, -edge:], exact[:, :, edge:])
