"""Workloads of the operators that train through attention: its backward pass on MXFP4 operands, and rotary positions.

``attention``  the gradients of Q, K and V from those of the output: the probabilities are recomputed from the quantized
               operands and the forward's log-sum-exp.  E2M1 codes with one E8M0 scale for each 32 x 32 block, as the forward takes
               them; grouped-query heads, causal or not, ALiBi slopes or a bias, sequences packed along the tokens.
``rotary``     the rotation of Q and K by their positions: forward alone, or forward and backward of a training step.  Half and
               interleaved pairs, all or part of the head, frequencies as they are or scaled for long contexts.

``run`` computes them in elementary torch operations in 32 bits; with ``own`` it calls this package.  A case is a dict of plain
values; ``listed`` gives the fixed ones, ``draw`` more of the same ranges.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _attention(name, B, Sq, Sk, Hq, Hk, D, Dv, causal, extra="none", seqs=0):
    return dict(name=name, kind="attention", B=B, Sq=Sq, Sk=Sk, Hq=Hq, Hk=Hk, D=D, Dv=Dv, causal=causal, extra=extra, seqs=seqs)


def _rotary(name, B, S, Hq, Hk, D, R, dtype, direction, layout="bshd", interleaved=False, scaling="none", start=0, fused=False, seqs=0):
    return dict(name=name, kind="rotary", B=B, S=S, Hq=Hq, Hk=Hk, D=D, R=R, dtype=dtype, direction=direction, layout=layout, interleaved=interleaved,
                scaling=scaling, start=start, fused=fused, seqs=seqs)


def listed():
    return [
        # two short sequences, a few heads: launches are all of it
        _attention("attention_short", 2, 96, 96, 4, 4, 64, 64, True),
        # one 2048-token sequence of an 8B model's attention, the everyday training shape
        _attention("attention_8b", 1, 2048, 2048, 32, 8, 128, 128, True),
        # a full micro batch of a model with 64 query heads on 8 key heads, the largest
        _attention("attention_large", 4, 2048, 2048, 64, 8, 128, 128, True),
        # one long sequence, few heads
        _attention("attention_long", 1, 8192, 8192, 16, 2, 128, 128, True),
        # documents of different lengths packed along the tokens, small heads
        _attention("attention_packed", 1, 3232, 3232, 16, 4, 64, 64, True, seqs=6),
        # keys of another sequence, wide query heads, padded batch: a bias of -inf hides keys, and leaves one sequence none
        _attention("attention_cross_bias", 3, 480, 1056, 8, 8, 192, 128, False, extra="bias"),
        # ALiBi slopes on a model with as many key heads as query heads
        _attention("attention_alibi", 2, 1024, 1024, 16, 16, 64, 64, True, extra="alibi"),
        # one decoded token of each of 16 sequences, far into a long context
        _rotary("rotary_decode", 16, 1, 32, 8, 128, 128, "bf16", "forward", start=100_000, scaling="yarn"),
        # a training step of an 8B model on one 2048-token sequence
        _rotary("rotary_8b", 1, 2048, 32, 8, 128, 128, "bf16", "train"),
        # a training step on a full micro batch whose Q and K are slices of one projection's output, the largest
        _rotary("rotary_large", 4, 2048, 64, 8, 128, 128, "bf16", "train", fused=True),
        # part of an odd-sized head, interleaved pairs, odd length, fp32
        _rotary("rotary_partial_fp32", 3, 1001, 10, 2, 80, 20, "fp32", "train", layout="bhsd", interleaved=True, scaling="linear"),
        # packed documents, each from position 0, half of the head, frequencies scaled by wavelength
        _rotary("rotary_packed", 1, 3232, 16, 4, 64, 32, "bf16", "forward", layout="thd", scaling="wavelength", seqs=6),
    ]


def _log(rng, lo, hi, step):
    """A multiple of ``step`` in [lo, hi], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi // step * step, max(-(-lo // step) * step, round(v / step) * step)))


def draw(rng: random.Random):
    if rng.random() < 0.6:
        while True:
            hk, packed = rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.random() < 0.3
            sq = _log(rng, 32, 8192, 32)
            causal = rng.random() < 0.7
            sk = sq if packed or rng.random() < 0.6 else _log(rng, sq if causal else 32, 8192, 32)
            c = _attention(None, 1 if packed else rng.choice([1, 2, 3, 4]), sq, sk, hk * rng.choice([1, 1, 2, 3, 4, 8]), hk, rng.choice([64, 64, 128, 128, 128, 192, 256]),
                           rng.choice([64, 128]), causal, "none" if packed else rng.choice(["none", "none", "none", "alibi", "bias"]), rng.randint(2, 8) if packed else 0)
            scores = c["B"] * c["Hq"] * sq * sk
            if scores * (3 * c["D"] + 2 * c["Dv"]) <= 256 * 2048 ** 2 * 640 and scores <= 256 * 2048 ** 2 and (c["extra"] != "bias" or scores <= 2 ** 28):
                c.pop("name")
                return c
    while True:
        layout, hk, d = rng.choice(["bshd", "bshd", "bhsd", "thd"]), rng.choice([1, 2, 4, 8]), rng.choice([64, 64, 128, 128, 128, 80, 96, 192, 256])
        decode = layout != "thd" and rng.random() < 0.25
        s = rng.choice([1, 1, 2, 3]) if decode else _log(rng, 17, 8192, 1)
        r = rng.choice([d, d, d, d // 2, d // 4])
        c = _rotary(None, rng.randint(1, 64) if decode else 1 if layout == "thd" else rng.choice([1, 2, 3, 4]), s, hk * rng.choice([1, 2, 4, 8]), hk, d, r,
                    rng.choice(["bf16", "bf16", "fp32"]), "forward" if decode else rng.choice(["forward", "train"]), layout, rng.random() < 0.3,
                    rng.choice(["none", "none", "linear", "yarn", "wavelength"]), rng.choice([0, 0, 1000, 1_000_000]), layout == "bshd" and rng.random() < 0.5,
                    rng.randint(2, 8) if layout == "thd" else 0)
        if c["B"] * s * (c["Hq"] + hk) * d * (2 if c["dtype"] == "fp32" else 1) <= 8192 * 72 * 128:
            c.pop("name")
            return c


# ------------------------------------------------------------------------------------------------------------- inputs
def _starts(case, seed, step):
    """Boundaries of the packed sequences: uneven lengths, none empty."""
    total = case["Sq"] if case["kind"] == "attention" else case["S"]
    rng, blocks = random.Random(seed), total // step
    n = min(case["seqs"], blocks)
    return [0] + [step * c for c in sorted(rng.sample(range(1, blocks), n - 1))] + [total]


def _quantized(gen, B, H, S, D):
    """N(0, 1) rounded to E2M1 with one power of two for each 32 x 32 block: codes [B, H, S, D], scale bytes [B, H, S/32, D/32]."""
    x = torch.randn((B, H, S, D), device=DEVICE, generator=gen)
    block = x.view(B, H, S // 32, 32, D // 32, 32)
    exponent = torch.floor(torch.log2(block.abs().amax(dim=(3, 5), keepdim=True))) - 2
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEVICE)
    code = torch.bucketize((block * torch.exp2(-exponent)).abs(), bounds, out_int32=True).to(torch.uint8) + (block < 0).to(torch.uint8) * 8
    return code.reshape(B, H, S, D), (exponent + 127).to(torch.uint8).reshape(B, H, S // 32, D // 32)


def _two_a_byte(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous()


def _frequencies(R, scaling):
    """Radians a position of each of the R/2 pairs, in 64 bits, and what cosine and sine are multiplied with: as they are (base 10000), all
    of them divided by 4, blended between the two by the rotations a pair makes in 4096 positions (factor 8), or by its wavelength
    against 8192 positions (base 500000, factor 8)."""
    i = torch.arange(0, R, 2, dtype=torch.float64)
    f = (500000.0 if scaling == "wavelength" else 10000.0) ** (-i / R)
    if scaling == "linear":
        return f / 4, 1.0
    if scaling == "yarn":
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f / 8 * (1 - keep) + f * keep, 0.1 * math.log(8) + 1
    if scaling == "wavelength":
        keep = ((8192 * f / (2 * math.pi) - 1) / (4 - 1)).clamp(0, 1)
        return f / 8 * (1 - keep) + f * keep, 1.0
    return f, 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    st = {"case": case}
    if case["kind"] == "attention":
        B, Sq, Sk, Hq, Hk, D, Dv = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D", "Dv"))
        st["sm_scale"] = D ** -0.5
        st["starts"] = _starts(case, seed, 32) if case["seqs"] else None
        (qc, st["qs"]), (kc, st["ks"]), (vc, st["vs"]) = _quantized(gen, B, Hq, Sq, D), _quantized(gen, B, Hk, Sk, D), _quantized(gen, B, Hk, Sk, Dv)
        st["q"], st["k"], st["v"] = _two_a_byte(qc), _two_a_byte(kc), _two_a_byte(vc.transpose(2, 3))   # V's codes are packed along the keys
        if case["extra"] == "alibi":
            st["alibi"] = torch.exp2(-8 * torch.arange(1, Hq + 1, device=DEVICE) / Hq)
        if case["extra"] == "bias":   # scores of some other kind, and -inf on each sequence's padding: all of the last one's keys
            length = torch.randint(1, Sk + 1, (B,), device=DEVICE, generator=gen)
            length[-1] = 0 if B > 1 else Sk
            pad = torch.arange(Sk, device=DEVICE) >= length[:, None]
            st["bias"] = torch.randn((B, 1, Sq, Sk), device=DEVICE, generator=gen).masked_fill_(pad[:, None, None, :], -math.inf)
        st["dout"] = torch.randn((B, Hq, Sq, Dv), device=DEVICE, generator=gen).to(torch.bfloat16)
        # what the forward left: output and log-sum-exp (0 and -inf in a row that sees no key)
        s = _scores(st)
        top = s.amax(-1, keepdim=True)
        s = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
        total = s.sum(-1, keepdim=True)
        st["out"] = (s @ _shared(_values(st["v"].contiguous(), st["vs"], True), Hq)).div_(total.clamp(min=1e-30)).to(torch.bfloat16)
        st["lse"] = (top + total.log()).squeeze(-1)
        return st
    B, S, Hq, Hk, D = (case[n] for n in ("B", "S", "Hq", "Hk", "D"))
    dt = DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, device=DEVICE, generator=gen).to(dt)  # noqa: E731
    dims = lambda h: {"bshd": (B, S, h, D), "bhsd": (B, h, S, D), "thd": (S, h, D)}[case["layout"]]  # noqa: E731
    if case["fused"]:   # [B, S, heads of Q, K and V]: Q and K are slices
        whole = normal(B, S, Hq + 2 * Hk, D)
        q, k = whole[:, :, :Hq], whole[:, :, Hq:Hq + Hk]
    else:
        q, k = normal(*dims(Hq)), normal(*dims(Hk))
    train = case["direction"] == "train"
    st.update(q=q.requires_grad_(train), k=k.requires_grad_(train))
    if train:
        st.update(dq=normal(*dims(Hq)), dk=normal(*dims(Hk)))
    freq, st["factor"] = _frequencies(case["R"], case["scaling"])
    st["inv_freq"] = freq.to(DEVICE)
    if case["layout"] == "thd":
        starts = _starts(case, seed, 1)
        st["positions"] = torch.cat([torch.arange(b - a) for a, b in zip(starts, starts[1:])]).to(DEVICE)
    elif case["start"]:
        st["positions"] = torch.arange(S, device=DEVICE) + torch.randint(case["start"] // 2, case["start"], (B, 1), device=DEVICE, generator=gen)
    else:
        st["positions"] = torch.arange(S, device=DEVICE)
    return st


# --------------------------------------------------------------------------------------------------------- plain forms
def _values(codes, scales, along_keys=False):
    """The numbers that codes and block scales stand for, fp32 [B, H, S, D]."""
    grid = torch.tensor(E2M1 + [-v for v in E2M1], device=codes.device)
    x = grid[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()]
    x = x.transpose(2, 3) if along_keys else x
    return x * torch.exp2(scales.float() - 127).repeat_interleave(32, dim=2).repeat_interleave(32, dim=3)


def _shared(x, heads):
    return x.repeat_interleave(heads // x.shape[1], dim=1)


def _scores(st):
    """Scaled scores with their additive terms, -inf where a row may not look."""
    case, q, k = st["case"], _values(st["q"], st["qs"]), _values(st["k"], st["ks"])
    Sq, Sk = q.shape[2], k.shape[2]
    s = (q @ _shared(k, q.shape[1]).transpose(2, 3)).mul_(st["sm_scale"])
    row, key = torch.arange(Sq, device=s.device)[:, None] + Sk - Sq, torch.arange(Sk, device=s.device)
    if case["extra"] == "alibi":
        s -= st["alibi"][:, None, None] * (row - key).abs()
    if case["extra"] == "bias":
        s += st["bias"]
    hidden = torch.zeros((Sq, Sk), dtype=torch.bool, device=s.device)
    if case["causal"]:
        hidden |= key > row
    if st["starts"]:
        at = torch.bucketize(key, torch.tensor(st["starts"][1:], device=s.device), right=True)
        hidden |= at[:, None] != at
    return s.masked_fill_(hidden, -math.inf)


def _attention_backward(st):
    dout, out, lse = st["dout"].float(), st["out"].float(), st["lse"]
    q, k, v = _values(st["q"], st["qs"]), _values(st["k"], st["ks"]), _values(st["v"], st["vs"], True)
    B, Hq, Sq, D = q.shape
    Hk, Sk, Dv = k.shape[1], k.shape[2], v.shape[3]
    p = _scores(st).sub_(lse.masked_fill(lse == -math.inf, 0.0)[..., None]).exp_()
    dv = p.transpose(2, 3) @ dout
    ds = (dout @ _shared(v, Hq).transpose(2, 3)).sub_((dout * out).sum(-1, keepdim=True)).mul_(p).mul_(st["sm_scale"])
    dq = ds @ _shared(k, Hq)
    dk = ds.transpose(2, 3) @ q
    group = lambda x: x.view(B, Hk, Hq // Hk, Sk, -1).sum(2)  # noqa: E731
    return {"dq": dq.to(torch.bfloat16), "dk": group(dk).to(torch.bfloat16), "dv": group(dv).to(torch.bfloat16)}


def _rotated(x, st, back):
    case = st["case"]
    angle = st["positions"].double()[..., None] * st["inv_freq"]      # [S or B x S, R/2]
    c, s = (torch.cos(angle) * st["factor"]).float(), (torch.sin(angle) * st["factor"]).float()
    s = -s if back else s
    if case["layout"] == "bhsd":
        c, s = (t.unsqueeze(-3) for t in (c, s))
    else:
        c, s = (t.unsqueeze(-2) for t in (c, s))
    R, f = case["R"], x.float()
    a, b = (f[..., 0:R:2], f[..., 1:R:2]) if case["interleaved"] else (f[..., :R // 2], f[..., R // 2:R])
    turned = (c * a - s * b, s * a + c * b)
    turned = torch.stack(turned, dim=-1).flatten(-2) if case["interleaved"] else torch.cat(turned, dim=-1)
    return torch.cat((turned, f[..., R:]), dim=-1).to(x.dtype)


# ------------------------------------------------------------------------------------------------------------ one pass
def run(st):
    case = st["case"]
    if case["kind"] == "attention":
        if own:
            import alto_amd.mxfp4 as mx
            dq, dk, dv = mx.attention_mxfp4_backward(st["dout"], st["q"], st["k"], st["v"], st["qs"], st["ks"], st["vs"], st["out"], st["lse"], st["sm_scale"],
                                                     case["causal"], bias=st.get("bias"), alibi_slopes=st.get("alibi"), cu_seqlens_q=st["starts"],
                                                     cu_seqlens_k=st["starts"])
            return {"dq": dq, "dk": dk, "dv": dv}
        return _attention_backward(st)
    if own:
        import alto_amd.mxfp4 as mx
        q, k = mx.apply_rotary(st["q"], st["k"], st["inv_freq"], st["positions"], interleaved=case["interleaved"], factor=st["factor"], layout=case["layout"])
        if case["direction"] == "forward":
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (st["q"], st["k"]), (st["dq"], st["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    result = {"q": _rotated(st["q"].detach(), st, False), "k": _rotated(st["k"].detach(), st, False)}
    if case["direction"] == "train":
        result.update(dq=_rotated(st["dq"], st, True), dk=_rotated(st["dk"], st, True))
    return result


# --------------------------------------------------------------------------------------------------------------- work
def _pairs(case):
    """(row, key) pairs that the mask leaves; packed sequences: on average over their possible lengths."""
    Sq, Sk = case["Sq"], case["Sk"]
    if case["seqs"]:
        pairs = 2 * Sq * Sq / (min(case["seqs"], Sq // 32) + 1)
        return pairs / 2 if case["causal"] else pairs
    return Sq * (Sk - Sq) + Sq * (Sq + 1) / 2 if case["causal"] else Sq * Sk


def work(case):
    """Bytes: each input read once, each output written once.  FLOPs of attention: its five products over the pairs that the mask
    leaves (2 per multiply-add); of a rotation six a pair of elements."""
    if case["kind"] == "attention":
        B, Sq, Sk, Hq, Hk, D, Dv = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D", "Dv"))
        codes = (Hq * Sq * D + Hk * Sk * (D + Dv)) * (1 / 2 + 1 / 1024)
        wide = 2 * (2 * Hq * Sq * Dv + Hq * Sq * D + Hk * Sk * (D + Dv)) + 4 * Hq * Sq + (4 * Sq * Sk if case["extra"] == "bias" else 0)
        return {"bytes": B * (codes + wide), "flops": 2 * B * Hq * (3 * D + 2 * Dv) * _pairs(case)}
    n = case["B"] * case["S"] * (case["Hq"] + case["Hk"])
    times = 2 if case["direction"] == "train" else 1
    return {"bytes": 2 * times * n * case["D"] * (4 if case["dtype"] == "fp32" else 2), "flops": 3 * times * n * case["R"]}


# -------------------------------------------------------------------------------------------------------------- exact
def _decoded(code, byte):
    """One head's codes (a uint8 for each) and its scale bytes, as fp64."""
    magnitude = torch.tensor(E2M1, dtype=torch.float64, device=code.device)[(code & 7).long()]
    signed = torch.where(code >= 8, -magnitude, magnitude)
    return (signed.unflatten(0, (-1, 32)).unflatten(2, (-1, 32)) * torch.pow(2.0, byte.double() - 127)[:, None, :, None]).flatten(2, 3).flatten(0, 1)


def _nibbles(packed):
    return torch.stack((packed % 16, packed // 16), dim=2).flatten(1, 2)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "attention":
        B, Sq, Sk, Hq, Hk, D, Dv = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hk", "D", "Dv"))
        dq = torch.zeros((B, Hq, Sq, D), dtype=torch.float64, device=DEVICE)
        dk = torch.zeros((B, Hk, Sk, D), dtype=torch.float64, device=DEVICE)
        dv = torch.zeros((B, Hk, Sk, Dv), dtype=torch.float64, device=DEVICE)
        spans = list(zip(st["starts"], st["starts"][1:])) if st["starts"] else [None]
        for b in range(B):
            for h in range(Hq):
                g = h // (Hq // Hk)
                q, k = _decoded(_nibbles(st["q"][b, h]), st["qs"][b, h]), _decoded(_nibbles(st["k"][b, g]), st["ks"][b, g])
                v = _decoded(_nibbles(st["v"][b, g]).t(), st["vs"][b, g])
                for span in spans:
                    rows, keys = (slice(*span), slice(*span)) if span else (slice(0, Sq), slice(0, Sk))
                    qi, kj, vj, do = q[rows], k[keys], v[keys], st["dout"][b, h, rows].double()
                    n, m = qi.shape[0], kj.shape[0]
                    x = torch.mm(qi, kj.t()) * st["sm_scale"]
                    away = torch.arange(n, device=DEVICE)[:, None] + (m - n) - torch.arange(m, device=DEVICE)[None, :]
                    if case["extra"] == "alibi":
                        x = x - st["alibi"][h].double() * away.abs()
                    if case["extra"] == "bias":
                        x = x + st["bias"][b, 0].double()
                    seen = (away >= 0) if case["causal"] else torch.ones_like(x, dtype=torch.bool)
                    lse = st["lse"][b, h, rows].double()[:, None]
                    p = torch.where(seen & (x > -math.inf), torch.exp(x - lse), torch.zeros_like(x))
                    inner = torch.mm(do, vj.t()) - torch.sum(do * st["out"][b, h, rows].double(), 1)[:, None]
                    ds = p * inner * st["sm_scale"]
                    dq[b, h, rows] = torch.mm(ds, kj)
                    dk[b, g, keys] += torch.mm(ds.t(), qi)
                    dv[b, g, keys] += torch.mm(p.t(), do)
        return {"dq": dq, "dk": dk, "dv": dv}
    R, axis = case["R"], 1 if case["layout"] == "bhsd" else -2

    def turned(x, sign):
        z = x.detach().double()
        turn = st["factor"] * torch.exp(1j * sign * st["positions"].double()[..., None] * st["inv_freq"])
        turn = turn.unsqueeze(0) if turn.dim() == 2 and case["layout"] != "thd" else turn
        turn = turn.unsqueeze(axis)
        if case["interleaved"]:
            w = turn * torch.view_as_complex(z[..., :R].reshape(*z.shape[:-1], R // 2, 2).contiguous())
            z[..., :R] = torch.view_as_real(w).reshape(*z.shape[:-1], R)
        else:
            w = turn * torch.complex(z[..., :R // 2].contiguous(), z[..., R // 2:R].contiguous())
            z[..., :R // 2], z[..., R // 2:R] = w.real, w.imag
        return z

    result = {"q": turned(st["q"], 1), "k": turned(st["k"], 1)}
    if case["direction"] == "train":
        result.update(dq=turned(st["dq"], -1), dk=turned(st["dk"], -1))
    return result
