"""Host code of the attention backward and of the rotary positions without a GPU: what the C entries refuse, and the workspace they ask for."""
import ctypes

import pytest

from alto_amd import _lib
from alto_amd.mxfp4.attention import _Backward
from alto_amd.mxfp4.rotary import _Args

MEMORY = ctypes.create_string_buffer(4096)   # stands for device memory: no call here gets as far as a launch
P = ctypes.addressof(MEMORY) + (-ctypes.addressof(MEMORY)) % 256


def ints(*values):
    return (ctypes.c_int32 * len(values))(*values)


def attention(**changes):
    args = dict(q_codes=P, q_scales=P, k_codes=P, k_scales=P, vt_codes=P, v_scales=P, dout=P, out=P, lse=P, dq=P, dk=P, dv=P, workspace=P, workspace_bytes=1 << 40,
                B=1, Hq=4, Hk=2, Sq=96, Sk=128, Sk_used=128, D=128, Dv=64, causal=1, sm_scale=0.1)
    return _Backward(**{**args, **changes})


def rotary(**changes):
    args = dict(q=P, k=P, q_out=P, k_out=P, inv_freq=P, B=1, S=4, Hq=2, Hk=1, D=64, R=64, factor=1.0)
    return _Args(**{**args, **changes})


def refused(entry, args, text, *more):
    lib = _lib.load()
    rc = getattr(lib, entry)(ctypes.byref(args), *more)
    assert rc < 0 and text in lib.alto_mxfp4_last_error().decode(), (rc, lib.alto_mxfp4_last_error())


SIZES = [
    (dict(Hq=3), "multiple of Hk"), (dict(Hk=0), "multiple of Hk"), (dict(B=0), "Hq="), (dict(Sq=0), "Sq=0"), (dict(Sq=33), "Sq=33"), (dict(Sk=-32), "Sk=-32"),
    (dict(D=32), "D=32"), (dict(D=320), "D=320"), (dict(Dv=96), "Dv=96"), (dict(Sk_used=160), "Sk_used"), (dict(Sk_used=0), "Sk_used"), (dict(Sk_used=40), "Sk_used"),
    (dict(Sq=160), "Sq <= Sk"), (dict(B=65536), "65536"), (dict(Sk=1 << 40, Sk_used=128), "below 65536"), (dict(Hq=1 << 32, Hk=1 << 31), "below 65536"),
    (dict(Hq=1 << 30, Hk=1 << 30), "too large"), (dict(n_seqs=-1), "negative number"), (dict(n_seqs=1), "boundaries"),
    (dict(n_seqs=1, cu_q=ints(0, 96), cu_k=ints(0, 128), B=2), "B = 1"), (dict(n_seqs=1, cu_q=ints(0, 64), cu_k=ints(0, 128)), "token counts"),
    (dict(n_seqs=2, cu_q=ints(0, 96, 96), cu_k=ints(0, 96, 128)), "increasing"), (dict(n_seqs=2, cu_q=ints(0, 40, 96), cu_k=ints(0, 64, 128)), "increasing"),
    (dict(n_seqs=2, cu_q=ints(0, 64, 96), cu_k=ints(0, 32, 128)), "Sq <= Sk"), (dict(n_seqs=2, cu_q=ints(0, -(1 << 31), 96), cu_k=ints(0, 64, 128)), "increasing"),
]


@pytest.mark.parametrize("changes,text", SIZES)
def test_attention_sizes(changes, text):
    refused("alto_mxfp4_attention_bwd", attention(**changes), text, None)
    refused("alto_mxfp4_attention_bwd_workspace_bytes", attention(**changes), text)


@pytest.mark.parametrize("changes,text", [
    *[(dict([(name, None)]), "null pointer") for name in ("q_codes", "q_scales", "k_codes", "k_scales", "vt_codes", "v_scales", "dout", "out", "lse", "workspace")],
    (dict(dq=None, dk=None, dv=None), "null pointer"), (dict(dk=None), "together"), (dict(dv=None), "together"), (dict(q_codes=P + 8), "aligned"), (dict(dout=P + 8), "aligned"),
    (dict(vt_codes=P + 4), "aligned"), (dict(dk=P + 8), "aligned"), (dict(lse=P + 2), "aligned"), (dict(bias=P + 2), "aligned"), (dict(dout_ss=12), "multiples of 8"),
    (dict(out_sb=-8), "multiples of 8"), (dict(dq_sh=12), "multiples of 8"), (dict(dv_ss=-8), "multiples of 8"), (dict(bias=P, bias_sm=1 << 24), "2^24"), (dict(bias=P, sm_scale=1e-20), "2^-64"), (dict(alibi_slopes=P, sm_scale=1e-20), "2^-64"), (dict(bias_sm=-1), "non-negative"), (dict(lse_sb=1 << 50), "non-negative"),
    (dict(sm_scale=0.0), "sm_scale"), (dict(sm_scale=-1.0), "sm_scale"), (dict(sm_scale=float("inf")), "sm_scale"), (dict(sm_scale=float("nan")), "sm_scale"),
    (dict(workspace_bytes=1024), "workspace"), (dict(workspace=P + 128), "workspace"),
])
def test_attention_operands(changes, text):
    refused("alto_mxfp4_attention_bwd", attention(**changes), text, None)


def test_attention_workspace():
    """It holds the tiles, and parts of sums only where lists are cut."""
    size = _lib.load().alto_mxfp4_attention_bwd_workspace_bytes

    def up(n):
        return -(-n // 256) * 256

    # one key block of 3 tiles by 2 heads: nothing to cut
    tiles = up(4 * 3 * 272) + up(2 * 4 * 16) + 2 * 128 * (128 + 64) * 2 + 4 * 96 * 64 * 2
    assert size(ctypes.byref(attention())) == tiles
    assert size(ctypes.byref(attention(n_seqs=1, cu_q=ints(0, 96), cu_k=ints(0, 128)))) == tiles
    # one head with one block of keys and 1024 tiles of rows: 16 parts
    long = dict(Hq=1, Hk=1, Sq=32768, causal=0)
    assert size(ctypes.byref(attention(**long))) == up(1024 * 272) + up(4 * 16) + 128 * 192 * 2 + 32768 * 64 * 2 + 2 * 16 * 128 * 192 * 4
    # one block of rows with 1024 tiles of keys: 32 parts
    few = dict(Hq=1, Hk=1, Sq=32, Sk=32768, Sk_used=32768)
    assert size(ctypes.byref(attention(**few))) == up(272) + up(1024 * 16) + 32768 * 192 * 2 + 32 * 64 * 2 + 32 * 128 * 128 * 4


@pytest.mark.parametrize("changes,text", [
    (dict(dtype=2), "dtype 2"), (dict(B=-1), "negative"), (dict(S=-1), "negative"), (dict(Hq=0), "query heads"), (dict(Hk=-1), "negative"), (dict(R=0), "R=0"), (dict(R=7), "R=7"),
    (dict(R=66), "R=66"), (dict(D=4096, R=2050), "R=2050"), (dict(D=1 << 20), "out of range"), (dict(B=1 << 20, S=1 << 21), "out of range"), (dict(q=None), "null"), (dict(k_out=None), "null"),
    (dict(inv_freq=None), "null"), (dict(q_sb=-1), "non-negative"), (dict(pos_ss=-1), "non-negative"), (dict(q=P + 1), "aligned"), (dict(positions=P + 4), "aligned"), (dict(inv_freq=P + 4), "aligned"),
])
def test_rotary_arguments(changes, text):
    refused("alto_mxfp4_rotary", rotary(**changes), text, None)


def test_rotary_of_no_tokens():
    lib = _lib.load()
    assert lib.alto_mxfp4_rotary(ctypes.byref(rotary(S=0, q=None, q_out=None, k=None, k_out=None)), None) == 0


def test_no_cpu_fallback():
    import torch

    import alto_amd.mxfp4 as mx
    codes, scales, rows = torch.zeros(1, 1, 32, 32, dtype=torch.uint8), torch.zeros(1, 1, 1, 2, dtype=torch.uint8), torch.zeros(1, 1, 32, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        mx.attention_mxfp4_backward(rows, codes, codes, codes.reshape(1, 1, 64, 16), scales, scales, scales, rows, torch.zeros(1, 1, 32), 0.125, True)
    with pytest.raises(RuntimeError):
        mx.apply_rotary(rows, rows, mx.rotary_frequencies(64)[0])
