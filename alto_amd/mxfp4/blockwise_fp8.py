"""8-bit floating point with one fp32 scale for each block of 128: quantizer, products, products grouped by expert, and the layers made of them.

For the layers of a model that do not stand 4 bits, next to the MXFP4 path and in its manner: :func:`convert_to_blockwise_fp8` /
:func:`quantize_blockwise_fp8_rowcol` make codes and scales, :func:`blockwise_fp8_gemm` and :func:`blockwise_fp8_grouped_gemm` multiply them,
:func:`blockwise_fp8_linear` and :func:`blockwise_fp8_grouped_linear` train with them.  Codes are ``torch.float8_e4m3fn`` or
``torch.float8_e5m2``; L is the largest (448, 57344).  Of a block's largest magnitude amax (taken as at least 2^-100 L)

    scale = amax / L,   code = x L / amax to the nearest code, ties to even;

a block with NaN or an infinity in it stands for NaN.  (Of bf16 data that is exact; of fp32 data a quotient within 2^-22 of halfway between two codes may go to
either.)  Activations and gradients have blocks of 1 x 128 along a product's reduction, weights blocks of 128 x 128, whose codes serve the forward product and,
stored transposed, the input gradient's.

The reference has such a path beside its MXFP4 one (``alto/kernels/blockwise_fp8/``).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _runtime as rt
from .._lib import check
from .linear import cached_weight_quantisation, unwrap_weight_wrapper, weight_cache_enabled

FP8_BLOCK_SIZE = 128

_LONGEST = 2 ** 22 - 16   # codes of a row, and bytes from row to row, that a native product takes
_PART = 2 ** 22 - 128     # whole blocks of them: longer reductions are taken in parts of this length

_CODES = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}


def _struct(name: str, pointers: str, longs: str, ints: str):
    """``name`` of include/alto_mxfp4.h."""
    fields = [(n, t) for names, t in ((pointers, ctypes.c_void_p), (longs, ctypes.c_int64), (ints, ctypes.c_int)) for n in names.split()]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


_Quantize = _struct("alto_mxfp4_fp8_quantize_t", "x row_codes col_codes row_scales col_scales offs", "B M C x_sb x_sm row_sb row_ld col_sb col_ld", "dtype code is_2d groups")
_Dequantize = _struct("alto_mxfp4_fp8_dequantize_t", "codes scales out", "B R C codes_sb ld s_sb s_r s_c out_sb ldo", "code is_2d out_dtype")
_Gemm = _struct("alto_mxfp4_fp8_gemm_t", "a b a_scales b_scales c", "M N K lda ldb a_ss_r a_ss_k b_ss_r b_ss_k ldc", "a_code a_is_2d b_is_2d c_dtype")
_Grouped = _struct("alto_mxfp4_fp8_grouped_gemm_t", "a w a_scales w_scales c offs", "M N K lda a_ss_r a_ss_k w_se ldw ws_e ws_r ws_k ldc", "a_code w_is_2d c_dtype groups")
_Weights = _struct("alto_mxfp4_fp8_grouped_gemm_weights_t", "go x go_scales x_scales dw offs", "tokens N K go_ld x_ld go_ss x_ss dw_se ld_dw", "go_code dw_dtype groups")


def _call(name: str, args: ctypes.Structure, device: torch.device) -> None:
    fn = getattr(rt.lib(), name)
    if device.index == torch.cuda.current_device():
        check(fn(ctypes.byref(args), rt.stream_ptr(device)), name)
    else:
        with torch.cuda.device(device):
            check(fn(ctypes.byref(args), rt.stream_ptr(device)), name)


@torch.compiler.disable
def _between_graphs(fn, *args):
    """(nothing of a call can be traced: a compiled caller breaks its graph here)"""
    return fn(*args)


def _blocks(n: int) -> int:
    return -(-n // FP8_BLOCK_SIZE)


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _code(dtype: torch.dtype, what: str = "codes") -> int:
    if dtype not in _CODES:
        raise AssertionError(f"{what} of type {dtype}: torch.float8_e4m3fn or torch.float8_e5m2")
    return _CODES[dtype]


def _same_device(*tensors: Optional[torch.Tensor]) -> None:
    rt.require_gpu(*tensors)
    first = tensors[0]
    for t in tensors[1:]:
        assert t is None or t.device == first.device, f"tensors on {first.device} and {t.device}"


def _no_gradients(what: str, *tensors: torch.Tensor) -> None:
    rt.refuse_transforms(what, *tensors)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise NotImplementedError(f"{what}: gradients of codes and scales are not implemented: detach them")


def _check_offsets(offsets: torch.Tensor) -> None:
    assert offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.shape[0] >= 2, "offsets: int32, one boundary more than there are groups"


# ------------------------------------------------------------------------------------------------------------ quantizer
def _rows_readable(x: torch.Tensor) -> torch.Tensor:
    """x [B, M, C] with unit stride along C (a copy where it has another, or where its numbers are memory's with the sign turned)."""
    x = x.resolve_neg()
    return x if x.shape[2] <= 1 or x.stride(2) == 1 else x.contiguous()


def _stride(t: torch.Tensor, d: int) -> int:
    return 0 if t.shape[d] <= 1 else t.stride(d)


def _quantize(x: torch.Tensor, want_row: bool, want_col: bool, is_2d: bool, dtype: torch.dtype, offsets: Optional[torch.Tensor] = None):
    """x [B, M, C] -> (row codes [B, M, C], row scales, col codes [B, tokens, C] as a view of [B, C, tokens] memory, col scales); None for a copy that
    is not wanted.  Rows of codes lie at multiples of 128 bytes."""
    x = _rows_readable(x)
    B, M, C = x.shape
    f32 = dict(dtype=torch.float32, device=x.device)
    tokens = M if offsets is None else FP8_BLOCK_SIZE * rt.lib().alto_mxfp4_fp8_token_blocks(M, offsets.shape[0] - 1)
    rq = rs = cq = cs = None
    if is_2d:
        rs = cs = torch.empty((B, _blocks(M), _blocks(C)), **f32)
    if want_row:
        pitch = _up(C, 128)
        rq = torch.empty((B, M, pitch), dtype=dtype, device=x.device)[..., :C]
        if not is_2d:
            rs = torch.empty((B, _blocks(C), M), **f32)
    if want_col:
        pitch = _up(tokens, 128)
        cq = torch.empty((B, C, pitch), dtype=dtype, device=x.device)[..., :tokens]
        if not is_2d:
            cs = torch.empty((B, _blocks(tokens), C), **f32)
    if C and B and (M or offsets is not None):
        a = _Quantize(x=x.data_ptr(), row_codes=rt.ptr(rq), col_codes=rt.ptr(cq), row_scales=rt.ptr(rs), col_scales=rt.ptr(cs), offs=rt.ptr(offsets), B=B, M=M, C=C,
                      x_sb=_stride(x, 0), x_sm=_stride(x, 1), dtype=rt.dtype_code(x.dtype), code=_code(dtype), is_2d=int(is_2d), groups=0 if offsets is None else offsets.shape[0] - 1)
        if want_row:
            a.row_sb, a.row_ld = rq.stride(0), rq.stride(1)
        if want_col:
            a.col_sb, a.col_ld = cq.stride(0), cq.stride(1)
        _call("alto_mxfp4_fp8_quantize", a, x.device)
    if want_col:
        cq = cq.transpose(1, 2)
    if want_row and not is_2d:
        rs = rs.transpose(1, 2)
    return rq, rs, cq, cs


def _copies(x: torch.Tensor, want_row: bool, want_col: bool, is_2d: bool, dtype: torch.dtype, offsets: Optional[torch.Tensor] = None):
    """:func:`_quantize` of x [M, C] or [B, M, C], the results with as many dims: in one native call, the general way where that declines."""
    out = rt.host().fp8_quantize(x, want_row, want_col, is_2d, dtype is torch.float8_e5m2, offsets)
    if out is not None:
        return out
    x = x.detach()
    if x.dim() == 3:
        return _quantize(x, want_row, want_col, is_2d, dtype, offsets)
    return tuple(t if t is None else t[0] for t in _quantize(x.unsqueeze(0), want_row, want_col, is_2d, dtype, offsets))


def _check_input(x: torch.Tensor, dtype: torch.dtype, dims: Tuple[int, ...]) -> None:
    rt.require_gpu(x)
    assert x.dtype in (torch.bfloat16, torch.float32), f"input of type {x.dtype}: bfloat16 or float32"
    assert x.dim() in dims, f"input of {x.dim()} dims"
    _code(dtype)


def convert_to_blockwise_fp8(data_hp: torch.Tensor, axis: int = -1, is_2d_block: bool = False, dtype: torch.dtype = torch.float8_e4m3fn) -> Tuple[torch.Tensor, torch.Tensor]:
    """bf16 / fp32 [M, C] or [B, M, C] of any sizes and strides -> (codes of its shape, fp32 scales).

    Blocks of 1 x 128 along ``axis``: scales [M, ceil(C/128)] for -1 (a view with the rows contiguous in memory), [ceil(M/128), C] for -2; blocks of 128 x 128
    with ``is_2d_block``: scales [ceil(M/128), ceil(C/128)].  With ``axis=-2`` the codes are a view of [C, M] memory, as a product that sums over M reads
    them.  Rows of codes lie at multiples of 128 bytes.  Codes and scales carry no gradient.
    """
    if torch.compiler.is_compiling():
        return _between_graphs(_convert_to, data_hp, axis, is_2d_block, dtype)
    return _convert_to(data_hp, axis, is_2d_block, dtype)


def _convert_to(x, axis, is_2d, dtype):
    if dtype in _CODES and axis in (-1, -2):   # (first of all the native call: it serves nothing that the checks below refuse)
        out = rt.host().fp8_quantize(x, axis == -1, axis == -2, bool(is_2d), dtype is torch.float8_e5m2, None)
        if out is not None:
            return out[:2] if axis == -1 else out[2:]
    rt.refuse_transforms("convert_to_blockwise_fp8", x)
    _check_input(x, dtype, (2, 3))
    assert axis in (-1, -2, x.dim() - 1, x.dim() - 2), f"axis {axis}: the last or the one before"
    last = axis in (-1, x.dim() - 1)
    out = _copies(x, last, not last, bool(is_2d), dtype)
    return out[:2] if last else out[2:]


def quantize_blockwise_fp8_rowcol(x: torch.Tensor, is_2d_block: bool = False, dtype: torch.dtype = torch.float8_e4m3fn,
                                  offsets: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`convert_to_blockwise_fp8` along both axes from one pass over x: (codes, scales) of ``axis=-1``, then those of ``axis=-2``.  With blocks of 128 x 128
    both come with the same scales (one tensor).

    ``offsets`` (int32 [E + 1] on the device; x [M, C], blocks of 1 x 128): the rows are grouped, and the blocks along them start anew with each group, as the weight
    gradients by group (:func:`blockwise_fp8_grouped_gemm_weights`) read them: the second pair is [P, C] and [P/128, C], P = 128 * ((M + 127 (E + 2)) // 128), with
    the rows ahead of the first group, of each group and behind the last one after another, each padded with zero codes to whole blocks.
    """
    if torch.compiler.is_compiling():
        return _between_graphs(_rowcol, x, is_2d_block, dtype, offsets)
    return _rowcol(x, is_2d_block, dtype, offsets)


def _rowcol(x, is_2d, dtype, offsets):
    if dtype in _CODES:
        out = rt.host().fp8_quantize(x, True, True, bool(is_2d), dtype is torch.float8_e5m2, offsets)
        if out is not None:
            return out
    rt.refuse_transforms("quantize_blockwise_fp8_rowcol", x)
    _check_input(x, dtype, (2, 3) if offsets is None else (2,))
    if offsets is not None:
        _same_device(x, offsets)
        _check_offsets(offsets)
        assert not is_2d, "groups of rows have blocks of 1 x 128"
        offsets = offsets.contiguous()
    return _copies(x, True, True, bool(is_2d), dtype, offsets)


def convert_from_blockwise_fp8(codes: torch.Tensor, scales: torch.Tensor, axis: int = -1, is_2d_block: bool = False,
                               output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers that codes [M, C] or [B, M, C] and their scales (as :func:`convert_to_blockwise_fp8` returns them for ``axis``) stand for, bf16 or fp32.  With
    ``axis=-2`` the result is a view of [C, M] memory like the codes."""
    if torch.compiler.is_compiling():
        return _between_graphs(_convert_from, codes, scales, axis, is_2d_block, output_dtype)
    return _convert_from(codes, scales, axis, is_2d_block, output_dtype)


def _convert_from(codes, scales, axis, is_2d, output_dtype):
    _no_gradients("convert_from_blockwise_fp8", codes, scales)
    _same_device(codes, scales)
    assert codes.dim() in (2, 3) and scales.dim() == codes.dim(), f"codes of {codes.dim()} dims and scales of {scales.dim()}"
    assert axis in (-1, -2, codes.dim() - 1, codes.dim() - 2), f"axis {axis}: the last or the one before"
    last = axis in (-1, codes.dim() - 1)
    scales = scales.resolve_neg()
    q, s = (codes, scales) if codes.dim() == 3 else (codes.unsqueeze(0), scales.unsqueeze(0))
    if not last:
        q, s = q.transpose(1, 2), s.transpose(1, 2)
    B, R, C = q.shape
    code, out_code = _code(codes.dtype), rt.dtype_code(output_dtype)
    exp = (B, _blocks(R) if is_2d else R, _blocks(C))
    assert s.shape == exp and s.dtype == torch.float32, f"scales of shape {tuple(scales.shape)} and type {scales.dtype} for codes of {tuple(codes.shape)}"
    if C > 1 and q.stride(2) != 1:
        q = q.contiguous()
    out = torch.empty((B, R, C), dtype=output_dtype, device=codes.device)
    for b in range(0, B if out.numel() else 0, 65535):   # (as many matrices as a launch takes)
        qb, sb, ob = (t[b:b + 65535] for t in (q, s, out))
        a = _Dequantize(codes=qb.data_ptr(), scales=sb.data_ptr(), out=ob.data_ptr(), B=qb.shape[0], R=R, C=C, codes_sb=_stride(q, 0), ld=_stride(q, 1), s_sb=_stride(s, 0), s_r=_stride(s, 1),
                        s_c=_stride(s, 2), out_sb=out.stride(0), ldo=out.stride(1), code=code, is_2d=int(bool(is_2d)), out_dtype=out_code)
        _call("alto_mxfp4_fp8_dequantize", a, codes.device)
    out = out if last else out.transpose(1, 2)
    return out if codes.dim() == 3 else out[0]


# ------------------------------------------------------------------------------------------------------------- products
def _operand(t: torch.Tensor) -> torch.Tensor:
    """Codes [..., rows, K] as a product reads them: unit stride along K, rows at multiples of 16 bytes and readable to the next one behind K; otherwise a copy that is."""
    rows, K = t.shape[-2], t.shape[-1]
    if t.numel() == 0:
        return t
    steps = [_stride(t, d) for d in range(t.dim() - 1)]
    if (K == 1 or t.stride(-1) == 1) and all(s % 16 == 0 and s >= 0 for s in steps) and (rows == 1 or steps[-1] >= K) and steps[-1] <= _LONGEST and t.data_ptr() % 16 == 0:
        end = t.storage_offset() + sum(s * (n - 1) for s, n in zip(steps, t.shape)) + _up(K, 16)
        if K % 16 == 0 or end <= t.untyped_storage().nbytes():
            return t
    out = torch.empty((*t.shape[:-1], max(_up(K, 16), min(_up(K, 128), _LONGEST))), dtype=t.dtype, device=t.device)[..., :K]
    out.view(torch.uint8).copy_(t.view(torch.uint8))
    return out


def _scales(s: torch.Tensor) -> torch.Tensor:
    """Scales [..., rows, blocks] at strides that a product takes."""
    s = s.resolve_neg()
    return s if all(0 <= _stride(s, d) for d in range(s.dim())) and _stride(s, -2) < 2 ** 21 else s.transpose(-1, -2).contiguous().transpose(-1, -2)


def _in_parts(K: int, product, dtype: torch.dtype) -> torch.Tensor:
    """A reduction longer than a native product's: ``product(lo, hi)`` over each part in fp32, summed in fp32 in their order and rounded once."""
    total = None
    for lo in range(0, K, _PART):
        part = product(lo, min(lo + _PART, K))
        total = part if total is None else total.add_(part)
    return total.to(dtype)


def _check_scales(name: str, s: torch.Tensor, expected) -> None:
    assert s.dtype == torch.float32, f"{name}: scales of type {s.dtype}, float32 is taken"
    assert tuple(s.shape) == tuple(expected), f"{name} has shape {tuple(s.shape)}, but {tuple(expected)} is expected."


def blockwise_fp8_gemm(a: torch.Tensor, a_s: torch.Tensor, b: torch.Tensor, b_s: torch.Tensor, use_2dblock_a: bool = False, use_2dblock_b: bool = False,
                       trans_a: bool = False, trans_b: bool = False, output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C = op(A) @ op(B) on 8-bit codes with fp32 scales for each 128 along the reduction K, fp32 accumulation, bf16 or fp32 results.

    ``a`` [M, K] ([K, M] with ``trans_a``) of ``float8_e4m3fn`` or ``float8_e5m2``, ``b`` [K, N] ([N, K] with ``trans_b``) of ``float8_e4m3fn``; ``a_s``, ``b_s`` in the same
    orientation: one scale for each row (column) and 128 of K, or with ``use_2dblock_*`` for each 128 x 128.  Any sizes and strides: operands
    with unit stride along K and rows at multiples of 16 bytes (what the quantizers return) are read as they are, others are copied first, and so is
    what lies 2^22 bytes or more from row to row (the quantizers' copies of more than 2^22 - 128).  K above 2^22 - 16 is taken in parts, whose sums are added
    in fp32.

    The matrix pipe adds the products of 8 neighbouring k aligned to the largest of them and cut at 2^-13 of it, whatever instruction or library asks: of Gaussian
    data an fp32 result is off by 3e-5 of the results' norm, a hundredth of a bf16 rounding.  The product of two scales is taken in fp32, whose normal range has to hold it.
    """
    if torch.compiler.is_compiling():
        return _between_graphs(_gemm, a, a_s, b, b_s, use_2dblock_a, use_2dblock_b, trans_a, trans_b, output_dtype)
    return _gemm(a, a_s, b, b_s, use_2dblock_a, use_2dblock_b, trans_a, trans_b, output_dtype)


def _gemm(a, a_s, b, b_s, a_2d, b_2d, trans_a, trans_b, output_dtype):
    if output_dtype is torch.bfloat16 or output_dtype is torch.float32:
        out = rt.host().fp8_gemm(a, a_s, b, b_s, bool(a_2d), bool(b_2d), bool(trans_a), bool(trans_b), output_dtype is torch.float32)
        if out is not None:
            return out
    _no_gradients("blockwise_fp8_gemm", a, a_s, b, b_s)
    _same_device(a, a_s, b, b_s)
    assert a.dim() == 2 and b.dim() == 2 and a_s.dim() == 2 and b_s.dim() == 2, "operands and scales of two dims"
    av, asv = (a.t(), a_s.t()) if trans_a else (a, a_s)
    bv, bsv = (b, b_s) if trans_b else (b.t(), b_s.t())
    (M, K), N = av.shape, bv.shape[0]
    assert bv.shape[1] == K, f"Input B has reduction shape ({bv.shape[1]}) but {(K)} is expected."
    a_code, c_dtype = _code(a.dtype, "A"), rt.dtype_code(output_dtype)
    assert b.dtype == torch.float8_e4m3fn, f"B of type {b.dtype}: torch.float8_e4m3fn"
    _check_scales("A scale", asv, (_blocks(M) if a_2d else M, _blocks(K)))
    _check_scales("B scale", bsv, (_blocks(N) if b_2d else N, _blocks(K)))
    if K > _LONGEST:
        blocks = lambda s, lo, hi: s[:, lo // FP8_BLOCK_SIZE:_blocks(hi)]  # noqa: E731
        return _in_parts(K, lambda lo, hi: _gemm(av[:, lo:hi], blocks(asv, lo, hi), bv[:, lo:hi], blocks(bsv, lo, hi), a_2d, b_2d, False, True, torch.float32), output_dtype)
    c = torch.empty((M, N), dtype=output_dtype, device=a.device)
    if K == 0:
        return c.zero_()
    if c.numel():
        av, bv, asv, bsv = _operand(av), _operand(bv), _scales(asv), _scales(bsv)
        args = _Gemm(a=av.data_ptr(), b=bv.data_ptr(), a_scales=asv.data_ptr(), b_scales=bsv.data_ptr(), c=c.data_ptr(), M=M, N=N, K=K, lda=_stride(av, 0), ldb=_stride(bv, 0),
                     a_ss_r=_stride(asv, 0), a_ss_k=_stride(asv, 1), b_ss_r=_stride(bsv, 0), b_ss_k=_stride(bsv, 1), ldc=N, a_code=a_code, a_is_2d=int(bool(a_2d)),
                     b_is_2d=int(bool(b_2d)), c_dtype=c_dtype)
        _call("alto_mxfp4_fp8_gemm", args, a.device)
    return c


def blockwise_fp8_grouped_gemm(a: torch.Tensor, a_s: torch.Tensor, w: torch.Tensor, w_s: torch.Tensor, offsets: torch.Tensor, use_2dblock_w: bool = True,
                               trans_weights: bool = True, output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[m] = a[m] . W[e]^T for the rows ``offsets[e] <= m < offsets[e + 1]`` of each expert e; rows of no expert are zero.

    ``a`` [M, K] with scales [M, ceil(K/128)]; ``w`` [E, N, K] (``trans_weights=False``: [E, K, N]) of ``float8_e4m3fn``, scales [E, ceil(N/128), ceil(K/128)]
    (with ``use_2dblock_w=False`` [E, N, ceil(K/128)]), in w's orientation; ``offsets`` int32 [E + 1] on the device, non-decreasing, at most M: groups of any size (boundaries outside are
    taken as the nearest that are), E at most 65535.  The input gradient is the same product with the transposed codes.
    """
    if torch.compiler.is_compiling():
        return _between_graphs(_grouped, a, a_s, w, w_s, offsets, use_2dblock_w, trans_weights, output_dtype)
    return _grouped(a, a_s, w, w_s, offsets, use_2dblock_w, trans_weights, output_dtype)


def _grouped(a, a_s, w, w_s, offsets, w_2d, trans_weights, output_dtype):
    if output_dtype is torch.bfloat16 or output_dtype is torch.float32:
        out = rt.host().fp8_grouped_gemm(a, a_s, w, w_s, offsets, bool(w_2d), bool(trans_weights), output_dtype is torch.float32)
        if out is not None:
            return out
    _no_gradients("blockwise_fp8_grouped_gemm", a, a_s, w, w_s)
    _same_device(a, a_s, w, w_s, offsets)
    assert a.dim() == 2 and w.dim() == 3 and a_s.dim() == 2 and w_s.dim() == 3, "a of two dims, w of three, scales alike"
    _check_offsets(offsets)
    wv, wsv = (w, w_s) if trans_weights else (w.transpose(1, 2), w_s.transpose(1, 2))
    (M, K), (E, N, KW) = a.shape, wv.shape
    assert KW == K, f"Input K ({K}) must match weight K ({KW})"
    assert offsets.shape[0] == E + 1, f"{offsets.shape[0]} offsets for {E} experts"
    a_code, c_dtype = _code(a.dtype, "a"), rt.dtype_code(output_dtype)
    assert w.dtype == torch.float8_e4m3fn, f"w of type {w.dtype}: torch.float8_e4m3fn"
    _check_scales("a scale", a_s, (M, _blocks(K)))
    _check_scales("w scale", wsv, (E, _blocks(N) if w_2d else N, _blocks(K)))
    if K > _LONGEST:
        blocks = lambda s, lo, hi: s[..., lo // FP8_BLOCK_SIZE:_blocks(hi)]  # noqa: E731
        return _in_parts(K, lambda lo, hi: _grouped(a[:, lo:hi], blocks(a_s, lo, hi), wv[..., lo:hi], blocks(wsv, lo, hi), offsets, w_2d, True, torch.float32), output_dtype)
    out = torch.empty((M, N), dtype=output_dtype, device=a.device)
    if K == 0:
        return out.zero_()
    if out.numel():
        av, wv, asv, wsv, offs = _operand(a), _operand(wv), _scales(a_s), _scales(wsv), offsets.contiguous()
        args = _Grouped(a=av.data_ptr(), w=wv.data_ptr(), a_scales=asv.data_ptr(), w_scales=wsv.data_ptr(), c=out.data_ptr(), offs=offs.data_ptr(), M=M, N=N, K=K, lda=_stride(av, 0),
                        a_ss_r=_stride(asv, 0), a_ss_k=_stride(asv, 1), w_se=_stride(wv, 0), ldw=_stride(wv, 1), ws_e=_stride(wsv, 0), ws_r=_stride(wsv, 1), ws_k=_stride(wsv, 2),
                        ldc=N, a_code=a_code, w_is_2d=int(bool(w_2d)), c_dtype=c_dtype, groups=E)
        _call("alto_mxfp4_fp8_grouped_gemm", args, a.device)
    return out


def blockwise_fp8_grouped_gemm_weights(grad_output: torch.Tensor, go_s: torch.Tensor, inputs: torch.Tensor, x_s: torch.Tensor, offsets: torch.Tensor,
                                       output_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Weight gradients by group, [E, N, K]: dW[e] = dY_e^T X_e over the rows of each group e (zeros for a group without rows).

    ``grad_output`` [P, N] and ``inputs`` [P, K] with scales [P/128, N] and [P/128, K] are the second pairs that :func:`quantize_blockwise_fp8_rowcol` returns with the
    same ``offsets``; the gradient may be ``float8_e5m2``.  P of 2^22 and more is taken in parts, whose sums are added in fp32.
    """
    if torch.compiler.is_compiling():
        return _between_graphs(_grouped_weights, grad_output, go_s, inputs, x_s, offsets, output_dtype)
    return _grouped_weights(grad_output, go_s, inputs, x_s, offsets, output_dtype)


def _grouped_weights(go, go_s, x, x_s, offsets, output_dtype):
    if output_dtype is torch.bfloat16 or output_dtype is torch.float32:
        out = rt.host().fp8_grouped_gemm_weights(go, go_s, x, x_s, offsets, output_dtype is torch.float32)
        if out is not None:
            return out
    _no_gradients("blockwise_fp8_grouped_gemm_weights", go, go_s, x, x_s)
    _same_device(go, go_s, x, x_s, offsets)
    assert go.dim() == 2 and x.dim() == 2 and go_s.dim() == 2 and x_s.dim() == 2, "operands and scales of two dims"
    _check_offsets(offsets)
    (P, N), K, E = go.shape, x.shape[1], offsets.shape[0] - 1
    assert x.shape[0] == P and P % FP8_BLOCK_SIZE == 0, f"{P} and {x.shape[0]} tokens: the same number, whole blocks of {FP8_BLOCK_SIZE}"
    go_code, dw_dtype = _code(go.dtype, "grad_output"), rt.dtype_code(output_dtype)
    assert x.dtype == torch.float8_e4m3fn, f"inputs of type {x.dtype}: torch.float8_e4m3fn"
    _check_scales("grad_output scale", go_s, (P // FP8_BLOCK_SIZE, N))
    _check_scales("input scale", x_s, (P // FP8_BLOCK_SIZE, K))
    if P > _PART:
        # the groups' tokens lie in whole blocks, one group's behind another's: a part's boundaries are theirs, cut off at its ends
        ends = torch.cummax(offsets.clamp(min=0).long(), 0).values
        padded = torch.cat([ends[:1], ends.diff()]).add_(FP8_BLOCK_SIZE - 1).div_(FP8_BLOCK_SIZE, rounding_mode="floor").cumsum(0).mul_(FP8_BLOCK_SIZE)
        blocks = lambda s, lo, hi: s[lo // FP8_BLOCK_SIZE:hi // FP8_BLOCK_SIZE]  # noqa: E731
        return _in_parts(P, lambda lo, hi: _grouped_weights(go[lo:hi], blocks(go_s, lo, hi), x[lo:hi], blocks(x_s, lo, hi), (padded - lo).clamp_(0, hi - lo).int(), torch.float32), output_dtype)
    dw = torch.empty((E, N, K), dtype=output_dtype, device=go.device)
    if P == 0:
        return dw.zero_()
    if dw.numel():
        gv, xv, offs = _operand(go.t()), _operand(x.t()), offsets.contiguous()
        gs, xs = (s if s.shape[1] == 1 or s.stride(1) == 1 else s.contiguous() for s in (go_s.resolve_neg(), x_s.resolve_neg()))
        args = _Weights(go=gv.data_ptr(), x=xv.data_ptr(), go_scales=gs.data_ptr(), x_scales=xs.data_ptr(), dw=dw.data_ptr(), offs=offs.data_ptr(), tokens=P, N=N, K=K,
                        go_ld=_stride(gv, 0), x_ld=_stride(xv, 0), go_ss=_stride(gs, 0), x_ss=_stride(xs, 0), dw_se=dw.stride(0), ld_dw=dw.stride(1), go_code=go_code,
                        dw_dtype=dw_dtype, groups=E)
        _call("alto_mxfp4_fp8_grouped_gemm_weights", args, go.device)
    return dw


# --------------------------------------------------------------------------------------------------------------- layers
def _quantized_weight(owner: torch.Tensor, w: torch.Tensor, want_transposed: bool):
    """(codes, scales, codes of the transposed storage) of w [N, K] or [E, N, K] in blocks of 128 x 128; the cache entry (``enable_weight_cache``, both copies) belongs
    to ``owner``."""
    both = want_transposed or weight_cache_enabled()

    def make():
        if torch.is_inference_mode_enabled() and weight_cache_enabled():   # (what is kept may serve a training step, whose graph cannot save tensors of that mode)
            with torch.inference_mode(False):
                return copies()
        return copies()

    def copies():
        if w.stride(-1) != 1 and w.stride(-2) == 1:   # (stored the other way round: a block is square, so the copies swap places)
            qt, s, q, _ = _copies(w.transpose(-1, -2), both, True, True, torch.float8_e4m3fn)
            return q.transpose(-1, -2), s.transpose(-1, -2), qt.transpose(-1, -2) if both else None
        q, s, qt, _ = _copies(w, True, both, True, torch.float8_e4m3fn)
        return q, s, qt
    return cached_weight_quantisation(owner, ("blockwise_fp8", tuple(w.shape), tuple(w.stride())), make)


class BlockwiseFP8LinearFunction(torch.autograd.Function):
    """y = x W^T, dX = dY W and dW = dY^T X, each on operands quantized along its reduction; x [M, K], W [N, K]."""

    @staticmethod
    def forward(ctx, x, weight, grad_dtype, training):
        w = unwrap_weight_wrapper(weight)
        want_dx, want_dw = (training and n for n in ctx.needs_input_grad[:2])   # (those say what requires gradients under no_grad as well)
        xq, xs, xt, xts = _copies(x, True, want_dw, False, torch.float8_e4m3fn)
        wq, ws, wt = _quantized_weight(weight, w, want_dx)
        ctx.save_for_backward(xt, xts, wt if want_dx else None, ws if want_dx else None)
        ctx.more = grad_dtype, x.dtype, w.dtype
        return _gemm(xq, xs, wq, ws, False, True, False, True, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xt, xts, wt, ws = ctx.saved_tensors
        grad_dtype, x_dtype, w_dtype = ctx.more
        want_dx, want_dw = ctx.needs_input_grad[:2]
        dq, ds, dt, dts = _copies(dy, want_dx, want_dw, False, grad_dtype)
        dx = _gemm(dq, ds, wt, ws, False, True, False, False, x_dtype) if want_dx else None
        dw = _gemm(dt, dts, xt, xts, False, False, True, False, w_dtype) if want_dw else None
        return dx, dw, None, None


def _check_layer(what: str, x: torch.Tensor, weight: torch.Tensor, grad_dtype: torch.dtype) -> None:
    rt.refuse_transforms(what, x, weight)
    rt.require_gpu(x, weight)
    for name, t in (("x", x), ("weight", weight)):
        assert t.dtype in (torch.bfloat16, torch.float32), f"{name} of type {t.dtype}: bfloat16 or float32"
    assert x.device == weight.device, f"tensors on {x.device} and {weight.device}"
    _code(grad_dtype, "gradients")


def blockwise_fp8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, grad_dtype: torch.dtype = torch.float8_e4m3fn) -> torch.Tensor:
    """``x @ weight.T (+ bias)`` with 8-bit operands in all three products of a training step; x [..., K], weight [N, K], bf16 or fp32, of any sizes.

    x and the gradient are quantized in blocks of 1 x 128 along each product's reduction (the gradient to ``grad_dtype``, E4M3 or E5M2), the weight in blocks
    of 128 x 128.  The result has x's type (with a bias of another, what torch's sum of them has), each gradient its tensor's; of fp32 tensors too
    the products hold what :func:`blockwise_fp8_gemm` says.  Without a graph to build only the forward product's operands are made.
    """
    if torch.compiler.is_compiling():
        return _between_graphs(_linear, x, weight, bias, grad_dtype)
    return _linear(x, weight, bias, grad_dtype)


def _linear(x, weight, bias, grad_dtype):
    _check_layer("blockwise_fp8_linear", x, weight, grad_dtype)
    assert weight.dim() == 2 and x.dim() >= 1 and x.shape[-1] == weight.shape[1], f"x of shape {tuple(x.shape)} and weight of {tuple(weight.shape)}"
    y = BlockwiseFP8LinearFunction.apply(x.reshape(-1, x.shape[-1]) if x.shape[-1] else x.reshape(x.shape[:-1].numel(), 0), weight, grad_dtype, torch.is_grad_enabled())
    y = y.view(*x.shape[:-1], weight.shape[0])
    return y if bias is None else y + bias


class BlockwiseFP8GroupedFunction(torch.autograd.Function):
    """y[m] = x[m] W[e]^T for the rows m of each expert e, and its gradients; x [M, K], W [E, N, K], or [E, K, N] without ``trans_weights``."""

    @staticmethod
    def forward(ctx, x, weight, offsets, grad_dtype, trans_weights, training):
        w = unwrap_weight_wrapper(weight)
        w = w if trans_weights else w.transpose(1, 2)
        want_dx, want_dw = (training and n for n in ctx.needs_input_grad[:2])
        xq, xs, xt, xts = _copies(x, True, want_dw, False, torch.float8_e4m3fn, offsets if want_dw else None)
        wq, ws, wt = _quantized_weight(weight, w, want_dx)
        ctx.save_for_backward(xt, xts, wt if want_dx else None, ws if want_dx else None, offsets)
        ctx.more = grad_dtype, x.dtype, w.dtype, trans_weights
        return _grouped(xq, xs, wq, ws, offsets, True, True, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xt, xts, wt, ws, offsets = ctx.saved_tensors
        grad_dtype, x_dtype, w_dtype, trans_weights = ctx.more
        want_dx, want_dw = ctx.needs_input_grad[:2]
        dq, ds, dt, dts = _copies(dy, want_dx, want_dw, False, grad_dtype, offsets if want_dw else None)
        dx = _grouped(dq, ds, wt, ws, offsets, True, False, x_dtype) if want_dx else None
        dw = None
        if want_dw and not trans_weights and grad_dtype is torch.float8_e4m3fn:   # (the products' second operand is E4M3)
            dw = _grouped_weights(xt, xts, dt, dts, offsets, w_dtype)
        elif want_dw:
            dw = _grouped_weights(dt, dts, xt, xts, offsets, w_dtype)
            dw = dw if trans_weights else dw.transpose(1, 2)
        return dx, dw, None, None, None, None


def blockwise_fp8_grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, grad_dtype: torch.dtype = torch.float8_e4m3fn,
                                 trans_weights: bool = True) -> torch.Tensor:
    """:func:`blockwise_fp8_linear` with rows grouped by expert: x [M, K], weight [E, N, K] (``trans_weights=False``: [E, K, N]), rows
    ``offsets[e] <= m < offsets[e + 1]`` meet weight[e].

    ``offsets``: int32 [E + 1] on the device, non-decreasing, at most M; groups of any size, E at most 65535.  Rows of no expert, and their gradients, are zero.  The blocks of the weight
    gradients' operands start anew with each group.
    """
    if torch.compiler.is_compiling():
        return _between_graphs(_grouped_linear, x, weight, offsets, grad_dtype, trans_weights)
    return _grouped_linear(x, weight, offsets, grad_dtype, trans_weights)


def _grouped_linear(x, weight, offsets, grad_dtype, trans_weights):
    _check_layer("blockwise_fp8_grouped_linear", x, weight, grad_dtype)
    _same_device(x, offsets)
    assert x.dim() == 2 and weight.dim() == 3 and x.shape[1] == weight.shape[2 if trans_weights else 1], f"x of shape {tuple(x.shape)} and weight of {tuple(weight.shape)}"
    _check_offsets(offsets)
    assert offsets.shape[0] == weight.shape[0] + 1, f"{offsets.shape[0]} offsets for {weight.shape[0]} experts"
    return BlockwiseFP8GroupedFunction.apply(x, weight, offsets.contiguous(), grad_dtype, bool(trans_weights), torch.is_grad_enabled())
