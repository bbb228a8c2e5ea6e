"""Calls on a wrapped weight of the 8-bit layers: arguments by position or by name reach the layers, what these do not offer is refused (the layers stood in for)."""
import pytest
import torch

import alto_amd.mxfp4 as mx
from alto_amd.mxfp4 import tensor as T

CONFIG = mx.TrainingOpConfig(precision="blockwise_fp8")
X, W, B = torch.zeros(4, 256), mx.BlockwiseFP8TrainingWeightWrapperTensor(torch.zeros(256, 8), CONFIG), torch.arange(8.0)
L = mx.BlockwiseFP8TrainingWeightWrapperTensor(torch.zeros(8, 256), CONFIG)
E, OFFS = mx.BlockwiseFP8TrainingWeightWrapperTensor(torch.zeros(2, 256, 8), CONFIG), torch.tensor([1, 4], dtype=torch.int32)


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(T, "blockwise_fp8_linear", lambda x, w, bias=None: made.append((x, tuple(w.shape), bias)) or torch.full((4, 8), 2.0))
    monkeypatch.setattr(T, "blockwise_fp8_grouped_linear", lambda x, w, offsets, trans_weights: made.append((x, tuple(w.shape), offsets.tolist(), trans_weights)) or torch.full((4, 8), 3.0))
    return made


@pytest.mark.parametrize("call,bias", [
    (lambda: torch.nn.functional.linear(X, L), None), (lambda: torch.nn.functional.linear(X, L, B), B), (lambda: torch.nn.functional.linear(input=X, weight=L, bias=B), B),
    (lambda: torch.nn.functional.linear(X, weight=L), None), (lambda: torch.mm(X, W), None), (lambda: torch.mm(X, mat2=W), None), (lambda: X.mm(mat2=W), None), (lambda: torch.mm(input=X, mat2=W), None),
    (lambda: X @ W, None), (lambda: torch.matmul(X, other=W), None), (lambda: torch.addmm(B, X, W), B), (lambda: B.addmm(X, W), B), (lambda: torch.addmm(B, X, mat2=W), B),
    (lambda: torch.addmm(input=B, mat1=X, mat2=W, beta=1, alpha=1), B), (lambda: torch.ops.aten.addmm(self=B, mat1=X, mat2=W), B), (lambda: torch.ops.aten.mm.default(X, W), None),
    (lambda: torch.mm(X, W, out_dtype=torch.float32), None),
])
def test_products(calls, call, bias):
    assert bool((call() == 2).all())
    (x, shape, given), = calls
    assert x is X and shape == (8, 256) and given is bias


@pytest.mark.parametrize("call", [
    lambda: torch._grouped_mm(X, E, OFFS), lambda: torch._grouped_mm(X, E, offs=OFFS), lambda: torch._grouped_mm(X, mat2=E, offs=OFFS), lambda: torch._grouped_mm(input=X, mat2=E, offs=OFFS),
    lambda: torch._grouped_mm(X, E, OFFS, None, None), lambda: torch._grouped_mm(X, E, OFFS, out_dtype=torch.float32), lambda: torch.nn.functional.grouped_mm(X, E, offs=OFFS),
])
def test_grouped_products(calls, call):
    assert bool((call() == 3).all())
    (x, shape, offsets, trans), = calls
    assert x is X and shape == (2, 256, 8) and offsets == [0, 1, 4] and trans is False


@pytest.mark.parametrize("call,text", [
    (lambda: torch._grouped_mm(X, E, offs=OFFS, out_dtype=torch.bfloat16), "out_dtype"), (lambda: torch._grouped_mm(X, E, OFFS, None, torch.bfloat16), "out_dtype"), (lambda: torch._grouped_mm(X, E, OFFS, B), "[Bb]ias"),
    (lambda: torch._grouped_mm(X, E, offs=OFFS, bias=B), "[Bb]ias"), (lambda: torch._grouped_mm(X, E), "offsets"), (lambda: torch._grouped_mm(X, W, OFFS), "offsets"),
    (lambda: torch.mm(X, W, out=torch.empty(4, 8)), "out"), (lambda: torch.matmul(X, W, out=torch.empty(4, 8)), "out"), (lambda: torch.addmm(B, X, W, out=torch.empty(4, 8)), "out"),
    (lambda: torch.mm(X, W, torch.float64), "arguments"), (lambda: torch.mm(X, W, out_dtype=torch.bfloat16), "out_dtype"), (lambda: torch.addmm(B, X, W, torch.bfloat16), "arguments"),
    (lambda: torch.addmm(B, X, W, out_dtype=torch.bfloat16), "out_dtype"), (lambda: torch.addmm(B, X, W, beta=2), "beta"), (lambda: torch.addmm(B, X, W, alpha=0), "alpha"),
    (lambda: torch.mm(W, X), "second operand"), (lambda: torch.addmm(W, X, X), "second operand"),
])
def test_what_the_layers_do_not_offer(calls, call, text):
    with pytest.raises(AssertionError, match=text):
        call()
    assert not calls
