"""The largest products of 8-bit operands that one launch holds, by way of the C entries in a process that sees no GPU: what the checks let through fails at the launch, by name."""
import json
import os
import subprocess
import sys

import pytest

PROGRAM = """
import ctypes, json, sys
import alto_amd.mxfp4
from alto_amd import _lib
from alto_amd.mxfp4 import blockwise_fp8 as F
memory = ctypes.create_string_buffer(4096)   # stands for device memory
P, lib = ctypes.addressof(memory) + (-ctypes.addressof(memory)) % 256, _lib.load()
for kind, args in json.load(sys.stdin):
    struct, entry = {"gemm": (F._Gemm, "gemm"), "grouped": (F._Grouped, "grouped_gemm"), "weights": (F._Weights, "grouped_gemm_weights")}[kind]
    pointers = {n: P for n, t in struct._fields_ if t is ctypes.c_void_p}
    rc = getattr(lib, "alto_mxfp4_fp8_" + entry)(ctypes.byref(struct(**pointers, **args)), None)
    print(json.dumps([rc, lib.alto_mxfp4_last_error().decode()]))
"""


def gemm(M, N, K):
    return "gemm", dict(M=M, N=N, K=K, lda=K, ldb=K, a_ss_r=1, a_ss_k=M, b_ss_r=1, b_ss_k=N, ldc=N, b_is_2d=1)


def grouped(M, N, K, groups):
    return "grouped", dict(M=M, N=N, K=K, lda=K, a_ss_r=1, a_ss_k=M, ldw=K, ws_r=1, ws_k=N, ldc=N, w_is_2d=1, groups=groups)


def weights(tokens, N, K, groups):
    return "weights", dict(tokens=tokens, N=N, K=K, go_ld=tokens, x_ld=tokens, go_ss=N, x_ss=K, dw_se=N * K, ld_dw=K, groups=groups)


LAUNCHED = {
    "2^22 tiles of 128 x 128": gemm(262144, 262272, 128),
    "2^24 of those, a quarter as many of 256 x 256": gemm(2 ** 19, 2 ** 19 + 128, 128),
    "2^22 tiles of 256 x 256": gemm(2 ** 19, 2 ** 19 + 256, 4096),
    "the most groups": grouped(131072, 8192, 1024, 65535),
    "by group, 2^24 tiles of 128 x 128, fewer of 256 x 256": grouped(2 ** 23 - 1, 22016, 1024, 32768),
    "by group, 2^22 tiles of 256 x 256": grouped(2 ** 23, 40960, 1024, 8),
    "weight gradients, 2^22 tiles of 256 x 256": weights(128, 2 ** 20, 2 ** 18 + 256, 1),
}
TOO_MANY = {
    "2^23 tiles of 256 x 256": gemm(2 ** 20, 2 ** 19, 4096),
    "by group, 2^23 tiles of 256 x 256": grouped(2 ** 23, 65536 + 256, 1024, 8),
    "weight gradients, 2^23 tiles of 256 x 256": weights(128, 2 ** 20, 2 ** 19, 1),
}


@pytest.fixture(scope="module")
def answers():
    env = dict(os.environ, HIP_VISIBLE_DEVICES="", ROCR_VISIBLE_DEVICES="", CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", PROGRAM], input=json.dumps([*LAUNCHED.values(), *TOO_MANY.values()]), capture_output=True, text=True, env=env, timeout=300,
                       cwd=os.path.join(os.path.dirname(__file__), ".."))
    assert r.returncode == 0, r.stderr[-3000:]
    return dict(zip([*LAUNCHED, *TOO_MANY], map(json.loads, r.stdout.splitlines())))


@pytest.mark.parametrize("name", LAUNCHED)
def test_reaches_its_launch(answers, name):
    rc, text = answers[name]
    assert rc < 0 and ("launch failed" in text or "could not reserve" in text), text


@pytest.mark.parametrize("name", TOO_MANY)
def test_too_many_tiles(answers, name):
    rc, text = answers[name]
    assert rc < 0 and "too many tiles" in text, text
