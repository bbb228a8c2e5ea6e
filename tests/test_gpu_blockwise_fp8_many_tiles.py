"""More than 2^22 tiles in one launch.  Codes that are whole numbers: sums exact in fp32 in any order, rounded once."""
import pytest
import torch

import alto_amd.mxfp4 as mx

pytestmark = pytest.mark.gpu


def whole(rows, K, seed):
    return torch.randint(-15, 16, (rows, K), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(torch.bfloat16).to(torch.float8_e4m3fn)


def test_by_group():
    E, M, N, K = 1024, 2048, 2 ** 19, 256   # 1034 pieces of rows at most, 4096 columns of tiles
    q, w, s, w_s = whole(M, K, 1), whole(N, K, 2), torch.ones((M, 2), device="cuda"), torch.ones((N // 128, 2), device="cuda")
    offsets = torch.arange(0, M + 1, 2, dtype=torch.int32, device="cuda")
    got = mx.blockwise_fp8_grouped_gemm(q, s, w.expand(E, N, K), w_s.expand(E, *w_s.shape), offsets)
    assert torch.equal(got, mx.blockwise_fp8_gemm(q, s, w, w_s, use_2dblock_b=True, trans_b=True))
    a, b = q.float(), w.float()
    for n in range(0, N, 2 ** 17):
        assert torch.equal(got[:, n:n + 2 ** 17], (a @ b[n:n + 2 ** 17].t()).to(torch.bfloat16))


def test_one_weight():
    M, N, K = 262144, 262272, 16   # 2048 x 2049 tiles of 128 x 128; the result alone is 128 GiB
    if torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved() - torch.cuda.memory_allocated() < 150 * 2 ** 30:
        pytest.skip("needs 150 GiB of device memory")
    torch.cuda.empty_cache()
    q, w = whole(M, K, 1), whole(N, K, 2)
    got = mx.blockwise_fp8_gemm(q, torch.ones((M, 1), device="cuda"), w, torch.ones((N // 128, 1), device="cuda"), use_2dblock_b=True, trans_b=True)
    a, b = q.float(), w.float()
    for m in range(0, M, 4096):
        assert torch.equal(got[m:m + 4096], (a[m:m + 4096] @ b.t()).to(torch.bfloat16)), m
    del got
    torch.cuda.empty_cache()
