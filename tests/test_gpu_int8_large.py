"""int8_gemm on operands whose bytes pass 32-bit offsets, as weights of many outputs and as tokens of a long prompt."""
import pytest
import torch

from tests.test_gpu_int8 import _check_gemm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(7, 600001, 8192), (200, 600000, 8192), (270000, 96, 16384), (2, 40000, 131056)])
def test_operands_past_32_bit_offsets(cuda, lib, M, N, K):
    import thunderkittens_b200.ops as ops
    g = torch.Generator(device=cuda).manual_seed(M)
    a = torch.randint(-128, 128, (M, K), generator=g, device=cuda, dtype=torch.int8)
    b = torch.randint(-128, 128, (N, K), generator=g, device=cuda, dtype=torch.int8)
    a_sc, b_sc = torch.rand(M, generator=g, device=cuda) * 2e-3, torch.rand(N, generator=g, device=cuda) * 2e-3 / K ** 0.5
    D = torch.full((M, N), float("nan"), device=cuda)
    ops.int8_gemm(a, a_sc, b, b_sc, D)

    def parts(n):                                    # the ends, and round the rows that begin at 2^31 and 2^32 bytes
        at = [c for e in (2 ** 31, 2 ** 32) for c in (e // K - 40, e // K + 40) if 0 < c < n]
        return [slice(0, 64), slice(max(0, n - 64), n)] + [slice(lo, hi) for lo, hi in zip(at[::2], at[1::2])]

    for rows in parts(M):
        for cols in parts(N):
            _check_gemm(D[rows, cols], a[rows], a_sc[rows], b[cols], b_sc[cols])
    assert not bool(torch.isnan(D).any())
