"""Layouts of the row kernels that depend on how many rows there are and on where they begin: several rows in a CTA, gates of sequences
staged two at a time, rows that begin anywhere, outputs that are larger than L2.  Tolerances as derived in test_gpu_norm."""
import pytest
import torch

from tests.int8_common import norm64, padded
from tests.test_gpu_norm import EPS, HALF, S, _check_block, _inputs

pytestmark = pytest.mark.gpu


def _ops():
    import thunderkittens_b200.ops as ops
    return ops


@pytest.mark.parametrize("M,G,K", [(4096, 2, 12288), (4096, 2, 11300), (4000, 4, 12001), (3400, 4, 10241), (5000, 2500, 6800), (300, 300, 12288), (600, 2, 1000)])
def test_block_norm_does_not_depend_on_which_outputs_are_asked_for(cuda, lib, M, G, K):
    """Y, the codes, or both: they are the same, and so is R.  Large calls with Y alone keep fewer rows in a CTA."""
    x, h, w1, w2 = _inputs(M, K, torch.bfloat16, cuda, 11)
    g = torch.Generator(device=cuda).manual_seed(K)
    gate = torch.randn(G, K, generator=g, device=cuda).to(torch.bfloat16)
    got = []
    for y, codes in ((True, False), (False, True), (True, True)):
        R = torch.zeros_like(x)
        Y = torch.zeros_like(x) if y else None
        q, sc = (padded(M, K, torch.int8, cuda)[0], torch.empty(M, device=cuda)) if codes else (None, None)
        _ops().block_norm(h, x, R, w1, gate, 0.5, w2, Y, q, sc, eps=EPS)
        got.append((R, Y, q, sc))
    assert torch.equal(got[0][0], got[2][0]) and torch.equal(got[1][0], got[2][0])
    assert torch.equal(got[0][1], got[2][1])
    assert torch.equal(got[1][2], got[2][2]) and torch.equal(got[1][3], got[2][3])
