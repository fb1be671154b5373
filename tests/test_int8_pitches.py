"""Row pitches that nothing reads are not judged.  The calls pass every check and stop at the missing device."""
import pytest

from thunderkittens_b200 import _lib as L

FAR = [0x7F0000001000 + (i << 32) for i in range(5)]
ALIGN, NO_DEVICE = 2, 3


def test_pitches_of_a_single_row(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where nothing can be launched")
    A, SA, B, SB, D = FAR
    f = lib.tkb_int8_gemm
    for lda in (0, 1, 40, 64, 4096):
        assert f(A, lda, SA, B, 0, SB, D, 0, L.DTYPE_BF16, 1, 8, 64, None) == NO_DEVICE
        assert f(A, lda, SA, B, 48, SB, D, 0, L.DTYPE_BF16, 1, 1, 50, None) == NO_DEVICE
    assert f(A, 0, SA, B, 0, SB, D, 3, L.DTYPE_FP32, 1, 8, 64, None) == NO_DEVICE
    assert f(A, 64, SA, B, 7, SB, D, 0, L.DTYPE_FP32, 4, 1, 64, None) == NO_DEVICE
    # several rows are judged
    assert f(A, 48, SA, B, 0, SB, D, 0, L.DTYPE_BF16, 2, 8, 64, None) == ALIGN
    assert f(A, 0, SA, B, 48, SB, D, 0, L.DTYPE_BF16, 1, 8, 64, None) == ALIGN
    assert f(A, 0, SA, B, 0, SB, D, 7, L.DTYPE_BF16, 2, 8, 64, None) == ALIGN
