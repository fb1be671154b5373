"""Refusals of the int8 and norm entries that need no device.  EVERY call below fails validation (or has no rows); none reaches a
launch, so the made-up addresses are never used, with or without a GPU."""
import pytest

from thunderkittens_b200 import _lib as L

P = 0x7F0000001000
FAR = [P + (i << 32) for i in range(8)]
INVALID, ALIGN = 1, 2
BF16, FP16, FP32 = L.DTYPE_BF16, L.DTYPE_FP16, L.DTYPE_FP32


def _msg(lib):
    return lib.tkb_last_error().decode()


def test_int8_quantize(lib):
    f = lib.tkb_int8_quantize
    A, Q, S = FAR[:3]
    assert f(None, 0, BF16, Q, 0, S, 4, 64, None) == INVALID and "null" in _msg(lib)
    assert f(A, 0, BF16, None, 0, S, 4, 64, None) == INVALID and f(A, 0, BF16, Q, 0, None, 4, 64, None) == INVALID
    assert f(A, 0, FP32, Q, 0, S, 4, 64, None) == INVALID and "dtype" in _msg(lib)
    assert f(A, 0, BF16, Q, 0, A + 256, 4, 64, None) == INVALID and f(A, 0, BF16, Q, 0, Q + 252, 4, 64, None) == INVALID and "overlap" in _msg(lib)
    assert f(A, 0, BF16, Q, 0, S, 2 ** 30 + 1, 64, None) == INVALID
    assert f(A, 0, BF16, Q, 0, S, -1, 64, None) == INVALID and f(A, 0, BF16, Q, 0, S, 4, 0, None) == INVALID
    assert f(A, 0, BF16, Q, 0, S, 4, 65537, None) == INVALID and "65536" in _msg(lib)
    assert f(A, 63, BF16, Q, 0, S, 4, 64, None) == ALIGN and f(A, 0, BF16, Q, 63, S, 4, 64, None) == ALIGN
    assert f(A + 1, 0, BF16, Q, 0, S, 4, 64, None) == ALIGN and f(A, 0, BF16, Q, 0, S + 2, 4, 64, None) == ALIGN
    assert f(A, 0, BF16, A, 0, S, 4, 64, None) == INVALID and "overlap" in _msg(lib)
    assert f(A, 0, BF16, A + 511, 0, S, 4, 64, None) == INVALID and f(A, 0, BF16, A - 255, 0, S, 4, 64, None) == INVALID
    assert f(A, 100, BF16, A + 128, 200, S, 4, 73, None) == INVALID            # a column slice that reaches the next row
    assert f(None, 0, BF16, None, 0, None, 0, 64, None) == 0                   # no rows


def test_int8_gemm(lib):
    f = lib.tkb_int8_gemm
    A, SA, B, SB, D = FAR[:5]
    for i in (0, 2, 3, 5, 6):
        args = [A, 0, SA, B, 0, SB, D, 0, BF16, 8, 8, 64, None]
        args[i] = None
        assert f(*args) == INVALID and "null" in _msg(lib)
    assert f(A, 0, SA, B, 0, SB, D, 0, 3, 8, 8, 64, None) == INVALID and "dtype" in _msg(lib)
    for M, N, K in ((-1, 8, 64), (8, 0, 64), (8, 8, 0), (2 ** 30 + 1, 8, 64), (8, 2 ** 31 - 1, 64), (8, 8, 131072)):
        assert f(A, 0, SA, B, 0, SB, D, 0, BF16, M, N, K, None) == INVALID
    assert "131071" in _msg(lib)
    assert f(A, 0, SA, B, 0, SB, D, 0, BF16, 8, 8, 72, None) == ALIGN and "padded" in _msg(lib)
    assert f(A, 48, SA, B, 0, SB, D, 0, BF16, 8, 8, 64, None) == ALIGN and f(A, 0, SA, B, 0, SB, D, 7, BF16, 8, 8, 64, None) == ALIGN
    assert f(A + 8, 0, SA, B, 0, SB, D, 0, BF16, 8, 8, 64, None) == ALIGN and f(A, 0, SA, B + 1, 0, SB, D, 0, BF16, 8, 8, 64, None) == ALIGN
    assert f(A, 0, SA + 1, B, 0, SB, D, 0, BF16, 8, 8, 64, None) == ALIGN and f(A, 0, SA, B, 0, SB, D + 2, 0, FP32, 8, 8, 64, None) == ALIGN
    for config in (-1, L.GEMM_PAIR_M512_N256, 99):
        assert lib.tkb_int8_gemm_ex(A, 0, SA, B, 0, SB, D, 0, BF16, 8, 8, 64, config, None) == INVALID and "config" in _msg(lib)
    assert f(None, 0, None, B, 0, SB, None, 0, BF16, 0, 8, 64, None) == 0      # no rows


def test_int8_gemm_output_over_an_operand(lib):
    f = lib.tkb_int8_gemm
    A, SA, B, SB, D = FAR[:5]
    for D in (A, A + 8 * 64 - 2, SA + 28, SA - 126, B + 64, SB):               # 8 x 8 bf16: 128 bytes
        assert f(A, 0, SA, B, 0, SB, D, 0, BF16, 8, 8, 64, None) == INVALID and "overlaps" in _msg(lib)


def test_rms_norm(lib):
    f = lib.tkb_rms_norm
    X, W, Y, Q, S = FAR[:5]
    assert f(None, 0, W, Y, 0, None, 0, None, BF16, 4, 64, 1e-6, None) == INVALID and f(X, 0, None, Y, 0, None, 0, None, BF16, 4, 64, 1e-6, None) == INVALID
    assert f(X, 0, W, None, 0, None, 0, None, BF16, 4, 64, 1e-6, None) == INVALID and "no output" in _msg(lib)
    assert f(X, 0, W, Y, 0, Q, 0, None, BF16, 4, 64, 1e-6, None) == INVALID and "together" in _msg(lib)
    assert f(X, 0, W, Y, 0, None, 0, None, BF16, 4, 16385, 1e-6, None) == INVALID and "16384" in _msg(lib)
    for eps in (-1e-6, float("nan"), float("inf")):
        assert f(X, 0, W, Y, 0, None, 0, None, BF16, 4, 64, eps, None) == INVALID and "eps" in _msg(lib)
    assert f(X, 0, W, X, 0, None, 0, None, BF16, 4, 64, 1e-6, None) == INVALID and "overlap" in _msg(lib)
    assert f(X, 0, W, Y, 0, Y + 100, 0, S, BF16, 4, 64, 1e-6, None) == INVALID and "overlap" in _msg(lib)
    assert f(X, 0, W + 1, Y, 0, None, 0, None, BF16, 4, 64, 1e-6, None) == ALIGN and f(X, 60, W, Y, 0, None, 0, None, BF16, 4, 64, 1e-6, None) == ALIGN
    assert f(None, 0, None, None, 0, None, 0, None, FP16, 0, 64, 1e-6, None) == 0


def test_block_norm(lib):
    f = lib.tkb_block_norm
    H, X, R, W, G, V, Y, Q = FAR

    def call(h=H, ldh=0, x=X, ldx=0, r=R, ldr=0, w_post=W, gate=G, ldg=0, per=4, rs=1.0, w_pre=V, y=Y, ldy=0, q=None, ldq=0, sc=None, dtype=BF16, M=4, K=64, eps=1e-6):
        return f(h, ldh, x, ldx, r, ldr, w_post, gate, ldg, per, rs, w_pre, y, ldy, q, ldq, sc, dtype, M, K, eps, None)

    for name in ("h", "x", "r"):
        assert call(**{name: None}) == INVALID and "null" in _msg(lib)
    assert call(w_pre=None) == INVALID and call(y=None) == INVALID and "second norm" in _msg(lib)
    assert call(per=0) == INVALID and "rows_per_gate" in _msg(lib)
    assert call(dtype=FP32) == INVALID and call(K=16385) == INVALID and call(q=Q) == INVALID
    assert call(r=H) == INVALID and call(r=X, ldr=128) == INVALID and call(r=X + 2) == INVALID and call(y=X) == INVALID and call(y=R) == INVALID and "overlap" in _msg(lib)
    assert call(y=V) == INVALID and call(r=W) == INVALID and call(y=G + 126) == INVALID and call(y=G - 510, per=1) == INVALID and "gate" in _msg(lib)
    assert call(rs=float("inf")) == INVALID and call(rs=float("nan")) == INVALID and "residual_scale" in _msg(lib)
    assert call(gate=G + 1) == ALIGN and call(ldg=63) == ALIGN and call(ldr=1) == ALIGN
    assert call(h=None, x=None, r=None, w_post=None, gate=None, w_pre=None, y=None, M=0) == 0


def test_without_a_device_it_is_an_error(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert lib.tkb_int8_quantize(FAR[0], 0, BF16, FAR[1], 0, FAR[2], 4, 64, None) == 3
    assert lib.tkb_int8_gemm(FAR[0], 0, FAR[1], FAR[2], 0, FAR[3], FAR[4], 0, BF16, 8, 8, 64, None) == 3
    assert lib.tkb_rms_norm(FAR[0], 0, FAR[1], FAR[2], 0, None, 0, None, BF16, 4, 64, 1e-6, None) == 3
    # column slices of one buffer do not overlap: accepted up to the missing device
    assert lib.tkb_rms_norm(P, 128, FAR[1], P + 128, 128, None, 0, None, BF16, 4, 64, 1e-6, None) == 3


def test_ops_refuse_tensors_off_the_gpu():
    import torch
    from thunderkittens_b200 import ops
    x, q, s = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.int8_quantize(x, q, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.int8_gemm(q, s, q, s, torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rms_norm(x, x[0], x.clone())
    with pytest.raises(RuntimeError, match="must be a torch.Tensor"):
        ops.block_norm(None, x, x)


def test_ops_refuse_sizes_past_c_ints():
    """2^32 + 4 rows would arrive as 4."""
    import torch
    from thunderkittens_b200 import ops

    class Sized(torch.Tensor):               # a size on a CUDA device, and no memory
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError(f"{func} on a tensor without memory")

    def sized(shape, dtype):
        return torch.Tensor._make_wrapper_subclass(Sized, shape, dtype=dtype, device="cuda:0")

    for M, K in ((2 ** 32 + 4, 1), (4, 2 ** 32 + 16)):
        with pytest.raises(RuntimeError, match="sizes up to"):
            ops.int8_quantize(sized((M, K), torch.bfloat16), sized((M, K), torch.int8), sized((M,), torch.float32))
        with pytest.raises(RuntimeError, match="sizes up to"):
            ops.rms_norm(sized((M, K), torch.float16), sized((K,), torch.float16), sized((M, K), torch.float16))
