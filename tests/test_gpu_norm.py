"""rms_norm and block_norm against their definitions in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32).  A sum of squares adds at most 64 products in a thread and 10 more times across
the CTA, each a rounding: it is off by at most 75 u relative.  The mean, + eps, the inverse root and two products add 5 u, and the root
halves what is under it: a norm is off by at most S = 45 u relative to its value.  Stored values add half a step of their type.
r = residual_scale * x + gate * p is off by (S + u)|gate * p| + u|r| at most, with cancellation between its terms, and y by that much times
its own factor, by the same over the whole row in its root mean square, and by S."""
import pytest
import torch

from tests.int8_common import block64, gemm64, norm64, padded

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
S = 45 * U
EPS = 1e-5
HALF = [torch.bfloat16, torch.float16]


def _ops():
    import thunderkittens_b200.ops as ops
    return ops


def _inputs(M, K, dtype, cuda, seed):
    g = torch.Generator(device=cuda).manual_seed(seed + 31 * M + K)
    x, h = (torch.randn(M, K, generator=g, device=cuda) * s for s in (1.0, 3.0))
    w1, w2 = (1 + 0.2 * torch.randn(K, generator=g, device=cuda) for _ in range(2))
    if M > 2:
        x[2] = 0.0; h[2] = 0.0                      # a padding row
    return [t.to(dtype) for t in (x, h, w1, w2)]


def _close(got, ref, tol, what):
    half_step = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0                 # half of the smallest subnormal step of fp16
    tol = tol * (1 + half_step) + ref.abs() * half_step + tiny + 2.0 ** -140
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: {int((err > tol).sum())} of {err.numel()} off, worst {float((err / tol).max()):.3f} of the tolerance"


def _check_codes(q, sc, y, tol):
    """Codes and steps against the y of 64 bits, itself known to `tol` (absolute, per element)."""
    amax = y.abs().amax(1).clamp_min(2.0 ** -100)
    d = tol.amax(1)
    assert bool(((sc.double() - amax / 127).abs() <= d / 127 + sc.double() * 2 * U).all())
    # code * step is within half a step of y, and y within tol of itself
    assert bool(((q.double() * sc.double()[:, None] - y).abs() <= 0.5 * sc.double()[:, None] * (1 + 1e-5) + tol + 127 * sc.double()[:, None] * 4 * U).all())


SIZES = [(1, 1), (1, 8), (3, 7), (5, 130), (64, 2048), (9, 2056), (33, 4096), (4, 5001), (3, 7168), (2, 8200), (3, 16384), (2, 16383), (1500, 512), (300, 7168)]


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("M,K", SIZES)
def test_rms_norm(cuda, lib, M, K, dtype):
    x, _, w, _ = _inputs(M, K, dtype, cuda, 1)
    y = norm64(x, w, EPS)
    Y = torch.full((M, K), float("nan"), dtype=dtype, device=cuda)
    q, buf = padded(M, K, torch.int8, cuda, fill=99)
    sc = torch.empty(M, device=cuda)
    _ops().rms_norm(x, w, Y, eps=EPS)
    _close(Y, y, y.abs() * S, "Y")
    _ops().rms_norm(x, w, Y_int8=q, Y_sc=sc, eps=EPS)
    _check_codes(q, sc, y, y.abs() * S)
    assert bool((buf[:, K:] == 99).all())
    # both at once are the same two
    Y2, q2, sc2 = torch.zeros_like(Y), padded(M, K, torch.int8, cuda)[0], torch.empty(M, device=cuda)
    _ops().rms_norm(x, w, Y2, q2, sc2, eps=EPS)
    assert torch.equal(Y, Y2) and torch.equal(q, q2) and torch.equal(sc, sc2)


def _check_block(x, h, w_post, w_pre, gate, rs, R, Y, q, sc):
    r = block64(h, x, w_post, gate, rs, EPS)
    gp = (r - rs * x.double()).abs()
    tr = (S + U) * gp + U * r.abs() + 2 * U * (rs * x.double()).abs()
    _close(R, r, tr, "R")
    if w_pre is None:
        return
    y = norm64(r, w_pre, EPS)
    rms = torch.sqrt((r * r).mean(1, keepdim=True) + EPS)
    off = torch.sqrt((tr * tr).mean(1, keepdim=True)) / rms                  # relative error that tr brings into the root mean square
    ty = y.abs() * (S + off) * (1 + 1e-3) + tr / rms * w_pre.double().abs()
    if Y is not None:
        _close(Y, y, ty, "Y")
    if q is not None:
        _check_codes(q, sc, y, ty)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("M,K", SIZES)
def test_block_norm(cuda, lib, M, K, dtype):
    x, h, w1, w2 = _inputs(M, K, dtype, cuda, 2)
    g = torch.Generator(device=cuda).manual_seed(M * K)
    for post, gates, rs, quant in ((True, 1, 1.0, False), (False, None, 0.5, True), (True, M, -0.25, True), (False, 1, 1.0, False)):
        gate = None if gates is None else (0.3 * torch.randn(gates, K, generator=g, device=cuda)).to(dtype)
        R, Y = (torch.full((M, K), float("nan"), dtype=dtype, device=cuda) for _ in range(2))
        q, sc = (padded(M, K, torch.int8, cuda)[0], torch.empty(M, device=cuda)) if quant else (None, None)
        w_post = w1 if post else None
        _ops().block_norm(h, x, R, w_post, gate[0] if gates == 1 else gate, rs, w2, Y, q, sc, eps=EPS)
        _check_block(x, h, w_post, w2, gate, rs, R, Y, q, sc)
    # without the second norm, in place
    X = x.clone()
    _ops().block_norm(h, X, X, w1, None, 1.0, eps=EPS)
    _check_block(x, h, w1, None, None, 1.0, X, None, None, None)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("K", [256, 301])
def test_block_norm_gate_for_each_sequence(cuda, lib, K, dtype):
    M, G = 60, 4
    x, h, w1, w2 = _inputs(M, K, dtype, cuda, 3)
    gate = torch.randn(G, 3 * K, device=cuda).to(dtype)[:, K:2 * K]          # as it comes out of a projection that makes three of them
    R, Y = torch.empty_like(x), torch.empty_like(x)
    _ops().block_norm(h, x, R, w1, gate, 1.0, w2, Y, eps=EPS)
    _check_block(x, h, w1, w2, gate, 1.0, R, Y, None, None)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("M,G,K", [(900, 4, 512), (900, 2, 1001), (1500, 10, 1000), (1501, 19, 777), (444, 3, 5001), (600, 2, 7168), (300, 2, 12001), (3001, 1, 303)])
def test_block_norm_gates_of_long_sequences(cuda, lib, M, G, K, dtype):
    """Many rows with a gate for each of a few sequences, where a CTA's rows end one sequence and begin the next."""
    x, h, w1, w2 = _inputs(M, K, dtype, cuda, 8)
    gate = torch.randn(G, 2 * K + 1, device=cuda).to(dtype)[:, 1:K + 1]
    per_row = gate.repeat_interleave(M // G, 0)
    R, Y = (torch.full((M, K), float("nan"), dtype=dtype, device=cuda) for _ in range(2))
    q, sc = padded(M, K, torch.int8, cuda)[0], torch.empty(M, device=cuda)
    _ops().block_norm(h, x, R, w1, gate, 0.5, w2, Y, eps=EPS)
    _check_block(x, h, w1, w2, per_row, 0.5, R, Y, None, None)
    X = x.clone()                                    # in place, without the first norm, quantized
    _ops().block_norm(h, X, X, None, gate, 1.0, w2, None, q, sc, eps=EPS)
    _check_block(x, h, None, w2, per_row, 1.0, X, None, q, sc)


def test_strides_offsets_and_neighbours(cuda, lib):
    """Column slices of one buffer as inputs and outputs; nothing outside them is written."""
    M, K = 37, 504
    for off, pitch in ((0, 1600), (8, 1608), (1, 1600), (4, 1555)):
        buf = torch.randn(M, pitch, device=cuda).to(torch.bfloat16)
        before = buf.clone()
        w1, w2 = torch.rand(2, K, device=cuda).to(torch.bfloat16)
        x, h, Y = (buf[:, off + i * K + i:off + i * K + i + K] for i in range(3))
        xs, hs = x.clone(), h.clone()
        _ops().block_norm(h, x, x, w1, None, 0.5, w2, Y, eps=EPS)            # r into x, y into a slice beside h
        _check_block(xs, hs, w1, w2, None, 0.5, x, Y, None, None)
        mask = torch.ones_like(buf, dtype=torch.bool)
        for i in (0, 2):
            mask[:, off + i * K + i:off + i * K + i + K] = False
        assert torch.equal(buf[mask], before[mask])


def test_rows_that_hold_no_numbers(cuda, lib):
    K = 700
    x, h, w1, w2 = _inputs(6, K, torch.bfloat16, cuda, 4)
    h[1, 5] = float("nan"); x[3, 699] = float("inf")
    R, Y = torch.empty_like(x), torch.empty_like(x)
    q, sc = padded(6, K, torch.int8, cuda)[0], torch.empty(6, device=cuda)
    _ops().block_norm(h, x, R, w1, None, 1.0, w2, Y, q, sc, eps=EPS)
    assert torch.isnan(Y[1]).all() and torch.isnan(sc[[1, 3]]).all() and bool((q[[1, 3]] == 0).all())
    ok = [0, 2, 4, 5]                                                        # the other rows do not see it
    _check_block(x[ok], h[ok], w1, w2, None, 1.0, R[ok], Y[ok], q[ok], sc[ok])
    assert float(Y[2].abs().sum()) == 0.0 and bool((q[2] == 0).all())


def test_without_rows(cuda, lib):
    e = torch.empty(0, 64, dtype=torch.float16, device=cuda)
    w = torch.ones(64, dtype=torch.float16, device=cuda)
    _ops().rms_norm(e, w, e.clone())
    _ops().block_norm(e, e, e, w, None, 1.0, w, e.clone())
    torch.cuda.synchronize()


def test_rows_past_32_bit_offsets(cuda, lib):
    M, K = 300000, 8192
    x = torch.zeros(M, K, dtype=torch.bfloat16, device=cuda)
    w = torch.ones(K, dtype=torch.bfloat16, device=cuda)
    part = torch.randn(100, K, device=cuda).to(torch.bfloat16)
    x[-100:] = part; x[262100:262200] = part
    q, sc = torch.empty(M, K, dtype=torch.int8, device=cuda), torch.empty(M, device=cuda)
    Y = torch.empty_like(x)
    _ops().rms_norm(x, w, Y, q, sc, eps=EPS)
    y = norm64(part, w, EPS)
    for rows in (slice(M - 100, M), slice(262100, 262200)):
        _close(Y[rows], y, y.abs() * S, "Y")
        _check_codes(q[rows], sc[rows], y, y.abs() * S)
    assert float(Y[5].abs().sum()) == 0.0 and bool((q[262099] == 0).all())


@pytest.mark.parametrize("M", [1, 24, 400])
def test_a_block_of_layers(cuda, lib, M):
    """rms_norm -> product -> block_norm -> product, as a transformer block with int8 weights runs it, captured and replayed."""
    ops, K, N = _ops(), 768, 1000
    dtype = torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(M)
    w_in, w_post, w_pre = (1 + 0.1 * torch.randn(K, generator=g, device=cuda).to(dtype) for _ in range(3))
    gate = torch.randn(K, generator=g, device=cuda).to(dtype)
    weights = []
    for n in (K, N):
        w = (0.05 * torch.randn(n, K, generator=g, device=cuda)).to(dtype)
        wq, wsc = torch.empty(n, K, dtype=torch.int8, device=cuda), torch.empty(n, device=cuda)
        ops.int8_quantize(w, wq, wsc)                                        # weights: a scale for each output channel
        weights.append((wq, wsc))
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    q1, q2 = (torch.empty(M, K, dtype=torch.int8, device=cuda) for _ in range(2))
    s1, s2 = (torch.empty(M, device=cuda) for _ in range(2))
    h, r, out = torch.empty_like(x), torch.empty_like(x), torch.empty(M, N, dtype=dtype, device=cuda)

    def run():
        ops.rms_norm(x, w_in, Y_int8=q1, Y_sc=s1, eps=EPS)
        ops.int8_gemm(q1, s1, *weights[0], h)
        ops.block_norm(h, x, r, w_post, gate, 1.0, w_pre, Y_int8=q2, Y_sc=s2, eps=EPS)
        ops.int8_gemm(q2, s2, *weights[1], out)

    def check():
        y = norm64(x, w_in, EPS)
        _check_codes(q1, s1, y, y.abs() * S)
        # each stage against 64 bits of what the stage before it stored
        half = torch.finfo(dtype).eps / 2
        ref = gemm64(q1, s1, *weights[0])
        assert bool(((h.double() - ref).abs() <= ref.abs() * (half + 4 * U) + 1e-30).all())
        _check_block(x, h, w_post, w_pre, gate[None], 1.0, r, None, q2, s2)
        ref = gemm64(q2, s2, *weights[1])
        assert bool(((out.double() - ref).abs() <= ref.abs() * (half + 4 * U) + 1e-30).all())

    run()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    x.copy_(torch.randn(M, K, generator=g, device=cuda))
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    check()


def test_refusals_on_tensors(cuda, lib):
    ops = _ops()
    x, h, w, _ = _inputs(6, 64, torch.bfloat16, cuda, 5)
    Y, q, sc = torch.zeros_like(x), torch.zeros(6, 64, dtype=torch.int8, device=cuda), torch.zeros(6, device=cuda)
    for args, word in [((x, w), "needs Y"), ((x, w.half(), Y), "dtype"), ((x, w[:60], Y), "shape"), ((x, w, x), "overlap"), ((x, w, None, q), "together"),
                       ((x.float(), w, Y), "dtype"), ((x, w, Y[:5]), "shape"), ((x, w, Y, q, sc[:4]), "shape"), ((x.t(), w, Y), "contiguous")]:
        with pytest.raises(RuntimeError, match=word):
            ops.rms_norm(*args)
    for args, word in [((h, x, h), "overlap"), ((h, x, Y, w, None, 1.0, w), "W_pre needs"), ((h, x, Y, w, None, 1.0, None, q.view(6, 64)), "need W_pre"),
                       ((h, x, Y, w, w[None].expand(4, 64).contiguous()), "multiple"), ((h, x, Y, w, None, 1.0, w, Y), "overlap"), ((h, x, Y, w, None, 1.0, w, h), "overlap"),
                       ((h, x.half(), Y), "dtype"), ((h, x, Y, w.cpu()), "CUDA")]:
        with pytest.raises(RuntimeError, match=word):
            ops.block_norm(*args)
    with pytest.raises(RuntimeError, match="eps"):
        ops.rms_norm(x, w, Y, eps=-1.0)
    with pytest.raises(RuntimeError, match="16384"):
        ops.rms_norm(torch.zeros(1, 16392, dtype=torch.bfloat16, device=cuda), torch.zeros(16392, dtype=torch.bfloat16, device=cuda), torch.zeros(1, 16392, dtype=torch.bfloat16, device=cuda))
    assert float(Y.abs().sum()) == 0.0
