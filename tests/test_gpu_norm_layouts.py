"""Layouts of the row kernels that depend on how many rows there are and on where they begin: several rows in a CTA, gates of sequences
staged two at a time, rows that begin anywhere, outputs that are larger than L2.  Tolerances as derived in test_gpu_norm."""
import pytest
import torch

from tests.int8_common import norm64, padded, quantize64
from tests.test_gpu_norm import EPS, HALF, S, _check_block, _check_codes, _close, _inputs

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


@pytest.mark.parametrize("M,G,K", [(6, 6, 64), (600, 600, 1000), (600, 4, 1001), (5, 5, 1)])
def test_block_norm_one_gate_row_expanded(cuda, lib, M, G, K):
    x, h, w1, w2 = _inputs(M, K, torch.bfloat16, cuda, 17)
    gate = torch.randn(K, device=cuda).to(torch.bfloat16)
    out = [[torch.full_like(x, float("nan")) for _ in range(2)] for _ in range(2)]
    for (R, Y), g in zip(out, (gate, gate.expand(G, K))):
        _ops().block_norm(h, x, R, w1, g, 0.5, w2, Y, eps=EPS)
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    _check_block(x, h, w1, w2, gate[None], 0.5, *out[1], None, None)
    with pytest.raises(RuntimeError, match="multiple"):
        _ops().block_norm(h, x, out[0][0], w1, gate.expand(M + 1, K))


def _at(t, off, pitch, guard=7.0):
    """(a view with the values of t whose rows begin `off` elements into rows of `pitch`, its buffer, a mask of what lies outside)."""
    M, K = t.shape
    buf = torch.full((M, pitch), guard, dtype=t.dtype, device=t.device)
    view = buf[:, off:off + K]
    view.copy_(t)
    outside = torch.ones(M, pitch, dtype=torch.bool, device=t.device)
    outside[:, off:off + K] = False
    return view, buf, outside


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("M,G,K", [(900, 4, 512), (900, 2, 1000), (1500, 10, 1024), (444, 3, 5000), (600, 2, 7168), (600, 2, 11264), (602, 2, 12288), (301, 7, 16384),
                                   (1600, 8, 8), (2000, 250, 2048)])
def test_block_norm_gates_of_aligned_rows(cuda, lib, M, G, K, dtype):
    """A gate for each of a few sequences, or of many short ones, where every row begins on 16 bytes."""
    x, h, w1, w2 = _inputs(M, K, dtype, cuda, 12)
    g = torch.Generator(device=cuda).manual_seed(M)
    gate = torch.randn(G, 3 * K, generator=g, device=cuda).to(dtype)[:, K:2 * K]
    per_row = gate.repeat_interleave(M // G, 0)
    R, Y = (torch.full((M, K), float("nan"), dtype=dtype, device=cuda) for _ in range(2))
    q, sc = padded(M, K, torch.int8, cuda)[0], torch.empty(M, device=cuda)
    _ops().block_norm(h, x, R, w1, gate, 0.5, w2, Y, eps=EPS)
    _check_block(x, h, w1, w2, per_row, 0.5, R, Y, None, None)
    X = x.clone()                                    # in place, without the first norm, quantized
    _ops().block_norm(h, X, X, None, gate, 1.0, w2, None, q, sc, eps=EPS)
    _check_block(x, h, None, w2, per_row, 1.0, X, None, q, sc)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("M,G,K", [(700, 1, 504), (700, 4, 1001), (1400, 700, 300), (600, 2, 5001), (300, 1, 12001), (300, 3, 16384), (299, 299, 2049)])
def test_block_norm_tensors_that_begin_differently(cuda, lib, M, G, K, dtype):
    """No two of the tensors begin alike within 16 bytes; many rows, with one gate, one for each sequence, one for each token."""
    x, h, w1, w2 = _inputs(M, K, dtype, cuda, 13)
    g = torch.Generator(device=cuda).manual_seed(M)
    gate = torch.randn(G, K, generator=g, device=cuda).to(dtype)
    per_row = gate.repeat_interleave(M // G, 0)
    pitch = K + 16 - K % 8
    hv, xv = _at(h, 1, pitch)[0], _at(x, 2, pitch)[0]
    (R, rb, ro), (Y, yb, yo) = (_at(torch.zeros_like(x), off, pitch) for off in (3, 5))
    Q, qb, qo = _at(torch.zeros(M, K, dtype=torch.int8, device=cuda), 3, pitch, 77)
    sc = torch.empty(M, device=cuda)
    _ops().block_norm(hv, xv, R, w1, gate, 0.5, w2, Y, Q, sc, eps=EPS)
    _check_block(x, h, w1, w2, per_row, 0.5, R, Y, Q, sc)
    assert bool((rb[ro] == 7).all() and (yb[yo] == 7).all() and (qb[qo] == 77).all())


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("offsets", [(0, 0), (3, 3), (1, 4)], ids=["contiguous", "shifted", "differently"])
@pytest.mark.parametrize("M,K", [(297, 303), (1500, 300), (700, 1001), (3000, 127), (400, 5001), (301, 12301), (300, 16383), (297, 16384), (600, 1)])
def test_rms_norm_rows_that_begin_anywhere(cuda, lib, M, K, offsets, dtype):
    """More rows than one for each CTA: contiguous rows of odd K, rows shifted alike, and a result that begins elsewhere."""
    x, _, w, _ = _inputs(M, K, dtype, cuda, 14)
    y = norm64(x, w, EPS)
    pitch = K if offsets == (0, 0) else K + 16 - K % 8
    xv = _at(x, offsets[0], pitch)[0]
    Y, yb, yo = _at(torch.zeros_like(x), offsets[1], pitch)
    q, qb = padded(M, K, torch.int8, cuda, fill=99)
    sc = torch.empty(M, device=cuda)
    _ops().rms_norm(xv, w, Y, eps=EPS)
    _close(Y, y, y.abs() * S, "Y")
    assert bool((yb[yo] == 7).all())
    _ops().rms_norm(xv, w, None, q, sc, eps=EPS)
    _check_codes(q, sc, y, y.abs() * S)
    assert bool((qb[:, K:] == 99).all())


@pytest.mark.parametrize("M,K", [(16400, 4096), (13500, 5001), (33000, 2048)])
def test_rms_norm_results_larger_than_l2(cuda, lib, M, K):
    """16-bit results of long prompts alone: over 256 MB read and written, where a CTA holds fewer rows."""
    x, _, w, _ = _inputs(M, K, torch.bfloat16, cuda, 15)
    Y = torch.full_like(x, float("nan"))
    _ops().rms_norm(x, w, Y, eps=EPS)
    for rows in torch.arange(M, device=cuda).split(4096):
        y = norm64(x[rows], w, EPS)
        _close(Y[rows], y, y.abs() * S, "Y")


@pytest.mark.parametrize("M,G,K", [(8200, 1, 4096), (6800, 4, 5001), (4800, 2, 7168), (2100, 3, 16384), (4800, 4800, 7168)])
def test_block_norm_results_larger_than_l2(cuda, lib, M, G, K):
    x, h, w1, w2 = _inputs(M, K, torch.bfloat16, cuda, 16)
    g = torch.Generator(device=cuda).manual_seed(M)
    gate = torch.randn(G, K, generator=g, device=cuda).to(torch.bfloat16)
    R, Y = torch.full_like(x, float("nan")), torch.full_like(x, float("nan"))
    _ops().block_norm(h, x, R, w1, gate, 0.5, w2, Y, eps=EPS)
    for rows in torch.arange(M, device=cuda).split(2048):
        _check_block(x[rows], h[rows], w1, w2, gate[rows // (M // G)], 0.5, R[rows], Y[rows], None, None)


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("off", [0, 1, 6])
@pytest.mark.parametrize("M,K", [(1000, 100), (777, 509), (400, 7), (3000, 1), (500, 1021), (400, 4001), (300, 8193), (300, 16001), (40, 65535), (300, 65529)])
def test_quantize_rows_that_begin_anywhere(cuda, lib, M, K, off, dtype):
    """Short rows, of which a warp holds one, to the longest, with codes that begin elsewhere; contiguous (off 0) and in wider rows."""
    g = torch.Generator(device=cuda).manual_seed(M + K)
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    x[3 % M] = 0.0
    pitch = K if off == 0 else K + 16 - K % 8
    xv = _at(x, off, pitch)[0]
    Q, qb, qo = _at(torch.zeros(M, K, dtype=torch.int8, device=cuda), 5 * (off > 0), pitch, 77)
    sc = torch.empty(M, device=cuda)
    _ops().int8_quantize(xv, Q, sc)
    codes, steps = quantize64(x)
    assert torch.equal(Q.double(), codes) and torch.equal(sc, steps.float())
    assert bool((qb[qo] == 77).all())


def test_row_lengths_in_turn_do_not_ask_the_driver_again(cuda, lib):
    """A model's hidden and inner rows go through one instance of the kernel; how many CTAs fit is asked for once for each length."""
    from torch.profiler import ProfilerActivity, profile
    calls = []
    for K in (2048, 7168, 5000):
        x = torch.randn(4, K, device=cuda).to(torch.bfloat16)
        calls.append((x, torch.empty(4, K, dtype=torch.int8, device=cuda), torch.empty(4, device=cuda)))
    for c in calls:
        _ops().int8_quantize(*c)
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        for _ in range(3):
            for c in calls:
                _ops().int8_quantize(*c)
        torch.cuda.synchronize()
    names = [e.name for e in p.events()]
    if sum("aunch" in n for n in names) < 9:
        pytest.skip("the profiler records no runtime calls here")
    assert not [n for n in names if "Occupancy" in n]
