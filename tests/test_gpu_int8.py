"""int8_quantize and int8_gemm against their definitions in 64 bits.

Tolerances.  Codes and steps of the quantizer are exact by definition (one fp32 division each, one rounding to an integer).
The product's int32 sum is exact; it is converted to fp32, multiplied by two scales and rounded to the output type, so an element
is off by at most 3 fp32 half steps and one half step of the output type, relative to its own value."""
import pytest
import torch

from tests.int8_common import gemm64, padded, quantize64

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]


def _ops():
    import thunderkittens_b200.ops as ops
    return ops


def _randn(shape, seed, cuda, std=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=cuda) * std


def _randint8(rows, k, seed, cuda):
    g = torch.Generator(device=cuda).manual_seed(seed)
    v, buf = padded(rows, k, torch.int8, cuda, fill=77)          # what lies behind a row must not matter
    v.copy_(torch.randint(-128, 128, (rows, k), generator=g, device=cuda, dtype=torch.int8))
    return v


def _check_quantize(x, q, sc):
    codes, steps = quantize64(x)
    assert torch.equal(q.double(), codes)
    assert torch.equal(torch.nan_to_num(sc, nan=-1.0), torch.nan_to_num(steps.float(), nan=-1.0))


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 7), (3, 16), (5, 129), (64, 2048), (33, 2056), (7, 5001), (2, 7168), (3, 16384), (4, 16392), (2, 28672), (2, 40001), (3, 65536),
                                 (2000, 256), (301, 8192)])
def test_quantize(cuda, lib, M, K, dtype):
    x = _randn((M, K), M + K, cuda).to(dtype)
    q, buf = padded(M, K, torch.int8, cuda, fill=99)
    sc = torch.full((M,), float("nan"), device=cuda)
    _ops().int8_quantize(x, q, sc)
    _check_quantize(x, q, sc)
    assert bool((buf[:, K:] == 99).all())


@pytest.mark.parametrize("dtype", HALF, ids=str)
def test_quantize_strided_and_misaligned(cuda, lib, dtype):
    for off, pitch, K in ((8, 520, 512), (3, 515, 512), (1, 900, 333)):
        buf = _randn((40, pitch + 8), off, cuda).to(dtype)
        x = buf[:, off:off + K]
        out = torch.full((40, pitch + 24), 55, dtype=torch.int8, device=cuda)
        q, sc = out[:, 5:5 + K], torch.empty(44, device=cuda)[3:43]
        _ops().int8_quantize(x, q, sc)
        _check_quantize(x, q, sc)
        assert bool((out[:, :5] == 55).all()) and bool((out[:, 5 + K:] == 55).all())


@pytest.mark.parametrize("dtype", HALF, ids=str)
@pytest.mark.parametrize("K", [64, 1027])
def test_quantize_special_rows(cuda, lib, dtype, K):
    """Zeros, the smallest and largest numbers, values on the border between two codes, infinities and NaN."""
    x = _randn((12, K), 5, cuda).to(dtype)
    x[0] = 0.0
    x[1] = 0.0; x[1, K - 1] = torch.finfo(dtype).smallest_normal / 4
    x[2] *= torch.finfo(dtype).max / 16; x[2, 3] = -torch.finfo(dtype).max
    x[2].clamp_(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    x[3] = torch.linspace(-1, 1, K, device=cuda).to(dtype); x[3, 0] = 2.0; x[3, 5] = 1.0; x[3, 6] = -1.0
    x[4] = -0.5; x[4, K // 2] = 1.0
    x[5] = (torch.arange(K, device=cuda) % 128 - 64).to(dtype) / 2; x[5, 1] = 63.5
    x[6, K // 3] = float("inf")
    x[7, 0] = float("-inf"); x[7, K - 1] = float("nan")
    x[8, K - 1] = float("nan")
    x[9] = -1.0
    q, _ = padded(12, K, torch.int8, cuda)
    sc = torch.empty(12, device=cuda)
    _ops().int8_quantize(x, q, sc)
    _check_quantize(x, q, sc)
    assert torch.isnan(sc[6:9]).all() and bool((q[6:9] == 0).all()) and bool((q[0] == 0).all()) and sc[0] > 0


def _check_gemm(D, a, a_sc, b, b_sc):
    ref = gemm64(a, a_sc, b, b_sc)
    half_step = torch.finfo(D.dtype).eps / 2
    tiny = 2.0 ** -25 if D.dtype == torch.float16 else 2.0 ** -134          # half of the smallest subnormal step
    tol = ref.abs() * (half_step + 3 * 2.0 ** -24) * (1 + 2.0 ** -10) + tiny * (1 + 2.0 ** -10)
    err = (D.double() - ref).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()} elements off, worst {float((err / ref.abs().clamp_min(1e-30)).max()):.3e} relative"


def _operands(M, N, K, cuda, seed=0):
    a, b = _randint8(M, K, 3 * seed + M + K, cuda), _randint8(N, K, 3 * seed + N + K + 1, cuda)
    g = torch.Generator(device=cuda).manual_seed(seed + 7)
    # scales of a range of sizes whose products stay inside fp16
    return a, torch.rand(M, generator=g, device=cuda) * 2e-3, b, torch.rand(N, generator=g, device=cuda) * 2e-3 / K ** 0.5


SHAPES = [(1, 1, 1), (1, 16, 16), (3, 5, 7), (1, 300, 4100), (2, 128, 129), (16, 130, 512), (17, 1000, 272), (33, 257, 1040), (64, 128, 128), (65, 77, 2000),
          (100, 4096, 64), (127, 129, 333), (128, 512, 4096), (129, 256, 128), (200, 64, 3000), (256, 256, 256), (300, 129, 1000), (513, 777, 640), (1024, 1040, 2048)]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(cuda, lib, M, N, K, out):
    a, a_sc, b, b_sc = _operands(M, N, K, cuda)
    D = torch.full((M, N), float("nan"), dtype=out, device=cuda)
    _ops().int8_gemm(a, a_sc, b, b_sc, D)
    _check_gemm(D, a, a_sc, b, b_sc)


@pytest.mark.parametrize("M", [9, 33, 48, 49, 70, 90, 110, 128])
@pytest.mark.parametrize("N,K", [(333, 2100), (5000, 2176), (9001, 2300), (19000, 2064), (40000, 2100)])
def test_gemm_streamed_weights(cuda, lib, M, N, K):
    """Few tokens: every padding of them, slabs of few and of many weight rows, K that ends inside a stage and inside a block."""
    a, a_sc, b, b_sc = _operands(M, N, K, cuda, seed=5)
    for out in (torch.float16, torch.float32):
        D = torch.full((M, N), float("nan"), dtype=out, device=cuda)
        _ops().int8_gemm(a, a_sc, b, b_sc, D)
        _check_gemm(D, a, a_sc, b, b_sc)


@pytest.mark.parametrize("cfg", ["pair_n256", "single_n256", "pair_n128", "single_n128"])
@pytest.mark.parametrize("M,N,K", [(1, 40, 48), (130, 264, 272), (600, 513, 900), (2048, 1536, 1024)])
def test_gemm_tiles(cuda, lib, M, N, K, cfg):
    a, a_sc, b, b_sc = _operands(M, N, K, cuda, seed=1)
    for out in (torch.bfloat16, torch.float32):
        D = torch.full((M, N), float("nan"), dtype=out, device=cuda)
        _ops().int8_gemm(a, a_sc, b, b_sc, D, cfg)
        _check_gemm(D, a, a_sc, b, b_sc)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("M", [5, 90, 300])
def test_gemm_writes_only_its_columns(cuda, lib, M, out):
    """D as columns of a wider tensor, at offsets that allow TMA stores and ones that do not."""
    N, K = 200, 400
    a, a_sc, b, b_sc = _operands(M, N, K, cuda, seed=2)
    for off, pitch in ((8, 216), (3, 216), (0, 211), (1, 201)):
        buf = torch.full((M + 2, pitch), 9.0, dtype=out, device=cuda)
        _ops().int8_gemm(a, a_sc, b, b_sc, buf[1:M + 1, off:off + N])
        _check_gemm(buf[1:M + 1, off:off + N], a, a_sc, b, b_sc)
        assert bool((buf[0] == 9).all() and (buf[M + 1] == 9).all() and (buf[:, :off] == 9).all() and (buf[:, off + N:] == 9).all())


@pytest.mark.parametrize("M,N", [(2, 3), (150, 140)])
def test_gemm_longest_sum_of_extremes(cuda, lib, M, N):
    """128 * 128 * 131071 still fits int32."""
    K = 131071
    a, b = padded(M, K, torch.int8, cuda)[0], padded(N, K, torch.int8, cuda)[0]
    a.fill_(-128); b.fill_(-128); b[1] = 127; a[1, ::2] = 127
    ones = torch.ones(max(M, N), device=cuda)
    D = torch.empty(M, N, device=cuda)
    _ops().int8_gemm(a, ones[:M], b, ones[:N], D)
    # sums over 2^24 are rounded once to fp32, times one: compare with the rounded exact sums
    assert torch.equal(D, (a.double() @ b.double().T).float())


@pytest.mark.parametrize("M", [4, 140])
def test_gemm_scales_that_are_no_numbers(cuda, lib, M):
    N, K = 140, 64
    a, a_sc, b, b_sc = _operands(M, N, K, cuda, seed=3)
    a_sc[1] = float("nan"); b_sc[3] = float("nan")
    D = torch.zeros(M, N, device=cuda)
    _ops().int8_gemm(a, a_sc, b, b_sc, D)
    nan = torch.isnan(D)
    assert bool(nan[1].all()) and bool(nan[:, 3].all()) and int(nan.sum()) == M + N - 1


def test_gemm_without_rows(cuda, lib):
    b, b_sc = _randint8(32, 64, 1, cuda), torch.ones(32, device=cuda)
    _ops().int8_gemm(torch.empty(0, 64, dtype=torch.int8, device=cuda), torch.empty(0, device=cuda), b, b_sc, torch.empty(0, 32, device=cuda))
    _ops().int8_quantize(torch.empty(0, 64, dtype=torch.bfloat16, device=cuda), torch.empty(0, 64, dtype=torch.int8, device=cuda), torch.empty(0, device=cuda))
    torch.cuda.synchronize()


def test_gemm_repeats_bit_for_bit(cuda, lib):
    for M in (7, 64, 700):
        a, a_sc, b, b_sc = _operands(M, 1500, 2000, cuda, seed=4)
        D = [torch.empty(M, 1500, device=cuda) for _ in range(3)]
        for d in D:
            _ops().int8_gemm(a, a_sc, b, b_sc, d)
        assert torch.equal(D[0], D[1]) and torch.equal(D[0], D[2])


@pytest.mark.parametrize("M,N,K", [(1, 96, 2048), (5, 2048, 1024), (33, 77, 2000), (65, 77, 2000), (128, 1000, 4096), (7, 6000, 1040), (100, 5000, 528)])
def test_gemm_of_few_tokens_many_times(cuda, lib, M, N, K):
    """Back to back, each launch beginning while the one before it ends."""
    a, a_sc, b, b_sc = _operands(M, N, K, cuda, seed=8)
    D = [torch.full((M, N), float("nan"), device=cuda) for _ in range(40)]
    for _ in range(10):
        for d in D:
            _ops().int8_gemm(a, a_sc, b, b_sc, d)
    _check_gemm(D[0], a, a_sc, b, b_sc)
    assert all(torch.equal(d, D[0]) for d in D[1:])


@pytest.mark.parametrize("N", [60000, 60001])
def test_gemm_output_past_32_bit_offsets(cuda, lib, N):
    M, K = 40000, 16
    a, a_sc, b, b_sc = _operands(M, N, K, cuda, seed=5)
    D = torch.empty(M, N, dtype=torch.bfloat16, device=cuda)
    _ops().int8_gemm(a, a_sc, b, b_sc, D)
    for rows in (slice(0, 64), slice(35780, 35860), slice(M - 64, M)):
        _check_gemm(D[rows], a[rows], a_sc[rows], b, b_sc)


@pytest.mark.parametrize("M", [3, 40, 300])
def test_linear_on_two_streams_and_in_graphs(cuda, lib, M):
    """Quantizer and product as a layer runs them: on two streams at once, and captured twice and replayed at once on new inputs."""
    ops, N, K = _ops(), 1111, 1500
    g = torch.Generator(device=cuda).manual_seed(M)
    b, b_sc = _operands(M, N, K, cuda, seed=6)[2:]

    class Layer:
        def __init__(self):
            self.x = torch.randn(M, K, generator=g, device=cuda).to(torch.bfloat16)
            self.q, self.sc = padded(M, K, torch.int8, cuda)[0], torch.empty(M, device=cuda)
            self.D = torch.empty(M, N, device=cuda)

        def run(self):
            ops.int8_quantize(self.x, self.q, self.sc)
            ops.int8_gemm(self.q, self.sc, b, b_sc, self.D)

        def check(self):
            codes, steps = quantize64(self.x)
            _check_gemm(self.D, codes, steps.float(), b, b_sc)

    layers, streams = [Layer(), Layer()], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for layer, s in zip(layers, streams):
            with torch.cuda.stream(s):
                layer.run()
    torch.cuda.synchronize()
    for layer in layers:
        layer.check()
    graphs = []
    for layer in layers:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            layer.run()
    for layer in layers:
        layer.x.copy_(torch.randn(M, K, generator=g, device=cuda))
        layer.D.fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for layer in layers:
        layer.check()


@pytest.mark.parametrize("M", [2, 30, 100, 260])
def test_linear_with_operands_that_change_every_call(cuda, lib, M):
    """Launches that begin while the ones before them end read what those wrote: the same buffers, other values, no waiting."""
    ops, N, K, R = _ops(), 700, 1024, 24
    g = torch.Generator(device=cuda).manual_seed(M)
    xs = torch.randn(R, M, K, generator=g, device=cuda).to(torch.bfloat16) * (1 + torch.arange(R, device=cuda).to(torch.bfloat16))[:, None, None]
    w = torch.randn(R, N, K, generator=g, device=cuda).to(torch.bfloat16)
    q, sc, b, b_sc = torch.empty(M, K, dtype=torch.int8, device=cuda), torch.empty(M, device=cuda), torch.empty(N, K, dtype=torch.int8, device=cuda), torch.empty(N, device=cuda)
    Ds = torch.empty(R, M, N, device=cuda)
    torch.cuda.synchronize()
    for i in range(R):
        ops.int8_quantize(w[i], b, b_sc)
        ops.int8_quantize(xs[i], q, sc)
        ops.int8_gemm(q, sc, b, b_sc, Ds[i])
    for i in range(R):
        codes, steps = quantize64(xs[i])
        w_codes, w_steps = quantize64(w[i])
        _check_gemm(Ds[i], codes, steps.float(), w_codes, w_steps.float())


def test_refusals_on_tensors(cuda, lib):
    ops = _ops()
    a, a_sc, b, b_sc = _operands(20, 32, 64, cuda)
    D = torch.zeros(20, 32, device=cuda)
    bad = [
        ((a.cpu(), a_sc, b, b_sc, D), "CUDA"), ((a.float(), a_sc, b, b_sc, D), "dtype"), ((a, a_sc[:5], b, b_sc, D), "shape"),
        ((a, a_sc, b[:, :48], b_sc, D), "shape"), ((a, a_sc, b, b_sc, D[:, :30]), "shape"), ((a, a_sc.double(), b, b_sc, D), "dtype"),
        ((a.expand(20, 64).t().contiguous().t(), a_sc, b, b_sc, D), "contiguous"), ((a[:1].expand(20, 64), a_sc, b, b_sc, D), "overlap"),
        ((a[:, 1:], a_sc, b[:, 1:], b_sc, D), "16 bytes"), ((a, a_sc, b, b_sc[::2].repeat(2)[::2], D), "shape"), ((a, a_sc, b, b_sc, D.double()), "dtype"),
    ]
    for args, word in bad:
        with pytest.raises(RuntimeError, match=word):
            ops.int8_gemm(*args)
    x, q, sc = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda), torch.zeros(4, 64, dtype=torch.int8, device=cuda), torch.zeros(4, device=cuda)
    for args, word in [((x.float(), q, sc), "dtype"), ((x, q[:3], sc), "shape"), ((x, x.view(torch.int8)[:, :64], sc), "overlaps"), ((x, q, sc[:3]), "shape"),
                       ((torch.zeros(2, 65537, dtype=torch.bfloat16, device=cuda), torch.zeros(2, 65537, dtype=torch.int8, device=cuda), sc[:2]), "65536")]:
        with pytest.raises(RuntimeError, match=word):
            ops.int8_quantize(*args)
    assert float(D.abs().sum()) == 0.0


def test_numbers_that_are_none(cuda, lib):
    """What is no number is refused by name; numbers of any Python type are taken."""
    ops = _ops()
    x, w, Y = torch.ones(4, 64, dtype=torch.bfloat16, device=cuda), torch.ones(64, dtype=torch.bfloat16, device=cuda), torch.empty(4, 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(RuntimeError, match="eps"):
        ops.rms_norm(x, w, Y, eps="small")
    with pytest.raises(RuntimeError, match="residual_scale"):
        ops.block_norm(x, x, Y, residual_scale=None)
    ops.block_norm(H=x, X=x, X_out=Y, residual_scale=2, eps=1)
    assert bool((Y == 3).all())
    with pytest.raises(RuntimeError, match="must be a torch.Tensor"):
        ops.rms_norm(x, [1.0] * 64, Y)
