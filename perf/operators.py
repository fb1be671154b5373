"""Cases of the 8-bit integer linear layer and of the norms around it: what is timed and what is compared.

Four kinds of case, all as a serving program runs them, with the weights quantized ahead of time:

  gemm    D = (A_sc (x) B_sc) * (A . B^T): int8 operands, one fp32 scale per token and one per output channel
  linear  the same product from 16-bit activations: every token is quantized on the fly, then multiplied
  norm    y = RMSNorm(x) * w, the norm before a block; with "N" > 0 its result is quantized and multiplied
  block   r = residual_scale * x + gate * RMSNorm(h) * w_post, y = RMSNorm(r) * w_pre: the norm after a block, its gate
          and residual, and the norm before the next block; with "N" > 0 y is quantized and multiplied

The codes of quantized activations are intermediate: they go into the product, whose result is returned beside the token
scales.  A token is quantized with the step amax / 127; its codes are the halves-to-even roundings of x * fl32(127 / amax).
"""
import torch

own = False
EPS = 1e-6
#: the smallest row maximum that a quantization step is made from
FLOOR = 2.0 ** -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, kind, M, K, N=0, dtype="bf16", out="bf16", gates=1, post=True, r_scale=1.0):
    return {"name": name, "kind": kind, "M": M, "K": K, "N": N, "dtype": dtype, "out": out, "gates": gates, "post": post, "r_scale": r_scale}


def listed():
    return [
        # one token through a small projection: latency counts
        _case("gemm one token", "gemm", 1, 7168, 2048),
        # a decode batch through the widest projection of this repository's benchmark: bound by reading the weights
        _case("gemm decode batch", "gemm", 16, 8192, 28672),
        # the last projection of a decode batch, to fp32 logits over an odd number of words
        _case("gemm logits", "gemm", 48, 2048, 50257, out="fp32"),
        # a few packed prompts: no size is a multiple of a tile, fp16
        _case("gemm ragged", "gemm", 333, 4112, 5001, out="fp16"),
        # a long prompt through the widest projection
        _case("gemm prefill", "gemm", 8192, 8192, 28672),
        # a few tokens, quantized on the fly, fp16
        _case("linear few tokens", "linear", 4, 2048, 7168, dtype="fp16", out="fp16"),
        # a prompt quantized on the fly
        _case("linear prompt", "linear", 2048, 8192, 8192),
        # the norm before a block, over a long prompt
        _case("norm prompt", "norm", 16384, 7168),
        # the norm of a small decode batch into the first projection of the block
        _case("norm decode linear", "norm", 32, 7168, 2048),
        # the boundary between two blocks of a small decode batch
        _case("block decode", "block", 8, 7168, r_scale=0.5),
        # the same over packed prompts with a gate for each of them, an odd width, fp16
        _case("block ragged", "block", 4098, 5001, dtype="fp16", out="fp16", gates=6),
        # the boundary between two blocks of a long prompt, quantized into the next block's first projection
        _case("block prompt linear", "block", 16384, 7168, 2048),
    ]


def _spread(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["gemm", "linear", "norm", "block"])
    M, K = _spread(rng, 1, 16384), _spread(rng, 128, 16384)
    if rng.random() < 0.6:
        K = max(16, K // 16 * 16)
    N = _spread(rng, 64, 28672) if kind in ("gemm", "linear") or rng.random() < 0.4 else 0
    if N and rng.random() < 0.6:
        N = N // 8 * 8
    while M * K > 16384 * 8192 or M * max(1, N) * K > 8192 * 8192 * 28672:
        M = (M + 1) // 2
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    c = _case("", kind, M, K, N, dtype, rng.choice([dtype, dtype, "fp32"]) if kind in ("gemm", "linear") else dtype)
    if kind == "block":
        c["gates"] = rng.choice([1, 1, 0, M, max(g for g in (2, 3, 5, 1) if M % g == 0)])
        c["post"] = rng.random() < 0.75
        c["r_scale"] = rng.choice([1.0, 0.5, 0.7071])
    del c["name"]
    return c


def _rows(n, k, device, dtype):
    """An [n, k] tensor whose rows begin 16 bytes apart, as both operands of the product need."""
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    return torch.empty(n, (k + per - 1) // per * per, dtype=dtype, device=device)[:, :k]


def _steps(x):
    """fp32 (127 / amax, amax / 127) of the rows of x, each rounded once: a division by a tensor is one, by a number is not."""
    amax = x.abs().amax(1, keepdim=True).clamp_min(FLOOR)
    top = torch.full_like(amax, 127.0)
    return top / amax, (amax / top).squeeze(1)


def _codes(x, device):
    """Symmetric int8 codes of the rows of x and their fp32 steps."""
    inverse, steps = _steps(x)
    q = _rows(x.shape[0], x.shape[1], device, torch.int8)
    q.copy_((x * inverse).round_())
    return q, steps


def _activations(M, K, g, device):
    """Token rows: a few channels stand out, as they do behind a norm, and padding rows are zeros."""
    x = torch.randn(M, K, generator=g, device=device)
    x *= 1.0 + 7.0 * (torch.rand(K, generator=g, device=device) < 0.01)
    x *= torch.exp(0.5 * torch.randn(M, 1, generator=g, device=device))
    if M > 64:
        x[M - M // 50:] = 0.0
    return x


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    M, N, K, t, out = case["M"], case["N"], case["K"], TYPES[case["dtype"]], TYPES[case["out"]]
    s = dict(case, seed=seed)
    x = _activations(M, K, g, device)
    if case["kind"] == "gemm":
        s["A"], s["A_sc"] = _codes(x, device)
    else:
        s["X"] = x.to(t)
        s["Q"], s["Q_sc"] = _rows(M, K, device, torch.int8), torch.empty(M, device=device)
    del x
    if N:
        s["B"], s["B_sc"] = _codes(torch.randn(N, K, generator=g, device=device).mul_(0.02), device)
        s["D"] = torch.empty(M, N, dtype=out, device=device)
    if case["kind"] in ("norm", "block"):
        s["W_pre"] = (1.0 + 0.1 * torch.randn(K, generator=g, device=device)).to(t)
        if not N:
            s["Y"] = torch.empty(M, K, dtype=t, device=device)
    if case["kind"] == "block":
        s["H"] = (3.0 * torch.randn(M, K, generator=g, device=device)).to(t)
        s["W_post"] = (1.0 + 0.1 * torch.randn(K, generator=g, device=device)).to(t) if case["post"] else None
        gates = case["gates"]
        s["gate"] = (0.3 * torch.randn(gates, K, generator=g, device=device)).to(t) if gates else None
        s["R"] = torch.empty(M, K, dtype=t, device=device)
    return s


def _plain_norm(x, w):
    return x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * w.float()


def _plain_product(q, q_sc, s):
    return ((q @ s["B"].float().T) * q_sc[:, None] * s["B_sc"]).to(s["D"].dtype)


def _plain_linear(x, s):
    inverse, q_sc = _steps(x)
    # a code next to a border is decided by the exact product, which 64 bits hold
    q = (x.double() * inverse.double()).round().float()
    return _plain_product(q, q_sc, s), q_sc


def _plain(s):
    if s["kind"] == "gemm":
        return _plain_product(s["A"].float(), s["A_sc"], s)
    x = s["X"].float()
    if s["kind"] == "linear":
        return _plain_linear(x, s)
    if s["kind"] == "norm":
        y = _plain_norm(x, s["W_pre"])
        return _plain_linear(y, s) if s["N"] else y.to(s["X"].dtype)
    h = s["H"].float()
    p = _plain_norm(h, s["W_post"]) if s["post"] else h
    if s["gates"]:
        p = (p.view(s["gates"], -1, s["K"]) * s["gate"].float()[:, None]).view(s["M"], -1)
    r = s["r_scale"] * x + p
    y = _plain_norm(r, s["W_pre"])
    return r.to(s["X"].dtype), (_plain_linear(y, s) if s["N"] else y.to(s["X"].dtype))


def run(s):
    if not own:
        return _plain(s)
    from thunderkittens_b200 import ops
    kind, N = s["kind"], s["N"]
    if kind == "gemm":
        ops.int8_gemm(s["A"], s["A_sc"], s["B"], s["B_sc"], s["D"])
        return s["D"]
    if kind == "linear":
        ops.int8_quantize(s["X"], s["Q"], s["Q_sc"])
    elif kind == "norm":
        if not N:
            ops.rms_norm(s["X"], s["W_pre"], s["Y"], eps=EPS)
            return s["Y"]
        ops.rms_norm(s["X"], s["W_pre"], Y_int8=s["Q"], Y_sc=s["Q_sc"], eps=EPS)
    elif not N:
        ops.block_norm(s["H"], s["X"], s["R"], s["W_post"], s["gate"], s["r_scale"], s["W_pre"], s["Y"], eps=EPS)
        return s["R"], s["Y"]
    else:
        ops.block_norm(s["H"], s["X"], s["R"], s["W_post"], s["gate"], s["r_scale"], s["W_pre"], Y_int8=s["Q"], Y_sc=s["Q_sc"], eps=EPS)
    ops.int8_gemm(s["Q"], s["Q_sc"], s["B"], s["B_sc"], s["D"])
    return (s["R"], (s["D"], s["Q_sc"])) if kind == "block" else (s["D"], s["Q_sc"])


def work(case):
    M, N, K = case["M"], case["N"], case["K"]
    out = 4 if case["out"] == "fp32" else 2
    size, flops = 0, 2.0 * M * N * K
    if case["kind"] == "gemm":
        size += M * K + 4 * M
    else:
        size += 2 * M * K                        # x
    if case["kind"] == "block":
        size += 2 * 2 * M * K                    # h, r
        size += 2 * K * (case["gates"] + int(case["post"]))
        flops += 4.0 * M * K
    if case["kind"] in ("norm", "block"):
        size += 2 * K                            # w_pre
        flops += 5.0 * M * K
        if not N:
            size += 2 * M * K                    # y
    if N:
        size += N * K + 4 * N + M * N * out
        if case["kind"] != "gemm":
            size += 4 * M                        # the token scales
    return {"bytes": float(size), "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64

    def norm(v, w):
        return torch.einsum("mk,m,k->mk", v, ((v ** 2).sum(1) / v.shape[1] + EPS) ** -0.5, w.to(f))

    def product(codes, steps):
        return torch.einsum("mn,m,n->mn", codes @ s["B"].to(f).T, steps.to(f), s["B_sc"].to(f))

    def linear(v):
        top = v.abs().max(1).values.clamp(min=FLOOR)
        inverse = (127.0 / top).to(torch.float32).to(f)          # held in 32 bits by definition
        steps = top / 127.0
        return product(torch.round(v * inverse[:, None]), steps), steps

    if case["kind"] == "gemm":
        return product(s["A"].to(f), s["A_sc"])
    v = s["X"].to(f)
    if case["kind"] == "linear":
        return linear(v)
    if case["kind"] == "block":
        b = norm(s["H"].to(f), s["W_post"]) if case["post"] else s["H"].to(f)
        if case["gates"]:
            b = b * s["gate"].to(f).repeat_interleave(case["M"] // case["gates"], 0)
        v = case["r_scale"] * v + b
    y = norm(v, s["W_pre"])
    y = linear(y) if case["N"] else y
    return (v, y) if case["kind"] == "block" else y
