"""The int8 linear layer and the norms around it in 64 bits, from their definitions, on whatever device the inputs are."""
import torch

FLOOR = 2.0 ** -100


def quantize64(x):
    """(codes as float64, steps as float64) of the rows of x, any float type: the exact product with the fp32 inverse step."""
    x = x.double()
    amax = x.abs().amax(1).clamp_min(FLOOR)
    inverse = torch.div(torch.full_like(amax, 127.0), amax.float().double()).float().double()
    codes = torch.round(x * inverse[:, None])
    steps = amax.float().double() / 127.0
    bad = ~torch.isfinite(x).all(1)
    codes[bad] = 0.0
    steps[bad] = float("nan")
    return codes, steps


def gemm64(a, a_sc, b, b_sc):
    return (a.double() @ b.double().T) * a_sc.double()[:, None] * b_sc.double()


def norm64(x, w, eps):
    x = x.double()
    return x / torch.sqrt((x * x).mean(1, keepdim=True) + eps) * w.double()


def block64(h, x, w_post, gate, residual_scale, eps):
    """r of block_norm; gate (G, K) or None."""
    p = norm64(h, w_post, eps) if w_post is not None else h.double()
    if gate is not None:
        p = p * gate.double().repeat_interleave(max(p.shape[0] // gate.shape[0], 1), 0)
    return residual_scale * x.double() + p


def padded(rows, k, dtype, device, fill=None):
    """A [rows, k] view whose rows begin 16 bytes apart, inside a buffer filled with `fill`; returns (view, buffer)."""
    per = 16 // torch.empty(0, dtype=dtype).element_size()
    buf = torch.empty(rows, (k + per - 1) // per * per, dtype=dtype, device=device)
    if fill is not None:
        buf.fill_(fill)
    return buf[:, :k], buf
