"""Plain forms of the 8-bit block operators and of the trainable layer norm: the block format in
fp32 (every step of it is an exactly rounded fp32 operation, so codes and scales must agree bit for
bit) and everything else in 64 bits, with the error bounds the GPU tests apply."""
from __future__ import annotations

import math

import torch

BLOCK = 128
U = 2.0**-24  # half a step of fp32, relative
FLOOR = 2.0**-100
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype) -> float:
    """Half the spacing of the type's subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def block_scale(amax):
    amax = torch.where(amax < FLOOR, torch.full_like(amax, FLOOR), amax)  # NaN stays
    top = torch.full_like(amax, 448.0)  # tensors on both sides: torch multiplies by the reciprocal of a number
    return top / amax, amax / top


def quantize_rows(x):
    """x [..., C] (fp32, on the CPU) -> codes as fp32 values [..., C], scale [..., ceil(C / 128)]."""
    x = x.float()
    c = x.shape[-1]
    n = -(-c // BLOCK)
    q = torch.empty_like(x)
    scale = torch.empty(*x.shape[:-1], n)
    for b in range(n):
        part = x[..., b * BLOCK:(b + 1) * BLOCK]
        inv, scale[..., b] = block_scale(part.abs().amax(-1))
        q[..., b * BLOCK:(b + 1) * BLOCK] = (part * inv[..., None]).to(torch.float8_e4m3fn).float()
    return q, scale


def quantize_tiles(x):
    x = x.float()
    rows, cols = x.shape
    q = torch.empty_like(x)
    scale = torch.empty(-(-rows // BLOCK), -(-cols // BLOCK))
    for r in range(scale.shape[0]):
        for c in range(scale.shape[1]):
            at = (slice(r * BLOCK, (r + 1) * BLOCK), slice(c * BLOCK, (c + 1) * BLOCK))
            inv, scale[r, c] = block_scale(x[at].abs().amax())
            q[at] = (x[at] * inv).to(torch.float8_e4m3fn).float()
    return q, scale


def spread(scale, shape, block_rows=1):
    """Scales repeated over their elements, 64 bits."""
    s = scale.double().repeat_interleave(BLOCK, -1)[..., : shape[-1]]
    return s if block_rows == 1 else s.repeat_interleave(BLOCK, 0)[: shape[0]]


def values(q, scale, block_rows=1):
    return q.double() * spread(scale, q.shape, block_rows)


def act(x, kind):
    """act(x), its slope and |z|, 64 bits (kind 0 GELU in its tanh form, 1 SiLU), through both sides of
    the sigmoid: 1 + tanh and 1 - tanh^2 would cancel, and leave 1e-16 where the slope is 1e-20."""
    x = x.double()
    c = 2 * math.sqrt(2 / math.pi)
    z, dz = (c * (x + 0.044715 * x**3), c * (1 + 3 * 0.044715 * x * x)) if kind == 0 else (x, torch.ones_like(x))
    s, rest = torch.sigmoid(z), torch.sigmoid(-z)
    return x * s, s + x * s * rest * dz, z.abs()


def slope_bound(x, kind):
    """How far an fp32 evaluation of the slope may be off: z is rounded a few times, so exp(-z) is
    off by (4 |z| + 16) half steps with the exponential's and the reciprocal's own; the slope's two
    terms are each off by at most that, relative."""
    x = x.double()
    _, slope, z = act(x, kind)
    s = torch.sigmoid(-z * torch.sign(-x))
    z = z.clamp(max=100.0)  # beyond, both terms are 0 or 1 in fp32
    return U * (16 + 4 * z) * (s + (slope - s).abs()) + 1e-30


def layer_norm(x, gamma, beta, eps):
    """y, xh, mean, rstd in 64 bits."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    return xh * gamma.double() + beta.double(), xh, mean, rstd


def layer_norm_bounds(x, gamma, beta, eps):
    """Bounds of xh's, mean's and rstd's error of an fp32 evaluation: a thread adds at most
    ceil(H / 32) terms and the partial sums are joined in at most 16 more additions, each off by a
    half step of a sum that is at most the sum of the terms' magnitudes; the terms are deviations
    from the row's first element."""
    x = x.double()
    _, xh, mean, rstd = layer_norm(x, gamma, beta, eps)
    steps = -(-x.shape[-1] // 32) + 16
    dev = (x - x[..., :1]).abs().mean(-1, keepdim=True)
    d_mean = U * (steps + 2) * dev + 2 * U * mean.abs()
    # the variance is taken around the computed mean: off by d_mean^2 and by its own additions
    d_rstd = rstd * (U * (steps + 8) + 0.5 * (d_mean * rstd) ** 2)
    d_xh = rstd * (d_mean + U * (x - mean).abs()) + xh.abs() * (d_rstd / rstd + 2 * U)
    return d_xh, d_mean, d_rstd


def layer_norm_grads(dy, xh, rstd, gamma):
    """dx, dgamma, dbeta in 64 bits from xh and rstd [..., 1]."""
    dy, g = dy.double(), dy.double() * gamma.double()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    flat = (-1, dy.shape[-1])
    return dx, (dy * xh).reshape(flat).sum(0), dy.reshape(flat).sum(0)


def layer_norm_grad_bounds(dy, xh, d_xh, rstd, gamma):
    """Bounds for dx, dgamma and dbeta in fp32 with xh off by d_xh: sums as in layer_norm_bounds,
    and over the rows one half step for each row and each of 16 joining additions."""
    dy, g = dy.double(), dy.double() * gamma.double()
    steps = -(-dy.shape[-1] // 32) + 16
    c1, c2 = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    d_c1 = U * (steps + 3) * c1
    d_c2 = U * (steps + 4) * c2 + (g.abs() * d_xh).mean(-1, keepdim=True)
    mean2 = (g * xh).mean(-1, keepdim=True).abs()
    d_dx = rstd * (4 * U * (g.abs() + c1 + xh.abs() * mean2) + d_c1 + xh.abs() * d_c2 + d_xh * (mean2 + d_c2))
    rows = dy.numel() // dy.shape[-1]
    flat = (-1, dy.shape[-1])
    n = rows + 16
    d_gamma = U * n * (dy * xh).abs().reshape(flat).sum(0) + (dy.abs() * d_xh).reshape(flat).sum(0)
    d_beta = U * n * dy.abs().reshape(flat).sum(0)
    return d_dx, d_gamma, d_beta


def assert_within(got, ref, bound, what, dtype=None):
    """Each element within `bound` of ref, and half a step of the output type where it is rounded."""
    dtype = dtype or got.dtype
    got, ref = got.double().cpu(), ref.double().cpu()
    bound = bound.double().cpu() + half_step(dtype) * (ref.abs() + bound.double().cpu()) + tiny(dtype)
    off = (got - ref).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((off / bound).max()):.3g} "
                           f"of the bound, first at {bad.nonzero()[0].tolist()}")
