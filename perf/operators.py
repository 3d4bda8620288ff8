"""Measured cases of the 8-bit block operators and the trainable layer norm.

The operators and the calls that a user makes of them (torch.ops.hc, see hc.load_torch_ops()):
  layer_norm_fwd_train / layer_norm_bwd          layer norm with its statistics, and its gradients
  layer_norm_ckpt / layer_norm_ckpt_bwd          the same, keeping the normalised rows in 8 bits
  activation_gelu_silu_ckpt / ..._ckpt_bwd       GELU or SiLU keeping its input in 8 bits, and its gradient from that
  quantize_fp8_block, matmul_fp8_block           e4m3 operands with a scale for each block of 128
"""
import math
import os
import sys

import torch

own = False

BLOCK = 128            # elements of a row that share a scale (and rows of a weight's block)
FP8_MAX = 448.0        # largest finite e4m3 value
AMAX_FLOOR = 2.0**-100  # a block's largest magnitude is taken as at least this
EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # A few tokens of one sequence while a model is tried out: launch cost is all that counts.
        {"name": "ln_train_few_rows", "kind": "ln_train", "rows": 8, "cols": 1024, "type": "f32"},
        # The layer norm benchmark's rows, one training step: forward, then all three gradients.
        {"name": "ln_train_large", "kind": "ln_train", "rows": 16384, "cols": 4096, "type": "bf16"},
        # Rows that are no multiple of 16 bytes, a row count that divides by nothing: a ragged token batch.
        {"name": "ln_train_odd", "kind": "ln_train", "rows": 1037, "cols": 1001, "type": "f16"},
        # A layer's forward under a memory limit: the normalised rows are kept in 8 bits.
        {"name": "ln_ckpt_forward", "kind": "ln_ckpt_fwd", "rows": 8192, "cols": 2048, "type": "bf16"},
        # The matching backward at a wide hidden size, from the 8-bit rows.
        {"name": "ln_ckpt_backward", "kind": "ln_ckpt_bwd", "rows": 8192, "cols": 8192, "type": "bf16"},
        # The activation benchmark's tensor: GELU in the forward pass of a feed-forward layer.
        {"name": "act_ckpt_forward", "kind": "act_ckpt_fwd", "rows": 16384, "cols": 4096, "type": "bf16", "act": 0},
        # SiLU's gradient from the 8-bit input, fp16 training.
        {"name": "act_ckpt_backward", "kind": "act_ckpt_bwd", "rows": 16384, "cols": 4096, "type": "f16", "act": 1},
        # A short fp32 batch whose rows end inside a block of 128.
        {"name": "act_ckpt_small", "kind": "act_ckpt_bwd", "rows": 33, "cols": 1000, "type": "f32", "act": 0},
        # Serving one token: the weight is read once, and that is the time.
        {"name": "matmul_one_token", "kind": "matmul", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False},
        # A ragged decode batch against an odd output width, K ending inside a block.
        {"name": "matmul_ragged", "kind": "matmul", "m": 77, "n": 10001, "k": 2064, "type": "f16", "bias": True},
        # The matmul benchmark's product.
        {"name": "matmul_large", "kind": "matmul", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False},
        # A prompt through a linear layer: its activations are quantised, then multiplied; fp32 logits.
        {"name": "linear_prompt", "kind": "linear", "m": 2048, "n": 4096, "k": 4096, "type": "f32", "bias": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["ln_train", "ln_ckpt_fwd", "ln_ckpt_bwd", "act_ckpt_fwd", "act_ckpt_bwd", "matmul", "linear"])
    case = {"kind": kind, "type": rng.choice(["bf16", "f16", "f32"])}
    if kind in ("matmul", "linear"):
        # Rows of the operands are multiples of 16 bytes, as hidden sizes are; M and N are anything.
        case.update(m=_log_int(rng, 1, 8192), n=_log_int(rng, 64, 8192), k=16 * _log_int(rng, 8, 512),
                    bias=rng.random() < 0.5)
        return case
    cols = _log_int(rng, 64, 8192)
    if rng.random() < 0.5:
        cols = max(64, cols // 64 * 64)
    rows = _log_int(rng, 1, min(16384, 16384 * 4096 // (cols * (2 if case["type"] == "f32" else 1))))
    case.update(rows=rows, cols=cols)
    if kind.startswith("act"):
        case["act"] = rng.randrange(2)
    return case


# ---------------------------------------------------------------------------------------------
# Plain forms: elementary torch operations in 32 bits, rounded once at the end
# ---------------------------------------------------------------------------------------------
def _blocks(x):
    """x [..., C] as [..., ceil(C / 128), 128], zeros behind the last column."""
    c = x.shape[-1]
    n = -(-c // BLOCK)
    x = torch.nn.functional.pad(x, (0, n * BLOCK - c))
    return x.reshape(*x.shape[:-1], n, BLOCK)


def _inverse_and_scale(amax):
    """448 / amax and amax / 448, each a division: with a Python number on one side torch would
    multiply by a rounded reciprocal."""
    top = torch.full_like(amax, FP8_MAX)
    return top / amax, amax / top


def _quantize(x):
    """Rows of x (32 bits) in e4m3 with a scale for each 128 elements of a row."""
    b = _blocks(x)
    amax = b.abs().amax(-1).clamp(min=AMAX_FLOOR)
    inverse, scale = _inverse_and_scale(amax)
    q = (b * inverse.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return q.reshape(*x.shape[:-1], -1)[..., : x.shape[-1]].contiguous(), scale


def _spread(scale, like, dtype):
    """Row-block scales [..., n] repeated over their columns."""
    return scale.to(dtype).repeat_interleave(BLOCK, -1)[..., : like.shape[-1]]


def _quantize_weight(w):
    """w [N, K] (32 bits) in e4m3 with a scale for each 128 x 128 block."""
    n, k = w.shape
    p = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    b = p.reshape(p.shape[0] // BLOCK, BLOCK, p.shape[1] // BLOCK, BLOCK)
    amax = b.abs().amax((1, 3)).clamp(min=AMAX_FLOOR)
    inverse, scale = _inverse_and_scale(amax)
    q = (b * inverse[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.reshape(p.shape)[:n, :k].contiguous(), scale


def _spread_weight(scale, like, dtype):
    s = scale.to(dtype).repeat_interleave(BLOCK, 0)[: like.shape[0]]
    return s.repeat_interleave(BLOCK, 1)[:, : like.shape[1]]


def _ln_stats(x):
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    return mean, centred * rstd, rstd


def _ln_grads(dy, xhat, rstd, gamma, dtype):
    g = dy * gamma
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx.to(dtype), (dy * xhat).sum(0), dy.sum(0)


def _act_parts(x, act):
    """sigmoid(z) and dz/dx with act(x) = x sigmoid(z): z = 2 sqrt(2/pi) (x + 0.044715 x^3) or x."""
    if act == 0:
        k = 2.0 * math.sqrt(2.0 / math.pi)
        return torch.sigmoid(k * (x + 0.044715 * x * x * x)), k * (1.0 + 3 * 0.044715 * x * x)
    return torch.sigmoid(x), torch.ones_like(x)


def _product(s, x_q, x_scale):
    a = x_q.float() * _spread(x_scale, x_q, torch.float32)
    b = s["w_q"].float() * _spread_weight(s["w_scale"], s["w_q"], torch.float32)
    c = a @ b.t()
    if s["bias"] is not None:
        c = c + s["bias"].float()
    return c.to(s["dtype"])


def _run_plain(s):
    kind = s["kind"]
    if kind == "ln_train":
        x, dy = s["x"].float(), s["dy"].float()
        _, xhat, rstd = _ln_stats(x)
        y = xhat * s["gamma"] + s["beta"]
        dx, dgamma, dbeta = _ln_grads(dy, xhat, rstd, s["gamma"], s["dtype"])
        return {"y": y.to(s["dtype"]), "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if kind == "ln_ckpt_fwd":
        _, xhat, rstd = _ln_stats(s["x"].float())
        q, scale = _quantize(xhat)
        return {"y": (xhat * s["gamma"] + s["beta"]).to(s["dtype"]), "q": q, "scale": scale, "rstd": rstd[..., 0]}
    if kind == "ln_ckpt_bwd":
        xhat = s["q"].float() * _spread(s["scale"], s["q"], torch.float32)
        dx, dgamma, dbeta = _ln_grads(s["dy"].float(), xhat, s["rstd"][:, None], s["gamma"], s["dtype"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if kind == "act_ckpt_fwd":
        x = s["x"].float()
        q, scale = _quantize(x)
        return {"y": (x * _act_parts(x, s["act"])[0]).to(s["dtype"]), "q": q, "scale": scale}
    if kind == "act_ckpt_bwd":
        x = s["q"].float() * _spread(s["scale"], s["q"], torch.float32)
        sig, dz = _act_parts(x, s["act"])
        return {"dx": (s["dy"].float() * (sig + x * sig * (1.0 - sig) * dz)).to(s["dtype"])}
    if kind == "matmul":
        return {"c": _product(s, s["x_q"], s["x_scale"])}
    q, scale = _quantize(s["x"].float())
    return {"c": _product(s, q, scale), "q": q, "scale": scale}


# ---------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------
_loaded = []


def _ops():
    if not _loaded:
        sys.path.insert(0, os.path.join(os.getcwd(), "ascend-npu-harness_b200"))
        import hc

        _loaded.append(hc.load_torch_ops())
    return _loaded[0]


def _run_own(s):
    ops, kind = _ops(), s["kind"]
    if kind == "ln_train":
        y, mean, rstd = ops.layer_norm_fwd_train(s["x"], s["gamma"], s["beta"], EPS)
        dx, dgamma, dbeta = ops.layer_norm_bwd(s["dy"], s["x"], s["gamma"], mean, rstd)
        return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if kind == "ln_ckpt_fwd":
        y, q, scale, rstd = ops.layer_norm_ckpt(s["x"], s["gamma"], s["beta"], EPS)
        return {"y": y, "q": q, "scale": scale, "rstd": rstd}
    if kind == "ln_ckpt_bwd":
        dx, dgamma, dbeta = ops.layer_norm_ckpt_bwd(s["dy"], s["q"], s["scale"], s["gamma"], s["rstd"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if kind == "act_ckpt_fwd":
        y, q, scale = ops.activation_gelu_silu_ckpt(s["x"], s["act"])
        return {"y": y, "q": q, "scale": scale}
    if kind == "act_ckpt_bwd":
        return {"dx": ops.activation_gelu_silu_ckpt_bwd(s["dy"], s["q"], s["scale"], s["act"])}
    if kind == "matmul":
        return {"c": ops.matmul_fp8_block(s["x_q"], s["x_scale"], s["w_q"], s["w_scale"], s["bias"], s["dtype"])}
    q, scale = ops.quantize_fp8_block(s["x"], 1)
    return {"c": ops.matmul_fp8_block(q, scale, s["w_q"], s["w_scale"], s["bias"], s["dtype"]), "q": q, "scale": scale}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, dtype = case["kind"], TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def activations(rows, cols):
        """Hidden states: channels of differing size, a few of them large, and a small offset."""
        size = torch.exp(0.4 * normal(cols)) * torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        return normal(rows, cols) * size + 0.2

    s = {"kind": kind, "dtype": dtype, "act": case.get("act", 0)}
    if kind in ("matmul", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        s["w_q"], s["w_scale"] = _quantize_weight(normal(n, k) / math.sqrt(k))
        s["bias"] = (0.1 * normal(n)).to(dtype) if case["bias"] else None
        x = activations(m, k)
        if kind == "linear":
            s["x"] = x.to(torch.bfloat16)
        else:
            s["x_q"], s["x_scale"] = _quantize(x)
        return s
    rows, cols = case["rows"], case["cols"]
    x = activations(rows, cols).to(dtype)
    if kind.startswith("ln"):
        s["gamma"], s["beta"] = 1.0 + 0.1 * normal(cols), 0.1 * normal(cols)
    if kind in ("ln_train", "ln_ckpt_bwd", "act_ckpt_bwd"):
        s["dy"] = (0.02 * normal(rows, cols)).to(dtype)
    if kind == "ln_ckpt_bwd":
        _, xhat, rstd = _ln_stats(x.float())
        s["q"], s["scale"] = _quantize(xhat)
        s["rstd"] = rstd[:, 0].contiguous()
    elif kind == "act_ckpt_bwd":
        s["q"], s["scale"] = _quantize(x.float())
    else:
        s["x"] = x
    return s


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    kind, e = case["kind"], BYTES[case["type"]]
    if kind in ("matmul", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        size = n * k + 4 * nb * kb + e * m * n + (e * n if case["bias"] else 0) + m * k + 4 * m * kb
        flops = 2 * m * n * k
        if kind == "linear":
            size += 2 * m * k  # bf16 activations in; their 8-bit form and its scales are outputs
            flops += 3 * m * k
        return {"bytes": size, "flops": flops}
    n, rows, cols = case["rows"] * case["cols"], case["rows"], case["cols"]
    ckpt = n + 4 * rows * -(-cols // BLOCK)
    return {
        "ln_train": {"bytes": 4 * e * n + 16 * cols, "flops": 22 * n},
        "ln_ckpt_fwd": {"bytes": 2 * e * n + ckpt + 4 * rows + 8 * cols, "flops": 11 * n},
        "ln_ckpt_bwd": {"bytes": 2 * e * n + ckpt + 4 * rows + 12 * cols, "flops": 15 * n},
        "act_ckpt_fwd": {"bytes": 2 * e * n + ckpt, "flops": 12 * n},
        "act_ckpt_bwd": {"bytes": 2 * e * n + ckpt, "flops": 16 * n},
    }[kind]


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]

    def d(name):
        return s[name].to(torch.float64)

    def per_column(scale, cols):
        return scale.to(torch.float64)[:, torch.arange(cols, device="cuda") // BLOCK]

    def block_amax(x):
        rows, cols = x.shape
        n = (cols + BLOCK - 1) // BLOCK
        p = torch.zeros(rows, n * BLOCK, dtype=torch.float64, device="cuda")
        p[:, :cols] = x.abs()
        return torch.clamp(p.view(rows, n, BLOCK).max(2).values, min=AMAX_FLOOR)

    if kind in ("matmul", "linear"):
        n, k = case["n"], case["k"]
        if kind == "linear":  # the 8-bit activations are those of the definition in 32 bits, exact as they stand
            q32, s32 = _quantize(s["x"].float())
            a, scale = q32.to(torch.float64) * per_column(s32, k), block_amax(d("x")) / FP8_MAX
        else:
            a, scale = d("x_q") * per_column(s["x_scale"], k), None
        rows = torch.arange(n, device="cuda") // BLOCK
        w = d("w_q") * per_column(s["w_scale"], k)[rows]
        c = torch.einsum("mk,nk->mn", a, w)
        if case["bias"]:
            c += d("bias")
        return {"c": c, "q": None, "scale": scale} if kind == "linear" else {"c": c}
    cols = case["cols"]
    if kind.startswith("act"):
        x = d("q") * per_column(s["scale"], cols) if kind == "act_ckpt_bwd" else d("x")
        if case["act"] == 0:
            c = math.sqrt(2.0 / math.pi)
            t = torch.tanh(c * (x + 0.044715 * x**3))
            y, slope = 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 0.134145 * x * x)
        else:
            e = torch.exp(-x)
            y, slope = x / (1 + e), (1 + e + x * e) / (1 + e) ** 2
        if kind == "act_ckpt_bwd":
            return {"dx": d("dy") * slope}
        return {"y": y, "q": None, "scale": block_amax(x) / FP8_MAX}
    gamma = d("gamma")
    if kind == "ln_ckpt_bwd":
        xhat, sigma = d("q") * per_column(s["scale"], cols), 1.0 / d("rstd")[:, None]
    else:
        x = d("x")
        var, mu = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sigma = torch.sqrt(var + EPS)
        xhat = (x - mu) / sigma
    y = None if kind == "ln_ckpt_bwd" else torch.addcmul(d("beta"), xhat, gamma)
    if kind == "ln_ckpt_fwd":
        return {"y": y, "q": None, "scale": block_amax(xhat) / FP8_MAX, "rstd": 1.0 / sigma[:, 0]}
    dy = d("dy")
    dxhat = dy * gamma
    total = dxhat.sum(1, keepdim=True) + xhat * torch.einsum("rc,rc->r", dxhat, xhat)[:, None]
    grads = {"dx": (dxhat - total / cols) / sigma, "dgamma": torch.einsum("rc,rc->c", dy, xhat), "dbeta": dy.sum(0)}
    return grads if kind == "ln_ckpt_bwd" else {"y": y, **grads}
