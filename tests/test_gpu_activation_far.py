"""GELU and SiLU far from zero on the GPU, where the sigmoid is 0 or 1 in every type."""
from __future__ import annotations

import pytest
import torch

import fp8_reference as R
import hc

pytestmark = pytest.mark.gpu

VALUES = [3e38, 1e30, 1e10, 6e4, 1e4, 300.0, 200.0, 100.0, 89.0, 88.5, 88.0, 87.5, 87.0, 50.0, 20.0, 12.0, 10.0, 9.9, 5.0, 1.0, 0.0]


def far(kind, cols):
    """The values of either sign that the type holds, repeated over a row."""
    top = torch.finfo(R.DTYPES[kind]).max
    v = torch.tensor([s * a for a in VALUES if a <= top for s in (1.0, -1.0)])
    return v.repeat(-(-cols // len(v)))[:cols].reshape(1, cols).to(R.DTYPES[kind])


@pytest.mark.parametrize("cols", [512, 501])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_far_values(cuda, kind, act, cols):
    """Against 64 bits.  exp(-|z|) is off by (16 + 4 |z|) half steps.  From z = -87 on (2^-126, the smallest normal
    number of fp32, is exp(-87.34)) a result anywhere between the exact one and 0 will do; the fp32 GELU forms 1 + tanh,
    which leaves 4 half steps of |x| below zero."""
    x = far(kind, cols)
    ref, _, z = R.act(x, 0 if act == "gelu" else 1)
    ref = torch.where(x.double() < -1e4, torch.zeros_like(ref), ref)  # exp(-z) is 0 in 64 bits, too
    rel = torch.where(x < 0, torch.where(z < 87, R.U * (16 + 4 * z), torch.ones_like(z)), torch.full_like(z, R.U * 16))
    bound = rel * ref.abs()
    if kind == "f32" and act == "gelu":
        bound = bound + torch.where((x < 0) & (x > -20), 4 * R.U * x.double().abs(), torch.zeros_like(bound))
    y, _, _ = hc.activation_gelu_silu_ckpt(x.cuda(), act)
    R.assert_within(y, ref, bound, "checkpointed")
    R.assert_within(hc.activation_gelu_silu(x.cuda(), act), ref, bound, "plain")


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_infinities_and_nan(cuda, kind, act):
    """x * sigmoid(x) at the infinities and at a NaN, as the 64-bit form has it: inf, NaN (inf * 0) and NaN."""
    x = torch.zeros(3, 256, dtype=R.DTYPES[kind], device="cuda")
    x[0, ::3], x[1, 1::3], x[2, 2::3] = float("inf"), float("-inf"), float("nan")
    for y in (hc.activation_gelu_silu_ckpt(x, act)[0], hc.activation_gelu_silu(x, act)):
        assert bool(y[0, ::3].isposinf().all()) and bool(y[1, 1::3].isnan().all()) and bool(y[2, 2::3].isnan().all())
        assert int((y == 0).sum()) == 3 * 256 - 86 - 85 - 85
