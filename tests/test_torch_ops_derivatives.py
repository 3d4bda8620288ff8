"""What torch's differentiation gets from the training and 8-bit ops, on Meta tensors: no derivative is dropped in
silence, and the backward formulas are made of ops that other dispatch layers can see."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwad

F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(hc_lib):
    if not hc_lib.TORCH_OPS_PATH.exists():
        import build

        build.build_torch()
    return hc_lib.load_torch_ops()


def meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


X, G, STAT, Q, S = meta(4, 256), meta(256), meta(4), meta(4, 256, dtype=F8), meta(4, 2)
DIFFERENTIABLE = {
    "layer_norm_fwd_train": lambda o, x: o.layer_norm_fwd_train(x, G, G, 1e-5),
    "layer_norm_fwd_train, gamma": lambda o, x: o.layer_norm_fwd_train(X, x[0].contiguous(), G, 1e-5),
    "layer_norm_fwd_train, beta": lambda o, x: o.layer_norm_fwd_train(X, G, x[0].contiguous(), 1e-5),
    "layer_norm_ckpt": lambda o, x: o.layer_norm_ckpt(x, G, G, 1e-5),
    "layer_norm_ckpt, beta": lambda o, x: o.layer_norm_ckpt(X, G, x[0].contiguous(), 1e-5),
    "activation_gelu_silu_ckpt": lambda o, x: o.activation_gelu_silu_ckpt(x, 0),
}
OTHERS = {
    "quantize_fp8_block": lambda o, x: o.quantize_fp8_block(x, 1),
    "dequantize_fp8_block": lambda o, x: o.dequantize_fp8_block(Q, x[:, :2].contiguous(), torch.float32, 1),
    "matmul_fp8_block": lambda o, x: o.matmul_fp8_block(Q, S, Q, meta(1, 2), x[0, :4].contiguous(), torch.float32),
    "activation_gelu_silu_ckpt_bwd": lambda o, x: o.activation_gelu_silu_ckpt_bwd(x, Q, S, 1),
    "layer_norm_bwd": lambda o, x: o.layer_norm_bwd(x, X, G, STAT, STAT),
    "layer_norm_ckpt_bwd": lambda o, x: o.layer_norm_ckpt_bwd(x, Q, S, G, STAT),
}
CALLS = {**DIFFERENTIABLE, **OTHERS}


def first(out):
    return out[0] if isinstance(out, (tuple, list)) else out


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", ["plain", "requires_grad", "no_grad"])
def test_forward_mode_is_refused(ops, name, grad):
    """A tangent that an op would drop is a wrong derivative of zero."""
    with fwad.dual_level(), torch.set_grad_enabled(grad != "no_grad"):
        x = fwad.make_dual(X.clone().requires_grad_(grad == "requires_grad"), torch.ones_like(X))
        with pytest.raises(NotImplementedError, match="forward"):
            CALLS[name](ops, x)
    first(CALLS[name](ops, X))  # without a tangent it runs as ever


@pytest.mark.parametrize("name", CALLS)
def test_functional_jvp_is_refused(ops, name):
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda x: first(CALLS[name](ops, x)), (X,), (torch.ones_like(X),))


@pytest.mark.parametrize("name", OTHERS)
def test_missing_reverse_formula_is_an_error(ops, name):
    """No op gives up a gradient with no more than a warning."""
    out = first(OTHERS[name](ops, X.clone().requires_grad_(True)))
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="not implemented"):
        out.float().sum().backward()
    assert not first(OTHERS[name](ops, X)).requires_grad
