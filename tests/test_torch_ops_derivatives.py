"""What torch's differentiation gets from the training and 8-bit ops, on Meta and fake tensors: no derivative is dropped in
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


# ------------------------------------------------------------------------------ backward formulas
STEPS = {  # op -> (inputs' shapes, call, the op its gradient is made of)
    "layer_norm_fwd_train": (((4, 256), (256,), (256,)), lambda o, *t: o.layer_norm_fwd_train(*t, 1e-5)[0], "layer_norm_bwd"),
    "layer_norm_ckpt": (((4, 256), (256,), (256,)), lambda o, *t: o.layer_norm_ckpt(*t, 1e-5)[0], "layer_norm_ckpt_bwd"),
    "activation_gelu_silu_ckpt": (((4, 256),), lambda o, x: o.activation_gelu_silu_ckpt(x, 1)[0], "activation_gelu_silu_ckpt_bwd"),
}


def leaves(shapes, device):
    return [torch.empty(s, device=device, requires_grad=True) for s in shapes]


@pytest.mark.parametrize("name", STEPS)
def test_backward_of_meta_tensors(ops, name):
    shapes, call, _ = STEPS[name]
    t = leaves(shapes, "meta")
    call(ops, *t).sum().backward()
    assert [tuple(x.grad.shape) for x in t] == list(shapes) and all(x.grad.device.type == "meta" for x in t)


@pytest.mark.gpu  # torch's engine asks the device of a fake CUDA tensor for its context
@pytest.mark.parametrize("name", STEPS)
def test_backward_of_fake_cuda_tensors(ops, name):
    from torch._subclasses import FakeTensorMode

    shapes, call, _ = STEPS[name]
    with FakeTensorMode():
        t = leaves(shapes, "cuda")
        grads = torch.autograd.grad(call(ops, *t), t, torch.empty(shapes[0], device="cuda"))
        assert [tuple(g.shape) for g in grads] == list(shapes) and all(g.device.type == "cuda" for g in grads)


@pytest.mark.parametrize("name", STEPS)
@pytest.mark.parametrize("device", ["meta", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_traced_step_holds_the_backward_op(ops, name, device):
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    shapes, call, bwd = STEPS[name]

    def step(dy, *t):
        t = [x.detach().requires_grad_(True) for x in t]
        return torch.autograd.grad(call(ops, *t), t, dy)

    with FakeTensorMode():
        args = [torch.empty(s, device=device) for s in (shapes[0], *shapes)]
        graph = make_fx(step)(*args).graph
    called = [str(n.target) for n in graph.nodes if n.op == "call_function"]
    assert f"hc.{name}.default" in called and f"hc.{bwd}.default" in called


@pytest.mark.parametrize("name", STEPS)
def test_dispatch_modes_see_both_directions(ops, name):
    from torch.utils._python_dispatch import TorchDispatchMode

    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    shapes, call, bwd = STEPS[name]
    t = leaves(shapes, "meta")
    with Mode():
        call(ops, *t).sum().backward()
    assert f"hc::{name}" in seen and f"hc::{bwd}" in seen


@pytest.mark.parametrize("name", STEPS)
def test_tangent_of_the_incoming_gradient_is_refused(ops, name):
    """Forward over reverse: a tangent that enters through the output's gradient."""
    shapes, call, _ = STEPS[name]
    t = leaves(shapes, "meta")
    y = call(ops, *t)
    with fwad.dual_level():
        dy = fwad.make_dual(torch.empty_like(y, requires_grad=False), torch.empty_like(y, requires_grad=False))
        with pytest.raises(NotImplementedError, match="forward"):
            torch.autograd.grad(y, t, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("name", STEPS)
def test_compiled_step(cuda, ops, name):
    """torch.compile without code generation: the traced forward and backward give the eager bits."""
    shapes, call, _ = STEPS[name]
    g = torch.Generator().manual_seed(5)
    values = [torch.randn(*s, generator=g).cuda() for s in shapes]
    dy = torch.randn(*shapes[0], generator=g).cuda()

    def step(f):
        t = [v.clone().requires_grad_(True) for v in values]
        y = f(*t)
        return [y.detach(), *torch.autograd.grad(y, t, dy)]

    eager = step(lambda *t: call(ops, *t))
    compiled = step(torch.compile(lambda *t: call(ops, *t), backend="aot_eager"))
    assert all(torch.equal(a, b) for a, b in zip(eager, compiled))
