"""Layer norm for training on the GPU: statistics, the 8-bit checkpoint, all three gradients against
64-bit forms and differences, and autograd."""
from __future__ import annotations

import pytest
import torch

import fp8_reference as R
import hc

pytestmark = pytest.mark.gpu

EPS = 1e-5
KINDS = ["f32", "f16", "bf16"]
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (4, 64), (9, 127), (1, 128), (37, 129), (2, 3, 136), (33, 768), (8, 1024), (65, 1000),
          (130, 1001), (700, 256), (40, 2048), (301, 520), (16, 4096), (3, 5120), (5, 8192), (3, 8200), (2, 16384), (2, 20000),
          (2, 20001), (2000, 72), (5000, 8), (600, 1536), (1300, 4096), (700, 6000), (450, 7001)]


@pytest.fixture(scope="module")
def ops(cuda):
    return hc.load_torch_ops()


def rnd(shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def inputs(shape, kind, offset=0.3):
    H = shape[-1]
    x = (rnd(shape, 1) * (1 + torch.arange(H) % 5) + offset).to(R.DTYPES[kind]).cuda()
    gamma, beta = 1 + 0.2 * rnd((H,), 2).cuda(), 0.3 * rnd((H,), 3).cuda()
    return x, gamma, beta, rnd(shape, 4).to(R.DTYPES[kind]).cuda()


def check_forward(x, gamma, beta, y, mean, rstd):
    ref, xh, m, r = R.layer_norm(x, gamma, beta, EPS)
    d_xh, d_mean, d_rstd = R.layer_norm_bounds(x, gamma, beta, EPS)
    R.assert_within(rstd, r[..., 0], d_rstd[..., 0], "rstd")
    if mean is not None:
        R.assert_within(mean, m[..., 0], d_mean[..., 0], "mean")
    g = gamma.double().abs()
    R.assert_within(y, ref, g * d_xh + 2 * R.U * (g * xh.abs() + beta.double().abs()), "y")
    return xh, d_xh


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(cuda, shape, kind):
    x, gamma, beta, dy = inputs(shape, kind)
    y, mean, rstd = hc.layer_norm_fwd_train(x, gamma, beta, EPS)
    check_forward(x, gamma, beta, y, mean, rstd)
    dx, dgamma, dbeta = hc.layer_norm_bwd(dy, x, gamma, mean, rstd)
    # the backward's own error, from the statistics it is given
    m, r = mean.double()[..., None], rstd.double()[..., None]
    xh = (x.double() - m) * r
    d_xh = 3 * R.U * r * (x.double().abs() + m.abs())
    ref = R.layer_norm_grads(dy, xh, r, gamma)
    bounds = R.layer_norm_grad_bounds(dy, xh, d_xh, r, gamma)
    for name, got, want, bound in zip(("dx", "dgamma", "dbeta"), (dx, dgamma, dbeta), ref, bounds):
        R.assert_within(got, want, bound, name)
    again = hc.layer_norm_bwd(dy, x, gamma, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dgamma, dbeta)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_checkpoint(cuda, shape, kind):
    x, gamma, beta, dy = inputs(shape, kind)
    y, q, scale, rstd = hc.layer_norm_ckpt(x, gamma, beta, EPS)
    xh, d_xh = check_forward(x, gamma, beta, y, None, rstd)
    # scale: the largest |xh| of the block, off by what xh is off; kept values: half a code step more
    n = scale.shape[-1]
    pad = torch.nn.functional.pad(xh, (0, n * 128 - shape[-1])).abs().reshape(*shape[:-1], n, 128)
    pad_d = torch.nn.functional.pad(d_xh, (0, n * 128 - shape[-1])).reshape(*shape[:-1], n, 128)
    amax = pad.amax(-1).clamp(min=R.FLOOR)
    assert bool(((scale.double() * 448 - amax).abs() <= pad_d.amax(-1) + 2 * R.U * amax).all())
    kept = R.values(q, scale)
    spread = R.spread(scale, shape)
    bound = d_xh + (xh.abs() + d_xh) * 2.0**-4 * (1 + 8 * R.U) + spread * 2.0**-10 * (1 + 8 * R.U)
    assert bool(((kept - xh).abs() <= bound).all())
    dx, dgamma, dbeta = hc.layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd)
    r = rstd.double()[..., None]
    ref = R.layer_norm_grads(dy, kept, r, gamma)
    bounds = R.layer_norm_grad_bounds(dy, kept, R.U * kept.abs(), r, gamma)
    for name, got, want, bound in zip(("dx", "dgamma", "dbeta"), (dx, dgamma, dbeta), ref, bounds):
        R.assert_within(got, want, bound, name)
    again = hc.layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd)
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dgamma, dbeta)))


@pytest.mark.parametrize("shape", [(9, 129), (33, 768)], ids=str)
def test_gradients_against_differences(cuda, shape):
    """Along random directions of x, gamma and beta: the 64-bit forward's central difference."""
    x, gamma, beta, dy = inputs(shape, "f32")
    y, mean, rstd = hc.layer_norm_fwd_train(x, gamma, beta, EPS)
    grads = hc.layer_norm_bwd(dy, x, gamma, mean, rstd)
    _, xh, m, r = R.layer_norm(x, gamma, beta, EPS)
    d_xh, _, d_rstd = R.layer_norm_bounds(x, gamma, beta, EPS)
    bounds = list(R.layer_norm_grad_bounds(dy, xh, d_xh + 3 * R.U * r * (x.double().abs() + m.abs()), r, gamma))
    ref = R.layer_norm_grads(dy, xh, r, gamma)
    bounds[0] = bounds[0] + ref[0].abs() * d_rstd / r
    at = [t.double() for t in (x, gamma, beta)]
    h = 1e-5
    for i, (g, bound) in enumerate(zip(grads, bounds)):
        v = rnd(tuple(at[i].shape), 5 + i).double().cuda()
        lo, hi = [t.clone() for t in at], [t.clone() for t in at]
        lo[i] -= h * v
        hi[i] += h * v
        diff = ((R.layer_norm(*hi, EPS)[0] - R.layer_norm(*lo, EPS)[0]) * dy.double()).sum() / (2 * h)
        # the difference itself: h^2 of a smooth function and 2^-53 / h of the values
        slack = ((bound + R.U * ref[i].abs()) * v.abs()).sum() + 1e-8 * (dy.double().abs()).sum()
        assert abs(float((g.double() * v).sum() - diff)) <= float(slack), i


@pytest.mark.parametrize("kind", KINDS)
def test_rows_near_a_large_constant(cuda, kind):
    """|mean| far above the spread: mean and variance over deviations keep their precision, and the
    checkpoint holds the normalised rows, not the offset."""
    x, gamma, beta, dy = inputs((6, 1024), kind, offset=300.0 if kind != "f32" else 3000.0)
    y, q, scale, rstd = hc.layer_norm_ckpt(x, gamma, beta, EPS)
    xh, _ = check_forward(x, gamma, beta, y, None, rstd)
    assert float((R.values(q, scale) - xh).abs().max()) <= float(xh.abs().max()) * 2.0**-4


@pytest.mark.parametrize("H", [8, 129, 1024])
def test_constant_and_nonfinite_rows(cuda, H):
    """A constant row gives xh = 0 and y = beta; a NaN or an infinity spoils its own row and, through the
    sums, the weights' gradients, but no other row."""
    x, gamma, beta, dy = inputs((5, H), "f32")
    x[1] = 3.5
    x[3, H // 2] = float("nan")
    x[4, 0] = float("inf")
    y, mean, rstd = hc.layer_norm_fwd_train(x, gamma, beta, EPS)
    assert torch.equal(y[1], beta) and bool(y[3].isnan().all()) and bool(y[4].isnan().all())
    assert bool(y[:3].isfinite().all())
    dx, dgamma, dbeta = hc.layer_norm_bwd(dy, x, gamma, mean, rstd)
    assert bool(dx[:3].isfinite().all()) and bool(dx[3:].isnan().all())
    assert bool(dgamma.isnan().all()) and bool(dbeta.isfinite().all())
    y2, q, scale, rstd = hc.layer_norm_ckpt(x, gamma, beta, EPS)
    assert torch.equal(y2[:3], y[:3]) and bool((R.values(q, scale)[1] == 0).all())
    assert bool(R.values(q, scale)[3:].isnan().all())
    dx, _, _ = hc.layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd)
    assert bool(dx[:3].isfinite().all()) and bool(dx[3:].isnan().all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("H", [5, 37, 136, 1000, 1001, 2056, 6000])
def test_constant_rows_of_large_values(cuda, H, kind):
    """mean * rstd above the largest fp32: x - mean is zero, and so is xh.  Rows that leave some of their
    threads' columns unused take no part of what those would compute."""
    _, gamma, beta, dy = inputs((6, H), kind)
    x = torch.full((6, H), 1e36, dtype=R.DTYPES[kind], device="cuda")
    y, mean, rstd = hc.layer_norm_fwd_train(x, gamma, beta, 1e-12)
    assert torch.equal(mean, x[:, 0].float()) and torch.equal(y, beta.to(y.dtype).expand_as(y))
    assert bool((mean * rstd).isinf().all())
    xh, r = torch.zeros(6, H, dtype=torch.float64, device="cuda"), rstd.double()[:, None]
    ref = R.layer_norm_grads(dy, xh, r, gamma)
    bounds = R.layer_norm_grad_bounds(dy, xh, xh, r, gamma)
    for name, got, want, bound in zip(("dx", "dgamma", "dbeta"), hc.layer_norm_bwd(dy, x, gamma, mean, rstd), ref, bounds):
        R.assert_within(got, want, bound, name)


@pytest.mark.parametrize("kind", KINDS)
def test_unaligned_buffers(cuda, kind):
    """Contiguous views that start off a 16-byte boundary."""
    x, gamma, beta, dy = inputs((6, 256), kind)

    def moved(t):
        return torch.empty(1 + t.numel(), dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    for f in range(4):
        a, g, b, d = (moved(t) if f in (i, 3) else t for i, t in enumerate((x, gamma, beta, dy)))
        if f == 2:
            b = moved(beta)
        y, mean, rstd = hc.layer_norm_fwd_train(a, g, b, EPS)
        check_forward(x, gamma, beta, y, mean, rstd)
        dx, dgamma, dbeta = hc.layer_norm_bwd(moved(d) if f == 2 else d, a, g, mean, rstd)
        m, r = mean.double()[..., None], rstd.double()[..., None]
        xh = (x.double() - m) * r
        bounds = R.layer_norm_grad_bounds(dy, xh, 3 * R.U * r * (x.double().abs() + m.abs()), r, gamma)
        for got, want, bound in zip((dx, dgamma, dbeta), R.layer_norm_grads(dy, xh, r, gamma), bounds):
            R.assert_within(got, want, bound, f"moved {f}")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,H", [(1, 768), (40, 768), (3, 6000), (20, 6000)])
def test_parameters_at_any_address(cuda, rows, H, kind):
    """gamma, beta, dgamma and dbeta 4 bytes behind a 16-byte boundary: the bits of the aligned call, and nothing
    written beside them."""
    x, gamma, beta, dy = inputs((rows, H), kind)
    off = [torch.cat([v[:1], v])[1:] for v in (gamma, beta)]
    assert all(v.data_ptr() % 16 == 4 for v in off)
    want = hc.layer_norm_fwd_train(x, gamma, beta, EPS)
    assert all(torch.equal(a, b) for a, b in zip(hc.layer_norm_fwd_train(x, *off, EPS), want))
    mean, rstd = want[1:]
    dx, dgamma, dbeta = hc.layer_norm_bwd(dy, x, gamma, mean, rstd)
    out, dx2 = torch.full((2, H + 8), 7.0, device="cuda"), torch.empty_like(dx)
    t = hc.LayerNormTiling(rows, H, 0, EPS)
    work = torch.empty(rows * 2 * H, device="cuda")
    hc.check(hc.load().hc_layer_norm_bwd_launch(
        dy.data_ptr(), x.data_ptr(), off[0].data_ptr(), mean.data_ptr(), rstd.data_ptr(), dx2.data_ptr(),
        out[0, 1:].data_ptr(), out[1, 1:].data_ptr(), work.data_ptr(), work.numel() * 4, t, hc.dtype_code(x),
        torch.cuda.current_stream().cuda_stream))
    assert torch.equal(dx2, dx) and torch.equal(out[0, 1:H + 1], dgamma) and torch.equal(out[1, 1:H + 1], dbeta)
    assert bool((out[:, 0] == 7.0).all()) and bool((out[:, H + 1:] == 7.0).all())


def test_no_rows(ops):
    x, gamma = torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda")
    y, mean, rstd = ops.layer_norm_fwd_train(x, gamma, gamma, EPS)
    dx, dgamma, dbeta = ops.layer_norm_bwd(y, x, gamma, mean, rstd)
    assert dx.shape == (0, 64) and bool((dgamma == 0).all()) and bool((dbeta == 0).all())
    y, q, scale, rstd = ops.layer_norm_ckpt(x, gamma, gamma, EPS)
    _, dgamma, dbeta = ops.layer_norm_ckpt_bwd(y, q, scale, gamma, rstd)
    assert bool((dgamma == 0).all()) and bool((dbeta == 0).all())


def test_autograd(ops):
    x, gamma, beta, dy = inputs((4, 33, 264), "bf16")
    leaves = [t.clone().requires_grad_(True) for t in (x, gamma, beta)]
    y, mean, rstd = ops.layer_norm_fwd_train(*leaves, EPS)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
    y.backward(dy)
    for leaf, want in zip(leaves, ops.layer_norm_bwd(dy, x, gamma, mean, rstd)):
        assert torch.equal(leaf.grad, want)
    y, q, scale, rstd = ops.layer_norm_ckpt(*leaves, EPS)
    got = torch.autograd.grad(y, leaves, dy)
    for a, want in zip(got, ops.layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd)):
        assert torch.equal(a, want)
    # a gradient that is not dense, a frozen weight, and no second derivative
    y, mean, rstd = ops.layer_norm_fwd_train(leaves[0], gamma, beta, EPS)
    (dx,) = torch.autograd.grad(y.sum(), leaves[0])
    assert torch.equal(dx, ops.layer_norm_bwd(torch.ones_like(x), x, gamma, mean, rstd)[0])
    y, _, _ = ops.layer_norm_fwd_train(*leaves, EPS)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y, leaves, dy, create_graph=True)


def test_checkpoint_keeps_no_input(ops):
    """The checkpointed forward saves the 8-bit rows and not x: about half of x's bytes in bf16."""
    x = torch.randn(2048, 4096, device="cuda").to(torch.bfloat16).requires_grad_(True)
    gamma = torch.ones(4096, device="cuda", requires_grad=True)
    beta = torch.zeros(4096, device="cuda", requires_grad=True)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.nbytes) or t, lambda t: t):
        y, *_ = ops.layer_norm_ckpt(x, gamma, beta, EPS)
        z, *_ = ops.activation_gelu_silu_ckpt(y, 1)
    n = x.numel()
    assert sum(kept) <= 2 * (n + n // 128 * 4) + 4096 * 8 + 2048 * 8


def test_training_step_in_a_graph(ops):
    """Forward and backward through autograd captured together and replayed on new inputs."""
    x, gamma, beta, dy = inputs((70, 520), "bf16")
    static = x.clone().requires_grad_(True)
    g, b = gamma.clone().requires_grad_(True), beta.clone().requires_grad_(True)

    def step():
        y, *_ = ops.layer_norm_ckpt(static, g, b, EPS)
        z, *_ = ops.activation_gelu_silu_ckpt(y, 1)
        return torch.autograd.grad(z, (static, g, b), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        with torch.no_grad():
            static.copy_(rnd((70, 520), 40 + turn).cuda())
        graph.replay()
        for a, want in zip(out, step()):
            assert torch.equal(a, want)


def test_explicit_backward_in_a_graph_beside_an_eager_graph(ops):
    """torch refuses to capture an autograd backward while an eager graph of the same leaves lives; the _bwd
    ops can be captured then, and the eager graph still gives its gradients afterwards."""
    x, gamma, beta, dy = inputs((70, 520), "bf16")
    leaf = x.clone().requires_grad_(True)
    alive = ops.layer_norm_fwd_train(leaf, gamma, beta, EPS)[0]

    def step():
        with torch.no_grad():
            y, q, scale, rstd = ops.layer_norm_ckpt(leaf, gamma, beta, EPS)
            return (y, *ops.layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    for a, want in zip(out, step()):
        assert torch.equal(a, want)
    alive.backward(dy)
    _, mean, rstd = ops.layer_norm_fwd_train(x, gamma, beta, EPS)
    assert torch.equal(leaf.grad, ops.layer_norm_bwd(dy, x, gamma, mean, rstd)[0])


@pytest.mark.parametrize("H", [264, 4104])
def test_more_than_32_bits_of_elements(ops, H):
    """Over 2^32 elements: the last rows of a tensor of repeated rows equal the first, and the weights'
    gradients are those of one copy times the number of copies, within the additions' error."""
    part, gamma, beta, dpart = inputs((256, H), "bf16")
    n = (1 << 32) // (256 * H) + 2
    x, dy = part.repeat(n, 1), dpart.repeat(n, 1)
    assert x.numel() > 1 << 32
    y0, q0, s0, r0 = ops.layer_norm_ckpt(part, gamma, beta, EPS)
    y, q, scale, rstd = ops.layer_norm_ckpt(x, gamma, beta, EPS)
    assert torch.equal(y[-256:], y0) and torch.equal(scale[-256:], s0) and torch.equal(rstd[-256:], r0)
    assert torch.equal(q[-256:].view(torch.uint8), q0.view(torch.uint8))
    dx0, _, _ = ops.layer_norm_ckpt_bwd(dpart, q0, s0, gamma, r0)
    dx, dgamma, dbeta = ops.layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd)
    assert torch.equal(dx[-256:], dx0)
    xh = R.values(q0, s0)
    bound = R.layer_norm_grad_bounds(dpart, xh, R.U * xh.abs(), r0.double()[:, None], gamma)
    _, dg, db = R.layer_norm_grads(dpart, xh, r0.double()[:, None], gamma)
    rows = x.shape[0] + 16  # additions, instead of the 256 + 16 of one copy
    R.assert_within(dgamma, n * dg, n * bound[1] * rows / (256 + 16), "dgamma")
    R.assert_within(dbeta, n * db, n * bound[2] * rows / (256 + 16), "dbeta")
    del y, q, dx
    y, mean, rstd = ops.layer_norm_fwd_train(x, gamma, beta, EPS)
    assert torch.equal(y[-256:], y0) and torch.equal(rstd[-256:], r0)
    dx, _, _ = ops.layer_norm_bwd(dy, x, gamma, mean, rstd)
    assert torch.equal(dx[-256:], dx[:256])
