"""8-bit blocks and layer norm for training without a GPU: refusals of the C entry points and of the
bindings, shapes of the torch ops, and the plain forms that the GPU tests compare with."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import fp8_reference as R
import hc

FAKE = C.c_void_p(0x1000)  # never dereferenced: every call below fails before device work
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib(hc_lib):
    return hc_lib.load()


@pytest.fixture(scope="module")
def ops(hc_lib):
    if not hc_lib.TORCH_OPS_PATH.exists():
        import build

        build.build_torch()
    return hc_lib.load_torch_ops()


def calls(lib):
    """name -> (call(tiling, dtype, pointers), pointer count, a valid tiling, an empty one)."""
    blk, mm = hc.Fp8BlockTiling, hc.MatmulFp8BlockTiling
    act, ln = hc.ActivationGeluSiluCkptTiling, hc.LayerNormTiling

    def plain(name):
        return lambda t, dt, p: getattr(lib, name)(*p, C.byref(t) if t is not None else None, dt, None)

    def matmul(t, dt, p):
        return lib.hc_matmul_fp8_block_launch(*p[:4], None, p[4], C.byref(t) if t is not None else None, dt, None)

    def ln_bwd(name):
        return lambda t, dt, p: getattr(lib, name)(*p, 1 << 30, C.byref(t) if t is not None else None, dt, None)

    def ln_fwd(t, dt, p):
        return lib.hc_layer_norm_fwd_train_launch(*p[:4], FAKE, p[4], None, None, C.byref(t) if t is not None else None,
                                                  dt, None)

    return {
        "quantize": (plain("hc_quantize_fp8_block_launch"), 3, blk(4, 128, 1), blk(0, 128, 1)),
        "dequantize": (plain("hc_dequantize_fp8_block_launch"), 3, blk(4, 128, 128), blk(4, 0, 128)),
        "act": (plain("hc_activation_gelu_silu_ckpt_launch"), 4, act(4, 128, 0), act(4, 0, 0)),
        "act_bwd": (plain("hc_activation_gelu_silu_ckpt_bwd_launch"), 4, act(4, 128, 1), act(0, 4, 1)),
        "matmul": (matmul, 5, mm(4, 128, 16), mm(0, 128, 16)),
        "ln": (ln_fwd, 5, ln(4, 128, 0, 1e-5), ln(0, 128, 0, 1e-5)),
        "ln_bwd": (ln_bwd("hc_layer_norm_bwd_launch"), 9, ln(4, 128, 0, 0.0), None),
        "ln_ckpt_bwd": (ln_bwd("hc_layer_norm_ckpt_bwd_launch"), 9, ln(4, 128, 0, 0.0), None),
    }


@pytest.mark.parametrize("name", ["quantize", "dequantize", "act", "act_bwd", "matmul", "ln", "ln_bwd", "ln_ckpt_bwd"])
def test_refusals(lib, name):
    call, n, good, empty = calls(lib)[name]
    ptrs = [FAKE] * n
    assert call(None, 2, ptrs) == hc.HC_ERR_INVALID
    for dt in (-1, 3, 4, 5, 9):
        assert call(good, dt, ptrs) == hc.HC_ERR_UNSUPPORTED, dt
    for i in range(n):
        some = list(ptrs)
        some[i] = None
        assert call(good, 2, some) == hc.HC_ERR_INVALID, i
        assert lib.hc_last_error_string()
    if empty is not None:
        assert call(empty, 2, [None] * n) == hc.HC_OK
    big = type(good)(*[getattr(good, f) for f, _ in good._fields_])
    setattr(big, good._fields_[0][0], 0x80000000)
    assert call(big, 2, ptrs) == hc.HC_ERR_UNSUPPORTED
    assert lib.hc_set_fault(b"launch:1") == hc.HC_OK
    try:
        assert call(good, 2, ptrs) == hc.HC_ERR_INJECTED
    finally:
        lib.hc_set_fault(None)


def test_refusals_of_values(lib):
    c = calls(lib)
    assert c["quantize"][0](hc.Fp8BlockTiling(4, 128, 64), 2, [FAKE] * 3) == hc.HC_ERR_INVALID
    assert b"blockRows" in lib.hc_last_error_string()
    assert c["act"][0](hc.ActivationGeluSiluCkptTiling(4, 128, 2), 2, [FAKE] * 4) == hc.HC_ERR_INVALID
    assert c["matmul"][0](hc.MatmulFp8BlockTiling(4, 0, 16), 2, [FAKE] * 5) == hc.HC_ERR_INVALID
    for eps in (-1e-5, float("nan"), float("inf")):
        assert c["ln"][0](hc.LayerNormTiling(4, 128, 0, eps), 2, [FAKE] * 5) == hc.HC_ERR_INVALID
    for name in ("ln", "ln_bwd", "ln_ckpt_bwd"):
        assert c[name][0](hc.LayerNormTiling(4, 0, 0, 1e-5), 2, [FAKE] * c[name][1]) == hc.HC_ERR_INVALID
    t = hc.LayerNormTiling(4, 128, 0, 1e-5)
    one = (FAKE, FAKE, FAKE, FAKE, None, FAKE)
    assert lib.hc_layer_norm_fwd_train_launch(*one, FAKE, None, C.byref(t), 2, None) == hc.HC_ERR_INVALID
    assert lib.hc_layer_norm_fwd_train_launch(*one, None, FAKE, C.byref(t), 2, None) == hc.HC_ERR_INVALID
    assert b"together" in lib.hc_last_error_string()


def test_layer_norm_workspace(lib):
    size = C.c_size_t()
    sizes = []
    for rows in (0, 1, 100, 100000):
        t = hc.LayerNormTiling(rows, 1000, 0, 0.0)
        assert lib.hc_layer_norm_bwd_workspace_size(C.byref(t), 2, C.byref(size)) == hc.HC_OK
        sizes.append(size.value)
    assert sizes == sorted(sizes) and sizes[1] >= 2 * 1000 * 4
    assert lib.hc_layer_norm_bwd_workspace_size(None, 2, C.byref(size)) == hc.HC_ERR_INVALID
    assert lib.hc_layer_norm_bwd_workspace_size(C.byref(t), 2, None) == hc.HC_ERR_INVALID
    assert lib.hc_layer_norm_bwd_workspace_size(C.byref(t), 9, C.byref(size)) == hc.HC_ERR_UNSUPPORTED
    lib.hc_layer_norm_bwd_workspace_size(C.byref(t), 2, C.byref(size))
    for ws, n in ((FAKE, size.value - 1), (C.c_void_p(0x1008), size.value)):  # too small; off a 16-byte boundary
        assert lib.hc_layer_norm_bwd_launch(*[FAKE] * 8, ws, n, C.byref(t), 2, None) == hc.HC_ERR_INVALID
        assert b"workspace" in lib.hc_last_error_string()


def test_bindings_refuse(hc_lib):
    x = torch.zeros(4, 128)
    q, s = torch.zeros(4, 128).to(F8), torch.ones(4, 1)
    for f in (lambda: hc.quantize_fp8_block(x), lambda: hc.dequantize_fp8_block(q, s, torch.float32),
              lambda: hc.activation_gelu_silu_ckpt(x, "gelu"), lambda: hc.activation_gelu_silu_ckpt(x, "relu"),
              lambda: hc.activation_gelu_silu_ckpt_bwd(x, q, s, "gelu"),
              lambda: hc.activation_gelu_silu_ckpt_bwd(x, x, s, "gelu"),
              lambda: hc.activation_gelu_silu_ckpt_bwd(x, q, torch.ones(4, 2), "gelu"),
              lambda: hc.matmul_fp8_block(q, s, torch.zeros(3, 64).to(F8), s),
              lambda: hc.matmul_fp8_block(q, torch.ones(4, 2), q, torch.ones(1, 1)),
              lambda: hc.matmul_fp8_block(q, s, q, s),
              lambda: hc.layer_norm_bwd(x, x.half(), torch.ones(128), s[:, 0], s[:, 0]),
              lambda: hc.layer_norm_bwd(x, x, torch.ones(127), s[:, 0], s[:, 0]),
              lambda: hc.layer_norm_fwd_train(x, torch.ones(128).half(), torch.ones(128), 1e-5),
              lambda: hc.quantize_fp8_block(x, 128)):
        with pytest.raises(hc.HcError):
            f()


OPS = ("quantize_fp8_block", "dequantize_fp8_block", "matmul_fp8_block", "activation_gelu_silu_ckpt",
       "activation_gelu_silu_ckpt_bwd", "layer_norm_fwd_train", "layer_norm_bwd", "layer_norm_ckpt", "layer_norm_ckpt_bwd")


def test_torch_ops_shapes(ops):
    for name in OPS:
        assert getattr(ops, name).default._schema.name == f"hc::{name}"
    m = {"device": "meta"}
    x, g = torch.empty(2, 5, 300, dtype=torch.bfloat16, **m), torch.empty(300, **m)
    q, s = ops.quantize_fp8_block(x)
    assert q.shape == x.shape and q.dtype == F8 and s.shape == (2, 5, 3) and s.dtype == torch.float32
    w_q, w_s = ops.quantize_fp8_block(torch.empty(260, 300, **m), 128)
    assert w_s.shape == (3, 3)
    assert ops.dequantize_fp8_block(q, s, torch.float16).dtype == torch.float16
    a_q, a_s = ops.quantize_fp8_block(torch.empty(7, 300, **m))
    c = ops.matmul_fp8_block(a_q, a_s, w_q, w_s, None, torch.float16)
    assert c.shape == (7, 260) and c.dtype == torch.float16
    y, q, s = ops.activation_gelu_silu_ckpt(x, 0)
    assert y.shape == x.shape and ops.activation_gelu_silu_ckpt_bwd(y, q, s, 0).shape == x.shape
    y, mean, rstd = ops.layer_norm_fwd_train(x, g, g, 1e-5)
    assert y.shape == x.shape and mean.shape == rstd.shape == (2, 5)
    y, q, s, rstd = ops.layer_norm_ckpt(x, g, g, 1e-5)
    assert q.dtype == F8 and s.shape == (2, 5, 3)
    for grads in (ops.layer_norm_bwd(y, x, g, mean, rstd), ops.layer_norm_ckpt_bwd(y, q, s, g, rstd)):
        assert [t.shape for t in grads] == [x.shape, g.shape, g.shape]
    with pytest.raises(RuntimeError, match="block_rows"):
        ops.quantize_fp8_block(x, 128)  # tiles are for 2-D weights


def test_torch_ops_have_no_cpu_kernel(ops):
    x, g = torch.ones(4, 128), torch.ones(128)
    for f in (lambda: ops.quantize_fp8_block(x), lambda: ops.activation_gelu_silu_ckpt(x, 0),
              lambda: ops.layer_norm_fwd_train(x, g, g, 1e-5),
              lambda: ops.layer_norm_ckpt(x.requires_grad_(True), g, g, 1e-5)):
        with pytest.raises(NotImplementedError):
            f()


def test_plain_gradients_against_autograd():
    """The 64-bit gradient formulas that the GPU tests use, against torch's differentiation of the forwards."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(7, 33, generator=g, dtype=torch.float64, requires_grad=True)
    gamma, beta = (torch.randn(33, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    dy = torch.randn(7, 33, generator=g, dtype=torch.float64)
    y, xh, _, rstd = R.layer_norm(x, gamma, beta, 1e-5)
    want = torch.autograd.grad(y, (x, gamma, beta), dy)
    for a, b in zip(R.layer_norm_grads(dy, xh.detach(), rstd.detach(), gamma.detach()), want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    for kind in (0, 1):
        y, slope, _ = R.act(x * 3, kind)
        (dx,) = torch.autograd.grad(y, x, dy)
        assert torch.allclose(dx, 3 * dy * slope, rtol=1e-12, atol=1e-12)


def test_plain_quantize_format():
    x = torch.tensor([[0.0, 448.0, -1.0, 3.0]])
    q, s = R.quantize_rows(x)
    assert float(s) == 1.0 and torch.equal(q, x)
    assert float(R.quantize_rows(torch.zeros(1, 4))[1]) == float(torch.tensor(R.FLOOR) / 448)
    q, s = R.quantize_rows(torch.tensor([[1.0, float("nan")]]))
    assert bool(R.values(q, s).isnan().all())
    q, s = R.quantize_rows(torch.tensor([[1.0, float("inf")]]))
    assert bool(R.values(q, s).isnan().all())


@pytest.mark.parametrize("K", [33, 128])
def test_failed_launch_leaves_the_path(lib, K):
    """hc_matmul_fp8_block_last_path() tells of successful launches; a thread of its own starts with none.  Without a
    GPU the launch fails; with one, an output type that the product does not have is refused before it."""
    import threading

    seen = []

    def call():
        t = hc.MatmulFp8BlockTiling(4, K, 16)
        dtype = 9 if torch.cuda.is_available() else 2
        seen.append(lib.hc_matmul_fp8_block_launch(FAKE, FAKE, FAKE, FAKE, None, FAKE, C.byref(t), dtype, None))
        seen.append(lib.hc_matmul_fp8_block_last_path())

    thread = threading.Thread(target=call)
    thread.start()
    thread.join()
    assert seen[0] != hc.HC_OK and seen[1] == 0
