"""Order around kernels that are set up while the one before them runs: inputs written just before a call, overwritten just
after it, and captured graphs whose branches join in front of one."""
from __future__ import annotations

import pytest
import torch

import hc

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(cuda):
    return hc.load_torch_ops()


def calls(ops, x, dy, gamma, w):
    """Every overlapped kernel, each behind one that writes what it reads."""
    y, q, scale, rstd = ops.layer_norm_ckpt(x, gamma, gamma, 1e-5)
    z, mean, rstd2 = ops.layer_norm_fwd_train(y, gamma, gamma, 1e-5)
    a, aq, a_scale = ops.activation_gelu_silu_ckpt(z, 0)
    da = ops.activation_gelu_silu_ckpt_bwd(dy, aq, a_scale, 0)
    dz = ops.layer_norm_bwd(da, y, gamma, mean, rstd2)
    dx = ops.layer_norm_ckpt_bwd(dz[0], q, scale, gamma, rstd)
    xq, x_scale = ops.quantize_fp8_block(dx[0], 1)
    wq, w_scale = ops.quantize_fp8_block(w, 128)
    c = ops.matmul_fp8_block(xq, x_scale, wq, w_scale, None, torch.float32)
    return [a, da, *dz, *dx, x_scale, w_scale, c, ops.dequantize_fp8_block(xq, x_scale, torch.float32, 1),
            ops.dequantize_fp8_block(wq, w_scale, torch.float32, 128)]


def inputs(rows, cols, n, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(t).cuda() for s, t in
            (((rows, cols), torch.bfloat16), ((rows, cols), torch.bfloat16), ((cols,), torch.float32), ((n, cols), torch.bfloat16))]


@pytest.mark.parametrize("rows,cols,n", [(4, 256, 512), (300, 1001, 130), (4000, 2048, 512), (3, 9000, 200)])
def test_inputs_change_around_the_calls(ops, rows, cols, n):
    """All buffers are rewritten between two runs without a wait on the host; each run gives what it gives alone."""
    sets = [inputs(rows, cols, n, seed) for seed in range(3)]
    want = []
    for s in sets:
        want.append([t.clone() for t in calls(ops, *s)])
        torch.cuda.synchronize()
    live, got = [t.clone() for t in sets[0]], []
    for turn in range(12):
        for a, b in zip(live, sets[turn % 3]):
            a.copy_(b)
        got.append(calls(ops, *live))
        for a in live:
            a.fill_(float("nan"))
    for turn, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[turn % 3])), turn


@pytest.mark.parametrize("rows,cols,n", [(4, 256, 512), (500, 1024, 512)])
def test_captured_branches_join(ops, rows, cols, n):
    """Two streams of a capture meet in front of a product; copies and fills stand between overlapped kernels."""
    x, dy, gamma, w = inputs(rows, cols, n, 7)
    out = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)

    def step():
        main, side = torch.cuda.current_stream(), torch.cuda.Stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            wq, w_scale = ops.quantize_fp8_block(w, 128)
        out.copy_(x)
        y, _, _ = ops.layer_norm_fwd_train(out, gamma, gamma, 1e-5)
        out.zero_()
        xq, x_scale = ops.quantize_fp8_block(y, 1)
        main.wait_stream(side)
        for t in (wq, w_scale):
            t.record_stream(main)
        c = ops.matmul_fp8_block(xq, x_scale, wq, w_scale, None, torch.bfloat16)
        return [c, y, *ops.layer_norm_bwd(dy, y, gamma, x_scale[:, 0].contiguous(), x_scale[:, 0].contiguous())]

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        for a, b in zip((x, dy, gamma, w), inputs(rows, cols, n, 20 + seed)):
            a.copy_(b)
        graph.replay()
        kept = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(kept, step())), seed
