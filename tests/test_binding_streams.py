"""The bindings' `stream` argument: buffers that a call allocates for itself have to outlive its kernels on that stream."""
from __future__ import annotations

import pytest
import torch

import hc

F8 = torch.float8_e4m3fn


class Launches:
    """The library with its layer norm backward replaced by a note of the workspace and stream it was given."""

    def __init__(self, lib):
        self.lib, self.seen = lib, []

    def __getattr__(self, name):
        if name not in ("hc_layer_norm_bwd_launch", "hc_layer_norm_ckpt_bwd_launch"):
            return getattr(self.lib, name)

        def launch(*args):
            self.seen.append((args[8], args[12]))  # workspace, stream
            return hc.HC_OK

        return launch


def backward(ckpt, stream):
    dy, gamma, rstd = torch.zeros(40, 256), torch.ones(256), torch.ones(40)
    if ckpt:
        return hc.layer_norm_ckpt_bwd(dy, torch.zeros(40, 256).to(F8), torch.ones(40, 2), gamma, rstd, stream=stream)
    return hc.layer_norm_bwd(dy, dy, gamma, rstd, rstd, stream=stream)


@pytest.mark.parametrize("ckpt", [False, True])
@pytest.mark.parametrize("stream", [None, 0, 0x5000])
def test_workspace_is_kept_for_the_stream(hc_lib, monkeypatch, ckpt, stream):
    lib, recorded = Launches(hc_lib.load()), []
    monkeypatch.setattr(hc, "load", lambda: lib)
    monkeypatch.setattr(hc, "_ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(hc, "_stream", lambda s: s)
    monkeypatch.setattr(hc, "_on", lambda x: torch.no_grad())
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda s, device=None: ("stream", s))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: recorded.append((t.data_ptr(), s)))
    backward(ckpt, stream)
    [(workspace, launched_on)] = lib.seen
    assert launched_on == stream
    assert recorded == ([] if stream is None else [(workspace, ("stream", stream))])


@pytest.mark.gpu
@pytest.mark.parametrize("ckpt", [False, True])
def test_backward_on_a_busy_stream(cuda, ckpt):
    """The side stream starts late; meanwhile tensors of the workspace's size are made and filled on the current one."""
    rows, H = 3000, 1024
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(rows, H, generator=g).cuda() for _ in range(2))
    gamma = torch.ones(H, device="cuda")
    y, q, scale, rstd = hc.layer_norm_ckpt(x, gamma, gamma, 1e-5)
    _, mean, rstd = hc.layer_norm_fwd_train(x, gamma, gamma, 1e-5)

    def call(stream=None):
        return hc.layer_norm_ckpt_bwd(dy, q, scale, gamma, rstd, stream) if ckpt else hc.layer_norm_bwd(dy, x, gamma, mean, rstd, stream)

    want = call()
    torch.cuda.synchronize()
    size = hc._sz()
    t = hc.LayerNormTiling(rows, H, 0, 0.0)
    hc.check(hc.load().hc_layer_norm_bwd_workspace_size(hc.C.byref(t), hc.DT_F32, hc.C.byref(size)))
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # some 10 ms
        got = call(side.cuda_stream)
        others = [torch.full((size.value // 4,), 7.0, device="cuda") for _ in range(8)]
        torch.cuda.current_stream().synchronize()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(bool((o == 7.0).all()) for o in others)
    got = call(0)  # the default stream by its handle
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
