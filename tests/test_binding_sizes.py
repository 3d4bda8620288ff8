"""Sizes that the C records' 32-bit fields cannot hold are refused by the bindings, not cut off."""
from __future__ import annotations

import pytest
import torch

import hc

F8, BF = torch.float8_e4m3fn, torch.bfloat16
BIG = 2**32 + 3  # ctypes would make 3 of it


def calls():
    def t(*shape, dtype=BF):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    f32 = torch.float32
    x, q, s, g = t(BIG, 1), t(BIG, 1, dtype=F8), t(BIG, 1, dtype=f32), t(1, dtype=f32)
    stat = t(BIG, dtype=f32)
    return {
        "quantize": lambda: hc.quantize_fp8_block(x),
        "quantize columns": lambda: hc.quantize_fp8_block(t(1, BIG)),
        "quantize more dimensions": lambda: hc.quantize_fp8_block(t(2**16, 2**16 + 1, 1)),
        "dequantize": lambda: hc.dequantize_fp8_block(q, s, BF),
        "act": lambda: hc.activation_gelu_silu_ckpt(x, "gelu"),
        "act_bwd": lambda: hc.activation_gelu_silu_ckpt_bwd(x, q, s, "silu"),
        "matmul M": lambda: hc.matmul_fp8_block(q, s, t(4, 1, dtype=F8), t(1, 1, dtype=f32)),
        "matmul N": lambda: hc.matmul_fp8_block(t(4, 1, dtype=F8), t(4, 1, dtype=f32), q, t(-(-BIG // 128), 1, dtype=f32)),
        "matmul K": lambda: hc.matmul_fp8_block(t(1, BIG, dtype=F8), t(1, -(-BIG // 128), dtype=f32), t(1, BIG, dtype=F8),
                                                t(1, -(-BIG // 128), dtype=f32)),
        "ln": lambda: hc.layer_norm_fwd_train(x, g, g, 1e-5),
        "ln_ckpt": lambda: hc.layer_norm_ckpt(x, g, g, 1e-5),
        "ln_bwd": lambda: hc.layer_norm_bwd(x, x, g, stat, stat),
        "ln_ckpt_bwd": lambda: hc.layer_norm_ckpt_bwd(x, q, s, g, stat),
    }


@pytest.mark.parametrize("name", ["quantize", "quantize columns", "quantize more dimensions", "dequantize", "act", "act_bwd",
                                  "matmul M", "matmul N", "matmul K", "ln", "ln_ckpt", "ln_bwd", "ln_ckpt_bwd"])
def test_sizes_past_32_bits(hc_lib, monkeypatch, name):
    from torch._subclasses import FakeTensorMode

    class Launched(Exception):
        pass

    class Lib:
        def __getattr__(self, entry):
            if entry.endswith("_size"):
                return lambda *args: hc.HC_OK

            def launch(*args):
                raise Launched(entry)

            return launch

    monkeypatch.setattr(hc, "load", Lib)
    monkeypatch.setattr(hc, "_ptr", lambda t: None)
    monkeypatch.setattr(hc, "_stream", lambda s: None)
    monkeypatch.setattr(hc, "_on", lambda x: torch.no_grad())
    with FakeTensorMode():
        with pytest.raises(hc.HcError, match="2\\^31") as e:
            calls()[name]()
    assert e.value.status == hc.HC_ERR_UNSUPPORTED
