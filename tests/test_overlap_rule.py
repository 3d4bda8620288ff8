"""Kernels that are set up while the one before them still runs (overlap.cuh) must not read their inputs through the
read-only path, nor with a load that the compiler may move in front of the wait."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "ascend-npu-harness_b200" / "csrc"
FILES = sorted(f for f in CSRC.glob("*.cu") if "launch_overlapped(" in f.read_text())


def code(path):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def test_files_are_found():
    assert {f.name for f in FILES} >= {"ops_fp8_block.cu", "ops_layer_norm_train.cu", "ops_matmul_fp8.cu"}


@pytest.mark.parametrize("path", FILES, ids=lambda f: f.name)
def test_inputs_are_read_coherently_behind_the_wait(path):
    text = code(path)
    for load in ("__ldg", "__ldcs", "__ldcg", "__ldca", "__ldlu", "ld_stream", "ld_cached", "ld.global.nc"):
        assert not re.search(rf"{re.escape(load)}\s*\(" if load[0] != "l" or "_" in load else re.escape(load), text), load
    # const and __restrict__ together let the compiler choose the read-only path
    assert not re.search(r"const\s+[\w:]+\s*\*\s*(const\s+)?__restrict__", text)


@pytest.mark.parametrize("path", FILES, ids=lambda f: f.name)
def test_every_overlapped_kernel_waits(path):
    text = code(path)
    kernels = re.findall(r"__global__[^;{]*?(\w+_kernel)\s*\(", text)
    assert kernels
    for name in kernels:
        body = text[re.search(rf"__global__[^;{{]*?\b{name}\s*\(", text).end():]
        assert "overlap_begin();" in body.split("__global__")[0], name


def test_the_wait_is_a_memory_barrier_for_the_compiler():
    text = code(CSRC / "overlap.cuh")
    assert re.search(r'asm volatile\("griddepcontrol\.wait;" ::: "memory"\)', text)
    for load in re.findall(r'asm( volatile)?\s*\(\s*"ld\.', text):
        assert load.strip() == "volatile"
