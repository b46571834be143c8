"""Matrices in 4 bits without a GPU: what must be refused or looked at before a kernel runs."""
import os
import re

import pytest
import torch

import chibillm_b200.csrc
from chibillm_b200.kernels.ops import CudaKernels, KernelError


def bare_kernels():
    """Kernels without a device: what stands before a launch."""
    k = CudaKernels.__new__(CudaKernels)
    k._device_index = 0
    return k


def test_both_matrices_of_a_pair_are_looked_at(monkeypatch):
    """Each tensor whose address a kernel gets has to be on the kernels' device."""
    k, seen = bare_kernels(), []
    monkeypatch.setattr(k, "_on_this_device", lambda what, *tensors: seen.extend(tensors))
    monkeypatch.setattr(k, "_packed_room", lambda *sizes: (_ for _ in ()).throw(KernelError("no room")))
    gate, up = torch.zeros(32, 64), torch.zeros(32, 64)
    with pytest.raises(KernelError, match="no room"):
        k.pack_gate_up(gate, up, 32)
    assert any(t is gate for t in seen) and any(t is up for t in seen)


def kernel_bodies(name):
    with open(os.path.join(os.path.dirname(chibillm_b200.csrc.__file__), name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    for m in re.finditer(r"__global__ void (?:__launch_bounds__\([^)]*\)\s*)?(\w+)\([^{;]*\)\n\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at]


def test_kernels_that_write_a_matrix_let_no_product_start_early():
    """bfloat16 products fetch their matrix before the kernel ahead of them has ended, so a kernel that makes one (its values read
    back are one, too) neither triggers the next launch nor ends with stores that a tile copy might miss."""
    bodies = dict(kernel_bodies("packed_weights.cu"))
    writers = ["pack_kernel", "pack_codes_kernel", "unpack_kernel"]
    assert set(writers) < set(bodies)
    for name in writers:
        assert "pdl_enter()" not in bodies[name] and "pdl_trigger" not in bodies[name], name
        assert bodies[name].lstrip().startswith("pdl_wait_now();") and "packed_done();" in bodies[name], name
