"""Matrices in 4 bits without a GPU: what must be refused or looked at before a kernel runs."""
import os
import re

import pytest
import torch

import chibillm_b200.csrc
from chibillm_b200.engine.runner import make_runtime
from chibillm_b200.kernels.ops import CudaKernels, KernelError
from chibillm_b200.kernels.packed import PackedWeights
from packed_models import PackedReferenceKernels


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


@pytest.mark.parametrize("paired", [False, True])
def test_records_that_are_not_all_there_are_refused(monkeypatch, paired):
    """A kernel reads as many bytes as the matrix's sizes say."""
    k = bare_kernels()
    monkeypatch.setattr(k, "_on_this_device", lambda what, *tensors: None)
    k._current_device = lambda: (_ for _ in ()).throw(AssertionError("a launch"))
    k.error, k.lib, k.packed_few_rows_max = torch.zeros(1, dtype=torch.int32), None, 16
    rows, columns, group = 40, 200, 64
    need = PackedWeights.bytes_for(rows, columns, group, paired)
    whole = torch.zeros(need + 16, dtype=torch.uint8)
    whole = whole[-whole.data_ptr() % 16:][:need]
    x, out = torch.zeros(3, columns), torch.zeros(2 * rows if paired else rows, columns)
    for data in (whole[:-1], whole[:0], whole[1:], torch.zeros(need, dtype=torch.int8), torch.zeros(2 * need, dtype=torch.uint8)[::2],
                 torch.cat([whole, whole])[1:]):
        w = PackedWeights(data, rows, columns, group, paired)
        with pytest.raises(KernelError, match="bytes"):
            k.unpack_weights(w, out)
        with pytest.raises(KernelError, match="bytes"):
            k._packed_call(x, w, torch.zeros(3, rows), "silu" if paired else None, False, "linear")


@pytest.mark.parametrize("group", [64.0, True, "64", None, 0, 48, 256])
def test_groups_are_whole_numbers_of_the_list(monkeypatch, group):
    k = bare_kernels()
    monkeypatch.setattr(k, "_on_this_device", lambda what, *tensors: None)
    w = torch.zeros(32, 64)
    for call in (lambda: k.pack_weights(w, group), lambda: k.pack_gate_up(w, w, group),
                 lambda: k.pack_codes(w.to(torch.int8), torch.zeros(32, 1, dtype=torch.bfloat16), group)):
        with pytest.raises(KernelError, match="groups of"):
            call()
    if group is not None:
        with pytest.raises(ValueError, match="weight_group"):
            make_runtime("bfloat16", "cpu", kernels=PackedReferenceKernels(), weight_group=group)
