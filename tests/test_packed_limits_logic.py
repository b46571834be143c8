"""Matrices in 4 bits without a GPU: what must be refused or looked at before a kernel runs."""
import pytest
import torch

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
