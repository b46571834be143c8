"""Matrices in 4 bits on the device: the calls at the edge of what the operators take.

Comparisons are with the definition in 64 bits.  What a product of few rows may be off by is ``off_by`` of
test_packed_weights_gpu.py; where whole numbers make every sum exact, bits have to be equal.
"""
import math

import pytest
import torch

from test_packed_weights_gpu import BF16, DEV, F32, close, gen, matrix, off_by, packed_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kernels():
    from chibillm_b200.kernels.ops import CudaKernels
    return CudaKernels(torch.device(DEV))


def test_a_pair_whose_second_matrix_is_elsewhere_is_refused(kernels):
    from chibillm_b200.kernels.ops import KernelError
    w = torch.zeros(32, 64, dtype=BF16, device=DEV)
    for gate, up in ((w, w.cpu()), (w.cpu(), w)):
        with pytest.raises(KernelError):
            kernels.pack_gate_up(gate, up, 32)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_values_read_back_are_the_next_products_matrix(kernels, m):
    """bfloat16 products fetch their matrix early: not before it has been written."""
    g = gen(50)
    x = torch.randn(m, 512, generator=g, device=DEV).to(BF16)
    matrices = [kernels.pack_weights(matrix(g, 2048, 512, BF16), 64) for _ in range(4)]
    values, out = torch.empty(2048, 512, dtype=BF16, device=DEV), torch.empty(m, 2048, device=DEV)
    want = []
    for packed in matrices:
        kernels.unpack_weights(packed, values)
        torch.cuda.synchronize()
        kernels.linear(x, values, out)
        want.append(out.clone())
    for turn in range(40):
        kernels.unpack_weights(matrices[turn % 4], values)
        kernels.linear(x, values, out)
        got = out.clone()
        assert torch.equal(got, want[turn % 4]), turn
