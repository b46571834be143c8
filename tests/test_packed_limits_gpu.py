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


def test_more_rows_of_x_than_a_grid_takes(kernels):
    """The second axis of a grid ends at 65,535 blocks of 16 rows: more 32-bit rows than that, and bfloat16 ones off 16 bytes."""
    g = gen(51)
    w = matrix(g, 8, 9, BF16)
    packed, pair = kernels.pack_weights(w, 32), kernels.pack_gate_up(w, w.flip(0).contiguous(), 32)
    values, other = packed_values(w, 32), packed_values(w.flip(0), 32)
    m = 65535 * 16 + 1000
    for dtype in (F32, BF16):
        x = torch.randn(m, 9, generator=g, device=DEV).to(dtype)
        out = torch.full((m, 8), math.nan, device=DEV)
        add = torch.randn(m, 8, generator=g, device=DEV)
        kernels.linear(x, packed, out, residual=add)
        product = x.double() @ values.t()
        want = product + add.double()
        close(out, want, off_by(x, values, 32, F32, product) + want.abs() * 2.0 ** -23)
        gated = torch.full((m, 8), math.nan, device=DEV)
        kernels.linear_swiglu(x, pair, gated)
        up = x.double() @ other.t()
        want = product * torch.sigmoid(product) * up
        # (as test_gated_pairs has it)
        a, b = off_by(x, values, 32, F32, product), off_by(x, other, 32, F32, up)
        bound = (1.13 * a + 8 * 2.0 ** -24 * product.abs()) * (up.abs() + b) + product.abs() * b + want.abs() * 2.0 ** -24 + 1e-30
        close(gated, want, bound)
    kernels.check_error_word()


@pytest.mark.parametrize("m", [5, 40, 300])
def test_rows_of_x_that_overlap(kernels, m):
    """One row for all (an expanded tensor), and rows that begin within the row before: what no tile copy is described for."""
    g = gen(52)
    w = matrix(g, 200, 256, BF16)
    packed, values = kernels.pack_weights(w, 64), packed_values(w, 64)
    line = torch.randn(8 * m + 256, generator=g, device=DEV).to(BF16)
    for x in (line[:256].expand(m, 256), line.as_strided((m, 256), (8, 1)), line.as_strided((m, 256), (3, 1))):
        out = torch.empty(m, 200, device=DEV)
        kernels.linear(x, packed, out)
        want = x.double() @ values.t()
        close(out, want, off_by(x, values, 64, F32, want))
    kernels.check_error_word()
