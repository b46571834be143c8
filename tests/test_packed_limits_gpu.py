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


def whole_numbers(g, m, n, k, group, x_dtype):
    """Codes, scales that are powers of two and x of small whole numbers: every sum is exact in 32 bits in any order
    (k * 8 * 15 * 2^3 < 2^24 steps)."""
    codes = torch.randint(-8, 8, (n, k), generator=g, device=DEV, dtype=torch.int8)
    scales = (2.0 ** torch.randint(-3, 1, (n, -(-k // group)), generator=g, device=DEV)).to(BF16)
    x = torch.randint(-15, 16, (m, k), generator=g, device=DEV).to(x_dtype)
    return codes, scales, x


def values_of(codes, scales, group):
    return codes.double() * scales.double().repeat_interleave(group, 1)[:, :codes.shape[1]]


@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 70, 200), (3, 2048, 1024), (8, 33, 4096), (11, 300, 1021), (16, 64, 2048), (1, 32, 8192),
                                   (20, 130, 2048), (90, 64, 512), (300, 2050, 264)])
def test_numbers_of_all_sizes_in_one_row(kernels, m, n, k, group, x_dtype):
    """A large number that meets only zeros leaves no trace, however small the others are."""
    g = gen(53 + m)
    codes, scales, x = whole_numbers(g, m, n, k, group, x_dtype)
    at = [0, k // 2, k - 1]
    codes[:, at] = 0
    packed = kernels.pack_codes(codes, scales, group)
    values = values_of(codes, scales, group)
    out = torch.empty(m, n, device=DEV)
    for small in (1.0, 2.0 ** -8, 2.0 ** -20, 2.0 ** -40, 2.0 ** -119):
        for large in (2.0 ** 9, 2.0 ** 20, 2.0 ** 50, 2.0 ** 126):
            rows = x * small
            rows[:, at] = large
            if m > 1:
                rows[1, at[1:]] = 0.0              # (a row of its own range)
            want = rows.double() @ values.t()
            kernels.linear(rows, packed, out)
            assert torch.equal(out.double(), want), (small, large)
    kernels.check_error_word()


@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 300, 4096), (4, 64, 20000), (16, 100, 1000)])
def test_rows_whose_sizes_run_from_the_smallest_to_the_largest(kernels, m, n, k, x_dtype):
    """Whatever part of a row a column of the matrix sees, its numbers have kept their bits: bfloat16 all of them, 32-bit ones all
    but 2^-23 of themselves, and 2^-16 where they are below 2^-16 of the row's largest (a float16's last half step, 2^-25,
    against numbers from 2^-9 on, multiplied so that the row's largest is 2^14 ... 2^15; smaller numbers are added apart)."""
    g = gen(54 + m)
    x = torch.randn(m, k, generator=g, device=DEV, dtype=torch.float64) * 2.0 ** torch.linspace(-100, 100, k, device=DEV, dtype=torch.float64)
    x = x.to(x_dtype)
    codes = torch.zeros(n, k, dtype=torch.int8, device=DEV)
    scales = torch.ones(n, -(-k // 32), dtype=BF16, device=DEV)
    start = torch.linspace(0, k - 8, n, device=DEV).long()
    for j in range(8):                             # row i of the matrix sees 8 neighbouring columns
        codes[torch.arange(n, device=DEV), start + j] = torch.randint(1, 8, (n,), generator=g, device=DEV, dtype=torch.int8)
    packed, values = kernels.pack_codes(codes, scales, 32), values_of(codes, scales, 32)
    out = torch.empty(m, n, device=DEV)
    kernels.linear(x, packed, out)
    want = x.double() @ values.t()
    own = (x.double().abs() @ values.t()) * (2.0 ** -16 if x_dtype == F32 else 0.0)
    close(out, want, off_by(x, values, 32, F32, want) + own)


def rows_beyond_32_bits(g, m, n, k, group, x_dtype):
    """(x, codes, scales): products whose sums are whole numbers, exact in 32 bits, on a way that passes 2^128.  Rows of x in turn:
    tiny ones that meet huge scales, huge ones that meet tiny scales, huge ones whose terms cancel."""
    codes = torch.randint(1, 8, (n, k), generator=g, device=DEV, dtype=torch.int8)
    codes[:, 1::2] = -codes[:, 0:-1:2] if k % 2 == 0 else torch.cat([-codes[:, 0:-1:2]], 1)[:, :codes[:, 1::2].shape[1]]
    codes[:, :4] = 7
    groups = -(-k // group)
    scales = torch.empty(n, groups, dtype=BF16, device=DEV)
    scales[0::2], scales[1::2] = 2.0 ** 110, 2.0 ** -100
    x = torch.zeros(m, k, device=DEV)
    x[0::3, :4] = 2.0 ** -104                     # 28 * 2^6 with the first scale, as multiplied 2^14 * 28 * 2^110
    x[1::3, :4] = 2.0 ** 120                      # 28 * 2^20 with the second
    x[2::3] = 2.0 ** 122                          # neighbours cancel: 28 * 2^22 and less with the second
    return x.to(x_dtype), codes, scales


@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 40, 64), (3, 70, 300), (7, 2048, 1024), (16, 33, 2048), (12, 64, 30000), (17, 40, 128), (20, 2048, 1024),
                                   (90, 130, 2048), (300, 200, 72), (500, 4128, 512)])
def test_sums_whose_way_passes_32_bits(kernels, m, n, k, group, x_dtype):
    g = gen(60 + m)
    x, codes, scales = rows_beyond_32_bits(g, m, n, k, group, x_dtype)
    packed, values = kernels.pack_codes(codes, scales, group), values_of(codes, scales, group)
    out = torch.empty(m, n, device=DEV)
    for rows in (x, x.flip(0).contiguous()):
        kernels.linear(rows, packed, out)
        want = (rows.double() @ values.t()).float()        # (what is beyond 2^128 is infinite)
        assert want.isfinite().any() and torch.equal(out, want)
    # what is no number in x stays what it is
    x[0, k - 1] = math.inf
    kernels.linear(x, packed, out)
    want = (x.double() @ values.t()).float()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(0.0), want.nan_to_num(0.0))
    # a pair: the gate's sum on such a way, up's plain
    ones = torch.zeros(n, k, dtype=torch.int8, device=DEV)
    ones[:, 0] = 1
    x, _, _ = rows_beyond_32_bits(g, m, n, k, group, x_dtype)
    pair = kernels.pack_codes(codes, scales, group, ones, torch.full_like(scales, 2.0 ** 100))
    gate, up = (x.double() @ values.t()), x[:, :1].double() * 2.0 ** 100
    want = gate * torch.sigmoid(gate) * up
    gated = torch.empty(m, n, device=DEV)
    kernels.linear_swiglu(x, pair, gated)
    fits = (gate.abs() < 2.0 ** 127) & (up.abs() < 2.0 ** 127) & (want.abs() < 2.0 ** 127)
    assert fits.any()
    # (expf and the division are good to 2 half steps each, the product to one; gate and up are exact)
    assert ((gated.double() - want).abs() <= want.abs() * 8 * 2.0 ** -24 + 2.0 ** -149)[fits].all()
    kernels.check_error_word()


@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m,n,k", [(1, 151936, 256), (1, 128, 32768), (2, 64, 65536), (16, 64, 20000), (9, 40, 65531), (40, 64, 20000),
                                   (300, 200, 4104), (1, 6144, 4096), (24, 6144, 4096), (70, 129, 1)])
def test_no_element_of_a_long_row_hides(kernels, m, n, k, group, x_dtype):
    """Whole numbers whose sums are exact (65,536 * 8 * 4 * 2 < 2^24 steps): an element that is dropped, taken twice or swapped with
    another shows, wherever it is."""
    g = gen(70 + m)
    codes = torch.randint(-8, 8, (n, k), generator=g, device=DEV, dtype=torch.int8)
    scales = (2.0 ** torch.randint(-1, 1, (n, -(-k // group)), generator=g, device=DEV)).to(BF16)
    x = torch.randint(-4, 5, (m, k), generator=g, device=DEV).to(x_dtype)
    out = torch.empty(m, n, device=DEV)
    kernels.linear(x, kernels.pack_codes(codes, scales, group), out)
    for at in range(0, n, 8192):
        assert torch.equal(out[:, at:at + 8192].double(), x.double() @ values_of(codes[at:at + 8192], scales[at:at + 8192], group).t())
    kernels.check_error_word()


@pytest.mark.parametrize("kind", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 70, 512), (5, 2730, 1024), (12, 33, 2048), (16, 64, 4096), (17, 65, 512), (60, 300, 1024), (200, 1000, 136)])
def test_no_element_of_a_pair_hides(kernels, m, n, k, x_dtype, kind):
    """Gates from 32 on come out of both activations as they are, in 32 bits (exp(-32) is below half a step of 1): exact again.  The
    largest, 4,096 * 7 * 3 * 2, times the largest up, 7 * 3, is below 2^24 halves."""
    g = gen(71 + m)
    codes = torch.randint(0, 8, (n, k), generator=g, device=DEV, dtype=torch.int8)
    few = torch.zeros(n, k, dtype=torch.int8, device=DEV)
    few[torch.arange(n, device=DEV), torch.randint(0, k, (n,), generator=g, device=DEV)] = 7
    scales = torch.ones(n, -(-k // 64), dtype=BF16, device=DEV)
    x = torch.randint(1, 4, (m, k), generator=g, device=DEV).to(x_dtype)
    gate, up = x.double() @ codes.double().t(), x.double() @ few.double().t()
    assert gate.min() > 32 and (gate * up).max() < 2.0 ** 24
    out = torch.empty(m, n, device=DEV)
    kernels.linear_swiglu(x, kernels.pack_codes(codes, scales, 64, few, scales), out, kind=kind)
    assert torch.equal(out.double(), gate * up)
    kernels.check_error_word()


@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("m", [1, 9, 16, 17, 60, 400])
def test_a_residual_beside_bfloat16_outputs(kernels, m, x_dtype):
    """The residual is added to the 32-bit sums, before they are rounded."""
    g = gen(72 + m)
    w = matrix(g, 300, 512, BF16)
    packed, values = kernels.pack_weights(w, 64), packed_values(w, 64)
    x = torch.randn(m, 512, generator=g, device=DEV).to(x_dtype)
    add = torch.randn(m, 640, generator=g, device=DEV)[:, 5:305]
    out = torch.empty(m, 300, dtype=BF16, device=DEV)
    kernels.linear(x, packed, out, residual=add)
    want = x.double() @ values.t()
    bound = off_by(x, values, 64, F32, want) + want.abs() * 2.0 ** -24
    want = want + add.double()
    close(out, want, bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8)


@pytest.mark.parametrize("m", [1, 16, 17, 200])
@pytest.mark.parametrize("scale", [2.0 ** -113, 2.0 ** -100, 2.0 ** 100, 2.0 ** 116])
def test_weights_of_every_size(kernels, m, scale):
    """Scales from 2^-113 to 2^116 (weights of 10^-33 to 10^36) with x of about one, and with x that brings the product back to one."""
    g = gen(73 + m)
    codes, _, x = whole_numbers(g, m, 70, 600, 64, BF16)
    scales = torch.full((70, 10), scale, dtype=BF16, device=DEV)
    packed, values = kernels.pack_codes(codes, scales, 64), values_of(codes, scales, 64)
    out = torch.empty(m, 70, device=DEV)
    for rows in (x if scale < 1 else x * 2.0 ** -10, (x.float() / scale).to(BF16)):
        kernels.linear(rows, packed, out)
        # (600 * 8 * 15 < 2^17 steps of the product's own size: exact, its smallest step above 2^-149)
        assert torch.equal(out.double(), rows.double() @ values.t())
