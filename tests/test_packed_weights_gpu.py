"""Matrices in 4 bits on the device: packing and reading back, products with few and many rows, gated pairs.

Everything is compared with the definition in 64 bits.  What a product may be off by, derived: whole numbers and bfloat16
make exact products.  A tensor-core instruction adds 16 products to its 32-bit sum, and each of the 17 terms may lose half
a step or a whole one (2^-23) of the largest: 17 * 2^-23 of the magnitudes added up, for every 16 columns of a group (three
times as many for 32-bit x, whose numbers are three parts).  The groups' sums are then multiplied and added in 32 bits: one
half step (2^-24) of the magnitudes for every group and every warp's sum.  The output's own rounding, half a step of its
type, comes on top.  (A single wrong element would be off by about 1 / columns of the magnitudes, a hundred times that.)
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def kernels():
    from chibillm_b200.kernels.ops import CudaKernels
    return CudaKernels(torch.device(DEV))


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def matrix(g, n, k, dtype, std=0.02):
    return (torch.randn(n, k, generator=g, device=DEV) * std).to(dtype)


def packed_values(w, group):
    """What packing makes of w, in 64 bits."""
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for at in range(0, w.shape[1], group):
        part = w[:, at:at + group].double()
        finite = torch.isfinite(part).all(dim=1, keepdim=True)
        part = torch.where(finite, part, 0.0)
        first = part.abs().argmax(dim=1, keepdim=True)
        scale = (part.gather(1, first) / -8).float().to(BF16).double()
        q = torch.where(scale == 0, 0.0, (part / torch.where(scale == 0, 1.0, scale)).round().clamp(-8, 7))
        out[:, at:at + group] = torch.where(finite, q * scale, math.nan)
    return out


def off_by(x, values, group, out_dtype, result):
    """The bound above for x @ values^T."""
    magnitudes = x.double().abs() @ values.abs().t()
    columns = x.shape[1]
    steps = math.ceil(min(group, columns) / 16) * (3 if x.dtype == F32 else 1)
    sums = math.ceil(columns / group) + 128
    return magnitudes * (17 * steps * 2.0 ** -23 + sums * 2.0 ** -24) + result.abs() * (torch.finfo(out_dtype).eps / 2) + 1e-300


def close(got, want, bound):
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


# ------------------------------------------------------------------ packing
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (33, 1000), (128, 31), (5, 4096), (300, 260)])
def test_packing_keeps_the_nearest_values(kernels, n, k, group, dtype):
    w = matrix(gen(n * k + group), n, k, dtype)
    packed = kernels.pack_weights(w, group)
    assert tuple(packed.shape) == (n, k) and packed.group == group
    out = torch.empty(n, k, device=DEV)
    kernels.unpack_weights(packed, out)
    want = packed_values(w, group)
    assert torch.equal(out.double(), want)
    rounded = torch.empty(n, k, dtype=BF16, device=DEV)
    kernels.unpack_weights(packed, rounded)
    assert torch.equal(rounded, want.float().to(BF16))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packing_ties_signs_and_what_is_no_number(kernels, dtype):
    w = torch.zeros(9, 64, device=DEV)
    w[0, :4] = torch.tensor([8.0, -8.0, 0.5, 1.5])              # the first of equals: scale -1; halves to even
    w[1, :4] = torch.tensor([-8.0, 8.0, 0.5, 1.5])              # scale 1: 8 is beyond 7
    w[2, :6] = torch.tensor([-8.0, 2.5, 3.5, -2.5, -7.5, 7.5])
    w[3] = 0.0                                                  # nothing
    w[4, 5] = math.inf
    w[5, 63] = math.nan
    w[6, 40] = -math.inf
    w[7, :3] = torch.tensor([1e-38, -2e-38, 5e-39])
    w[8, :2] = torch.tensor([3e38, -1e38])
    w = w.to(dtype)
    packed = kernels.pack_weights(w, 32)
    out = torch.empty(9, 64, device=DEV)
    kernels.unpack_weights(packed, out)
    want = packed_values(w, 32)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.double().nan_to_num(0.0), want.nan_to_num(0.0))
    assert out[0, :4].tolist() == [8.0, -7.0, 0.0, 2.0] and out[1, :4].tolist() == [-8.0, 7.0, 0.0, 2.0]
    assert not out[3].signbit().any()


def test_a_32_bit_quotient_that_rounds_onto_a_half(kernels):
    """w just beside 2.5 scales: the 32-bit quotient is 2.5 itself, the element is not."""
    scale = torch.tensor(1.0 + 2.0 ** -7, dtype=F32)
    w = torch.zeros(2, 32, device=DEV)
    w[:, 0] = (-8 * scale).item()
    w[0, 1] = torch.nextafter(2.5 * scale, torch.tensor(10.0)).item()
    w[1, 1] = torch.nextafter(2.5 * scale, torch.tensor(0.0)).item()
    w[:, 2] = (2.5 * scale).item()
    out = torch.empty(2, 32, device=DEV)
    kernels.unpack_weights(kernels.pack_weights(w, 32), out)
    assert torch.equal(out.double(), packed_values(w, 32))
    assert (out[:, 1] / scale.item()).tolist() == [3.0, 2.0] and (out[:, 2] / scale.item()).tolist() == [2.0, 2.0]


@pytest.mark.parametrize("n,k,group", [(8, 128, 64), (13, 200, 32), (70, 64, 128)])
def test_a_pair_and_given_codes(kernels, n, k, group):
    g = gen(n)
    gate, up = matrix(g, n, k, BF16), matrix(g, n, k, BF16, 0.05)
    out = torch.empty(2 * n, k, device=DEV)
    packed = kernels.pack_gate_up(gate, up, group)
    kernels.unpack_weights(packed, out)
    assert packed.paired and tuple(packed.shape) == (2 * n, k)
    assert torch.equal(out.double(), torch.cat([packed_values(gate, group), packed_values(up, group)]))
    groups = -(-k // group)
    q = [torch.randint(-8, 8, (n, k), generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
    s = [matrix(g, n, groups, BF16) for _ in range(2)]
    values = [a.double() * b.double().repeat_interleave(group, 1)[:, :k] for a, b in zip(q, s)]
    kernels.unpack_weights(kernels.pack_codes(q[0], s[0], group, q[1], s[1]), out)
    assert torch.equal(out.double(), torch.cat(values))
    kernels.unpack_weights(kernels.pack_codes(q[0], s[0], group), out[:n])
    assert torch.equal(out[:n].double(), values[0])


def test_packing_rows_with_strides(kernels):
    g = gen(3)
    wide = matrix(g, 40, 515, F32)
    for view in (wide[:, 1:300], wide[3:20, :256], wide[::2, 2:514]):
        out = torch.empty(view.shape[0], view.shape[1] + 7, device=DEV)[:, 3:3 + view.shape[1]]
        kernels.unpack_weights(kernels.pack_weights(view, 64), out)
        assert torch.equal(out.double(), packed_values(view, 64))


# ------------------------------------------------------------------ products
def check_product(kernels, m, n, k, group, x_dtype, out_dtype, residual=False, seed=0, x=None):
    g = gen(seed + m)
    w = matrix(g, n, k, BF16)
    packed = kernels.pack_weights(w, group)
    values = packed_values(w, group)
    if x is None:
        x = torch.randn(m, k, generator=g, device=DEV).to(x_dtype)
    out = torch.full((m, n), math.nan, dtype=out_dtype, device=DEV)
    add = torch.randn(m, n, generator=g, device=DEV) if residual else None
    want = x.double() @ values.t()
    bound = off_by(x, values, group, out_dtype, want)
    if residual:
        want = want + add.double()
        bound = bound + want.abs() * 2.0 ** -23
    kernels.linear(x, packed, out, residual=add)
    kernels.check_error_word()
    close(out, want, bound)
    return packed, x, out


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_dtype,out_dtype", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("m,n,k", [(1, 2048, 1024), (1, 16, 128), (2, 17, 130), (7, 2051, 1021), (8, 100, 4096), (9, 512, 384),
                                   (16, 1000, 2000), (17, 96, 512), (40, 300, 1024), (1, 1, 1), (3, 5000, 64), (5, 64, 12288)])
def test_products(kernels, m, n, k, group, x_dtype, out_dtype):
    check_product(kernels, m, n, k, group, x_dtype, out_dtype, residual=out_dtype == F32 and m % 2 == 1)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(17, 128, 128), (32, 257, 1024), (33, 1000, 2056), (64, 40, 4096), (65, 4096, 512), (128, 128, 72), (129, 300, 1000),
                                   (300, 2051, 1024), (1000, 1024, 2048), (20, 6144, 4096), (2000, 4128, 264), (18, 5, 8),
                                   (48, 1000, 640), (49, 1000, 640), (96, 200, 1664), (97, 200, 1664), (192, 4096, 384), (193, 4096, 384)])
def test_products_with_many_rows(kernels, m, n, k, group, out_dtype):
    check_product(kernels, m, n, k, group, BF16, out_dtype, residual=out_dtype == F32 and m % 2 == 1)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k,kind", [(17, 64, 128, "silu"), (40, 1000, 512, "gelu_tanh"), (64, 12288, 1024, "silu"), (130, 77, 2000, "silu"),
                                        (700, 2730, 1024, "gelu_tanh"), (19, 3, 40, "silu")])
def test_gated_pairs_with_many_rows(kernels, m, n, k, kind, group):
    check_gated(kernels, m, n, k, group, BF16, kind)
    check_gated(kernels, m, n, k, group, BF16, kind, out_dtype=F32)


@pytest.mark.parametrize("m,n,k", [(1, 151936, 256), (1, 128, 32768), (16, 64, 20000), (2, 64, 65536)])
@pytest.mark.parametrize("x_dtype", [BF16, F32])
def test_products_of_far_ends(kernels, m, n, k, x_dtype):
    """Many rows of the matrix, and more columns than a CTA's shared memory holds of x at first."""
    check_product(kernels, m, n, k, 64, x_dtype, F32)


@pytest.mark.parametrize("x_dtype", [BF16, F32])
def test_rows_of_x_and_out_with_strides_and_the_residual_in_place(kernels, x_dtype):
    g = gen(8)
    w = matrix(g, 200, 320, BF16)
    packed, values = kernels.pack_weights(w, 64), packed_values(w, 64)
    for m in (1, 6, 33, 150):
        wide = torch.randn(2 * m, 336, generator=g, device=DEV).to(x_dtype)
        for x in (wide[::2, 1:321], wide[:m, 8:328], wide[:m, :320], wide[:m, 16:].contiguous()):
            room = torch.full((m, 230), 7.0, device=DEV)
            out = room[:, 5:205]
            start = torch.randn(m, 200, generator=g, device=DEV)
            out.copy_(start)
            kernels.linear(x, packed, out, residual=out)
            want = start.double() + x.double() @ values.t()
            close(out, want, off_by(x, values, 64, F32, want) + want.abs() * 2.0 ** -23)
            assert (room[:, :5] == 7).all() and (room[:, 205:] == 7).all()


def test_32_bit_rows_of_every_size(kernels):
    """Rows whose numbers are tiny, huge, or both keep all of their bits (what a sum may lose counts its own magnitudes)."""
    g = gen(9)
    w = matrix(g, 64, 512, BF16)
    packed, values = kernels.pack_weights(w, 64), packed_values(w, 64)
    x = torch.randn(6, 512, generator=g, device=DEV)
    x *= torch.tensor([1e-36, 1e-30, 1.0, 1e20, 1e36, 1e37], device=DEV)[:, None]
    x[2, :100] *= 1e-25
    out = torch.empty(6, 64, device=DEV)
    kernels.linear(x, packed, out)
    want = x.double() @ values.t()
    close(out, want, off_by(x, values, 64, F32, want) + 2.0 ** -126)


@pytest.mark.parametrize("x_dtype", [BF16, F32])
def test_what_is_no_number_stays_with_its_row(kernels, x_dtype):
    g = gen(10)
    w = matrix(g, 96, 256, BF16)
    packed, values = kernels.pack_weights(w, 32), packed_values(w, 32)
    x = torch.randn(5, 256, generator=g, device=DEV).to(x_dtype)
    clean = torch.empty(5, 96, device=DEV)
    kernels.linear(x, packed, clean)
    x[1, 17], x[3, 200], x[4, 3] = math.inf, math.nan, -math.inf
    out = torch.empty(5, 96, device=DEV)
    kernels.linear(x, packed, out)
    assert torch.equal(out[[0, 2]], clean[[0, 2]])
    assert out[3].isnan().all()
    for row, at, sign in ((1, 17, 1.0), (4, 3, -1.0)):
        v = values[:, at]
        assert out[row][v == 0].isnan().all()
        assert torch.equal(out[row][v != 0], (sign * v[v != 0].sign() * math.inf).float())


def test_a_group_that_is_no_number_spoils_its_rows_alone(kernels):
    g = gen(11)
    w = matrix(g, 40, 300, BF16)
    w[7, 299] = math.nan
    packed = kernels.pack_weights(w, 64)
    x = torch.randn(3, 300, generator=g, device=DEV).to(BF16)
    out = torch.empty(3, 40, device=DEV)
    kernels.linear(x, packed, out)
    assert out[:, 7].isnan().all() and not out[:, torch.arange(40, device=DEV) != 7].isnan().any()


@pytest.mark.parametrize("m", [5, 40, 300])
def test_no_rows_and_the_same_bits_twice(kernels, m):
    packed, x, out = check_product(kernels, m, 1000, 2048, 64, BF16, F32)
    again = torch.empty_like(out)
    kernels.linear(x, packed, again)
    assert torch.equal(out, again)
    launches = kernels.launches
    kernels.linear(x[:0], packed, out[:0])
    assert kernels.launches == launches


# ------------------------------------------------------------------ gated pairs
def check_gated(kernels, m, n, k, group, dtype, kind, out_dtype=None, seed=0):
    g = gen(seed + 100 + m)
    gate, up = matrix(g, n, k, BF16, 0.05), matrix(g, n, k, BF16, 0.05)
    packed = kernels.pack_gate_up(gate, up, group)
    vg, vu = packed_values(gate, group), packed_values(up, group)
    x = torch.randn(m, k, generator=g, device=DEV).to(dtype)
    out = torch.full((m, n), math.nan, dtype=out_dtype or dtype, device=DEV)
    assert kernels.linear_swiglu(x, packed, out, **({} if kind == "silu" else {"kind": kind}))
    kernels.check_error_word()
    a, b = x.double() @ vg.t(), x.double() @ vu.t()
    act = a * torch.sigmoid(a) if kind == "silu" else 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
    want = act * b
    # the activations' slopes are below 1.13 in size; in 32 bits they are good to a few half steps of |a| (expf and tanhf to
    # two, and 1 + tanh loses no more than one of 1), the product to one
    ea, eb = off_by(x, vg, group, F32, a), off_by(x, vu, group, F32, b)
    bound = (1.13 * ea + 8 * 2.0 ** -24 * a.abs()) * (b.abs() + eb) + act.abs() * eb + want.abs() * (torch.finfo(out.dtype).eps / 2) + 1e-30
    close(out, want, bound)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k,kind", [(1, 2048, 1024, "silu"), (1, 8, 128, "gelu_tanh"), (3, 9, 130, "silu"), (8, 2730, 1024, "silu"),
                                        (12, 100, 2049, "gelu_tanh"), (16, 64, 4096, "silu"), (21, 77, 300, "silu"), (1, 1, 1, "silu")])
def test_gated_pairs(kernels, m, n, k, kind, dtype, group):
    check_gated(kernels, m, n, k, group, dtype, kind)


def test_a_gated_pair_with_an_output_of_the_other_type(kernels):
    check_gated(kernels, 4, 100, 256, 64, BF16, "silu", out_dtype=F32)
    check_gated(kernels, 4, 100, 256, 64, F32, "silu", out_dtype=BF16)


# ------------------------------------------------------------------ how they are called
def test_a_captured_product_replays_with_new_rows_of_x(kernels):
    g = gen(20)
    w = matrix(g, 700, 904, BF16)
    packed, values = kernels.pack_weights(w, 32), packed_values(w, 32)
    pair = kernels.pack_gate_up(w, w.flip(0).contiguous(), 32)
    stream = torch.cuda.Stream()
    graphs = []
    for m in (1, 11, 50):
        x = torch.randn(m, 904, generator=g, device=DEV).to(BF16)
        out, gated = torch.empty(m, 700, device=DEV), torch.empty(m, 700, dtype=BF16, device=DEV)
        with torch.cuda.stream(stream):
            kernels.linear(x, packed, out)
            kernels.linear_swiglu(x, pair, gated)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            kernels.linear(x, packed, out)
            kernels.linear_swiglu(x, pair, gated)
        graphs.append((graph, x, out, gated))
    for _ in range(3):
        for graph, x, out, gated in graphs:
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
            graph.replay()
        torch.cuda.synchronize()
        for graph, x, out, gated in graphs:
            want = x.double() @ values.t()
            close(out, want, off_by(x, values, 32, F32, want))
            again = torch.empty_like(gated)
            kernels.linear_swiglu(x, pair, again)
            assert torch.equal(gated, again)


def test_two_streams_at_once(kernels):
    g = gen(21)
    w = matrix(g, 4096, 2048, BF16)
    packed = kernels.pack_weights(w, 64)
    x = torch.randn(2, 4, 2048, generator=g, device=DEV).to(BF16)
    want = [torch.empty(4, 4096, device=DEV) for _ in range(2)]
    for i in range(2):
        kernels.linear(x[i], packed, want[i])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty(4, 4096, device=DEV) for _ in range(20)] for _ in range(2)]
    for j in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                kernels.linear(x[i], packed, outs[i][j])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


def test_refusals(kernels):
    from chibillm_b200.kernels.ops import KernelError
    w = torch.zeros(32, 64, dtype=BF16, device=DEV)
    packed, pair = kernels.pack_weights(w, 32), kernels.pack_gate_up(w, w, 32)
    x, out = torch.zeros(2, 64, dtype=BF16, device=DEV), torch.zeros(2, 32, dtype=BF16, device=DEV)
    codes, scales = torch.zeros(32, 64, dtype=torch.int8, device=DEV), torch.zeros(32, 2, dtype=BF16, device=DEV)
    for call in (lambda: kernels.pack_weights(w, 16), lambda: kernels.pack_weights(w.half(), 32), lambda: kernels.pack_weights(w.t(), 32),
                 lambda: kernels.pack_weights(w[:, :0], 32), lambda: kernels.pack_weights(w.cpu(), 32),
                 lambda: kernels.pack_gate_up(w, w[:5], 32), lambda: kernels.pack_gate_up(w, w.float(), 32),
                 lambda: kernels.pack_codes(codes + 8, scales, 32), lambda: kernels.pack_codes(codes - 9, scales, 32),
                 lambda: kernels.pack_codes(codes, scales, 64), lambda: kernels.pack_codes(codes, scales.float(), 32),
                 lambda: kernels.pack_codes(codes.int(), scales, 32), lambda: kernels.pack_codes(codes, scales, 32, codes),
                 lambda: kernels.pack_codes(codes, scales, 32, codes[:9], scales[:9]),
                 lambda: kernels.linear(x, pair, out), lambda: kernels.linear_swiglu(x, packed, out),
                 lambda: kernels.linear_swiglu(x, pair, out, kind="relu"),
                 lambda: kernels.linear(x[:, :32], packed, out), lambda: kernels.linear(x, packed, out[:, :31]),
                 lambda: kernels.linear(x.half(), packed, out), lambda: kernels.linear(x, packed, out.half()),
                 lambda: kernels.linear(x, packed, out, residual=out), lambda: kernels.linear(x.cpu(), packed, out),
                 lambda: kernels.linear(x, packed, out.t().contiguous().t()),
                 lambda: kernels.unpack_weights(packed, w[:5]), lambda: kernels.unpack_weights(pair, w)):
        with pytest.raises(KernelError):
            call()
    assert kernels.linear_partial(x, packed) is None


def test_the_first_call_may_be_captured(kernels):
    """Nothing that a product asks of the device on its first call stands in a capture's way."""
    g = gen(30)
    w = matrix(g, 333, 640, BF16)
    values = packed_values(w, 64)
    stream = torch.cuda.Stream()
    for m, dtype in ((3, BF16), (90, BF16), (5, F32)):
        packed = kernels.pack_weights(w, 64)
        x = torch.randn(m, 640, generator=g, device=DEV).to(dtype)
        out = torch.empty(m, 333, device=DEV)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            kernels.linear(x, packed, out)
        graph.replay()
        torch.cuda.synchronize()
        want = x.double() @ values.t()
        close(out, want, off_by(x, values, 64, F32, want))


def test_packing_inside_a_capture_and_its_product_at_once(kernels):
    g = gen(31)
    w = matrix(g, 256, 512, BF16)
    x = torch.randn(4, 512, generator=g, device=DEV).to(BF16)
    out = torch.empty(4, 256, device=DEV)
    kernels.linear(x, kernels.pack_weights(w, 32), out)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        packed = kernels.pack_weights(w, 32)
        kernels.linear(x, packed, out)
    for _ in range(20):
        w.copy_(matrix(g, 256, 512, BF16))
        graph.replay()
        torch.cuda.synchronize()
        values = packed_values(w, 32)
        want = x.double() @ values.t()
        close(out, want, off_by(x, values, 32, F32, want))


@pytest.mark.parametrize("m", [1, 9, 60])
def test_the_first_rows_of_a_matrix(kernels, m):
    g = gen(32)
    w = matrix(g, 300, 256, BF16)
    packed = kernels.pack_weights(w, 64)
    x = torch.randn(m, 256, generator=g, device=DEV).to(BF16)
    whole = torch.empty(m, 300, device=DEV)
    kernels.linear(x, packed, whole)
    for n in (1, 32, 45, 299, 300):
        out = torch.full((m, n + 3), 5.0, device=DEV)
        kernels.linear(x, packed[:n], out[:, :n])
        values = packed_values(w, 64)[:n]
        want = x.double() @ values.t()
        close(out[:, :n], want, off_by(x, values, 64, F32, want))
        assert (out[:, n:] == 5).all()


def test_rows_whose_factor_is_still_to_be_applied(kernels):
    """A norm's output without its rows' factor, as the bfloat16 products of many rows leave it."""
    g = gen(33)
    a, w0 = torch.randn(300, 256, generator=g, device=DEV).to(BF16), matrix(g, 512, 256, BF16)
    residual = torch.randn(300, 512, generator=g, device=DEV)
    norm = torch.ones(512, device=DEV)
    scaled = kernels.linear_residual_norm(a, w0, residual, norm, 1e-6, 0.0, torch.empty(300, 512, dtype=BF16, device=DEV))
    assert scaled is not None
    w = matrix(g, 200, 512, BF16)
    packed, values = kernels.pack_weights(w, 64), packed_values(w, 64)
    out = torch.empty(300, 200, device=DEV)
    kernels.linear(scaled, packed, out)
    x = scaled.materialise()
    want = x.double() @ values.t()
    close(out, want, off_by(x, values, 64, F32, want))


@pytest.mark.parametrize("m", [4, 40])
def test_bfloat16_rows_of_every_size(kernels, m):
    g = gen(34)
    w = matrix(g, 100, 384, BF16)
    packed, values = kernels.pack_weights(w, 64), packed_values(w, 64)
    x = torch.randn(m, 384, generator=g, device=DEV)
    x *= (10.0 ** torch.linspace(-30, 30, m, device=DEV))[:, None]
    x[0, :200] *= 1e-4
    x = x.to(BF16)
    out = torch.empty(m, 100, device=DEV)
    kernels.linear(x, packed, out)
    want = x.double() @ values.t()
    # (few rows: numbers below 2^-29 of a row's largest are off by 2^-40 of it, 2^-25 where that is 1 ... 2^15)
    small = x.double().abs().amax(1, keepdim=True) * 2.0 ** -25 * values.abs().sum(1)[None, :]
    close(out, want, off_by(x, values, 64, F32, want) + small)


def test_infinities_in_many_rows(kernels):
    g = gen(35)
    w = matrix(g, 130, 256, BF16)
    packed, values = kernels.pack_weights(w, 32), packed_values(w, 32)
    x = torch.randn(50, 256, generator=g, device=DEV).to(BF16)
    clean, out = torch.empty(50, 130, device=DEV), torch.empty(50, 130, device=DEV)
    kernels.linear(x, packed, clean)
    x[11, 17], x[30, 200], x[49, 3] = math.inf, math.nan, -math.inf
    kernels.linear(x, packed, out)
    rest = [i for i in range(50) if i not in (11, 30, 49)]
    assert torch.equal(out[rest], clean[rest]) and out[30].isnan().all()
    for row, at, sign in ((11, 17, 1.0), (49, 3, -1.0)):
        v = values[:, at]
        assert out[row][v == 0].isnan().all()
        assert torch.equal(out[row][v != 0], (sign * v[v != 0].sign() * math.inf).float())


def test_outputs_and_matrices_beyond_32_bits(kernels):
    """More than 2^31 outputs, and a matrix of more than 2^31 elements."""
    g = gen(36)
    w = matrix(g, 151936, 64, BF16)
    packed = kernels.pack_weights(w, 64)
    m = 14200
    x = torch.randn(m, 64, generator=g, device=DEV).to(BF16)
    out = torch.empty(m, 151936, dtype=BF16, device=DEV)
    kernels.linear(x, packed, out)
    rows = [0, 1, m // 2, m - 2, m - 1]
    few = torch.empty(len(rows), 151936, dtype=BF16, device=DEV)
    kernels.linear(x[rows].contiguous(), packed, few)
    # (other orders of the sums: a rounding apart at most)
    assert ((out[rows].float() - few.float()).abs() <= few.float().abs() * 2.0 ** -7 + 1e-6).all()
    del out
    n, k = 70016, 32768
    w = torch.empty(n, k, dtype=BF16, device=DEV).normal_(0.0, 0.02, generator=g)
    packed = kernels.pack_weights(w, 128)
    x = torch.randn(2, k, generator=g, device=DEV).to(BF16)
    out = torch.empty(2, n, device=DEV)
    kernels.linear(x, packed, out)
    for at in (0, 35000, n - 40):
        part = w[at:at + 40].contiguous()
        values = packed_values(part, 128)
        want = x.double() @ values.t()
        close(out[:, at:at + 40], want, off_by(x, values, 128, F32, want))
    kernels.check_error_word()


def test_calls_from_two_threads(kernels):
    import threading
    g = gen(37)
    w = matrix(g, 1000, 1024, BF16)
    packed = kernels.pack_weights(w, 64)
    x = {m: torch.randn(m, 1024, generator=g, device=DEV).to(BF16) for m in range(1, 60)}
    want = {}
    for m in x:
        want[m] = torch.empty(m, 1000, device=DEV)
        kernels.linear(x[m], packed, want[m])
    torch.cuda.synchronize()
    packed.calls.clear()
    wrong = []

    def work(order):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = []
            for m in order:
                out = torch.empty(m, 1000, device=DEV)
                kernels.linear(x[m], packed, out)
                outs.append((m, out))
        stream.synchronize()
        wrong.extend(m for m, out in outs if not torch.equal(out, want[m]))

    threads = [threading.Thread(target=work, args=(list(x)[::step],)) for step in (1, -1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("m", [1, 10, 30])
def test_small_numbers_beside_a_large_one_that_no_weight_sees(kernels, m, x_dtype):
    """A row's largest number meets zeros; the others are float16 subnormals beside it.  bfloat16 of few rows: off by 2^-25 of the
    largest (2^-40 where it is beyond 2^15); 32-bit: by 2^-40."""
    g = gen(40)
    w = matrix(g, 64, 384, BF16)
    w[:, 7] = 0.0
    packed, values = kernels.pack_weights(w, 64), packed_values(w, 64)
    assert (values[:, 7] == 0).all()
    for largest in (1.5, 3e4, 1e8):
        x = (torch.randn(m, 384, generator=g, device=DEV) * (1e-5 * largest)).to(x_dtype)
        x[:, 7] = largest
        out = torch.empty(m, 64, device=DEV)
        kernels.linear(x, packed, out)
        want = x.double() @ values.t()
        unseen = x.clone()
        unseen[:, 7] = 0.0
        step = largest * 2.0 ** -25 if x_dtype == BF16 and largest < 2.0 ** 15 else largest * 2.0 ** -40
        close(out, want, off_by(unseen, values, 64, F32, want) + step * values.abs().sum(1)[None, :])


@pytest.mark.parametrize("x_dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(700, 65, 515), (2400, 100, 129), (5000, 33, 1001)])
def test_more_blocks_of_rows_than_run_at_once(kernels, m, n, k, x_dtype):
    """Odd widths and 32-bit rows: 16 rows of x a CTA, more CTAs than there are SMs."""
    check_product(kernels, m, n, k, 64, x_dtype, F32, residual=True)
    check_gated(kernels, m, n, k, 64, x_dtype, "silu")
