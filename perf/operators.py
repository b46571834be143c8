"""What is timed of the products with matrices held in 4 bits.

Three kinds of cases:

* ``product``: x[M, K] times a matrix [N, K] in 4 bits with a scale per group of columns, through ``CudaKernels.linear``:
  a layer's projections and the vocabulary's, for one token, a batch of tokens, and prompts.
* ``gated``: act(x gate^T) * (x up^T) over two such matrices, through ``CudaKernels.linear_swiglu``: the first half
  of a gated feed-forward block.
* ``pack``: a matrix put into 4 bits and read back as the values that it then stands for, through
  ``CudaKernels.pack_weights`` and ``CudaKernels.unpack_weights``: what loading a model does to each matrix.

The numbers: within a group of ``group`` neighbouring columns of a row (a row's last group may be shorter) a value is
q * s, q a whole number of -8 ... 7 and s a bfloat16.  s is the element of largest magnitude (the first of equals) over
-8, rounded to bfloat16, and q = w / s rounded to the nearest whole number (ties to even) and kept within -8 ... 7.

Widths are those of Qwen3 0.6B (1,024) and 8B (4,096, feed-forward 12,288, vocabulary 151,936) and of ``bench.py``'s designs.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False
DEV = "cuda:0"
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one token through a projection of the 0.6B layer: the smallest call of a decode step
        dict(name="product token small", kind="product", rows=1, n=2048, k=1024, group=64, dtype="bfloat16", out="bfloat16", residual=False),
        # one token through the down projection of the 8B layer, added to the residual
        dict(name="product token down", kind="product", rows=1, n=4096, k=12288, group=128, dtype="bfloat16", out="float32", residual=True),
        # the logits of four requests
        dict(name="product logits", kind="product", rows=4, n=151936, k=4096, group=64, dtype="bfloat16", out="float32", residual=False),
        # a decode step of 24 requests through q | k | v
        dict(name="product batch", kind="product", rows=24, n=6144, k=4096, group=32, dtype="bfloat16", out="bfloat16", residual=False),
        # a prompt portion whose rows fill no whole tile
        dict(name="product prompt", kind="product", rows=1999, n=6144, k=4096, group=64, dtype="bfloat16", out="bfloat16", residual=False),
        # the 32-bit path, sizes that are multiples of nothing
        dict(name="product odd 32-bit", kind="product", rows=7, n=2051, k=1021, group=32, dtype="float32", out="float32", residual=True),
        # one token through the feed-forward of the 8B layer, and a step of 64 requests
        dict(name="gated token", kind="gated", rows=1, n=12288, k=4096, group=64, dtype="bfloat16", act="silu"),
        dict(name="gated batch", kind="gated", rows=64, n=12288, k=4096, group=128, dtype="bfloat16", act="silu"),
        # a prompt through the feed-forward of a layer of width 2,048, gelu as the gate
        dict(name="gated prompt", kind="gated", rows=2048, n=6144, k=2048, group=64, dtype="bfloat16", act="gelu_tanh"),
        # a small 32-bit batch
        dict(name="gated 32-bit", kind="gated", rows=12, n=2730, k=1024, group=64, dtype="float32", act="silu"),
        # a matrix of the 8B layer while it is loaded, and a small 32-bit one with a ragged last group
        dict(name="pack bf16", kind="pack", n=12288, k=4096, group=64, dtype="bfloat16"),
        dict(name="pack 32-bit", kind="pack", n=1023, k=2000, group=32, dtype="float32"),
    ]


def _log(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["product", "product", "product", "gated", "gated", "pack"])
    dtype = "float32" if rng.random() < 0.3 else "bfloat16"
    group = rng.choice([32, 64, 128])
    n, k = _log(rng, 500, 12288), _log(rng, 250, 12288)
    if rng.random() < 0.75:                                  # (most widths are multiples of 64; the others anything)
        n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
    if kind == "pack":
        return dict(kind=kind, n=n, k=k, group=group, dtype=dtype)
    rows = _log(rng, 1, 64) if rng.random() < 0.6 else _log(rng, 64, 2000)
    if dtype == "float32":
        rows = min(rows, 300)
    rows = max(1, min(rows, int(4e10) // (n * k)))
    if kind == "gated":
        return dict(kind=kind, rows=rows, n=n, k=k, group=group, dtype=dtype, act=rng.choice(["silu", "silu", "gelu_tanh"]))
    residual = rng.random() < 0.4
    out = "float32" if residual or dtype == "float32" or rng.random() < 0.3 else "bfloat16"
    return dict(kind=kind, rows=rows, n=n, k=k, group=group, dtype=dtype, out=out, residual=residual)


# ------------------------------------------------------------------ inputs
def _groups(k, group):
    return -(-k // group)


def _codes(g, n, k, group):
    """Whole numbers and scales as a quantised matrix has them (weights of about 0.02, the largest of a group at 8)."""
    q = torch.randn(n, k, generator=g, device=DEV).mul_(3.1).round_().clamp_(-8, 7).to(torch.int8)
    s = (torch.rand(n, _groups(k, group), generator=g, device=DEV) * 0.006 + 0.004)
    sign = torch.rand(n, _groups(k, group), generator=g, device=DEV) < 0.5
    return q, torch.where(sign, s, -s).to(torch.bfloat16)


def _activations(g, rows, k, dtype):
    """A norm's output: values of about one, a few columns much larger."""
    x = torch.randn(rows, k, generator=g, device=DEV)
    loud = torch.rand(k, generator=g, device=DEV) < 0.004
    return torch.where(loud, x * 20.0, x).to(TYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) + 4711)
    s = SimpleNamespace(case=case)
    n, k, group = case["n"], case["k"], case["group"]
    if own:
        from chibillm_b200.engine.runner import make_runtime
        s.kernels = make_runtime(case["dtype"], DEV).kernels
    if case["kind"] == "pack":
        w = torch.randn(n, k, generator=g, device=DEV) * 0.02
        far = torch.rand(n, k, generator=g, device=DEV) < 0.002
        s.w = torch.where(far, w * 8.0, w).to(TYPES[case["dtype"]])
        s.out = torch.empty(n, k, device=DEV)
        return s
    s.codes, s.scales = _codes(g, n, k, group)
    s.x = _activations(g, case["rows"], k, case["dtype"])
    if case["kind"] == "gated":
        s.up_codes, s.up_scales = _codes(g, n, k, group)
        s.out = torch.empty(case["rows"], n, dtype=TYPES[case["dtype"]], device=DEV)
        if own:
            s.packed = s.kernels.pack_codes(s.codes, s.scales, group, s.up_codes, s.up_scales)
        return s
    s.residual = torch.randn(case["rows"], n, generator=g, device=DEV) if case["residual"] else None
    s.out = torch.empty(case["rows"], n, dtype=TYPES[case["out"]], device=DEV)
    if own:
        s.packed = s.kernels.pack_codes(s.codes, s.scales, group)
    return s


# ------------------------------------------------------------------ a pass
def _values(codes, scales, group, dtype):
    """The matrix that codes and scales stand for."""
    k = codes.shape[1]
    return codes.to(dtype) * scales.to(dtype).repeat_interleave(group, dim=1)[:, :k]


def _activate(z, act):
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def _packed_values(w, group):
    """A matrix after its numbers were put into 4 bits.  Which whole number is nearest is decided in 64 bits."""
    n, k = w.shape
    full = torch.zeros(n, _groups(k, group) * group, dtype=torch.float32, device=w.device)
    full[:, :k] = w
    full = full.view(n, -1, group)
    largest = full.abs().argmax(dim=2, keepdim=True)          # the first of equals
    scales = (full.gather(2, largest) / -8.0).to(torch.bfloat16).float()
    ratio = full.double() / torch.where(scales == 0, torch.ones_like(scales), scales).double()
    q = torch.where(scales == 0, torch.zeros_like(ratio), ratio.round().clamp(-8, 7))
    return (q.float() * scales).view(n, -1)[:, :k].contiguous()


def run(s):
    case = s.case
    if own:
        k = s.kernels
        if case["kind"] == "pack":
            k.unpack_weights(k.pack_weights(s.w, case["group"]), s.out)
        elif case["kind"] == "gated":
            k.linear_swiglu(s.x, s.packed, s.out, kind=case["act"])
        else:
            k.linear(s.x, s.packed, s.out, residual=s.residual)
        return s.out
    if case["kind"] == "pack":
        return _packed_values(s.w, case["group"])
    x = s.x.float()
    product = x @ _values(s.codes, s.scales, case["group"], torch.float32).t()
    if case["kind"] == "gated":
        up = x @ _values(s.up_codes, s.up_scales, case["group"], torch.float32).t()
        return (_activate(product, case["act"]) * up).to(TYPES[case["dtype"]])
    if s.residual is not None:
        product = product + s.residual
    return product.to(TYPES[case["out"]])


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    group = case["group"]
    if case["kind"] == "pack":
        w = s.w.double()
        out = torch.empty_like(w)
        for at in range(0, w.shape[1], group):
            part = w[:, at:at + group]
            low, high = part.amin(dim=1), part.amax(dim=1)
            first_low = (part == low[:, None]).double().argmax(dim=1)
            first_high = (part == high[:, None]).double().argmax(dim=1)
            take_low = (-low > high) | ((-low == high) & (first_low <= first_high))
            scale = (torch.where(take_low, low, high) / -8.0).to(torch.float32).to(torch.bfloat16).double()[:, None]
            q = torch.round(part / torch.where(scale == 0, 1.0, scale)).clamp(-8.0, 7.0)
            out[:, at:at + group] = torch.where(scale == 0, 0.0, q * scale)
        return out
    x = s.x.double()

    def product(codes, scales):
        out = torch.empty(x.shape[0], codes.shape[0], dtype=torch.float64, device=x.device)
        for at in range(0, codes.shape[0], 8192):
            q, scale = codes[at:at + 8192].double(), scales[at:at + 8192].double()
            columns = torch.arange(q.shape[1], device=q.device) // group
            out[:, at:at + 8192] = torch.einsum("mk,nk->mn", x, q * scale[:, columns])
        return out

    a = product(s.codes, s.scales)
    if case["kind"] == "product":
        return a if s.residual is None else a + s.residual.double()
    b = product(s.up_codes, s.up_scales)
    if case["act"] == "silu":
        return a * torch.sigmoid(a) * b
    return a * 0.5 * (1.0 + torch.tanh(0.7978845608028654 * (a + 0.044715 * a ** 3))) * b


def work(case):
    n, k = case["n"], case["k"]
    weights = n * k / 2 + 2 * n * _groups(k, case["group"])
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "pack":
        # the matrix read, its 4-bit form written and read, the values written
        return {"bytes": n * k * size + 2 * weights + 4 * n * k, "flops": 4.0 * n * k}
    rows = case["rows"]
    moved = rows * k * size
    if case["kind"] == "gated":
        return {"bytes": 2 * weights + moved + rows * n * size, "flops": 4.0 * rows * n * k}
    moved += rows * n * (4 if case["out"] == "float32" else 2) + (rows * n * 4 if case["residual"] else 0)
    return {"bytes": weights + moved, "flops": 2.0 * rows * n * k}
