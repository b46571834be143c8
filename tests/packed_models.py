"""Matrices in 4 bits for the tests of whole models: a plain restatement of packing, the weights of a model folder as packing
leaves them, and stand-in kernels for a machine without a GPU."""
import torch

from reference_ops import ReferenceKernels

PACKED = ("q_proj.weight", "k_proj.weight", "v_proj.weight", "o_proj.weight", "gate_proj.weight", "up_proj.weight", "down_proj.weight")


def packed_values(w: torch.Tensor, group: int) -> torch.Tensor:
    """The values that w [rows, columns] stands for in 4 bits (32-bit; which whole number is nearest is decided in 64 bits)."""
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for at in range(0, w.shape[1], group):
        part = w[:, at:at + group].double()
        first = part.abs().argmax(dim=1, keepdim=True)
        scale = (part.gather(1, first) / -8).float().to(torch.bfloat16).double()
        out[:, at:at + group] = torch.where(scale == 0, 0.0, (part / torch.where(scale == 0, 1.0, scale)).round().clamp(-8, 7) * scale)
    return out.float()


def packed_weights(weights: dict, group: int) -> dict:
    """A Qwen3 folder's weights (32-bit) as a run with matrices in 4 bits has them."""
    out = {name: packed_values(w, group) if name.endswith(PACKED) else w for name, w in weights.items()}
    out["lm_head.weight"] = packed_values(weights.get("lm_head.weight", weights["model.embed_tokens.weight"]), group)
    return out


class PackedReference:
    """What ``PackedReferenceKernels`` hand out for PackedWeights: the values."""

    dtype = None

    def __init__(self, values, paired=False):
        self.values, self.paired = values, paired

    @property
    def shape(self):
        return self.values.shape

    def __getitem__(self, rows):
        return PackedReference(self.values[rows])


class PackedReferenceKernels(ReferenceKernels):
    def pack_weights(self, w, group=64):
        self._count("pack_weights")
        return PackedReference(packed_values(w, group))

    def pack_gate_up(self, gate, up, group=64):
        self._count("pack_gate_up")
        return PackedReference(torch.cat([packed_values(gate, group), packed_values(up, group)]), paired=True)

    def linear(self, x, w, out, residual=None, **kw):
        if not isinstance(w, PackedReference):
            return super().linear(x, w, out, residual, **kw)
        assert not w.paired
        self._count("packed product")
        return super().linear(x, w.values, out, residual, **kw)

    def linear_swiglu(self, x, w, out, kind="silu"):
        assert w.paired and kind in ("silu", "gelu_tanh")
        self._count("packed gate and up")
        both = x.float() @ w.values.t()
        gate, up = both[:, :out.shape[1]], both[:, out.shape[1]:]
        act = torch.nn.functional.silu(gate) if kind == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
        out.copy_((act * up).to(out.dtype))
        return True
