"""Matrices held in 4 bits, and how the product with few rows of x shares their work out.

A value is q * s: q a whole number of -8 ... 7, s a bfloat16 scale shared by ``group`` neighbouring columns of a row
(32, 64 or 128; a row's last group may be shorter).  ``csrc/packed.cuh`` says how they lie in memory.  The reference
makes such matrices while it loads a model (``--quantize q4``, src/cli_options.cc:13-25; affine groups of 64,
src/tensor/matrix.h:32-108).
"""
from __future__ import annotations

from typing import Callable, NamedTuple, Optional

import torch

GROUPS = (32, 64, 128)
BLOCK_ROWS, BLOCK_COLS = 16, 128
FEW_WARPS = 16                    # warps of a CTA of the product with few rows
FEW_TOKENS = 16                   # rows of x that such a CTA takes at most
FEW_SMEM_KB = 227


class PackedWeights:
    """A matrix [rows, columns] in 4 bits, or a pair of such matrices (``paired``: gate and up, whose product with x
    ``linear_swiglu`` activates and multiplies).  ``shape`` is that of the matrix, gate's rows and up's counted both.
    ``CudaKernels.pack_weights``, ``pack_gate_up`` and ``pack_codes`` make them; their bytes are constant from then on."""

    dtype = None                     # neither bfloat16 nor 32-bit

    def __init__(self, data: torch.Tensor, rows: int, columns: int, group: int, paired: bool):
        self.data, self.rows, self.columns, self.group, self.paired = data, rows, columns, group, paired

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows * (2 if self.paired else 1), self.columns))

    @property
    def device(self) -> torch.device:
        return self.data.device

    @staticmethod
    def bytes_for(rows: int, columns: int, group: int, paired: bool = False) -> int:
        each = BLOCK_ROWS // 2 if paired else BLOCK_ROWS
        return -(-rows // each) * -(-columns // BLOCK_COLS) * (BLOCK_ROWS * BLOCK_COLS // 2 + BLOCK_COLS // group * 2 * BLOCK_ROWS)


class FewRowsPlan(NamedTuple):
    """See FewRows in csrc/packed_weights.cu."""
    splits: int
    along_k: int
    batch: int
    depth: int
    tokens: int
    clusters: int


def few_rows_plan(rows: int, columns: int, paired: bool, m: int, smem_kb: Callable[[int, int, int, int], int],
                  most_clusters: Callable[[int, int, int], int]) -> Optional[FewRowsPlan]:
    """How CTAs and warps share a product of m rows of x.  ``smem_kb(tokens, splits, batch, depth)`` is a CTA's shared
    memory, ``most_clusters(tokens, splits, kb)`` how many clusters run at once.  None if nothing fits."""
    blocks = -(-rows // (BLOCK_ROWS // 2 if paired else BLOCK_ROWS))
    chunks = -(-columns // BLOCK_COLS)
    tokens = -(-m // -(-m // FEW_TOKENS))
    while tokens >= 1:
        best = None
        token_blocks = -(-m // tokens)
        for splits in (1, 2, 4, 8):
            if splits > chunks:
                break
            mine = -(-chunks // splits)
            for depth in (4, 3, 2):
                if smem_kb(tokens, splits, 1, depth) <= FEW_SMEM_KB:
                    break
            else:
                continue
            at_once = most_clusters(tokens, splits, smem_kb(tokens, splits, 1, depth))
            if at_once < 1:
                continue
            for along_k in (16, 8, 4, 2, 1):
                if along_k > 1 and along_k // 2 >= mine:
                    continue                     # half of the warps would have nothing
                per_unit = FEW_WARPS // along_k
                units = -(-blocks // per_unit)
                clusters = min(units, max(1, at_once // token_blocks))
                rounds = -(-units // clusters)
                cost = rounds * (per_unit * mine + 2) + (20 if splits > 1 else 0)
                if best is None or cost < best[0]:
                    best = (cost, splits, along_k, depth, clusters, rounds)
        if best is not None:
            _, splits, along_k, depth, clusters, rounds = best
            batch = 1
            while batch < min(rounds, 8) and smem_kb(tokens, splits, batch + 1, depth) <= FEW_SMEM_KB:
                batch += 1
            return FewRowsPlan(splits, along_k, batch, depth, tokens, clusters)
        tokens //= 2
    return None
