"""Matrices held in 4 bits, and how the product with few rows of x shares their work out.

A value is q * s: q a whole number of -8 ... 7, s a bfloat16 scale shared by ``group`` neighbouring columns of a row
(32, 64 or 128; a row's last group may be shorter).  ``csrc/packed.cuh`` says how they lie in memory.  The reference
makes such matrices while it loads a model (``--quantize q4``, src/cli_options.cc:13-25; affine groups of 64,
src/tensor/matrix.h:32-108).
"""
from __future__ import annotations

from typing import Callable, NamedTuple, Optional, Tuple

import torch

GROUPS = (32, 64, 128)
BLOCK_ROWS, BLOCK_COLS = 32, 128
FEW_TOKENS = 16                   # rows of x that such a CTA takes at most
FEW_SMEM_KB = 226


class PackedWeights:
    """A matrix [rows, columns] in 4 bits, or a pair of such matrices (``paired``: gate and up, whose product with x
    ``linear_swiglu`` activates and multiplies).  ``shape`` is that of the matrix, gate's rows and up's counted both.
    ``CudaKernels.pack_weights``, ``pack_gate_up`` and ``pack_codes`` make them; their bytes are constant from then on."""

    dtype = None                     # neither bfloat16 nor 32-bit

    def __init__(self, data: torch.Tensor, rows: int, columns: int, group: int, paired: bool):
        self.data, self.rows, self.columns, self.group, self.paired = data, rows, columns, group, paired
        self._parts = {}
        self.calls = {}              # (kernels, rows of x, types, activation) -> the arguments that stay the same

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows * (2 if self.paired else 1), self.columns))

    def __getitem__(self, rows: slice) -> "PackedWeights":
        """The matrix's first rows, ``w[:n]`` (no copy)."""
        if self.paired or not isinstance(rows, slice) or rows.start is not None or rows.step is not None \
                or not 0 < (self.rows if rows.stop is None else rows.stop) <= self.rows:
            raise IndexError("the first rows of a matrix in 4 bits, w[:n], and nothing else")
        n = self.rows if rows.stop is None else rows.stop
        return self._parts.setdefault(n, PackedWeights(self.data, n, self.columns, self.group, False))

    @property
    def device(self) -> torch.device:
        return self.data.device

    @staticmethod
    def bytes_for(rows: int, columns: int, group: int, paired: bool = False) -> int:
        each = BLOCK_ROWS // 2 if paired else BLOCK_ROWS
        return -(-rows // each) * -(-columns // BLOCK_COLS) * (BLOCK_ROWS * BLOCK_COLS // 2 + BLOCK_COLS // group * 2 * BLOCK_ROWS)


class FewRowsPlan(NamedTuple):
    """See FewRows in csrc/packed_weights.cu."""
    warps: int
    splits: int
    along_k: int
    batch: int
    depth: int
    run: int
    tokens: int
    clusters: int


def few_rows_plan(rows: int, columns: int, paired: bool, m: int, wide: bool, smem_kb: Callable[..., int],
                  most_clusters: Callable[[int, int, int, int], int], sms: int) -> Optional[FewRowsPlan]:
    """How CTAs and warps share a product of m rows of x (``wide``: 32-bit ones).  ``smem_kb(tokens, warps, splits, batch, depth,
    run)`` is a CTA's shared memory, ``most_clusters(tokens, warps, splits, kb)`` how many clusters run at once (0: none).  None if
    nothing fits.

    The cut with the least time by a rough model, in ns, fitted to sweeps of all cuts (1 to 16 rows of x, matrices of 2,048 x 1,024
    to 151,936 x 4,096): a record takes an SM 60 and a warp 530 (what instructions it issues, and their latency), two instructions
    for every 8 rows of x more of it; adding up the sums of a round 400; a cluster that adds up across CTAs 1,200.  About 64
    records are to be on their way to an SM (at 32, 4,096 x 12,288 took 13.3 us instead of 10.2), and no more room is taken than
    a warp's records need, so that the next kernel's CTAs fit beside (2,051 x 1,021: 6.2 us with four places a warp, 4.4 with one).

    With more rows of x than a CTA holds, their blocks are the grid's second axis, and what does not run at once runs after it:
    counted as whole waves (32-bit prompts, and bfloat16 ones of odd widths; uncounted, larger clusters looked as cheap as none: 1,024
    bfloat16 rows of 4,096 x 4,095 401 us instead of 185, 2,000 32-bit rows 1,015 instead of 589)."""
    blocks = -(-rows // (BLOCK_ROWS // 2 if paired else BLOCK_ROWS))
    chunks = -(-columns // BLOCK_COLS)
    tokens = -(-m // -(-m // FEW_TOKENS))
    while tokens >= 1:
        best = None
        token_blocks = -(-m // tokens)
        issue = 60 * (1.4 if tokens > 8 else 1.0) * (1.5 if wide else 1.0)
        for warps, resident in ((8, 2), (8, 1), (16, 1)):
            if tokens > warps:
                continue
            room = FEW_SMEM_KB // resident
            for splits in (1, 2, 4, 8):
                if splits > chunks:
                    break
                mine = -(-chunks // splits)
                for along_k in (16, 8, 4, 2, 1):
                    if along_k > warps:
                        continue
                    per_unit = warps // along_k
                    each = -(-mine // along_k)
                    units = -(-blocks // per_unit)
                    run = max(r for r in ((1, 2, 3, 4) if warps * resident == 8 else (1, 2)) if each % r == 0)
                    rounds = -(-units // max(1, min(units, resident * sms // splits // token_blocks)))
                    depth = min(-(-64 // (warps * resident * run)), rounds * (each // run))
                    while depth > 1 and smem_kb(tokens, warps, splits, 1, depth, run) > room:
                        depth -= 1
                    kb = smem_kb(tokens, warps, splits, 1, depth, run)
                    if kb > room:
                        continue
                    at_once = most_clusters(tokens, warps, splits, kb)
                    if at_once < 1:
                        continue
                    clusters = min(units, max(1, at_once // token_blocks))
                    rounds = -(-units // clusters)
                    waves = -(-clusters * token_blocks // at_once)
                    on_sm = -(-clusters * splits // sms)
                    busy = on_sm * per_unit * min(along_k, mine)
                    time = waves * (on_sm * rounds * per_unit * mine * max(issue, 530 / busy) + rounds * 400
                                    + (1200 if splits > 1 else 0) + mine * 16 * tokens / (warps * 32) * 30)
                    if best is None or time < best[0]:
                        best = (time, FewRowsPlan(warps, splits, along_k, 1, depth, run, tokens, clusters), rounds, room)
        if best is not None:
            _, plan, rounds, room = best
            batch = 1
            while batch < min(rounds, 8) and smem_kb(tokens, plan.warps, plan.splits, batch + 1, plan.depth, plan.run) <= room:
                batch += 1
            return plan._replace(batch=batch)
        tokens //= 2
    return None


class ManyRowsCut(NamedTuple):
    """See chibi_packed_many_rows in csrc/packed_tcgen05.cu."""
    tokens: int
    rounds: int
    splits: int
    clusters: int


def many_rows_cut(rows: int, columns: int, paired: bool, m: int, most_clusters: Callable[[int], int]) -> Optional[ManyRowsCut]:
    """How tiles of the product with many rows of x are shared out: whole rounds of tiles on all SMs, what is left by clusters
    whose CTAs share a tile's columns.  ``most_clusters(splits)``: how many clusters of so many CTAs run at once (the larger
    they are, the fewer SMs they reach).  None if the device runs none of any size."""
    tokens = 48 if m <= 48 else 96 if m <= 96 else 192
    tiles = -(-rows // (64 if paired else 128)) * -(-m // tokens)
    chunks = -(-columns // BLOCK_COLS)
    best = None
    for splits in range(1, min(8, chunks) + 1):
        clusters = most_clusters(splits)
        if clusters < 1:
            continue
        if splits == 1:
            clusters = min(clusters, tiles)
            cost, cut = -(-tiles // clusters) * chunks, ManyRowsCut(tokens, -(-tiles // clusters), 1, clusters)
        else:
            rounds, left = divmod(tiles, clusters * splits)
            if left == 0 or left > clusters:
                continue
            if rounds == 0:
                clusters = left
            # (adding a shared tile's sums up costs about as much as three blocks of columns)
            cost, cut = rounds * chunks + -(-chunks // splits) + 3, ManyRowsCut(tokens, rounds, splits, clusters)
        if best is None or cost < best[0]:
            best = (cost, cut)
    return best[1] if best is not None else None
