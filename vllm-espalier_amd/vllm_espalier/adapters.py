"""Low-rank adapters of many requests beside a shared layer (esp_lora, csrc/lora.hip): the base layer runs once for the whole
batch (dense.Dense, linear.TrellisLinear), then every row gets its own request's adapter, whatever adapters a batch mixes.

An Adapters store holds the adapters of one layer in slots of fixed size, so a captured graph keeps its addresses while
adapters come and go: load and clear write into the slots, and the rows of a batch name slots. A slot holds, for each of the
layer's matrices (q/k/v, gate/up, ...), A [rank, in] and B [out, rank] of any rank up to max_rank and a scale; a matrix that an
adapter does not touch has rank 0.
"""
from __future__ import annotations

import torch

from .experts import ext

MAX_MATRICES = 4             # matrices of a layer, as one dense launch takes
MAX_RANK = 256
RANK_TILE = 16               # slots are laid out in whole tiles of ranks,
K_UNIT, COLUMN_TILE = 32, 128   # units of k (A) and tiles of a matrix's columns (B): esp_lora's layout


def _padded(t: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """t in the corner of a [rows, cols] of zeros (whole tiles)."""
    up = lambda n, m: -(-n // m) * m  # noqa: E731
    return torch.nn.functional.pad(t, (0, up(t.shape[1], cols) - t.shape[1], 0, up(t.shape[0], rows) - t.shape[0]))


def pack_a(low: torch.Tensor) -> torch.Tensor:
    """A [rank, in] as esp_lora reads it: [rank tiles, k units, 4, 16, 8]."""
    t = _padded(low, RANK_TILE, K_UNIT)
    return t.reshape(-1, RANK_TILE, t.shape[1] // K_UNIT, 4, 8).permute(0, 2, 3, 1, 4)


def pack_b(high: torch.Tensor) -> torch.Tensor:
    """B [out, rank] as esp_lora reads it: [column tiles, rank tiles, 8, 2, 16, 8]."""
    t = _padded(high, COLUMN_TILE, RANK_TILE)
    return t.reshape(-1, 16, 8, t.shape[1] // RANK_TILE, 2, 8).permute(0, 3, 2, 4, 1, 5)


class Adapters:
    """The adapters of a layer in_features -> sum(out_features), whose matrices' columns stand side by side in its output (the
    Dense layout). in_features and out_features are multiples of 16; dtype is that of the rows (bf16 or fp16).

    Memory: slots * max_rank * (matrices * in_features + sum(out_features)) elements, max_rank rounded up to 16, in_features to
    32 and every matrix's columns to 128."""

    def __init__(self, in_features: int, out_features, slots: int, max_rank: int, dtype=torch.bfloat16, device="cuda"):
        self.in_features, self.out_features = int(in_features), [int(n) for n in out_features]
        self.slots, self.max_rank = int(slots), int(max_rank)
        if not 1 <= len(self.out_features) <= MAX_MATRICES:
            raise ValueError(f"a layer has 1 to {MAX_MATRICES} matrices, got {len(self.out_features)}")
        if any(n <= 0 or n % 16 for n in [self.in_features, *self.out_features]):
            raise ValueError("in_features and out_features must be positive multiples of 16")
        if self.slots < 1 or not 1 <= self.max_rank <= MAX_RANK:
            raise ValueError(f"at least one slot and a max_rank of 1 to {MAX_RANK}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("adapters are bf16 or fp16")
        tiles, S, self.n = -(-self.max_rank // RANK_TILE), len(self.out_features), sum(self.out_features)
        self.col_tiles = [-(-n // COLUMN_TILE) for n in self.out_features]
        units = -(-self.in_features // K_UNIT)
        self.a = torch.zeros((self.slots, S, tiles, units, 4, 16, 8), dtype=dtype, device=device)
        self.b = torch.zeros((self.slots, sum(self.col_tiles), tiles, 8, 2, 16, 8), dtype=dtype, device=device)
        self.ranks = torch.zeros((self.slots, S), dtype=torch.int32, device=device)
        self.scales = torch.zeros((self.slots, S), dtype=torch.float32, device=device)

    def to(self, device):
        """The store on another device (its dtypes stay); where it is there already, its addresses stay too."""
        for name in ("a", "b", "ranks", "scales"):
            setattr(self, name, getattr(self, name).to(device))
        return self

    @torch.no_grad()
    def load(self, slot: int, a, b, scale: float = 1.0) -> None:
        """Put an adapter into a slot: a[s] [rank_s, in_features] and b[s] [out_features[s], rank_s] for matrix s, None for
        both where it leaves the matrix alone; its product with a row is scaled by `scale` (alpha / rank). Values are copied:
        tensors that require grad may be given, and the store keeps nothing of them. Runs on the current stream; rows that name
        the slot must not be in flight on another one."""
        self._slot(slot)
        if len(a) != len(self.out_features) or len(b) != len(self.out_features):
            raise ValueError(f"an adapter has one A and one B for each of the {len(self.out_features)} matrices")
        for s, (low, high) in enumerate(zip(a, b)):
            if (low is None) != (high is None):
                raise ValueError(f"matrix {s}: A and B go together")
            if low is None:
                continue
            rank = low.shape[0]
            if (low.dim() != 2 or high.dim() != 2 or not 0 < rank <= self.max_rank or low.shape[1] != self.in_features or
                    tuple(high.shape) != (self.out_features[s], rank)):
                raise ValueError(f"matrix {s}: expected A [rank, {self.in_features}] and B [{self.out_features[s]}, rank] of a "
                                 f"rank of 1 to {self.max_rank}, got {tuple(low.shape)} and {tuple(high.shape)}")
        self.clear(slot)
        col = 0
        for s, (low, high) in enumerate(zip(a, b)):
            if low is not None:
                rank = low.shape[0]
                tiles = -(-rank // RANK_TILE)
                self.a[slot, s, :tiles].copy_(pack_a(low))
                self.b[slot, col:col + self.col_tiles[s], :tiles].copy_(pack_b(high))
                self.scales[slot, s] = float(scale)
                self.ranks[slot, s] = rank
            col += self.col_tiles[s]

    @torch.no_grad()
    def clear(self, slot: int) -> None:
        """Empty a slot: its rows are left as the base layer made them."""
        self._slot(slot)
        self.ranks[slot].zero_()

    def _slot(self, slot: int) -> None:
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} is outside [0, {self.slots})")

    def apply(self, x: torch.Tensor, y: torch.Tensor, rows: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """y [T, at least sum(out_features)] plus, for every row, the product of x [T, in_features] with the adapter in slot
        rows[t] (int32 [T], on the device; outside [0, slots): none, and the row keeps y's bits). In place unless `out` is
        given; what is written may not overlap x, nor y without being y. Columns past the matrices' are not touched. A row's bits
        do not depend on the other rows."""
        out = y if out is None else out
        ext().lora(x, y, out, rows, self.a, self.b, self.ranks, self.scales, self.out_features, self.in_features)
        return out
