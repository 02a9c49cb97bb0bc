"""Low-rank adapters beside the shared projections.

``AdapterBank`` stacks the adapters of one projection in fixed slots; ``AdapterPlan`` groups the rows of one step by
adapter slot, once for all projections.  ``ops.kernels.lora_add`` adds the deltas to a projection's output."""
from __future__ import annotations

import numpy as np
import torch

MAX_SLICES = 8
MAX_RANK = 256


class AdapterBank:
    """a [L, S, R, K], b [L, N, R] bf16; scale fp32 [L] (alpha / rank); ranks int32 [L] (an adapter uses its first
    ranks[l] of the R rows, 0 = empty slot); slices: the S + 1 offsets of the merged projection's parts in 0 .. N.
    The tensors are used as they are (not copied): writing a slot between steps changes that adapter."""

    def __init__(self, a, b, scale, ranks, slices):
        slices = [int(o) for o in slices]
        if a.dim() != 4 or b.dim() != 3 or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
            raise ValueError("adapters: a [L, S, R, K] and b [L, N, R] in bf16")
        L, S, R, K = a.shape
        if b.shape[0] != L or b.shape[2] != R or min(L, S, R, K, b.shape[1]) < 1:
            raise ValueError(f"adapters: a {tuple(a.shape)} and b {tuple(b.shape)} do not belong together")
        if S > MAX_SLICES or R > MAX_RANK:
            raise ValueError(f"adapters: at most {MAX_SLICES} slices and rank {MAX_RANK}, got {S} and {R}")
        if len(slices) != S + 1 or slices[0] != 0 or slices[-1] != b.shape[1] or \
                any(u >= v for u, v in zip(slices, slices[1:])):
            raise ValueError(f"adapters: slices {slices} do not cut 0 .. {b.shape[1]} into {S} parts")
        if scale.dtype != torch.float32 or ranks.dtype != torch.int32 or scale.shape != (L,) or ranks.shape != (L,):
            raise ValueError("adapters: scale fp32 [L], ranks int32 [L]")
        if not all(t.is_contiguous() for t in (a, b, scale, ranks)):
            raise ValueError("adapters: contiguous tensors")
        if len({t.device for t in (a, b, scale, ranks)}) != 1:
            raise ValueError("adapters: tensors on one device")
        self.a, self.b, self.scale, self.ranks, self.slices = a, b, scale, ranks, slices
        self.L, self.S, self.R, self.K, self.N = L, S, R, K, b.shape[1]
        self.device = a.device
        self.handle = None
        if a.is_cuda:
            from ..ops._ext import ext
            from ..ops.kernels import status_word
            self.handle = ext().LoraBank(a, b, scale, ranks, slices, status_word(a.device))


class AdapterPlan:
    """The rows of one step by adapter slot, in tiles of at most ``tile_rows`` rows of one adapter.  buf int32: [0] tiles
    in use, from 4 on (slot, rows, 1 if the rows are consecutive, 0) per tile, then ``tile_rows`` row numbers per tile."""

    # rows per tile: decode batches (few rows per adapter), prompts
    TILE_DECODE, TILE_PROMPT = 16, 128

    def __init__(self, buf: torch.Tensor, num_rows: int, max_tiles: int, tile_rows: int, num_slots: int, slots=None):
        self.buf, self.num_rows, self.max_tiles = buf, num_rows, max_tiles
        self.tile_rows, self.num_slots = tile_rows, num_slots
        self.slots = slots                       # host copy (CPU path)
        self.handle = None
        if buf.is_cuda:
            from ..ops._ext import ext
            self.handle = ext().LoraPlan(buf, num_rows, max_tiles, tile_rows, num_slots)

    @staticmethod
    def words(max_tiles: int, tile_rows: int) -> int:
        return 4 + (4 + tile_rows) * max_tiles

    @staticmethod
    def pack(slots: np.ndarray, num_slots: int, out=None, max_tiles=None, tile_rows=None):
        """-> (int32 words of the plan, max_tiles, tile_rows).  slots: adapter slot of each row, -1 = none."""
        slots = np.asarray(slots)
        T = slots.shape[0]
        if slots.ndim != 1 or (T and (slots.min() < -1 or slots.max() >= num_slots)):
            raise ValueError(f"adapter slots: one per row, in -1 .. {num_slots - 1}")
        order = np.argsort(slots, kind="stable")
        srt = slots[order]
        starts = np.flatnonzero(np.r_[True, srt[1:] != srt[:-1]]) if T else np.zeros(0, np.int64)
        counts = np.diff(np.r_[starts, T])
        if tile_rows is None:
            tile_rows = AdapterPlan.TILE_PROMPT if T > 32 * max(1, len(starts)) else AdapterPlan.TILE_DECODE
        per = (counts + tile_rows - 1) // tile_rows
        n = int(per.sum())
        if max_tiles is None:
            max_tiles = max(1, n)
        if n > max_tiles:
            raise ValueError(f"adapter plan: {n} tiles, room for {max_tiles}")
        grp = np.repeat(np.arange(len(starts)), per)
        j = np.arange(n) - np.repeat(np.cumsum(per) - per, per)
        first = starts[grp] + j * tile_rows
        rows = np.minimum(counts[grp] - j * tile_rows, tile_rows)
        words = np.zeros(AdapterPlan.words(max_tiles, tile_rows), np.int32) if out is None else out
        words[:4] = (n, 0, 0, 0)
        tiles = words[4:4 + 4 * n].reshape(n, 4)
        tiles[:, 0], tiles[:, 1], tiles[:, 3] = srt[starts[grp]], rows, 0
        tiles[:, 2] = order[first + rows - 1] - order[first] == rows - 1       # the order within a tile is ascending
        at = 4 + 4 * max_tiles + np.repeat(np.arange(n) * tile_rows - first, rows) + np.arange(T)
        words[at] = order
        return words, max_tiles, tile_rows

    @staticmethod
    def build(slots, num_slots: int, device) -> "AdapterPlan":
        slots = slots.cpu().numpy() if isinstance(slots, torch.Tensor) else np.asarray(slots)
        words, max_tiles, tile_rows = AdapterPlan.pack(slots, num_slots)
        return AdapterPlan(torch.from_numpy(words).to(device), slots.shape[0], max_tiles, tile_rows, num_slots,
                           slots=slots)
