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
    """The rows of one step by adapter slot, in tiles of one adapter each: full tiles of 128 rows, what remains in one
    more of them or, where it is short, in tiles of 16 (decode batches).  buf int32 holds the 16-row list, then the
    128-row list: [0] tiles in use, [1] those of rows without an adapter, which come first; from 4 on (slot, rows, 1 if
    the rows are consecutive, 0) per tile, then the row numbers, 16 or 128 per tile."""

    # rows of an adapter that are worth a 128-row tile: below, the 16-row kernels need less time
    TALL_FROM = 49
    # up to so many remainders go into 128-row tiles too, where there are such tiles: less time than two more launches
    FEW = 24

    def __init__(self, buf: torch.Tensor, num_rows: int, tiles16: int, tiles128: int, num_slots: int, slots=None):
        self.buf, self.num_rows, self.tiles16, self.tiles128 = buf, num_rows, tiles16, tiles128
        self.num_slots = num_slots
        self.slots = slots                       # host copy (CPU path)
        self.handle = None
        if buf.is_cuda:
            from ..ops._ext import ext
            self.handle = ext().LoraPlan(buf, num_rows, tiles16, tiles128, num_slots)

    @staticmethod
    def words(tiles16: int, tiles128: int) -> int:
        return 4 + (4 + 16) * tiles16 + 4 + (4 + 128) * tiles128

    @staticmethod
    def pack(slots: np.ndarray, num_slots: int, out=None, tiles16=None, tiles128=None, tall_from=None):
        """-> (int32 words of the plan, tiles16, tiles128).  slots: adapter slot of each row, -1 = none; tiles16 and
        tiles128: room for so many tiles (default: as many as there are); tiles128 = 0 packs 16-row tiles only."""
        slots = np.asarray(slots)
        T = slots.shape[0]
        if slots.ndim != 1 or (T and (slots.min() < -1 or slots.max() >= num_slots)):
            raise ValueError(f"adapter slots: one per row, in -1 .. {num_slots - 1}")
        order = np.argsort(slots, kind="stable")
        srt = slots[order]
        starts = np.flatnonzero(np.r_[True, srt[1:] != srt[:-1]]) if T else np.zeros(0, np.int64)
        counts = np.diff(np.r_[starts, T])
        if tall_from is None:
            tall_from = AdapterPlan.TALL_FROM
        full = counts // 128
        tall = full + (counts % 128 >= tall_from) if tiles128 != 0 else 0 * counts
        if tall.any() and np.count_nonzero(counts > tall * 128) <= AdapterPlan.FEW and tall_from < 128:
            tall = (counts + 127) // 128
        in_tall = np.minimum(tall * 128, counts)
        short = (counts - in_tall + 15) // 16
        n16, n128 = int(short.sum()), int(tall.sum())
        tiles16 = n16 if tiles16 is None else tiles16
        tiles128 = n128 if tiles128 is None else tiles128
        if n16 > tiles16 or n128 > tiles128:
            raise ValueError(f"adapter plan: {n16} and {n128} tiles, room for {tiles16} and {tiles128}")
        words = np.zeros(AdapterPlan.words(tiles16, tiles128), np.int32) if out is None else out
        at = 0
        for height, per, first0, cnt, room in ((16, short, starts + in_tall, counts - in_tall, tiles16),
                                               (128, tall, starts, in_tall, tiles128)):
            n = int(per.sum())
            grp = np.repeat(np.arange(len(starts)), per)
            j = np.arange(n) - np.repeat(np.cumsum(per) - per, per)
            first = first0[grp] + j * height
            rows = np.minimum(cnt[grp] - j * height, height)
            tile_slots = srt[first] if n else np.zeros(0, np.int64)
            words[at:at + 4] = (n, np.count_nonzero(tile_slots < 0), 0, 0)
            tiles = words[at + 4:at + 4 + 4 * n].reshape(n, 4)
            tiles[:, 0], tiles[:, 1], tiles[:, 3] = tile_slots, rows, 0
            tiles[:, 2] = order[first + rows - 1] - order[first] == rows - 1       # a tile's rows ascend
            pos = np.arange(int(rows.sum())) - np.repeat(np.cumsum(rows) - rows, rows)   # of each row in its tile
            words[at + 4 + 4 * room + np.repeat(np.arange(n) * height, rows) + pos] = order[np.repeat(first, rows) + pos]
            at += 4 + (4 + height) * room
        return words, tiles16, tiles128

    @staticmethod
    def build(slots, num_slots: int, device) -> "AdapterPlan":
        slots = slots.cpu().numpy() if isinstance(slots, torch.Tensor) else np.asarray(slots)
        words, tiles16, tiles128 = AdapterPlan.pack(slots, num_slots)
        return AdapterPlan(torch.from_numpy(words).to(device), slots.shape[0], tiles16, tiles128, num_slots, slots=slots)
