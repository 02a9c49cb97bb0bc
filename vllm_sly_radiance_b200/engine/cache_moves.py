"""Pages and state slots moved inside the GPU caches: forking a sequence, compacting the pool.

A forked sequence shares its parent's full pages (reference counts, ``KVCacheManager.fork``); its partly filled page
and the GDN layers' state, which both sequences will write, are copied.  Compacting moves the pages in use to the front
of the pool, so that the pages behind them are free in one piece.  ``CacheMover`` runs either as one launch over all
layers, pages and states together (``csrc/cache_moves.cu``).  ``CacheMover.compact`` is for callers that keep block tables
of their own; the engine's ``compact_cache`` plans from its reference counts (``KVCacheManager.compact``), moves the
pages of its prefix cache too, and calls ``copy``."""
from __future__ import annotations

import numpy as np
import torch

from ..models.hybrid import ModelCaches

PIECE_BYTES = 16384          # of an item, copied by one CTA (csrc/cache_moves.cu)


def plan_compaction(used: np.ndarray):
    """used: bool per block (block 0 is reserved and stays).  -> (src, dst, n): the blocks in use behind the first n =
    number in use, ascending, and the free blocks among 1 .. n they move to, ascending."""
    n = int(np.count_nonzero(used[1:]))
    src = n + 1 + np.flatnonzero(used[n + 1:])
    dst = 1 + np.flatnonzero(~used[1:n + 1])
    return src, dst, n


class _Items:
    """One kind of item (pages or slots) over its cache tensors."""

    def __init__(self, name: str, tensors: list, paged: bool):
        self.name, self.tensors, self.paged = name, tensors, paged
        self.num = tensors[0].shape[0] if tensors else 0
        self.rows = tensors[0].shape[2] if paged and tensors else 0
        self.cuda = bool(tensors) and tensors[0].is_cuda
        table, pieces = [], []
        for i, t in enumerate(tensors):
            if t.shape[0] != self.num or t.device != tensors[0].device:
                raise ValueError(f"cache moves: {name} tensors of one length on one device")
            if (not t[:1].is_contiguous()) or (paged and (t.dim() != 4 or t.shape[2] != self.rows)):
                raise ValueError(f"cache moves: {name} tensor {i} of shape {tuple(t.shape)}")
            es = t.element_size()
            nbytes = t[0].numel() * es if self.num else 0
            if paged:
                table.append([t.data_ptr(), t.stride(0) * es, t.shape[1], t.shape[2] * t.shape[3] * es,
                              t.shape[3] * es, t.shape[2]])
            else:
                table.append([t.data_ptr(), t.stride(0) * es, 1, nbytes, 0, 0])
            n = (nbytes + PIECE_BYTES - 1) // PIECE_BYTES
            pieces.append(np.stack([np.full(n, i, np.int32), np.arange(n, dtype=np.int32)], 1))
        self.handle = None
        if self.cuda:
            from ..ops._ext import ext
            from ..ops.kernels import status_word
            dev = tensors[0].device
            self.handle = ext().CacheItems(name, torch.tensor(table, dtype=torch.int64, device=dev),
                                           torch.from_numpy(np.concatenate(pieces)).to(dev),
                                           status_word(dev), self.num, self.rows)

    def move(self, moves):
        """On the CPU: (src, dst) or, of pages, (src, dst, tokens) rows, with the checks of csrc/cache_moves.cu."""
        try:
            m = np.asarray(moves)
        except ValueError:                       # rows of several lengths
            m = np.zeros(0)
        if m.dtype.kind not in "iu":
            raise ValueError(f"cache moves: {self.name} as rows of whole numbers")
        m = m.astype(np.int64)
        if m.ndim != 2 or m.shape[1] not in ((2, 3) if self.paged else (2,)):
            raise ValueError(f"cache moves: {self.name} as (src, dst{', tokens' if self.paged else ''}) rows")
        src, dst = m[:, 0], m[:, 1]
        tokens = m[:, 2] if m.shape[1] == 3 else np.full(len(m), self.rows)
        if m[:, :2].min() < 0 or m[:, :2].max() >= self.num:
            raise ValueError(f"cache moves: {self.name} outside 0 .. {self.num - 1}")
        if self.paged and (tokens.min() < 0 or tokens.max() > self.rows):
            raise ValueError(f"cache moves: 0 .. {self.rows} tokens of a page")
        if len(np.unique(dst)) != len(dst):
            raise ValueError(f"cache moves: {self.name}: a destination twice")
        if np.isin(src, dst).any():
            raise ValueError(f"cache moves: {self.name}: both source and destination")
        return src, dst, tokens

    def apply(self, src, dst, tokens):
        for s, d, n in zip(src, dst, tokens):
            for t in self.tensors:
                if self.paged:
                    t[d, :, :n] = t[s, :, :n]
                else:
                    t[d] = t[s]


class CacheMover:
    """Copies inside ``caches`` (whose tensors must stay where they are).  No item of a call may be a source and a
    destination, or a destination twice; everything is checked before anything moves.  Asynchronous on the current
    stream, without a host synchronisation."""

    def __init__(self, caches: ModelCaches):
        self.blocks = _Items("blocks", list(caches.k) + list(caches.v), True)
        self.slots = _Items("slots", list(caches.conv) + list(caches.ssm), False)
        self.cuda = self.blocks.cuda or self.slots.cuda

    def copy(self, blocks=(), slots=()):
        """blocks: (src, dst) pages or (src, dst, tokens) for the first tokens of a page; slots: (src, dst)."""
        if self.cuda:
            from ..ops._ext import ext
            ext().cache_copy(self.blocks.handle, blocks, self.slots.handle, slots)
            return
        todo = [(k, k.move(m)) for k, m in ((self.blocks, blocks), (self.slots, slots)) if len(m)]
        for k, m in todo:
            k.apply(*m)

    def compact(self, tables: np.ndarray):
        """tables: int32 or int64 [sequences, pages] block ids (<= 0: no page).  Moves the pages they name to blocks
        1 .. n and returns (the new tables, n)."""
        tables = np.ascontiguousarray(tables)
        if tables.dtype not in (np.int32, np.int64):
            raise ValueError(f"cache moves: tables of int32 or int64, got {tables.dtype}")
        if self.blocks.cuda:
            from ..ops._ext import ext
            return ext().cache_compact(self.blocks.handle, tables)
        if tables.size and tables.max() >= self.blocks.num:
            raise ValueError(f"cache moves: blocks outside 0 .. {self.blocks.num - 1}")
        used = np.zeros(self.blocks.num, bool)
        used[tables[tables > 0]] = True
        src, dst, n = plan_compaction(used)
        if len(src):
            self.copy(np.stack([src, dst], 1))
        to = np.arange(self.blocks.num, dtype=tables.dtype)
        to[src] = dst
        return np.where(tables > 0, to[np.maximum(tables, 0)], tables), n
