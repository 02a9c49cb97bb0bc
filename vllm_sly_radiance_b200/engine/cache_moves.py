"""Pages and state slots moved inside the GPU caches: forking a sequence, compacting the pool.

A forked sequence shares its parent's full pages (reference counts, ``KVCacheManager.fork``); its partly filled page
and the GDN layers' state, which both sequences will write, are copied.  Compacting moves the pages in use to the front
of the pool, so that the pages behind them are free in one piece.  ``CacheMover`` runs either as one launch per item
kind over all layers (``csrc/cache_moves.cu``)."""
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
            pieces += [[i, j] for j in range((nbytes + PIECE_BYTES - 1) // PIECE_BYTES)]
        if self.cuda:
            dev = tensors[0].device
            self.table = torch.tensor(table, dtype=torch.int64, device=dev)
            self.pieces = torch.tensor(pieces, dtype=torch.int32, device=dev)

    def move(self, moves):
        """moves: (src, dst) or, of pages, (src, dst, tokens) rows."""
        m = np.asarray(moves, dtype=np.int64)
        if m.ndim != 2 or m.shape[1] not in ((2, 3) if self.paged else (2,)):
            raise ValueError(f"cache moves: {self.name} as (src, dst{', tokens' if self.paged else ''}) rows")
        src, dst = m[:, 0], m[:, 1]
        tokens = m[:, 2] if m.shape[1] == 3 else np.full(len(m), self.rows)
        if m[:, :2].min() < 0 or m[:, :2].max() >= self.num:
            raise ValueError(f"cache moves: {self.name} outside 0 .. {self.num - 1}")
        if self.paged and (tokens.min() < 0 or tokens.max() > self.rows):
            raise ValueError(f"cache moves: 0 .. {self.rows} tokens of a page")
        taken = np.zeros(self.num, np.int8)
        taken[src] = 1
        if taken[dst].any():
            raise ValueError(f"cache moves: {self.name} both source and destination")
        taken[dst] = 2
        if np.count_nonzero(taken == 2) != len(dst):
            raise ValueError(f"cache moves: {self.name} a destination twice")
        if not self.cuda:
            for s, d, n in zip(src, dst, tokens):
                for t in self.tensors:
                    if self.paged:
                        t[d, :, :n] = t[s, :, :n]
                    else:
                        t[d] = t[s]
            return
        # the destinations of one (source, tokens) side by side: the source is read once
        order = np.lexsort((tokens, src))
        src, dst, tokens = src[order], dst[order], tokens[order]
        new = np.r_[True, (src[1:] != src[:-1]) | (tokens[1:] != tokens[:-1])]
        at = np.flatnonzero(new)
        groups = np.stack([src[at], at, np.diff(np.r_[at, len(src)]), tokens[at]], 1)
        if groups[:, 2].max() > 128:
            raise ValueError(f"cache moves: at most 128 destinations of one source")
        from ..ops._ext import ext
        from ..ops.kernels import status_word
        ext().cache_move(self.table, self.pieces, status_word(self.table.device), self.num,
                         torch.from_numpy(groups.astype(np.int32)), torch.from_numpy(dst.astype(np.int32)))


class CacheMover:
    """Copies inside ``caches`` (whose tensors must stay where they are).  All copies of a call read before any of
    them writes: no item may be a source and a destination, or a destination twice.  Asynchronous on the current
    stream, without a host synchronisation."""

    def __init__(self, caches: ModelCaches):
        self.blocks = _Items("blocks", list(caches.k) + list(caches.v), True)
        self.slots = _Items("slots", list(caches.conv) + list(caches.ssm), False)

    def copy(self, blocks=(), slots=()):
        """blocks: (src, dst) pages or (src, dst, tokens) for the first tokens of a page; slots: (src, dst)."""
        if len(blocks):
            self.blocks.move(blocks)
        if len(slots):
            self.slots.move(slots)

    def compact(self, tables: np.ndarray):
        """tables: int [sequences, pages] block ids (<= 0: no page).  Moves the pages they name to blocks 1 .. n and
        returns (the new tables, n)."""
        tables = np.asarray(tables)
        if tables.size and tables.max() >= self.blocks.num:
            raise ValueError(f"cache moves: blocks outside 0 .. {self.blocks.num - 1}")
        used = np.zeros(self.blocks.num, bool)
        used[tables[tables > 0]] = True
        src, dst, n = plan_compaction(used)
        if len(src):
            self.blocks.move(np.stack([src, dst], 1))
        to = np.arange(self.blocks.num, dtype=tables.dtype)
        to[src] = dst
        return np.where(tables > 0, to[np.maximum(tables, 0)], tables), n
