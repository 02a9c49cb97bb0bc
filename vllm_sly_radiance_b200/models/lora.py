"""Low-rank adapters beside the shared projections.

``AdapterBank`` stacks the adapters of one projection in fixed slots; ``AdapterPlan`` groups the rows of one step by
adapter slot, once for all projections.  ``ops.kernels.lora_add`` adds the deltas to a projection's output.
``ModelAdapters`` keeps the banks of a ``HybridModel`` and loads adapters in the PEFT layout (``adapter_config.json``,
``adapter_model.safetensors``)."""
from __future__ import annotations

import json
import os
import re

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

    # Rows of an adapter that are worth a 128-row tile.  B200, 5120 -> 17408 features, 16-row against 128-row tiles: 48 rows
    # of one adapter 7.6 / 15.6 us at rank 16 and 17.0 / 16.0 at rank 64; 48 rows each of 8 adapters 15.9 / 24.4 and
    # 37.8 / 27.0; 64 rows each 20.1 / 24.9 and 49.9 / 27.9.
    TALL_FROM = 49
    # Where there are 128-row tiles, up to so many remainders go into such tiles too, rather than two more launches: beside
    # 2048 rows, 16 remainders of 3 rows 58 / 63 us at rank 16 and 65 / 83 at rank 64, 24 of them 68 / 61 and 78 / 92.
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


class _Step:
    """The plan of the forward in progress, shared by all adapted linears (None: no row has an adapter)."""
    plan = None


class LinearAdapters:
    """The adapters of one ``Linear``: its bank and the model's current step."""

    def __init__(self, bank: AdapterBank, step: _Step):
        self.bank, self.step = bank, step

    @property
    def active(self) -> bool:
        return self.step.plan is not None

    def add(self, y, x):
        from ..ops import kernels as K
        return K.lora_add(y, x, self.bank, self.step.plan, out=y)


# checkpoint module -> (linear of a layer, slice of its merged output)
_MODULES = {
    "self_attn.q_proj": ("qkv", 0), "self_attn.k_proj": ("qkv", 1), "self_attn.v_proj": ("qkv", 2),
    "self_attn.o_proj": ("o_proj", 0), "linear_attn.in_proj_qkvz": ("in_proj", 0),
    "linear_attn.in_proj_ba": ("in_proj", 1), "linear_attn.out_proj": ("out_proj", 0),
    "mlp.gate_proj": ("gate_up", 0), "mlp.up_proj": ("gate_up", 1), "mlp.down_proj": ("down", 0),
}


# settings of an adapter_config.json under which the delta is not alpha / r times B A of every matrix
_UNSUPPORTED = ("use_dora", "bias", "lora_bias", "modules_to_save", "alpha_pattern", "rank_pattern", "layer_replication",
                "trainable_token_indices", "alora_invocation_tokens")


class ModelAdapters:
    """Banks for every projection of a model's layers (the mixers' and the dense MLP's), ``max_loras`` slots of up to
    ``max_rank`` each.  Tensor parallelism and expert weights are not covered."""

    def __init__(self, model, max_loras: int, max_rank: int):
        if model.tp.size > 1:
            raise ValueError("adapters with tensor parallelism are not supported")
        if max_loras < 1 or not 1 <= max_rank <= MAX_RANK:
            raise ValueError(f"adapters: at least one slot and a rank of 1 .. {MAX_RANK}")
        self.model, self.max_loras, self.max_rank = model, max_loras, (max_rank + 7) // 8 * 8
        self.step = _Step()
        self.slots: dict = {}                    # name -> slot
        self.reserved: frozenset = frozenset()   # names that mean the model without an adapter (the server's)
        self.salts: dict = {}                    # name -> what its cached prefixes are told apart by
        self._loads = 0
        cfg, dev = model.cfg, model.device
        self.banks: list = []                    # per layer: linear name -> bank
        for layer in model.layers:
            lins = {}
            m = layer.mixer
            if layer.is_attn:
                q = m.Hq * m.hd * (2 if m.gated else 1)
                lins["qkv"] = (m.qkv, [0, q, q + m.Hkv * m.hd, q + 2 * m.Hkv * m.hd])
                lins["o_proj"] = (m.o_proj, [0, m.o_proj.N])
            else:
                lins["in_proj"] = (m.in_proj, [0, m.conv_dim + m.value_dim, m.in_proj.N])
                lins["out_proj"] = (m.out_proj, [0, m.out_proj.N])
            if hasattr(layer.mlp, "gate_up"):
                lins["gate_up"] = (layer.mlp.gate_up, [0, layer.mlp.gate_up.N // 2, layer.mlp.gate_up.N])
                lins["down"] = (layer.mlp.down, [0, layer.mlp.down.N])
            banks = {}
            for name, (lin, sl) in lins.items():
                S, R = len(sl) - 1, self.max_rank
                banks[name] = AdapterBank(
                    torch.zeros(max_loras, S, R, lin.K, dtype=torch.bfloat16, device=dev),
                    torch.zeros(max_loras, lin.N, R, dtype=torch.bfloat16, device=dev),
                    torch.zeros(max_loras, device=dev), torch.zeros(max_loras, dtype=torch.int32, device=dev), sl)
                lin.lora = LinearAdapters(banks[name], self.step)
            self.banks.append(banks)
        self._perm = None
        if any(not layer.is_attn for layer in model.layers):
            from ..quant.loaders import gdn_in_proj_permutation
            self._perm = gdn_in_proj_permutation(cfg)

    @property
    def nbytes(self) -> int:
        return sum(2 * (b.a.numel() + b.b.numel()) for banks in self.banks for b in banks.values())

    def add(self, name: str, path: str) -> int:
        """Load the PEFT adapter in directory ``path`` under ``name``; returns its slot."""
        from safetensors import safe_open
        with open(os.path.join(path, "adapter_config.json")) as f:
            cfg = json.load(f)
        odd = [k for k in _UNSUPPORTED if cfg.get(k) not in (None, False, "none", [], {})]
        odd += ["peft_type"] if cfg.get("peft_type", "LORA") != "LORA" else []
        if odd:
            raise ValueError(f"adapter {name!r}: only plain low-rank matrices with one rank and one alpha are supported, "
                             f"not {', '.join(odd)}")
        rank = int(cfg["r"])
        alpha = float(cfg.get("lora_alpha", rank))
        scale = alpha / rank ** 0.5 if cfg.get("use_rslora") else alpha / rank
        with safe_open(os.path.join(path, "adapter_model.safetensors"), framework="pt", device="cpu") as f:
            return self.add_tensors(name, {k: f.get_tensor(k) for k in f.keys()}, rank, scale)

    def add_tensors(self, name: str, tensors: dict, rank: int, scale: float) -> int:
        """tensors: ``...layers.<i>.<module>.lora_A.weight`` [rank, in] and ``lora_B.weight`` [out, rank]."""
        if name in self.slots:
            raise ValueError(f"adapter {name!r} is loaded already")
        if name in self.reserved:
            raise ValueError(f"adapter {name!r}: the model itself is served under this name")
        if not 1 <= rank <= self.max_rank:
            raise ValueError(f"adapter {name!r}: rank {rank}, room for {self.max_rank}")
        free = sorted(set(range(self.max_loras)) - set(self.slots.values()))
        if not free:
            raise ValueError(f"adapter {name!r}: all {self.max_loras} slots are taken")
        slot = free[0]
        parts: dict = {}
        for key, t in tensors.items():
            m = re.search(r"layers\.(\d+)\.(.+)\.lora_([AB])(?:\.default)?\.weight$", key)
            if m is None or m.group(2) not in _MODULES or int(m.group(1)) >= len(self.banks) or \
                    _MODULES[m.group(2)][0] not in self.banks[int(m.group(1))]:
                raise ValueError(f"adapter {name!r}: no projection for {key}")
            parts.setdefault((int(m.group(1)), m.group(2)), {})[m.group(3)] = t
        for (i, module), p in parts.items():     # everything is checked before a slot is written
            lin, s = _MODULES[module]
            bank = self.banks[i][lin]
            n = self._rows(module, bank, s)
            if set(p) != {"A", "B"} or tuple(p["A"].shape) != (rank, bank.K) or tuple(p["B"].shape) != (n, rank):
                raise ValueError(f"adapter {name!r}: layer {i} {module} does not fit [{rank}, {bank.K}] and [{n}, {rank}]")
        for banks in self.banks:
            for b in banks.values():
                b.a[slot].zero_()
                b.b[slot].zero_()
                b.scale[slot] = scale
                b.ranks[slot] = 0
        for (i, module), p in parts.items():
            lin, s = _MODULES[module]
            bank = self.banks[i][lin]
            w = p["B"]
            if self._perm is not None and module.startswith("linear_attn.in_proj"):
                w = w[self._perm[s]]             # the checkpoint groups these rows per key head
            n0 = bank.slices[s]
            bank.a[slot, s, :rank] = p["A"].to(bank.a)
            bank.b[slot, n0:n0 + w.shape[0], :rank] = w.to(bank.b)
            bank.ranks[slot] = rank
        self._loads += 1
        self.slots[name] = slot
        self.salts[name] = f"{name}#{self._loads}"
        return slot

    def _rows(self, module: str, bank: AdapterBank, s: int) -> int:
        if module == "linear_attn.in_proj_ba":   # the merged projection is padded to a multiple of 8
            return len(self._perm[1])
        return bank.slices[s + 1] - bank.slices[s]

    def remove(self, name: str):
        if name not in self.slots:
            raise ValueError(f"adapter {name!r} is not loaded")
        self.slots.pop(name)
        self.salts.pop(name)
