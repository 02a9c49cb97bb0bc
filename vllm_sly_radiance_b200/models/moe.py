"""Mixture-of-experts block (256 routed experts, softmax top-8 with renormalised weights, one shared
expert behind a sigmoid gate; Qwen3-Next MoE semantics, served TP-sharded by the reference through
vLLM fused_moe, ``moe-configs/E=256,...``; sigmoid scores, a balance bias and expert groups by
configuration).

On the GPU: ``K.moe_route`` picks the experts, ``K.moe_plan`` sorts the (token, slot) pairs by expert,
and routed experts run as ONE launch per projection -- the tcgen05 grouped W4A8 GEMM
(``mxfp4_grouped_gemm`` in ``csrc/mxfp4_gemm.cu``) over rows gathered in that order, or the bf16
product of ``csrc/linear_fused.cu``, which picks its rows by token and ends in SwiGLU.
``K.moe_combine`` adds the rows up per token.

Expert parallelism: the tensor-parallel ranks already hold every token of the step (attention is
head-sharded), so each of the `size` ranks owns E/size experts and a 1/size slice of the shared
expert, evaluates them for all tokens, and its output is a partial sum.  Dispatch is then a local
selection and the combine is the all-reduce the model runs after every MLP, which on NVLink is
the fused all-reduce + residual add + RMSNorm + e4m3 kernel (``csrc/comm.cu``).
"""
from __future__ import annotations

from typing import Optional

import torch

from ..config import ModelConfig
from ..ops import kernels as K
from ..ops import reference as ref
from ..quant.mxfp4 import MXFP4Weight, cat_rows
from .layers import Linear, LinearBank


class MoEBlock:
    def __init__(self, cfg: ModelConfig, tp, quant: str, W, prefix: str, ep=None):
        H = cfg.hidden_size
        E = cfg.num_experts
        I = cfg.moe_intermediate_size
        self.cfg = cfg
        self.E, self.H, self.I = E, H, I
        self.top_k = cfg.num_experts_per_tok
        self.quant = quant
        groups, tops = cfg.moe_num_groups, cfg.moe_top_groups
        if cfg.moe_score not in ("softmax", "sigmoid"):
            raise ValueError(f"MoE router: scores softmax or sigmoid, got {cfg.moe_score!r}")
        if not 1 <= self.top_k <= E:
            raise ValueError(f"MoE router: {self.top_k} experts a token of {E}")
        if not 1 <= groups <= 32 or E % groups or not 1 <= tops <= groups or tops * (E // groups) < self.top_k:
            raise ValueError(f"MoE router: {self.top_k} experts in {tops} of {groups} groups of {E} experts")
        if cfg.moe_router_bias and groups > 1 and E // groups < 2:
            raise ValueError("MoE router: with a bias a group's value is that of two experts")
        # experts owned by this rank: expert parallel over the tensor-parallel group (tokens
        # replicated, partial sums all-reduced), or over a data-parallel group `ep` (tokens
        # local to each rank, rows exchanged by the EP transport's dispatch / combine)
        self.ep = ep.transport if ep is not None else None
        size = ep.size if ep is not None else (tp.size if tp is not None else 1)
        rank = ep.rank if ep is not None else (tp.rank if tp is not None else 0)
        assert E % size == 0, (E, size)
        self.e0, self.e_local = rank * (E // size), E // size
        router = W.tensor(prefix + "router", (E, H), "linear_bf16") if hasattr(W, "tensor") else None
        self.router = router.to(torch.bfloat16).contiguous()
        gu, dn = [], []
        for e in range(self.e0, self.e0 + self.e_local):
            gu.append(W.linear(prefix + f"experts.{e}.gate_up", 2 * I, H))
            dn.append(W.linear(prefix + f"experts.{e}.down", H, I))
        if quant == "mxfp4":
            to_mx = lambda w: w if isinstance(w, MXFP4Weight) else MXFP4Weight.from_float(w)
            self.w_gate_up = cat_rows([to_mx(w) for w in gu])      # [E_local*2I, H/2] stacked
            self.w_down = cat_rows([to_mx(w) for w in dn])         # [E_local*H, I/2]
            self.dense_gu = self.dense_dn = None
        else:
            deq = lambda w: (w.dequantize() if isinstance(w, MXFP4Weight) else w).to(torch.bfloat16)
            self.dense_gu = torch.stack([deq(w) for w in gu])      # [E_local, 2I, H]
            self.dense_dn = torch.stack([deq(w) for w in dn])      # [E_local, H, I]
            self.w_gate_up = self.w_down = None
        del gu, dn
        Is = cfg.shared_expert_intermediate_size
        from .hybrid import _cat_sections, make_linear
        from .weights import slice_cols
        wsg = W.linear(prefix + "shared.gate_up", 2 * Is, H)
        self.shared_gate_up = make_linear(_cat_sections(wsg, [Is, Is], tp), quant, "sh_gate_up")
        wsd = W.linear(prefix + "shared.down", H, Is)
        s0, per = tp.shard(Is)
        self.shared_down = make_linear(slice_cols(wsd, s0, per), quant, "sh_down")
        self.shared_gate = W.tensor(prefix + "shared_gate", (1, H), "linear_bf16").to(torch.bfloat16)
        # added to the scores when experts are ranked, not to the weights
        self.router_bias = W.tensor(prefix + "router_bias", (E,), "router_bias").float() if cfg.moe_router_bias else None
        self._prepare()

    def _prepare(self):
        """On the GPU: router and shared gate as one weight [rows in whole 8, H]; bf16 weights as ``K.linear_fused`` takes
        them, in place -- the shared expert's two products (None in another format) and the routed experts'."""
        self._gates = self._banks = None
        if not self.router.is_cuda:
            return
        both = torch.cat([self.router, self.shared_gate])
        self._gates = torch.cat([both, both.new_zeros(-both.shape[0] % 8, self.H)])
        if (self.dense_gu is not None and self.H % 8 == 0 and self.I % 8 == 0 and self.e_local <= K.MOE_MAX_EXPERTS):
            up, down = self.shared_gate_up, self.shared_down
            bf16 = up.quant == "bf16" and down.K % 8 == 0 and down.K > 0          # K is 0 without a shared expert
            self._banks = (LinearBank(up.w, act="swiglu") if bf16 else None, LinearBank(down.w) if bf16 else None,
                           LinearBank(self.dense_gu, act="swiglu"), LinearBank(self.dense_dn))

    def to(self, device):
        for k, v in list(vars(self).items()):
            if isinstance(v, torch.Tensor):
                setattr(self, k, v.to(device))
            elif isinstance(v, MXFP4Weight):
                setattr(self, k, v.to(device))
            elif isinstance(v, Linear):
                v.to(device)
        self._prepare()
        return self

    # ------------------------------------------------------------------------------------------
    # More experts, or more a token, than the router's and the plan's kernels take: plain torch operations, without a stop for the host
    def _choose(self, logits: torch.Tensor):
        cfg = self.cfg
        route = K.moe_route if self.E <= K.MOE_MAX_EXPERTS and self.top_k <= K.MOE_MAX_TOP_K else ref.moe_route
        return route(logits, self.top_k, score=cfg.moe_score, bias=self.router_bias, groups=cfg.moe_num_groups,
                     top_groups=cfg.moe_top_groups, renormalize=cfg.moe_renormalize, scale=cfg.moe_routed_scale)

    def _plan(self, ids: torch.Tensor, tile: int = 0) -> K.MoEPlan:
        if self.e_local <= K.MOE_MAX_EXPERTS:
            return K.moe_plan(ids, self.e_local, first=self.e0, tile=tile)
        order, pos, counts, starts = ref.moe_plan(ids, self.e_local, self.e0)
        items = K.moe_work_items(counts.long(), tile, (ids.numel() + tile - 1) // tile + self.e_local) if tile else None
        return K.MoEPlan(ids.shape[1], order, pos, counts, starts, items, tile)

    def route(self, x_bf16: torch.Tensor):
        """Scores over all experts, top-k, weights (``K.moe_route``) -> (ids [T,k], weights [T,k])."""
        return self._choose(x_bf16.float() @ self.router.float().t())

    def _route_and_gate(self, xb: torch.Tensor):
        """-> (ids, weights, the shared expert's gate before its sigmoid [T]); on the GPU the router and the gate are one
        product of bf16 numbers, summed in 32 bits."""
        if not xb.is_cuda:
            return *self.route(xb), (xb.float() @ self.shared_gate.float().t())[:, 0]
        logits = torch.mm(xb, self._gates.t(), out_dtype=torch.float32)
        return *self._choose(logits[:, :self.E]), logits[:, self.E]

    def forward(self, x):
        """x: (q, scale) from the fused producer or bf16 [T, H] -> bf16 [T, H]."""
        if isinstance(x, tuple):
            q, s = x
            xb = (q.float() * s[:, None]).to(torch.bfloat16)
        else:
            xb = x
            q, s = K.quant_fp8(x) if self.quant == "mxfp4" else (None, None)
        ids, w, gate = self._route_and_gate(xb)
        if (xb.is_cuda and self._banks is not None and self._banks[0] is not None
                and not (self.shared_gate_up._adapted() or self.shared_down._adapted())):
            # bf16 weights: SwiGLU ends the shared expert's first product, gate and routed sum its second
            up, down, _, _ = self._banks
            routed = self._experts(xb, (q, s), ids, w)
            return K.linear_fused(K.linear_fused(xb, up), down, scale=torch.sigmoid(gate), residual=routed, out=routed)
        sh = self.shared_down(K.silu_mul_quant(self.shared_gate_up((q, s) if q is not None else xb))
                              if self.quant == "mxfp4" else K.silu_mul(self.shared_gate_up(xb)))
        if self.ep is None and self._on_kernels(xb):
            return self.local_experts(xb, (q, s), ids, w, shared=sh, gate=gate)
        routed = self._experts(xb, (q, s), ids, w)
        return (routed.float() + torch.sigmoid(gate)[:, None] * sh.float()).to(torch.bfloat16)

    def _on_kernels(self, x: torch.Tensor) -> bool:
        """The routed experts run as grouped products (bf16 rows have to be whole 16 bytes)."""
        return x.is_cuda and (self.w_gate_up is not None or self._banks is not None)

    def _experts(self, xb, qs, ids, w):
        if self.ep is not None:
            return self.ep.dispatch_combine(self, xb, qs, ids, w)
        return self.local_experts(xb, qs, ids, w)

    def expert_rows(self, q, s, xb, le):
        """Unweighted outputs of this rank's experts for rows routed to them: row i goes through
        local expert le[i] (any order; rows of one expert are grouped internally)."""
        n = le.shape[0]
        dev = le.device
        if n == 0:
            return torch.zeros(0, self.H, dtype=torch.bfloat16, device=dev)
        y = torch.empty(n, self.H, dtype=torch.bfloat16, device=dev)
        if self.w_gate_up is None and self._on_kernels(le):
            _, _, up, down = self._banks
            plan = K.moe_plan(le[:, None], self.e_local)
            y[plan.order.long()] = K.linear_fused(K.linear_fused(xb, up, plan=plan, by_token=True), down, plan=plan)
            return y
        order = torch.argsort(le, stable=True)
        counts = torch.bincount(le, minlength=self.e_local)
        if self.w_gate_up is not None and le.is_cuda:
            y[order] = K.moe_grouped_mlp(q[order], s[order], counts, self.w_gate_up, self.w_down,
                                         self.I, self.H)
            return y
        starts = torch.cumsum(counts, 0) - counts
        for e in range(self.e_local):
            c = int(counts[e])
            if c == 0:
                continue
            idx = order[int(starts[e]):int(starts[e]) + c]
            if self.w_gate_up is not None:
                gsl = slice(e * 2 * self.I, (e + 1) * 2 * self.I)
                dsl = slice(e * self.H, (e + 1) * self.H)
                gu = K.mxfp4_gemm(q[idx], s[idx], self.w_gate_up.packed[gsl], None,
                                  self.w_gate_up.scales[gsl], 2 * self.I, fmt=self.w_gate_up.fmt)
                a = K.silu_mul_quant(gu)
                y[idx] = K.mxfp4_gemm(a[0], a[1], self.w_down.packed[dsl], None,
                                      self.w_down.scales[dsl], self.H, fmt=self.w_down.fmt)
            else:
                gu = xb[idx].float() @ self.dense_gu[e].float().t()
                a = K.silu_mul(gu.to(torch.bfloat16)).float()
                y[idx] = (a @ self.dense_dn[e].float().t()).to(torch.bfloat16)
        return y

    def local_experts(self, xb, qs, ids, w, shared=None, gate=None):
        """Experts [e0, e0+e_local) applied to every (token, slot) routed to them; the other
        slots contribute zero (they belong to another rank's experts).  As grouped products,
        shared rows times sigmoid(gate) join the sum.

        Each expert's row is rounded to bf16 between the down product and the weighted sum, which halves what the sum
        reads; the loop over bf16 experts below keeps it in 32 bits, but rounds gate, up and their product where the
        grouped products round the product alone.  Against 64 bits (K 512 and 256, top-8) the block's result is off by
        2.9e-3 with the grouped products, 3.6e-3 with the loop, in the 2-norm."""
        if self._on_kernels(xb):
            # fixed shapes, no host sync (CUDA-graph safe)
            if self.w_gate_up is None:
                _, _, up, down = self._banks
                plan = self._plan(ids)
                rows = K.linear_fused(K.linear_fused(xb, up, plan=plan, by_token=True), down, plan=plan)
            else:
                plan = self._plan(ids, tile=K.moe_tile(ids.numel(), self.e_local))
                q, s = K.moe_gather(qs, plan)
                rows = K.moe_grouped_mlp(q, s, plan, self.w_gate_up, self.w_down, self.I, self.H)
            return K.moe_combine(rows, plan, w, shared=shared, gate=gate)
        T, k = ids.shape
        dev = xb.device
        flat_e = ids.reshape(-1) - self.e0
        flat_t = torch.arange(T, device=dev).repeat_interleave(k)
        flat_w = w.reshape(-1)
        own = (flat_e >= 0) & (flat_e < self.e_local)
        out = torch.zeros(T, self.H, dtype=torch.float32, device=dev)
        flat_e, flat_t, flat_w = flat_e[own], flat_t[own], flat_w[own]
        if flat_e.numel() == 0:
            return out.to(torch.bfloat16)
        order = torch.argsort(flat_e, stable=True)
        se, st, sw = flat_e[order], flat_t[order], flat_w[order]
        counts = torch.bincount(se, minlength=self.e_local)
        y = torch.empty(se.shape[0], self.H, dtype=torch.float32, device=dev)
        starts = torch.cumsum(counts, 0) - counts
        for e in range(self.e_local):
            c = int(counts[e])
            if c == 0:
                continue
            r0 = int(starts[e])
            rows = xb[st[r0:r0 + c]]
            if self.w_gate_up is not None:     # CPU W4A8 oracle
                qq, ss = qs[0][st[r0:r0 + c]], qs[1][st[r0:r0 + c]]
                gsl = slice(e * 2 * self.I, (e + 1) * 2 * self.I)
                dsl = slice(e * self.H, (e + 1) * self.H)
                gu = K.mxfp4_gemm(qq, ss, self.w_gate_up.packed[gsl], None,
                                  self.w_gate_up.scales[gsl], 2 * self.I, fmt=self.w_gate_up.fmt)
                a = K.silu_mul_quant(gu)
                y[r0:r0 + c] = K.mxfp4_gemm(a[0], a[1], self.w_down.packed[dsl], None,
                                            self.w_down.scales[dsl], self.H, fmt=self.w_down.fmt).float()
            else:
                gu = rows.float() @ self.dense_gu[e].float().t()
                a = K.silu_mul(gu.to(torch.bfloat16)).float()
                y[r0:r0 + c] = a @ self.dense_dn[e].float().t()
        out.index_add_(0, st, y.float() * sw[:, None])
        return out.to(torch.bfloat16)
