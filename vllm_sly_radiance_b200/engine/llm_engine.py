"""LLMEngine: scheduler + KV/state cache manager + model runner (+ speculative decoding).

API (vLLM-compatible subset): ``add_request``, ``abort_request``, ``step`` ->
``list[RequestOutput]``, ``has_unfinished_requests``; ``add_adapter`` / ``remove_adapter`` for the
low-rank adapters that requests name, ``compact_cache``.  A request with ``SamplingParams.n`` > 1
prefills its prompt once; before the prompt's last token its cache is forked (full pages shared,
the partly filled page and the GDN state copied) and the samples run as requests of their own.  With tensor parallelism every rank runs
the same engine on the same request stream (SPMD); rank 0 returns outputs.
"""
from __future__ import annotations

import logging
import time
from typing import Optional, Union

import numpy as np
import torch

from ..config import EngineConfig, ModelConfig
from ..models.hybrid import HybridModel, TPInfo
from ..ops import kernels as K
from ..utils.metrics import EngineMetrics
from .kv_cache import KVCacheManager
from .model_runner import ModelRunner
from .request import CompletionOutput, Request, RequestOutput, RequestStatus, SamplingParams
from .scheduler import Scheduler
from .tokenizer import IncrementalDetokenizer, get_tokenizer

log = logging.getLogger("radiance.engine")


class EngineStepError(RuntimeError):
    """A step could not complete (e.g. a collective failed because a peer rank left); every open
    request was aborted."""


class LLMEngine:
    def __init__(self, config: EngineConfig, model: Optional[HybridModel] = None,
                 tokenizer=None, tp: Optional[TPInfo] = None, tokenizer_path: Optional[str] = None):
        self.config = config
        self.device = torch.device(config.device if (config.device != "cuda" or torch.cuda.is_available()) else "cpu")
        mcfg: ModelConfig = config.model_config()
        self.model_config = mcfg
        self.tp = tp or TPInfo()
        t0 = time.time()
        if model is None:
            quant = config.quantization if config.gemm_backend == "native" else "fp8"
            if quant == "nvfp4":
                quant = "mxfp4"
            model = HybridModel(mcfg, quant=quant, device=self.device, seed=config.seed, tp=self.tp,
                                lm_head_quant=config.lm_head_quant,
                                embed_quant=config.embed_quant)
        self.model = model
        self.load_time = time.time() - t0
        self.tokenizer = tokenizer or get_tokenizer(tokenizer_path, mcfg.vocab_size)
        self.eos_token_id = getattr(self.tokenizer, "eos_token_id", None)
        # ---- adapters (before the caches are sized by what memory is left) ----
        self.adapters = None
        lora_items = config.lora_items()
        if config.max_loras:
            from ..models.lora import ModelAdapters
            self.adapters = model.adapters = ModelAdapters(model, config.max_loras, config.max_lora_rank)
            for name, path in lora_items:
                self.adapters.add(name, path)
        # ---- cache sizing ----
        bs = config.block_size
        num_slots = config.max_num_seqs + 2
        pin = None
        if not config.num_kv_blocks and self.device.type == "cuda":
            # a pool size measured on this device by `calibrate-kv`, when one exists
            from ..entrypoints.hw import lookup_pin
            pin = lookup_pin(torch.cuda.get_device_name(self.device), config.model,
                             config.tensor_parallel_size, config.max_num_seqs,
                             config.max_num_batched_tokens)
        if config.num_kv_blocks:
            num_blocks = config.num_kv_blocks
        elif pin:
            num_blocks = pin
        elif self.device.type == "cuda":
            torch.cuda.synchronize()
            free, total = torch.cuda.mem_get_info(self.device)
            per_block = max(1, model.cache_bytes_per_block(bs, config.kv_cache_dtype))
            n_snap_b = config.prefix_snapshot_slots if config.enable_prefix_caching else 0
            state = model.state_bytes_per_slot(config.ssm_state_dtype) * (num_slots + n_snap_b)
            activ = 4 << 30   # activations / graphs headroom
            budget = int(free - (1 - config.gpu_memory_utilization) * total) - state - activ
            need = (config.max_model_len + bs - 1) // bs * config.max_num_seqs + 1
            num_blocks = max(8, min(budget // per_block, need * 4))
        else:
            num_blocks = (config.max_model_len + bs - 1) // bs * config.max_num_seqs + 1
        self.num_blocks = int(num_blocks)
        n_snap = config.prefix_snapshot_slots if config.enable_prefix_caching else 0
        if n_snap and config.speculative_method == "dflash2":
            raise ValueError("prefix caching with the DFlash2 drafter is not supported: a cached "
                             "prefix would skip the target forward that feeds the drafter context")
        self.caches = model.make_caches(self.num_blocks, bs, num_slots + n_snap,
                                        config.kv_cache_dtype, config.ssm_state_dtype)
        self.kv = KVCacheManager(self.num_blocks, bs, num_slots, config.enable_prefix_caching,
                                 num_snapshots=n_snap,
                                 snapshot_interval=config.prefix_snapshot_interval)
        if config.enable_prefix_caching and (config.kv_offload_gb > 0 or config.kv_offload_disk_dir):
            from .kv_offload import OffloadManager
            self.kv.offload = OffloadManager(
                self.caches, int(config.kv_offload_gb * (1 << 30)), config.kv_offload_disk_dir,
                int(config.kv_offload_disk_gb * (1 << 30)), config.kv_offload_policy,
                state_fraction=config.kv_offload_state_fraction)
        k = config.num_speculative_tokens if config.speculative_method else 0
        self.scheduler = Scheduler(self.kv, config.max_num_seqs, config.max_num_batched_tokens,
                                   config.max_model_len, num_spec_tokens=k)
        self.runner = ModelRunner(model, self.caches, max_num_seqs=config.max_num_seqs,
                                  max_num_tokens=config.max_num_batched_tokens,
                                  max_model_len=config.max_model_len, device=self.device,
                                  enable_graphs=config.enable_cuda_graphs,
                                  graph_max_bs=config.cuda_graph_max_bs, num_spec_tokens=k)
        from .cache_moves import CacheMover
        self.mover = CacheMover(self.caches)
        if self.adapters is not None:
            self.runner.enable_adapters(config.max_loras)
        if config.capture_graphs_at_start and self.device.type == "cuda":
            t1 = time.time()
            self.runner.capture_all()
            log.info("captured %d decode graphs in %.1fs", len(self.runner.graphs), time.time() - t1)
        self.spec = None
        if config.speculative_method:
            from ..spec_decode.proposer import build_proposer
            self.spec = build_proposer(config, self)
        self.requests: dict[str, Request] = {}
        # n > 1: request id -> its samples' outputs; sample's own id -> (request id, index)
        self.groups: dict[str, dict] = {}
        self.member: dict[str, tuple] = {}
        self.detok: dict[str, IncrementalDetokenizer] = {}
        self.metrics = EngineMetrics()
        from ..utils.step_trace import StepTrace
        self.trace = StepTrace(device=self.device)     # RADIANCE_STEP_TRACE=N
        self.faults = 0
        self.kv_tokens_capacity = self.num_blocks * bs
        log.info("engine ready: %d KV blocks (%d tokens), %d state slots, load %.1fs",
                 self.num_blocks, self.kv_tokens_capacity, num_slots, self.load_time)

    # ------------------------------------------------------------------------------------------
    def add_request(self, prompt: Union[str, list[int]], params: Optional[SamplingParams] = None,
                    request_id: Optional[str] = None, adapter: Optional[str] = None,
                    share_prompt: bool = True) -> str:
        """adapter: the name of a loaded adapter (add_adapter) that the request runs with.
        share_prompt: the n samples of a request start from one prefill of their prompt; without it
        each prefills the prompt itself, the only form that speculative decoding has."""
        params = params or SamplingParams()
        ids = self.tokenizer.encode(prompt) if isinstance(prompt, str) else list(prompt)
        if adapter is not None and adapter not in self.adapter_names:
            raise ValueError(f"adapter {adapter!r} is not loaded")
        if params.n > 1 and share_prompt and self.spec is not None:
            raise ValueError("n > 1 from one prefill is not supported with speculative decoding")
        req = Request(ids, params, request_id, eos_token_id=self.eos_token_id)
        reqs = [req]
        for i in range(1, params.n):
            r = Request(ids, params, f"{req.request_id}#{i}", eos_token_id=self.eos_token_id,
                        arrival_time=req.arrival_time)
            if params.seed is not None:
                r.seed = params.seed + i
            reqs.append(r)
        for r in reqs:
            if adapter is not None:
                r.adapter, r.adapter_slot = adapter, self.adapters.slots[adapter]
                r.cache_salt = self.adapters.salts[adapter]
        self.scheduler.add(req)
        if params.n > 1:
            rid = req.request_id
            self.groups[rid] = dict(ids=[r.request_id for r in reqs], done=set(),
                                    outs=[CompletionOutput(i, "", [], None) for i in range(params.n)])
            self.member.update({r.request_id: (rid, i) for i, r in enumerate(reqs)})
            if len(ids) == 1 or not share_prompt:          # no cache to share
                for r in reqs[1:]:
                    self.scheduler.add(r)
            else:
                req.fork_children = reqs[1:]
        for r in reqs:
            self.requests[r.request_id] = r
            self.detok[r.request_id] = IncrementalDetokenizer(self.tokenizer, params.stop)
        self.metrics.on_arrival()
        return req.request_id

    # ---- adapters ----
    @property
    def adapter_names(self) -> list:
        """Names that requests can give as their adapter."""
        return list(self.adapters.slots) if self.adapters is not None else []

    def add_adapter(self, name: str, path: str):
        """Load a low-rank adapter (PEFT directory) that requests can name."""
        if self.adapters is None:
            raise ValueError("the engine was started without adapter slots (max_loras)")
        self.adapters.add(name, path)

    def remove_adapter(self, name: str):
        """Free an adapter's slot; refused while an open request uses it."""
        if self.adapters is None:
            raise ValueError("the engine was started without adapter slots (max_loras)")
        if any(r.adapter == name for r in self.requests.values()):
            raise ValueError(f"adapter {name!r} is in use")
        self.adapters.remove(name)

    # ---- cache ----
    def compact_cache(self) -> int:
        """Between steps: move the KV blocks in use to the front of the pool.  Returns their number;
        every block behind them is free."""
        if self.spec is not None and self.spec.drafter is not None:
            raise ValueError("compacting with a drafter is not supported: its own cache follows the "
                             "target's blocks")
        live = {id(r): r for q in (self.scheduler.running, self.scheduler.waiting) for r in q}
        (src, dst), n = self.kv.compact(live.values())
        if len(src):
            self.mover.copy(np.stack([src, dst], 1))
        return n

    def _copy_state(self, src: int, dst: int):
        if self.mover.slots.num:
            self.mover.copy(slots=[(src, dst)])

    def _fork(self, parent: Request):
        """The samples of a prompt start from its cache; one that finds no room waits and recomputes."""
        children, parent.fork_children = parent.fork_children, []
        blocks, slots = [], []
        for c in children:
            got = None
            if len(self.scheduler.running) < self.scheduler.max_num_seqs:
                got = self.kv.fork(parent, c)
            if got is None:
                self.scheduler.add(c)
                continue
            blocks += got[0]
            slots += got[1]
            c.status = RequestStatus.RUNNING
            self.scheduler.running.append(c)
        if self.kv.offload is not None:
            self.kv.flush_offload()              # a block evicted for the copies is saved first
        self.mover.copy(blocks, slots if self.mover.slots.num else [])

    def abort_request(self, request_id: str) -> bool:
        group = self.groups.pop(request_id, None)
        if group is not None:
            ok = False
            for rid in group["ids"]:
                self.member.pop(rid, None)
                ok = self.abort_request(rid) or ok
            return ok
        ok = self.scheduler.abort(request_id)
        self.requests.pop(request_id, None)
        self.detok.pop(request_id, None)
        return ok

    def has_unfinished_requests(self) -> bool:
        return self.scheduler.has_unfinished()

    # ------------------------------------------------------------------------------------------
    def step(self) -> list[RequestOutput]:
        t0 = time.perf_counter()
        tr = self.trace.begin()
        sched = self.scheduler.schedule()
        self.trace.mark(tr, "t_sched")
        if self.kv.offload is not None:
            self.kv.flush_offload()    # write-backs of blocks evicted by this schedule
        if sched.is_empty:
            return []
        for s in sched.seqs:         # prefix-cache hits resume from a GDN state snapshot
            if s.req.restore_snapshot is not None:
                self._copy_state(s.req.restore_snapshot, s.req.state_slot)
                self.kv.release_restore(s.req)     # the copy is on the stream: slot reusable
        for s in sched.seqs:
            if s.req.fork_children and s.req.num_computed_tokens == s.req.num_prompt_tokens - 1:
                self._fork(s.req)
        try:
            if self.spec is not None:
                result = self.spec.execute(sched)
            else:
                result = self.runner.execute(sched)
            code = self.runner.read_status()
            if K._CANARY:
                K.check_canaries()          # debug mode: no kernel wrote past its workspace
        except Exception as e:
            # a failed collective (a peer rank that left or timed out) or any other step error:
            # the step's outputs are lost, so no open request can continue
            n = self._abort_all()
            log.error("step failed (%r): %d open requests failed", e, n)
            raise EngineStepError(f"engine step failed: {e!r}") from e
        if code:
            self._fail_open_requests(code)
        self.trace.mark(tr, "t_exec")
        finished = self.scheduler.update(sched, result.sampled)
        if self.kv.num_snapshots:
            for s in sched.seqs:
                if not s.is_decode and s.req.state_slot is not None:
                    sid = self.kv.take_snapshot(s.req)
                    if sid is not None:
                        self._copy_state(s.req.state_slot, sid)
        self.metrics.on_step(sched, result, time.perf_counter() - t0, self.kv.usage,
                             len(self.scheduler.running), len(self.scheduler.waiting))
        outs = []
        progressed = {}
        fin_ids = {r.request_id for r in finished}
        for s in sched.seqs:
            req = s.req
            rid = req.request_id
            if rid not in result.sampled and rid not in fin_ids:
                continue
            det = self.detok.get(rid)
            if det is not None:
                det.update(req.output_token_ids)
                if det.stopped and not req.status.finished:
                    self.scheduler.abort(rid)
                    req.status = RequestStatus.FINISHED_STOPPED
                    fin_ids.add(rid)
            done = req.status.finished
            text = det.text if det else ""
            gid, index = self.member.get(rid, (None, 0))
            comp = CompletionOutput(index, text, list(req.output_token_ids),
                                    req.status.value if done else None)
            met = dict(arrival=req.arrival_time, first_token=req.first_token_time,
                       finish=req.finish_time, num_preemptions=req.num_preemptions)
            if gid is None:
                outs.append(RequestOutput(request_id=rid, prompt_token_ids=req.prompt_token_ids,
                                          outputs=[comp], finished=done, metrics=met))
            else:
                self.groups[gid]["outs"][index] = comp
                if done:
                    self.groups[gid]["done"].add(index)
                progressed[gid] = (req.prompt_token_ids, met)
            if done:
                self.metrics.on_finish(req)
                self.requests.pop(rid, None)
                self.detok.pop(rid, None)
        for gid, (prompt_ids, met) in progressed.items():      # n > 1: all samples in one output
            g = self.groups[gid]
            done = len(g["done"]) == len(g["ids"])
            outs.append(RequestOutput(request_id=gid, prompt_token_ids=prompt_ids, outputs=list(g["outs"]),
                                      finished=done, metrics=met))
            if done:
                self.groups.pop(gid)
                for rid in g["ids"]:
                    self.member.pop(rid, None)
        self.trace.end(tr, result.num_tokens)
        return outs

    def _fail_open_requests(self, code: int):
        """A kernel of this step recorded an error (a bounded wait expired or a bad index was
        refused): its outputs are not valid.  Every open request is aborted and the step raises;
        the OpenAI server turns this into an error for each client and reports itself unhealthy."""
        from ..ops.kernels import KernelFaultError, reset_status
        reset_status(self.device)
        n = self._abort_all()
        log.error("kernel fault (status %d): %d open requests failed", code, n)
        self.faults += 1
        raise KernelFaultError(code)

    def _abort_all(self) -> int:
        ids = list(self.requests)
        for rid in ids:
            self.abort_request(rid)
        return len(ids)

    def generate(self, prompts, params=None, adapters=None) -> list[RequestOutput]:
        """adapters: a loaded adapter's name for all prompts, or one name (or None) per prompt."""
        if isinstance(params, SamplingParams) or params is None:
            params = [params or SamplingParams()] * len(prompts)
        if adapters is None or isinstance(adapters, str):
            adapters = [adapters] * len(prompts)
        if len(adapters) != len(prompts):
            raise ValueError(f"{len(adapters)} adapters for {len(prompts)} prompts")
        order = [self.add_request(p, sp, adapter=a, share_prompt=self.spec is None)
                 for p, sp, a in zip(prompts, params, adapters)]
        final = {}
        while self.has_unfinished_requests():
            for o in self.step():
                if o.finished:
                    final[o.request_id] = o
        return [final[r] for r in order]
