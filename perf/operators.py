"""Cases that measure the multi-adapter projection and the cache page moves.

Three operators: "adapters" adds the low-rank deltas of many requests' adapters to the output of a shared projection;
"fork" copies pages (whole or their first tokens) and recurrent state slots of a cache to one or several destinations;
"compact" moves the pages in use to the front of the pool and rewrites the block tables.

`run` computes them in plain torch operations, or with the framework's kernels where `own` is true."""
import numpy as np
import torch

own = False

DEVICE = "cuda"

# Output features of the merged projections of the 27B hybrid geometry (hidden 5120, SwiGLU 8704) and of the MoE hybrid
# (hidden 2048), as (input features, slices).
PROJECTIONS = {
    "qkv": (5120, "12288,1024,1024"),
    "in_proj": (5120, "16384,96"),
    "o_proj": (6144, "5120"),
    "gate_up": (5120, "8704,8704"),
    "down": (8704, "5120"),
    "moe_in_proj": (2048, "12288,64"),
    "moe_qkv": (2048, "8192,512,512"),
}

# Cache geometries: attention layers, kv heads, bytes of a token's row in one head (fp8 256, bf16 512, 4-bit 128 + 64),
# tokens of a page; GDN layers, bytes of a slot's conv and SSM state in one layer.
POOLS = {
    "fp8": dict(layers=16, heads=4, row=256, page=64, gdn=48, conv=10240 * 3 * 2, ssm=48 * 128 * 128 * 4),
    "int4": dict(layers=16, heads=4, row=192, page=16, gdn=48, conv=10240 * 3 * 2, ssm=48 * 128 * 128 * 4),
    "bf16": dict(layers=10, heads=2, row=512, page=64, gdn=30, conv=8192 * 3 * 2, ssm=32 * 128 * 128 * 4),
}


def _adapters(name, proj, rows, rank, used, kind, x, none=0.0, mixed=False, K=0, slices=""):
    k, sl = PROJECTIONS[proj] if proj else (K, slices)
    c = {"op": "adapters", "rows": rows, "K": k, "slices": sl, "rank": rank, "used": used, "kind": kind, "x": x,
         "none": none, "mixed": mixed}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one request's decode step through the attention projection, the smallest call
        _adapters("adapters decode 1", "qkv", 1, 16, 1, "decode", "e4m3"),
        # the default batch of the engine, every request with an adapter of its own
        _adapters("adapters decode 8", "gate_up", 8, 16, 8, "decode", "e4m3"),
        # a full decode batch: adapters of different ranks, some shared, some rows without one
        _adapters("adapters decode 64", "in_proj", 64, 32, 24, "decode", "e4m3", none=0.125, mixed=True),
        # sizes that no vector width divides, ranks from 1 to 8
        _adapters("adapters odd", "", 37, 8, 5, "decode", "bf16", none=0.1, mixed=True, K=1250, slices="777,130,35"),
        # one prompt of 1.5k tokens
        _adapters("adapters prompt 1500", "down", 1500, 64, 1, "prompt", "bf16"),
        # a step of the engine's token budget: three prompts' chunks and 61 decoding requests
        _adapters("adapters mixed 4096", "in_proj", 4096, 16, 64, "mixed", "e4m3", none=0.02),
        # the largest: two budgets' rows of several prompts through the widest projection
        _adapters("adapters prompt 8192", "gate_up", 8192, 64, 8, "prompt", "bf16", none=0.05),
        # the second sample of a request over a 4-bit cache: one partly filled page, no GDN state
        {"name": "fork 1 page", "op": "fork", "pool": "int4", "blocks": 64, "slots": 0, "parents": 1, "children": 1},
        # eight samples of one request: the partly filled page and the state of every GDN layer
        {"name": "fork 8 samples", "op": "fork", "pool": "fp8", "blocks": 64, "slots": 10, "parents": 1, "children": 8},
        # several requests fork at once, other geometry, lengths that end anywhere in a page
        {"name": "fork 5 requests", "op": "fork", "pool": "bf16", "blocks": 131, "slots": 25, "parents": 5, "children": 3},
        # a small pool after a few requests left
        {"name": "compact 61", "op": "compact", "pool": "fp8", "blocks": 61, "live": 0.4, "seqs": 3},
        # a long-context 4-bit pool, half of it freed in no order
        {"name": "compact 6000", "op": "compact", "pool": "int4", "blocks": 6000, "live": 0.5, "seqs": 24},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["adapters", "adapters", "adapters", "fork", "compact"])
    if op == "adapters":
        kind = rng.choice(["decode", "prompt", "mixed"])
        rows = _log(rng, 1, 256) if kind == "decode" else _log(rng, 65, 8192)
        rank = rng.choice([8, 16, 32, 64])
        x = rng.choice(["bf16", "e4m3"])
        none = rng.choice([0.0, 0.05, 0.3])
        used = min(rows, _log(rng, 1, 64))
        mixed = rng.random() < 0.4
        proj = rng.choice(sorted(PROJECTIONS) + [""])
        if proj:
            return _adapters("", proj, rows, rank, used, kind, x, none, mixed)
        n = [_log(rng, 8, 9000) for _ in range(rng.randint(1, 3))]
        return _adapters("", "", rows, rank, used, kind, x, none, mixed, K=_log(rng, 16, 8704), slices=",".join(map(str, n)))
    pool = rng.choice(sorted(POOLS))
    if op == "fork":
        parents, children = rng.randint(1, 4), rng.randint(1, 4)
        while parents * (children + 1) > 9:
            parents, children = rng.randint(1, 4), rng.randint(1, 4)
        blocks = rng.randint(parents * (children + 1) + 1, 200)
        slots = rng.choice([0, parents * (children + 1) + 1])
        return {"op": "fork", "pool": pool, "blocks": blocks, "slots": slots, "parents": parents, "children": children}
    blocks = _log(rng, 30, 5900) if pool == "int4" else _log(rng, 30, 1100)
    return {"op": "compact", "pool": pool, "blocks": blocks, "live": rng.choice([0.2, 0.4, 0.6, 0.8]), "seqs": rng.randint(1, 32)}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _slices(case):
    return np.concatenate([[0], np.cumsum([int(n) for n in case["slices"].split(",")])]).tolist()


def _row_slots(case, seed):
    """Adapter slot of each row (-1: none): decode rows in any order, a prompt's rows side by side."""
    rng = np.random.default_rng(seed)
    T, used = case["rows"], case["used"]
    if case["kind"] == "decode":
        s = rng.permutation(np.concatenate([np.arange(used), rng.integers(0, used, T - used)]))
        s[rng.random(T) < case["none"]] = -1
        return s.astype(np.int32)
    # decoding requests first, then the prompts' chunks
    nd = min(max(0, used - 3), T // 4) if case["kind"] == "mixed" else 0
    prompts = min(used - nd, T - nd)
    cuts = np.sort(rng.choice(np.arange(1, T - nd), prompts - 1, replace=False)) if prompts > 1 else np.zeros(0, int)
    runs = np.repeat(np.arange(prompts), np.diff(np.concatenate([[0], cuts, [T - nd]])))
    s = np.concatenate([prompts + np.arange(nd), runs])
    if case["none"] > 0:
        # some requests use no adapter: a share of the decoding ones, or the last prompt's tail
        s[:nd][rng.random(nd) < case["none"]] = -1
        s[T - max(1, int(case["none"] * T)):] = -1
    return s.astype(np.int32)


def _prepare_adapters(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    T, K, R = case["rows"], case["K"], case["rank"]
    slices = _slices(case)
    S, N = len(slices) - 1, slices[-1]
    slots = _row_slots(case, seed)
    L = case["used"] + 1                                        # a slot that no row uses
    ranks = np.random.default_rng(seed + 1).integers(1, R + 1, L) if case["mixed"] else np.full(L, R)

    def normal(*shape, std):
        return torch.randn(*shape, device=DEVICE, generator=g) * std

    r = torch.tensor(ranks, dtype=torch.int32, device=DEVICE)
    keep = torch.arange(R, device=DEVICE)[None, :] < r[:, None]  # [L, R]: ranks beyond an adapter's own are zero
    a = (normal(L, S, R, K, std=K ** -0.5) * keep[:, None, :, None]).to(torch.bfloat16)
    b = (normal(L, N, R, std=0.05) * keep[:, None, :]).to(torch.bfloat16)
    scale = torch.rand(L, device=DEVICE, generator=g) * 2 + 0.5
    y = normal(T, N, std=1.0).to(torch.bfloat16)
    x = normal(T, K, std=1.0)
    if case["x"] == "e4m3":
        sx = x.abs().amax(1) / 448
        x = ((x / sx[:, None]).to(torch.float8_e4m3fn), sx)
    else:
        x = x.to(torch.bfloat16)
    state = {"op": "adapters", "x": x, "y": y, "a": a, "b": b, "scale": scale, "ranks": r, "slices": slices, "slots": slots}
    # rows of one adapter in tiles of at most 128, padded with row T
    groups = [np.flatnonzero(slots == s) for s in range(L)]
    width = max(1, min(128, max(len(q) for q in groups)))
    tiles = [(s, q[i:i + width]) for s, q in enumerate(groups) for i in range(0, len(q), width)] or [(0, np.zeros(0, int))]
    index = np.full((len(tiles), width), T)
    for i, (_, q) in enumerate(tiles):
        index[i, :len(q)] = q
    state["index"] = torch.tensor(index, device=DEVICE)
    state["tile_slot"] = torch.tensor([s for s, _ in tiles], device=DEVICE)
    if own:
        # kept by a serving program: the stacked adapters of this projection, and the step's rows by adapter
        from vllm_sly_radiance_b200.models.lora import AdapterBank, AdapterPlan
        state["bank"] = AdapterBank(a, b, scale, r, slices)
        state["plan"] = AdapterPlan.build(slots, L, DEVICE)
    return state


def _pool(case, seed):
    """Cache tensors of all layers as whole numbers (pages are moved bit by bit): k, v [layers, blocks, heads, page,
    row / 8], conv, ssm [gdn layers, slots, bytes / 8]."""
    p = POOLS[case["pool"]]
    g = torch.Generator(DEVICE).manual_seed(seed)

    def bits(*shape):
        return torch.randint(-2 ** 62, 2 ** 62, shape, device=DEVICE, generator=g, dtype=torch.int64)

    slots = case.get("slots", 0)
    s = {"k": bits(p["layers"], case["blocks"], p["heads"], p["page"], p["row"] // 8),
         "v": bits(p["layers"], case["blocks"], p["heads"], p["page"], p["row"] // 8)}
    if slots:
        s["conv"] = bits(p["gdn"], slots, p["conv"] // 8)
        s["ssm"] = bits(p["gdn"], slots, p["ssm"] // 8)
    if own:
        # kept by a serving program: the mover over its caches
        from vllm_sly_radiance_b200.engine.cache_moves import CacheMover
        from vllm_sly_radiance_b200.models.hybrid import ModelCaches
        s["mover"] = CacheMover(ModelCaches(list(s["k"]), list(s["v"]), list(s["conv"]) if slots else [],
                                            list(s["ssm"]) if slots else [], p["page"]))
    return s


def _fork_moves(case, seed):
    rng = np.random.default_rng(seed)
    n, c = case["parents"], case["children"]
    ids = 1 + rng.permutation(case["blocks"] - 1)[:n * (c + 1)].reshape(n, c + 1)
    tokens = rng.integers(1, POOLS[case["pool"]]["page"] + 1, n)
    blocks = [(int(r[0]), int(d), int(t)) for r, t in zip(ids, tokens) for d in r[1:]]
    slots = []
    if case["slots"]:
        sid = 1 + rng.permutation(case["slots"] - 1)[:n * (c + 1)].reshape(n, c + 1)
        slots = [(int(r[0]), int(d)) for r in sid for d in r[1:]]
    return blocks, slots


def _tables(case, seed):
    """Block tables of the sequences in use, padded with -1: blocks in no order, a page of the first sequence shared."""
    rng = np.random.default_rng(seed)
    n = max(case["seqs"], int((case["blocks"] - 1) * case["live"]))
    ids = 1 + rng.permutation(case["blocks"] - 1)[:n]
    parts = np.array_split(ids, case["seqs"])
    width = max(len(p) for p in parts) + 1
    t = np.full((len(parts), width), -1, dtype=np.int32)
    for i, p in enumerate(parts):
        row = np.concatenate([[parts[0][0]], p]) if i else p
        t[i, :len(row)] = row
    return t


def prepare(case, seed):
    if case["op"] == "adapters":
        return _prepare_adapters(case, seed)
    s = _pool(case, seed)
    s["op"] = case["op"]
    if case["op"] == "fork":
        s["moves"], s["slot_moves"] = _fork_moves(case, seed)
    else:
        s["tables"] = _tables(case, seed)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _adapters_plain(s):
    x = s["x"]
    x = x[0].float() * x[1][:, None] if isinstance(x, tuple) else x.float()
    idx, slot, sl = s["index"], s["tile_slot"], s["slices"]
    y = s["y"].float()
    xt = torch.cat([x, x.new_zeros(1, x.shape[1])])[idx]                             # [tiles, width, K]
    a = s["a"][slot].float()
    v = torch.bmm(xt, a.flatten(1, 2).transpose(1, 2)) * s["scale"][slot][:, None, None]
    v = v.unflatten(2, a.shape[1:3])                                                # [tiles, width, S, R]
    b = s["b"][slot].float()
    d = torch.cat([torch.bmm(v[:, :, i], b[:, sl[i]:sl[i + 1]].transpose(1, 2)) for i in range(len(sl) - 1)], 2)
    out = torch.cat([y, y.new_zeros(1, y.shape[1])])
    out[idx] = out[idx] + d
    return out[:-1].to(torch.bfloat16)


def _copy_plain(c, blocks):
    """Rows < tokens of every head of block dst = those of src, in all layers."""
    src, dst, n = (torch.tensor(q, device=c.device) for q in zip(*blocks))
    m, t = (torch.arange(c.shape[3], device=c.device)[None] < n[:, None]).nonzero(as_tuple=True)
    c[:, dst[m], :, t] = c[:, src[m], :, t]


def _fork_plain(s):
    _copy_plain(s["k"], s["moves"])
    _copy_plain(s["v"], s["moves"])
    if s["slot_moves"]:
        src, dst = (torch.tensor(q, device=DEVICE) for q in zip(*s["slot_moves"]))
        s["conv"][:, dst] = s["conv"][:, src]
        s["ssm"][:, dst] = s["ssm"][:, src]


def _compact_plain(s):
    t, blocks = s["tables"], s["k"].shape[1]
    used = np.zeros(blocks, bool)
    used[t[t > 0]] = True
    n = int(used.sum())
    src = n + 1 + np.flatnonzero(used[n + 1:])
    dst = 1 + np.flatnonzero(~used[1:n + 1])
    to = np.arange(blocks)
    to[src] = dst
    s["new_tables"] = np.where(t > 0, to[t], t).astype(np.int32)
    src, dst = torch.tensor(src, device=DEVICE), torch.tensor(dst, device=DEVICE)
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["new_tables"], n


def run(s):
    if s["op"] == "adapters":
        if own:
            from vllm_sly_radiance_b200.ops import kernels
            return kernels.lora_add(s["y"], s["x"], s["bank"], s["plan"])
        return _adapters_plain(s)
    caches = [s[n] for n in ("k", "v", "conv", "ssm") if n in s]
    if s["op"] == "fork":
        if own:
            s["mover"].copy(s["moves"], s["slot_moves"])
        else:
            _fork_plain(s)
        return caches
    tables, n = s["mover"].compact(s["tables"]) if own else _compact_plain(s)
    return caches, tables, n


def work(case):
    if case["op"] == "adapters":
        T, K, R = case["rows"], case["K"], case["rank"]
        slices = _slices(case)
        S, N = len(slices) - 1, slices[-1]
        r = (R + 1) / 2 if case["mixed"] else R                 # ranks are drawn from 1 .. R
        rows = T * (1 - case["none"])
        e = 1 if case["x"] == "e4m3" else 2
        return {"bytes": rows * K * e + 4 * T * N + 2 * case["used"] * r * (S * K + N), "flops": 2 * rows * r * (S * K + N)}
    p = POOLS[case["pool"]]
    page = 2 * p["layers"] * p["heads"] * p["page"] * p["row"]
    if case["op"] == "fork":
        state = p["gdn"] * (p["conv"] + p["ssm"]) if case["slots"] else 0
        return {"bytes": case["parents"] * (1 + case["children"]) * (page / 2 + state), "flops": 0}
    n = case["blocks"] * case["live"]                           # as many of the live pages as lie beyond the first n move
    return {"bytes": 2 * page * max(1, n * (1 - case["live"])), "flops": 0}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] != "adapters":
        return None                                             # pages are whole numbers: they have to be equal
    s = _prepare_adapters(case, seed)
    x = s["x"][0].double() * s["x"][1].double()[:, None] if isinstance(s["x"], tuple) else s["x"].double()
    out = s["y"].double()
    for l in sorted(set(s["slots"].tolist()) - {-1}):
        rows = torch.tensor(np.flatnonzero(s["slots"] == l), device=DEVICE)
        for i, (n0, n1) in enumerate(zip(s["slices"], s["slices"][1:])):
            low = x[rows] @ s["a"][l, i].double().T
            out[rows, n0:n1] += s["scale"][l].double() * (low @ s["b"][l, n0:n1].double().T)
    return out
