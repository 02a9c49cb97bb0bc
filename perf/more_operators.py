"""Cases that measure the mixture-of-experts operators: router, sorting plan, product with an epilogue, weighted sum.

Four operators: "route" picks each token's experts and their weights from the router's logits; "plan" sorts the (token,
slot) pairs by expert; "linear" multiplies rows by their expert's weight (or all rows by one weight) with bias, SwiGLU,
row scale and residual in the epilogue; "combine" adds up each token's expert rows by weight, beside the shared expert's.

`run` computes them in plain torch operations, or with the framework's kernels where `own` is true."""
import numpy as np
import torch

own = False

DEVICE = "cuda"


def _route(name, rows, experts, k, score, dtype="fp32", bias=False, groups=1, top_groups=1, renorm=True, scale=1.0):
    c = {"op": "route", "rows": rows, "experts": experts, "k": k, "score": score, "dtype": dtype, "bias": bias,
         "groups": groups, "top_groups": top_groups, "renorm": renorm, "scale": scale}
    return {"name": name, **c} if name else c


def _plan(name, rows, experts, k, first=0, local=0):
    c = {"op": "plan", "rows": rows, "experts": experts, "k": k, "first": first, "local": local or experts}
    return {"name": name, **c} if name else c


def _linear(name, rows, K, N, experts=1, k=1, act="none", by_token=False, bias=False, residual=False, scale=False):
    c = {"op": "linear", "rows": rows, "K": K, "N": N, "experts": experts, "k": k, "act": act, "by_token": by_token,
         "bias": bias, "residual": residual, "scale": scale}
    return {"name": name, **c} if name else c


def _combine(name, rows, width, k, experts, shared):
    c = {"op": "combine", "rows": rows, "width": width, "k": k, "experts": experts, "shared": shared}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one request's decode step: the MoE hybrid's 256 experts, top-8 of a softmax
        _route("route 1", 1, 256, 8, "softmax"),
        # a batch of odd size, 60 experts, bf16 logits with ties, weights left as they are
        _route("route odd", 61, 60, 4, "softmax", dtype="bf16", renorm=False),
        # a long prompt's step, sigmoid scores with a balance bias, 4 of 8 groups
        _route("route 8192 groups", 8192, 256, 8, "sigmoid", bias=True, groups=8, top_groups=4, scale=2.5),
        # a full decode batch
        _plan("plan 64", 64, 256, 8),
        # two long prompts' tokens on a rank that owns half of the experts
        _plan("plan 16384 half", 16384, 256, 8, first=128, local=128),
        # one request's decode step: eight experts' gate and up rows, SwiGLU
        _linear("experts up 1", 1, 2048, 1024, 256, 8, act="swiglu", by_token=True),
        # a full decode batch: most experts in use, one to a few rows each
        _linear("experts down 64", 64, 512, 2048, 256, 8),
        # small experts of sizes that no tile divides, with a bias
        _linear("experts odd", 37, 200, 154, 10, 3, act="swiglu", by_token=True, bias=True),
        # the largest: 8192 tokens, 256 rows an expert on average, from 30 to over 1000
        _linear("experts up 8192", 8192, 2048, 1024, 256, 8, act="swiglu", by_token=True),
        # the shared expert's second product at the engine's token budget: gated, added to the routed sum
        _linear("shared down 4096", 4096, 512, 2048, residual=True, scale=True),
        # a full decode batch
        _combine("combine 64", 64, 2048, 8, 256, False),
        # a long prompt, with the shared expert's gated rows
        _combine("combine 8192", 8192, 2048, 8, 256, True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["route", "plan", "linear", "linear", "linear", "combine"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        experts = groups * _log(rng, 8, 512) if groups == 1 else groups * rng.randint(4, 48)
        k = rng.randint(1, 8)
        tops = 1 if groups == 1 else rng.randint(2, groups)
        return _route("", _log(rng, 1, 8192), experts, k, rng.choice(["softmax", "sigmoid"]), rng.choice(["fp32", "bf16"]),
                      rng.random() < 0.5, groups, tops, rng.random() < 0.7, rng.choice([1.0, 2.5]))
    if op == "plan":
        experts = _log(rng, 8, 512)
        part = rng.choice([1, 1, 2, 4])
        local = experts // part
        return _plan("", _log(rng, 1, 16384), experts, rng.randint(1, 8), local * rng.randrange(part), local)
    if op == "combine":
        return _combine("", _log(rng, 1, 8192), 8 * _log(rng, 8, 256), rng.randint(1, 8), _log(rng, 8, 256), rng.random() < 0.5)
    kind = rng.choice(["up", "down", "odd", "shared"])
    rows = _log(rng, 1, 4096)
    if kind == "up":
        return _linear("", rows, 2048, 1024, 256, 8, act="swiglu", by_token=True)
    if kind == "down":
        return _linear("", rows, 512, 2048, 256, 8)
    if kind == "shared":
        up = rng.random() < 0.5
        return _linear("", rows, 2048 if up else 512, 1024 if up else 2048, act="swiglu" if up else "none", residual=not up,
                       scale=not up)
    experts = rng.randint(1, 64)
    return _linear("", rows, 8 * _log(rng, 2, 160), 2 * _log(rng, 4, 700), experts, rng.randint(1, min(8, experts)),
                   rng.choice(["none", "swiglu"]), rng.random() < 0.5, rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(DEVICE).manual_seed(seed)


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, device=DEVICE, generator=g) * std


def _logits(g, rows, experts):
    """Router logits: some experts are more popular than others."""
    return _normal(g, rows, experts) * 1.5 + _normal(g, experts, std=0.5)


def _ids(g, rows, experts, k):
    return torch.topk(_logits(g, rows, experts), k, dim=1).indices


def _sorted(ids):
    """order: (token, slot) number of each row, rows of one expert side by side; starts of the experts; row of each pair."""
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(len(order), device=order.device)
    return order, flat[order], pos.view(ids.shape)


def _own_plan(ids, experts):
    from vllm_sly_radiance_b200.ops import kernels
    return kernels.moe_plan(ids, experts)


def _prepare_linear(case, seed):
    g = _gen(seed)
    T, K, N, E, k = case["rows"], case["K"], case["N"], case["experts"], case["k"]
    w = torch.empty(E, N, K, dtype=torch.bfloat16, device=DEVICE)
    for part in w.split(32):
        part.copy_(torch.randn(part.shape, device=DEVICE, generator=g) * K ** -0.5)
    s = {"op": "linear", "act": case["act"], "w": w, "bias": _normal(g, E, N, std=0.1).to(torch.bfloat16) if case["bias"] else None}
    ids = _ids(g, T, E, k)
    order, expert, _ = _sorted(ids)
    R, width = T * k, N // 2 if case["act"] == "swiglu" else N
    s["x"] = _normal(g, T if case["by_token"] else R, K).to(torch.bfloat16)
    s["by_token"] = case["by_token"]
    s["residual"] = _normal(g, R, width).to(torch.bfloat16) if case["residual"] else None
    s["scale"] = torch.rand(R, device=DEVICE, generator=g) if case["scale"] else None
    # rows in tiles of one expert, at most 128 each, padded with row R
    e = expert.cpu().numpy()
    groups = [np.flatnonzero(e == i) for i in np.unique(e)]
    wide = min(128, max(len(q) for q in groups))
    tiles = [(int(e[q[0]]), q[i:i + wide]) for q in groups for i in range(0, len(q), wide)]
    index = np.full((len(tiles), wide), R)
    for i, (_, q) in enumerate(tiles):
        index[i, :len(q)] = q
    s["index"] = torch.tensor(index, device=DEVICE)
    s["tile_expert"] = torch.tensor([t for t, _ in tiles], device=DEVICE)
    s["row_in"] = order // k if case["by_token"] else torch.arange(R, device=DEVICE)
    if own:
        # kept by a serving program: the layer's weights, and the step's plan
        from vllm_sly_radiance_b200.models.layers import LinearBank
        s["bank"] = LinearBank(w, s["bias"], act=case["act"])
        s["plan"] = _own_plan(ids, E) if E > 1 else None
    return s


def prepare(case, seed):
    if case["op"] == "linear":
        return _prepare_linear(case, seed)
    g = _gen(seed)
    T, k = case["rows"], case["k"]
    if case["op"] == "route":
        dtype = {"fp32": torch.float32, "bf16": torch.bfloat16}[case["dtype"]]
        s = {n: case[n] for n in ("op", "k", "score", "groups", "top_groups", "renorm", "scale")}
        s["logits"] = _logits(g, T, case["experts"]).to(dtype)
        s["bias"] = _normal(g, case["experts"], std=0.1) if case["bias"] else None
        return s
    ids = _ids(g, T, case["experts"], k)
    if case["op"] == "plan":
        return {"op": "plan", "ids": ids, "first": case["first"], "local": case["local"]}
    s = {"op": "combine", "weights": torch.softmax(_normal(g, T, k), 1)}
    s["rows"] = _normal(g, T * k, case["width"]).to(torch.bfloat16)
    s["shared"] = _normal(g, T, case["width"]).to(torch.bfloat16) if case["shared"] else None
    s["gate"] = _normal(g, T) if case["shared"] else None
    s["pos"] = _sorted(ids)[2]
    if own:
        s["plan"] = _own_plan(ids, case["experts"])             # kept from the step's experts
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _route_plain(s):
    """The choice is made in 64 bits: scores next to one another decide which expert a token goes to."""
    l = s["logits"].double()
    score = torch.softmax(l, 1) if s["score"] == "softmax" else torch.sigmoid(l)
    c = score + s["bias"].double() if s["bias"] is not None else score
    if s["groups"] > 1:
        g = c.view(len(c), s["groups"], -1)
        value = torch.topk(g, 2, dim=2).values.sum(2) if s["bias"] is not None else g.amax(2)
        best = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, best, True)
        c = torch.where(keep[:, :, None], g, -torch.inf).reshape(c.shape)
    ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :s["k"]]
    w = torch.gather(score, 1, ids)
    if s["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return ids, (w * s["scale"]).float()


def _plan_plain(s):
    flat = s["ids"].reshape(-1) - s["first"]
    here = (flat >= 0) & (flat < s["local"])
    key = torch.where(here, flat, s["local"])
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(s["local"] + 1, dtype=torch.long, device=key.device).scatter_add_(0, key, torch.ones_like(key))
    row = torch.empty_like(order)
    row[order] = torch.arange(len(order), device=order.device)
    pos = torch.where(here, row, -1).view(s["ids"].shape)
    return torch.where(here[order], order, -1).int(), pos.int(), counts[:-1].int()


def _linear_plain(s):
    idx, e = s["index"], s["tile_expert"]
    R = len(s["row_in"])
    x = s["x"].float()[s["row_in"]]
    x = torch.cat([x, x.new_zeros(1, x.shape[1])])[idx]                              # [tiles, width, K]
    y = torch.bmm(x, s["w"][e].float().transpose(1, 2))
    if s["bias"] is not None:
        y = y + s["bias"][e].float()[:, None]
    if s["act"] == "swiglu":
        gate, up = y.chunk(2, 2)
        y = gate / (1 + torch.exp(-gate)) * up
    out = y.new_empty(R + 1, y.shape[2])
    out[idx] = y
    out = out[:R]
    if s["scale"] is not None:
        out = out * s["scale"][:, None]
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(torch.bfloat16)


def _combine_plain(s):
    out = torch.bmm(s["weights"][:, None], s["rows"][s["pos"]].float())[:, 0]
    if s["shared"] is not None:
        out = out + s["shared"].float() / (1 + torch.exp(-s["gate"]))[:, None]
    return out.to(torch.bfloat16)


def run(s):
    if not own:
        return {"route": _route_plain, "plan": _plan_plain, "linear": _linear_plain, "combine": _combine_plain}[s["op"]](s)
    from vllm_sly_radiance_b200.ops import kernels
    if s["op"] == "route":
        return kernels.moe_route(s["logits"], s["k"], score=s["score"], bias=s["bias"], groups=s["groups"],
                                 top_groups=s["top_groups"], renormalize=s["renorm"], scale=s["scale"])
    if s["op"] == "plan":
        plan = kernels.moe_plan(s["ids"], s["local"], first=s["first"])
        return plan.order, plan.pos, plan.counts
    if s["op"] == "linear":
        return kernels.linear_fused(s["x"], s["bank"], plan=s["plan"], by_token=s["by_token"] and s["plan"] is not None,
                                    scale=s["scale"], residual=s["residual"])
    return kernels.moe_combine(s["rows"], s["plan"], s["weights"], shared=s["shared"], gate=s["gate"])


def work(case):
    T, k = case["rows"], case["k"]
    if case["op"] == "route":
        e = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": T * case["experts"] * e + 12 * T * k, "flops": 2 * T * case["experts"]}
    if case["op"] == "plan":
        return {"bytes": 16 * T * k, "flops": 0}
    if case["op"] == "combine":
        rows = T * k + T + (T if case["shared"] else 0)
        return {"bytes": 2 * rows * case["width"] + 8 * T * k, "flops": 2 * T * k * case["width"]}
    K, N, E, R = case["K"], case["N"], case["experts"], T * k
    used = E * (1 - (1 - k / E) ** T)                           # experts that some token goes to, were they all alike
    width = N // 2 if case["act"] == "swiglu" else N
    rows = 2 * K * (T if case["by_token"] else R) + 2 * R * width * (2 if case["residual"] else 1)
    return {"bytes": 2 * used * N * K + rows, "flops": 2 * R * N * K}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def _route_exact(s):
    l = s["logits"].double().cpu().numpy()
    with np.errstate(over="ignore"):
        score = 1 / (1 + np.exp(-l))
    if s["score"] == "softmax":
        score = np.exp(l - l.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    c = score + (s["bias"].double().cpu().numpy() if s["bias"] is not None else 0)
    if s["groups"] > 1:
        parts = np.sort(c.reshape(len(c), s["groups"], -1), axis=2)
        value = parts[:, :, -2:].sum(2) if s["bias"] is not None else parts[:, :, -1]
        rank = np.argsort(np.argsort(-value, axis=1, kind="stable"), axis=1)
        c = np.where(np.repeat(rank < s["top_groups"], parts.shape[2], axis=1), c, -np.inf)
    ids = np.argsort(-c, axis=1, kind="stable")[:, :s["k"]]
    w = np.take_along_axis(score, ids, 1)
    if s["renorm"]:
        w = w / w.sum(1, keepdims=True)
    return None, torch.tensor(w * s["scale"], device=DEVICE)


def exact(case, seed):
    if case["op"] == "plan":
        return None                                             # whole numbers: they have to be equal
    s = prepare(case, seed)
    if case["op"] == "route":
        return _route_exact(s)
    if case["op"] == "combine":
        w, pos = s["weights"].double(), s["pos"]
        out = torch.zeros(len(w), s["rows"].shape[1], dtype=torch.double, device=DEVICE)
        for j in range(w.shape[1]):
            out += w[:, j:j + 1] * s["rows"][pos[:, j]].double()
        if s["shared"] is not None:
            out += torch.sigmoid(s["gate"].double())[:, None] * s["shared"].double()
        return out
    row_in, idx = s["row_in"], s["index"]
    R = len(row_in)
    out = None
    for e in sorted(set(s["tile_expert"].tolist())):
        rows = idx[s["tile_expert"] == e].flatten()
        rows = rows[rows < R]
        y = s["x"][row_in[rows]].double() @ s["w"][e].double().T
        if s["bias"] is not None:
            y += s["bias"][e].double()
        if s["act"] == "swiglu":
            n = y.shape[1] // 2
            y = y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
        if out is None:
            out = torch.zeros(R, y.shape[1], dtype=torch.double, device=DEVICE)
        out[rows] = y
    if s["scale"] is not None:
        out *= s["scale"].double()[:, None]
    if s["residual"] is not None:
        out += s["residual"].double()
    return out
