"""Definitions of the mixture-of-experts operators in 64 bits, and how far their kernels may be from them."""
import torch

BF16 = 2.0 ** -8            # half a step of bf16, relative


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, renorm=True, scale=1.0):
    l = logits.double().cpu()
    s = torch.softmax(l, 1) if score == "softmax" else 1 / (1 + torch.exp(-l))
    c = s if bias is None else s + bias.double().cpu()
    T, E = l.shape
    ids, w = torch.empty(T, k, dtype=torch.long), torch.empty(T, k, dtype=torch.double)
    for t in range(T):
        cand = list(range(E))
        if groups > 1:
            n = E // groups
            vals = []
            for g in range(groups):
                v = sorted(c[t, g * n:(g + 1) * n].tolist(), reverse=True)
                vals.append(v[0] if bias is None else v[0] + v[1])
            best = sorted(range(groups), key=lambda g: (-vals[g], g))[:top_groups]
            cand = [e for g in sorted(best) for e in range(g * n, (g + 1) * n)]
        order = sorted(cand, key=lambda e: (-float(c[t, e]), e))[:k]
        ids[t] = torch.tensor(order)
        w[t] = s[t, order]
    if renorm:
        w = w / w.sum(1, keepdim=True)
    return ids, w * scale


def plan(ids, E, first=0):
    T, k = ids.shape
    rows = sorted((int(e) - first, f) for f, e in enumerate(ids.flatten().tolist()) if first <= e < first + E)
    order = [f for _, f in rows] + [-1] * (T * k - len(rows))
    pos = [-1] * (T * k)
    for r, (_, f) in enumerate(rows):
        pos[f] = r
    counts = [sum(1 for e, _ in rows if e == i) for i in range(E)]
    return order, torch.tensor(pos, dtype=torch.long).view(T, k).tolist(), counts


def linear(x, w, bias, act, rows, experts, scale=None, residual=None):
    """Row i of out: x[rows[i]] with weight experts[i].  -> value and bound of the error, both in 64 bits.

    Sums of K products in 32 bits, aligned and cut off by the tensor cores: at most K 2^-23 of the sum of magnitudes.
    exp, its argument and the quotient: 2^-19 of g / (1 + e^-g).  Scale and residual: three roundings in 32 bits."""
    x, w = x.double(), w.double()
    y = torch.einsum("rk,rnk->rn", x[rows], w[experts]) if len(rows) else x.new_zeros(0, w.shape[1])
    e = torch.einsum("rk,rnk->rn", x[rows].abs(), w[experts].abs()) * (w.shape[2] * 2.0 ** -23) if len(rows) else y
    if bias is not None:
        y = y + bias.double()[experts]
        e = e + y.abs() * 2.0 ** -24
    if act == "swiglu":
        n = y.shape[1] // 2
        g, u, eg, eu = y[:, :n], y[:, n:], e[:, :n], e[:, n:]
        s = g * torch.sigmoid(g)
        y = s * u
        e = 1.1 * eg * (u.abs() + eu) + s.abs() * eu + 2.0 ** -19 * y.abs()
    if scale is not None:
        y, e = y * scale.double()[:, None], e * scale.double().abs()[:, None]
        e = e + 2.0 ** -24 * y.abs()
    if residual is not None:
        y = y + residual.double()
    e = e + 2.0 ** -23 * y.abs()
    return y, e + BF16 * (y.abs() + e) + 1e-38


def combine(rows, pos, w, shared=None, gate=None):
    pos = torch.as_tensor(pos)
    T, k = pos.shape
    out = torch.zeros(T, rows.shape[1], dtype=torch.double, device=rows.device)
    mag = torch.zeros_like(out)
    for t in range(T):
        for j in range(k):
            if pos[t, j] >= 0:
                v = float(w[t, j]) * rows[pos[t, j]].double()
                out[t] += v
                mag[t] += v.abs()
    if shared is not None:
        v = shared.double() if gate is None else torch.sigmoid(gate.double())[:, None] * shared.double()
        out += v
        mag += v.abs() * 2.0 ** 5                  # the gate's exp and quotient: 2^-19 of it
    e = (k + 2) * 2.0 ** -24 * mag
    return out, e + BF16 * (out.abs() + e) + 1e-38


def near(got, want, bound):
    """Everything within its bound; names the worst place otherwise."""
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}: got "
                           f"{float(got[tuple(bad.nonzero()[0])])}, want {float(want[tuple(bad.nonzero()[0])])}")
