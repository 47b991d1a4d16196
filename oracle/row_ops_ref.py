"""The training step's row operators in float64 on the CPU, from their formulas, with the
gradients written out and, beside each result, the scale its rounding errors go by (the sum of
the magnitudes that meet in it), from which the tests derive their tolerances."""

from __future__ import annotations

import torch

INF = float("inf")


def _turn(x, cos, sin, interleaved, back=False):
    """The rotation (or its transpose) of x (..., tokens, heads, dim); cos, sin (..., tokens, half)."""
    half = cos.shape[-1]
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    s = -s if back else s
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y


def angles(q, cos, sin, positions):
    """Rows of the tables for q's tokens, NaN outside the tables; None without tables."""
    if cos is None:
        return None
    t = torch.arange(q.shape[-3]) if positions is None else positions.long()
    t = t.expand(q.shape[:-2])
    inside = (t >= 0) & (t < cos.shape[0])
    row = t.clamp(0, max(cos.shape[0] - 1, 0))
    return [torch.where(inside[..., None], x.double()[row], float("nan")) for x in (cos, sin)]


def norm_rope(x, w, turned, eps, interleaved):
    """(y, scale) of queries or keys."""
    x = x.double()
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r * (1 if w is None else w.double())
    y = n if turned is None else _turn(n, *turned, interleaved)
    if turned is not None:
        y = torch.where(turned[0].isnan().any(-1)[..., None, None], float("nan"), y)
    return y, n.abs().amax(-1, keepdim=True).expand_as(n)


def norm_rope_grad(x, w, dy, turned, eps, interleaved):
    """(dx, its scale, dw, its scale)."""
    x, dy = x.double(), dy.double()
    ww = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    u = dy if turned is None else _turn(dy, *turned, interleaved, back=True)
    g = u * ww
    dx = r * (g - x * r * r * (g * x).mean(-1, keepdim=True))
    top = g.abs().amax(-1, keepdim=True)
    lead = tuple(range(x.dim() - 1))
    return (dx, r * top * (1 + (x * r).abs()), (u * x * r).sum(lead), (u * x * r).abs().sum(lead))


def route(z, k, mask=None, normalize=True):
    """dict of gates, experts, counts, balance, z and what the gradient needs."""
    z = z.double()
    n, e = z.shape
    on = ~((z == -INF).all(1)) if mask is None else mask & ~((z == -INF).all(1))
    experts = torch.full((n, k), -1)
    gates = torch.zeros(n, k, dtype=torch.float64)
    p = torch.zeros_like(z)
    lse = torch.zeros(n, dtype=torch.float64)
    for t in range(n):
        if not on[t]:
            continue
        row = z[t]
        order = sorted(range(e), key=lambda i: (0, 0, i) if row[i].isnan() else (1, -float(row[i]), i))
        order = [i for i in order if row[i] != -INF][:k]
        m = row.max()
        p[t] = torch.exp(row - m) / torch.exp(row - m).sum()
        lse[t] = m + torch.log(torch.exp(row - m).sum())
        experts[t, :len(order)] = torch.tensor(order)
        chosen = p[t, order]
        gates[t, :len(order)] = chosen / chosen.sum() if normalize else chosen
    kept = int(on.sum())
    counts = torch.bincount(experts[experts >= 0], minlength=e)
    mean = p.sum(0) / kept if kept else torch.zeros(e, dtype=torch.float64)
    balance = e * (counts.double() / (k * kept) * mean).sum() if kept else torch.zeros((), dtype=torch.float64)
    zloss = lse.square().sum() / kept if kept else torch.zeros((), dtype=torch.float64)
    return dict(gates=gates, experts=experts, counts=counts, balance=balance, z=zloss, p=p, lse=lse,
                on=on, kept=kept, normalize=normalize)


def route_grad(r, dgates, dbalance, dz):
    """(dlogits, scale) for a result of route()."""
    n, e = r["p"].shape
    k, kept, p = r["experts"].shape[1], r["kept"], r["p"]
    if not kept:
        return torch.zeros_like(p), torch.zeros_like(p)
    a = dbalance * e * r["counts"].double() / (k * kept * kept)
    zpart = 2 * dz / kept * r["lse"][:, None]
    d = p * (a - (p * a).sum(1, keepdim=True) + zpart)
    scale = p * (a.abs().max() * 2 + zpart.abs())
    dgates = torch.where(r["experts"] >= 0, dgates.double(), 0.0)
    g = r["gates"]
    inner = (g * dgates).sum(1, keepdim=True)
    size = (g * dgates).abs().sum(1, keepdim=True)
    at = torch.where(r["experts"] >= 0, r["experts"], e)

    def put(v):
        return torch.zeros(n, e + 1, dtype=torch.float64).scatter_(1, at, v)[:, :e]

    if r["normalize"]:
        d = d + put(g * (dgates - inner))
    else:
        d = d + put(g * dgates) - p * inner
        scale = scale + p * size
    scale = scale + put(g * (dgates.abs() + size))
    off = ~r["on"][:, None]
    return d.masked_fill(off, 0.0), scale.masked_fill(off, 0.0)


def logprobs(x, tokens, temperature=1.0):
    """(logp, p): rows with a negative token 0, tokens past the end NaN."""
    z = x.double() / temperature
    v = z.shape[1]
    ls = torch.log_softmax(z, 1)
    got = ls.gather(1, tokens.clamp(0, v - 1)[:, None])[:, 0]
    got = torch.where(tokens >= v, float("nan"), got)
    return torch.where(tokens < 0, 0.0, got), ls.exp()


def logprobs_grad(p, tokens, g, temperature=1.0):
    """(dx, scale) of sum g logp; rows with g = 0 or a negative token are 0."""
    n, v = p.shape
    g = torch.where(tokens < 0, 0.0, g.double()) / temperature
    one = torch.zeros(n, v + 1, dtype=torch.float64).scatter_(
        1, torch.where((tokens < 0) | (tokens >= v), v, tokens)[:, None], 1.0)[:, :v]
    d = g[:, None] * (one - p)
    d = torch.where((tokens >= v)[:, None] & (g != 0)[:, None], float("nan"), d)
    out = (g == 0)[:, None]
    return d.masked_fill(out, 0.0), (g.abs()[:, None] * (one + p)).masked_fill(out, 0.0)


def policy(logp, old, adv, w, ref, low, high, beta):
    """(loss, slope g, scale of the loss per unit of logp's error) from the rows' logp."""
    on = w != 0
    old, adv, w = old.double(), adv.double(), torch.where(on, w.double(), 0.0)
    r = torch.exp(logp - old)
    term = -torch.minimum(r * adv, r.clamp(1 - low, 1 + high) * adv)
    cut = torch.where(adv >= 0, r > 1 + high, r < 1 - low)
    slope = torch.where(cut, 0.0, -r * adv)
    size = (r * adv).abs()
    if ref is not None:
        ahead = ref.double() - logp
        term = term + beta * (torch.exp(ahead) - ahead - 1)
        slope = slope + beta * (1 - torch.exp(ahead))
        size = size + beta * (torch.exp(ahead) + ahead.abs() + 1)

    def kept(v):
        return torch.where(on, w * v, 0.0)

    return kept(term).sum(), kept(slope), torch.where(on, w.abs() * size, 0.0).sum(), \
        torch.where(on, w.abs() * size, 0.0)
