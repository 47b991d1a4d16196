"""Tokens sorted by expert and back, the experts' products and the AdamW step in float64 on the CPU,
from their definitions, with the gradients written out and, beside a result, the scale its rounding
errors go by (the sum of the magnitudes that meet in it), from which the tests derive tolerances."""

from __future__ import annotations

import torch


def order(experts, n):
    """(slots, offsets) of (tokens, k) experts: a choice's row is the number of kept choices of lower
    experts and of earlier ones of its own; an empty one's is behind them all."""
    flat = [e if 0 <= e < n else n for e in experts.flatten().tolist()]
    counts = [flat.count(e) for e in range(n + 1)]
    starts = [sum(counts[:e]) for e in range(n + 1)]
    seen, slots = [0] * (n + 1), []
    for e in flat:
        row = starts[e] + seen[e]
        seen[e] += 1
        slots.append(row if e < n else -1 - row)
    return (torch.tensor(slots, dtype=torch.int32).view(experts.shape),
            torch.tensor(starts, dtype=torch.int32))


def choices(slots):
    """(token, choice, row) of every kept choice, as three index tensors."""
    t, j = (slots >= 0).nonzero(as_tuple=True)
    return t, j, slots[t, j].long()


def dispatch(x, slots):
    rows = torch.zeros(slots.numel(), x.shape[1], dtype=torch.float64)
    t, _, at = choices(slots)
    rows[at] = x.double()[t]
    return rows


def combine(rows, slots, gates):
    """(y, scale)."""
    t, j, at = choices(slots)
    part = rows.double()[at]
    if gates is not None:
        part = part * gates.double()[t, j, None]
    y = torch.zeros(slots.shape[0], rows.shape[1], dtype=torch.float64)
    return y.index_add(0, t, part), y.index_add(0, t, part.abs())


def combine_grad(rows, slots, gates, dy):
    """(drows, dgates, scale of dgates)."""
    t, j, at = choices(slots)
    d = dy.double()[t]
    drows = torch.zeros(rows.shape, dtype=torch.float64)
    drows[at] = d * gates.double()[t, j, None]
    part = d * rows.double()[at]
    dgates, scale = (torch.zeros(slots.shape, dtype=torch.float64) for _ in range(2))
    dgates[t, j], scale[t, j] = part.sum(1), part.abs().sum(1)
    return drows, dgates, scale


def spans(offsets):
    return list(zip(offsets.tolist(), offsets.tolist()[1:]))


def linear(rows, weight, offsets):
    """(y, scale)."""
    y, scale = (torch.zeros(rows.shape[0], weight.shape[1], dtype=torch.float64) for _ in range(2))
    for (a, b), w in zip(spans(offsets), weight.double()):
        x = rows[a:b].double()
        y[a:b], scale[a:b] = x @ w.T, x.abs() @ w.abs().T
    return y, scale


def linear_grad(rows, weight, offsets, dy):
    """(drows, its scale, dweight, its scale)."""
    dx, sx = (torch.zeros(rows.shape, dtype=torch.float64) for _ in range(2))
    dw, sw = (torch.zeros(weight.shape, dtype=torch.float64) for _ in range(2))
    for e, (a, b) in enumerate(spans(offsets)):
        x, d, w = rows[a:b].double(), dy[a:b].double(), weight[e].double()
        dx[a:b], sx[a:b] = d @ w, d.abs() @ w.abs()
        dw[e], sw[e] = d.T @ x, d.abs().T @ x.abs()
    return dx, sx, dw, sw


def adamw(p, g, m, v, step, lr, wd, betas, eps, maximize=False):
    """(p, m, v, root of v, size of the change) after step number `step` (1 is the first)."""
    b1, b2 = betas
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = -g if maximize else g
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    change = lr / (1 - b1**step) * m / (v.sqrt() / (1 - b2**step) ** 0.5 + eps)
    return (1 - lr * wd) * p - change, m, v, v.sqrt(), change
