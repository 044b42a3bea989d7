"""Plain 64-bit code that the tests of the 8-bit products, the sampling distributions and the
verification of drafts compare with."""
from __future__ import annotations

import math

import numpy as np
import torch


# -- products ------------------------------------------------------------------
def rows_to_8_bits(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(integers as float64, scales as float64) of the rows of x (any float type)."""
    x = x.detach().cpu().float().numpy()
    m = np.abs(x).max(1)
    with np.errstate(all="ignore"):
        s = np.where(np.isfinite(m), m, np.float32(np.nan)).astype(np.float32) / np.float32(127)
        q = np.rint(x / s[:, None])
    q = np.where((s > 0)[:, None], np.clip(q, -127, 127), 0)
    return torch.from_numpy(q).double(), torch.from_numpy(s).double()


def linear(x, w, bias=None):
    """(y, how far fp32 scaling may be off) in float64, before y's own rounding."""
    (qx, sx), (qw, sw) = rows_to_8_bits(x), rows_to_8_bits(w)
    y = (qx @ qw.T) * sx[:, None] * sw
    b = torch.zeros(len(sw), dtype=torch.float64) if bias is None else bias.detach().cpu().double()
    # the sum as fp32, the scales' product, the product of both, the bias added: half a step each
    return y + b, 2.0**-24 * (3.001 * y.abs() + (y + b).abs())


# -- distributions ----------------------------------------------------------------
def probs(row: np.ndarray, temp: float, top_k: int = -1, top_p: float = 1.0, min_p: float = 0.0) -> np.ndarray:
    """One row's distribution in float64, from float32 logits."""
    row = row.astype(np.float32) + np.float32(0)
    out = np.zeros(len(row))
    ok = ~np.isnan(row)
    if not (ok & (row > -np.inf)).any():
        return out
    if np.float32(temp) < np.float32(1e-5):
        out[int(np.argmax(np.where(ok, row, -np.inf)))] = 1.0
        return out
    with np.errstate(all="ignore"):
        top = np.finfo(np.float32).max
        x = np.where(np.isfinite(row), np.clip(row / np.float32(temp), -top, top), row)  # what is finite stays finite
        x = np.where(ok, x, -np.inf).astype(np.float64)
        m = x.max()
        e = np.where(x == m, 1.0, np.exp(x - m))
    e[~ok] = 0.0
    order = np.argsort(-x, kind="stable")
    order = order[ok[order]]
    if min_p > 0:
        order = order[e[order] >= float(np.float32(min_p))]
    if 0 < top_k < len(row):
        order = order[:top_k]
    if np.float32(top_p) < 1:
        total, cum = math.fsum(e[order]), np.cumsum(e[order])
        order = order[cum - e[order] < float(np.float32(top_p)) * total]
    out[order] = e[order] / math.fsum(e[order])
    return out


# -- verification -------------------------------------------------------------------
def verify_tree(tokens, parents, P, Q, u, distinct=False) -> list[int]:
    """The targets of one tree (lists; P and Q float64 arrays [rows, V]), -1 off the path."""
    n, V = len(tokens), P.shape[1]
    out = [-1] * n
    at = 0
    while True:
        A, c, before, nxt = 0.0, 1.0, 0.0, None
        for i in range(at + 1, n):
            if parents[i] != at:
                continue
            x = tokens[i]
            p, q = (P[at, x], Q[at, x]) if 0 <= x < V else (0.0, 0.0)
            scale = c
            if distinct and max(1.0 - before, q) > 0:
                scale = c / max(1.0 - before, q)
            if u[i] * q * scale < max(p - A * q, 0.0):
                nxt = i
                break
            A, before = A + scale, before + q
            c = np.maximum(P[at] - A * Q[at], 0.0).sum()
        if nxt is not None:
            out[at] = tokens[nxt]
            at = nxt
            continue
        w = np.maximum(P[at] - A * Q[at], 0.0) if A else P[at]
        if not w.sum() > 0:
            w = P[at]
        if not w.sum() > 0:
            return out
        cum = np.cumsum(w)
        t = u[0] * cum[-1]
        hits = np.nonzero((cum > t) & (w > 0))[0]
        out[at] = int(hits[0]) if len(hits) else int(np.nonzero(w > 0)[0][-1])
        follow = [i for i in range(at + 1, n) if parents[i] == at and tokens[i] == out[at]]
        if not follow:
            return out
        at = follow[0]


def verify(tokens, parents, P, Q, u, starts, max_nodes, distinct=False, before=-1) -> list[int]:
    """The targets of a step's rows; `before` where a row is no sequence's."""
    P, Q = P.cpu().double().numpy(), Q.cpu().double().numpy()
    tokens, parents, u, starts = tokens.tolist(), parents.tolist(), u.double().tolist(), starts.tolist()
    out = [before] * len(tokens)
    for a, e in zip(starts[:-1], starts[1:]):
        a = min(max(a, 0), len(tokens))
        e = min(max(min(e, len(tokens)), a), a + max_nodes)
        if e > a:
            out[a:e] = verify_tree(tokens[a:e], parents[a:e], P[a:e], Q[a:e], u[a:e], distinct)
    return out


def draft_case(counts, V, seed, width=1, distinct=False, near=0.5, scale=3.0, spare=3, keep=None):
    """A step's rows: tokens drawn from the drafter's distributions, parents, both models'
    distributions, uniforms and starts, on the CPU.  `keep`: tokens with weight, of each row."""
    g = torch.Generator().manual_seed(seed)
    starts = torch.tensor([0] + counts).cumsum(0).int()
    rows = int(starts[-1]) + spare
    x = torch.randn((rows, V), generator=g) * scale
    y = x + torch.randn((rows, V), generator=g) * scale * near
    if keep:
        x, y = (torch.where(t >= t.topk(min(keep, V)).values[:, -1:], t, -math.inf) for t in (x, y))
    P, Q = x.double().softmax(1).float(), y.double().softmax(1).float()
    parents = torch.full((rows,), -1, dtype=torch.int32)
    tokens = torch.randint(0, V, (rows,), generator=g)
    for a, e in zip(starts[:-1].tolist(), starts[1:].tolist()):
        kids = [[] for _ in range(e - a)]
        for i in range(1, e - a):
            free = [j for j in range(max(0, i - 6), i) if len(kids[j]) < width]
            up = free[int(torch.randint(0, len(free), (1,), generator=g))] if free else i - 1
            parents[a + i] = up
            q = Q[a + up].double().clone()
            if distinct:
                q[kids[up]] = 0.0
            if not q.sum() > 0:
                q[:] = 1.0
            tokens[a + i] = int(torch.multinomial(q, 1, generator=g))
            kids[up].append(int(tokens[a + i]))
    return dict(tokens=tokens, parents=parents, target_probs=P, draft_probs=Q,
                uniforms=torch.rand(rows, generator=g), row_starts=starts, max_nodes=max(max(counts), 1))
