"""Operators of speculative decoding with an 8-bit drafter, as cases that can be timed:
a copy of the model with 8-bit weights drafts tokens, the model itself verifies them by
given random numbers, and what comes out is distributed as the model's own samples.

  linear  linear_int8: y = x W^T (+ bias) as a product of 8-bit integers.  Every row of x and
          every row of W (an output channel) has a scale of its own,
            s = max |x| / 127,  q = rint(x / s)  (both quotients in single precision),
            y[m, n] = s_x[m] s_w[n] sum_k q_x[m, k] q_w[n, k] + bias[n]
  probs   sampling_probs: the distribution that sample_tokens draws a row's token from.
          x = logits / temperature (in single precision), tokens ordered by x descending, then
          index ascending; of them stay those with exp(x - max x) >= min_p, of these the first
          top_k, and of these the ones before which less than top_p of their sum stands
  verify  verify_draft_tree: which drafted tokens stay, and the token behind them.  At a row
          with target distribution p and drafter's distribution q its children are tested in
          order: with weights w = max(p - A q, 0) and c their sum (A = 0, c = 1 at first) the child's
          token x stays if u q(x) c < w(x); if not, A grows by c.  Children drawn without
          replacement have c divided by what q leaves to the tokens before them.  Where no
          child stays, the token is the first whose cumulative w exceeds u (of row 0) of the sum

Shapes are those of bench.py and the tests (hidden 896, intermediate 4864, 14 query and 2 kv
heads of 64 channels, T = 4, vocabulary 151,936) and generic ones around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
VOCAB = 151936


# -- the cases -----------------------------------------------------------------
def _linear(M, N, K, dtype="bf16", out="bf16", bias=False):
    return dict(op="linear", M=M, N=N, K=K, dtype=dtype, out=out, bias=bias)


def _probs(rows, V, dtype, top_k=-1, top_p=1.0, min_p=0.0, scale=3.0, temperature=0.8, mixed=False):
    return dict(op="probs", rows=rows, V=V, dtype=dtype, top_k=top_k, top_p=top_p, min_p=min_p, scale=scale,
                temperature=temperature, mixed=mixed)


def _verify(n, nodes, V, width=1, ragged=False, distinct=False, near=0.5, cut=False):
    return dict(op="verify", n=n, nodes=nodes, V=V, width=width, ragged=ragged, distinct=distinct, near=near,
                cut=cut)


def listed():
    return [
        # one token of one user through the q/k/v projection (T = 4 rows): latency only
        dict(_linear(4, 1152, 896, bias=True), name="linear_qkv_one"),
        # the drafter's logits for a full batch: bound by reading the weight
        dict(_linear(64, VOCAB, 896), name="linear_head_64"),
        # a prompt of 2,047 tokens through gate|up, and one of 4,096 through down: bound by arithmetic
        dict(_linear(4 * 2047, 9728, 896), name="linear_gate_up_prompt"),
        dict(_linear(4 * 4096, 896, 4864), name="linear_down_prompt"),
        # no size a multiple of anything, fp16 in, fp32 out
        dict(_linear(333, 1001, 777, "f16", "f32", True), name="linear_odd"),
        # one user's draft of four tokens and the token before it: top-p 0.9
        dict(_probs(5, VOCAB, "bf16", top_p=0.9), name="probs_one_user"),
        # 64 users' drafts of four tokens, top-k 50 and top-p 0.9
        dict(_probs(320, VOCAB, "bf16", 50, 0.9), name="probs_320"),
        # requests of every kind in one batch, fp32 logits of an odd vocabulary, nearly flat
        dict(_probs(77, 50257, "f32", 40, 0.95, 0.02, 1.0, 1.1, True), name="probs_mixed_f32"),
        # one user's chain of four drafted tokens
        dict(_verify(1, 5, VOCAB), name="verify_one_chain"),
        # a chat server's chains of uneven lengths: bound by reading a pair of rows each
        dict(_verify(64, 8, VOCAB, ragged=True), name="verify_64_chains"),
        # trees of drafted tokens, distributions cut as by top-p
        dict(_verify(16, 25, VOCAB, 3, cut=True), name="verify_trees_16"),
        # a small odd vocabulary, siblings drawn without replacement, a poor drafter
        dict(_verify(7, 13, 32003, 4, True, True, 1.5), name="verify_distinct"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear"] * 3 + ["probs"] * 2 + ["verify"] * 2)
    if op == "linear":
        N, K = rng.choice([(1152, 896), (896, 896), (9728, 896), (896, 4864), (VOCAB, 896)] +
                          [(_log(rng, 16, 9728), _log(rng, 16, 4864)) for _ in range(5)])
        M = _log(rng, 1, 16384)
        M = max(1, min(M, 16384 * 896 * 4864 // (N * K), 8188 * 9728 // N))
        return _linear(M, N, K, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["bf16", "bf16", "f16", "f32"]),
                       rng.random() < 0.4)
    V = rng.choice([VOCAB, VOCAB, 32000, 50257, _log(rng, 300, 200000)])
    if op == "probs":
        rows = max(1, min(_log(rng, 1, 512), 320 * VOCAB // V))
        k, p, m = rng.choice([(-1, 1.0, 0.0), (50, 0.9, 0.0), (20, 1.0, 0.0), (-1, 0.9, 0.0), (-1, 1.0, 0.05),
                              (1000, 0.95, 0.0), (-1, 0.6, 0.01)])
        return _probs(rows, V, rng.choice(["bf16", "bf16", "f16", "f32"]), k, p, m, rng.choice([1.0, 3.0, 6.0]),
                      round(rng.uniform(0.5, 1.3), 3), rng.random() < 0.4)
    nodes = _log(rng, 1, 64)
    width = rng.choice([1, 1, 2, 3, 5])
    n = max(1, min(_log(rng, 1, 128), 64 * 8 * VOCAB // (nodes * V * (1 if width == 1 else 2))))
    return _verify(n, nodes, V, width, rng.random() < 0.5, width > 1 and rng.random() < 0.5,
                   rng.choice([0.2, 0.5, 1.5]), rng.random() < 0.4)


# -- inputs --------------------------------------------------------------------
def _gens(seed):
    return torch.Generator().manual_seed(seed), torch.Generator(device=DEV).manual_seed(seed + 1)


def _rows_to_8_bits(x):
    """(integers in -127..127 as float32, scales): the formula above on the rows of x."""
    x = x.float()
    scale = x.abs().amax(-1, keepdim=True) / x.new_full((1, 1), 127.0)
    q = torch.where(scale > 0, torch.round(x / scale), 0.0).clamp_(-127.0, 127.0)
    return q, scale[:, 0]


def _row_starts(n, most, ragged, g):
    counts = torch.randint(1, most + 1, (n,), generator=g) if ragged else torch.full((n,), most)
    counts[0] = most
    return torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int()


def _parents(starts, width, g):
    """A chain for width 1; else node i's parent is one of those before it that have fewer than `width` children,
    the later the likelier."""
    parents = []
    for s, e in zip(starts[:-1].tolist(), starts[1:].tolist()):
        free = []
        for i in range(e - s):
            if i:
                u = torch.rand(1, generator=g).item()
                at = len(free) - 1 - int(u * u * min(len(free), 6))
                parents.append(free[at][0])
                free[at][1] += 1
                if free[at][1] == width:
                    free.pop(at)
            else:
                parents.append(-1)
            free.append([i, 0])
    return parents


def _ancestors(starts, parents, words):
    """Bitmasks int64 [rows, words] of each node's ancestors and itself, as the attention of a tree takes them."""
    rows = []
    for s, e in zip(starts[:-1].tolist(), starts[1:].tolist()):
        at = []
        for i in range(e - s):
            p = parents[s + i]
            at.append((at[p] if p >= 0 else 0) | 1 << i)
        rows += at
    part = lambda m, w: (m >> 64 * w) % 2**64
    sign = lambda x: x - 2**64 if x >= 2**63 else x
    return torch.tensor([[sign(part(m, w)) for w in range(words)] for m in rows], dtype=torch.int64)


@torch.no_grad()
def prepare(case, seed):
    c, (gc, g) = case, _gens(seed)
    normal = lambda *shape: torch.empty(shape, device=DEV).normal_(generator=g)
    if c["op"] == "linear":
        # rows of different sizes and a few large channels, as activations have them
        x = normal(c["M"], c["K"]) * torch.exp(0.5 * normal(c["M"], 1)) * (1 + 9 * (normal(1, c["K"]) > 2.5))
        w = (normal(c["N"], c["K"]) * 0.02).bfloat16()
        s = dict(c=c, x=x.to(DTYPES[c["dtype"]]), bias=normal(c["N"]).to(DTYPES[c["out"]]) if c["bias"] else None)
        q, scale = _rows_to_8_bits(w)
        s.update(wq=q.to(torch.int8), ws=scale)
        if own:
            from spikeinfer_amd.kernels import pack_linear_int8

            s["packed"] = pack_linear_int8(w)
        return s
    if c["op"] == "probs":
        rows = c["rows"]
        logits = (normal(rows, c["V"]) * c["scale"] + 2.0 * normal(1, c["V"])).to(DTYPES[c["dtype"]])
        kind = torch.arange(rows) % 5 if c["mixed"] else torch.full((rows,), 9)
        f32 = lambda v: v.float().to(DEV)
        return dict(c=c, logits=logits,
                    # of a mixed batch's rows the first kind is greedy, the second draws from everything, ...
                    temperature=f32(torch.where(kind == 0, 0.0, c["temperature"] + 0.05 * (torch.arange(rows) % 3))),
                    top_k=torch.where((kind == 1) | (kind == 2), -1, c["top_k"]).int().to(DEV),
                    top_p=f32(torch.where((kind == 1) | (kind == 3), 1.0, c["top_p"])),
                    min_p=f32(torch.where((kind == 1) | (kind == 4), 0.0, c["min_p"])))
    n, V = c["n"], c["V"]
    starts = _row_starts(n, c["nodes"], c["ragged"], gc)
    parents = _parents(starts, c["width"], gc)
    used = int(starts[-1])
    rows = n * c["nodes"] + 3  # a buffer is seldom exactly full
    x = normal(rows, V) * 3.0
    y = x + normal(rows, V) * (3.0 * c["near"])
    if c["cut"]:  # less than a thousandth of the largest: as a min-p or top-p cut leaves it
        x, y = (torch.where(t > t.amax(1, keepdim=True) - 7.0, t, -math.inf) for t in (x, y))
    target, draft = x.softmax(1), y.softmax(1)
    del x, y
    drawn = torch.multinomial(draft, c["width"], replacement=not c["distinct"], generator=g).cpu()
    tokens = torch.randint(0, V, (rows,), generator=gc)
    first, seen = starts[:-1].tolist(), {}
    for t, s in enumerate(first):
        for r in range(s, int(starts[t + 1])):
            if parents[r] >= 0:
                k = seen[s + parents[r]] = seen.get(s + parents[r], -1) + 1
                tokens[r] = drawn[s + parents[r], k]
    masks = torch.zeros((rows, -(-c["nodes"] // 64)), dtype=torch.int64)
    masks[:used] = _ancestors(starts, parents, masks.shape[1])
    parents = torch.tensor(parents + [-1] * (rows - used), dtype=torch.int32)
    return dict(c=c, tokens=tokens.to(DEV), parents=parents.to(DEV), target=target, draft=draft,
                uniforms=torch.rand(rows, generator=gc).to(DEV), starts=starts.to(DEV), masks=masks.to(DEV), out=torch.zeros(rows, dtype=torch.int64, device=DEV))


# -- the plain forms -------------------------------------------------------------
def _plain_linear(s):
    q, scale = _rows_to_8_bits(s["x"])
    y = q.double() @ s["wq"].double().T  # sums past 2^24: whole in 64 bits
    y *= scale.double()[:, None] * s["ws"].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y.to(DTYPES[s["c"]["out"]])


def _plain_probs(s):
    temp = s["temperature"][:, None]
    logits = s["logits"].float()
    greedy = temp < 1e-5
    x, order = torch.sort(torch.where(greedy, logits, logits / temp), dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device=x.device)
    limit = torch.where(s["top_k"] < 1, x.shape[1], s["top_k"])
    limit = torch.where(greedy[:, 0], 1, limit)[:, None]
    down = x.double() - x[:, :1].double()
    # a border of a cut lies between two neighbours: 64 bits
    w = torch.exp(down) * ((rank < limit) & (down >= torch.log(s["min_p"].double())[:, None]))
    top_p = torch.where(greedy | (s["top_p"][:, None] >= 1), math.inf, s["top_p"][:, None].double())
    w = w * (w.cumsum(1) - w < top_p * w.sum(1, keepdim=True))
    w = (w / w.sum(1, keepdim=True)).float()
    return torch.empty_like(w).scatter_(1, order, w)


def _plain_verify(s):
    c = s["c"]
    P, Q, dev = s["target"], s["draft"], s["target"].device
    most, last = c["nodes"], P.shape[0] - 1
    i = torch.arange(most, device=dev)
    count = (s["starts"][1:] - s["starts"][:-1])[:, None]
    at = (s["starts"][:-1, None].long() + i).clamp(max=last)  # [n, nodes]
    live = i < count
    up = torch.where(live, s["parents"][at].long(), -1)
    twin = (up[:, :, None] == up[:, None]) & (i < i[:, None])  # an earlier child of the same row
    rank, has = twin.sum(-1), up >= 0
    token = s["tokens"][at]
    above = at.gather(1, up.clamp(min=0))  # rows of p and q that test each node
    p, q, u = P[above, token].double(), Q[above, token].double(), s["uniforms"][at].double()
    before = (twin * q[:, None]).sum(-1) if c["distinct"] else torch.zeros_like(q)
    A, mass = torch.zeros_like(p), torch.ones_like(p)  # of the rows as parents
    pick = torch.full_like(up, -1)  # the child that stays
    for k in range(c["width"]):  # one sibling after the other: each test needs the sum that the one before left
        if k:
            w = torch.empty_like(A)
            for part in range(0, c["n"], 8):  # a few trees at a time: the rows in 64 bits are large
                rows = at[part:part + 8]
                w[part:part + 8] = (P[rows].double() - A[part:part + 8, :, None] * Q[rows]).clamp_(min=0).sum(-1)
            mass = torch.where(A > 0, w, mass)
        mine = has & (rank == k)
        parent = up.clamp(min=0)
        scale = mass.gather(1, parent) / (1 - before)
        left = A.gather(1, parent)
        stays = mine & (pick.gather(1, parent) < 0) & (u * q * scale < (p - left * q).clamp(min=0))
        grow = mine & ~stays & (pick.gather(1, parent) < 0)
        A = A.scatter_add(1, parent, torch.where(grow, scale, 0.0))
        pick = pick.scatter_reduce(1, parent, torch.where(stays, i, -1), "amax")
    ok = (pick.gather(1, up.clamp(min=0)) == i) | (i == 0)
    sees = ((s["masks"][at][:, :, i // 64] >> (i % 64)) & 1).bool()
    on = (ok[:, None] | ~sees).all(-1) & live
    end = (on & (pick < 0)).long().argmax(1, keepdim=True)  # one a tree
    row = at.gather(1, end)[:, 0]
    w = (P[row].double() - A.gather(1, end) * Q[row]).clamp_(min=0).cumsum(1)
    t = s["uniforms"][at[:, 0]].double()[:, None] * w[:, -1:]
    drawn = (w <= t).sum(1, keepdim=True)
    targets = torch.where(pick >= 0, token.gather(1, pick.clamp(min=0)), drawn)
    targets = torch.where(on, targets, -1)
    keep = torch.where(live, at, last)  # the spare row behind the trees takes what is no tree's
    value = torch.where(live, targets, s["out"][last])
    s["out"][keep.view(-1)] = value.view(-1)
    return s["out"]


def _own(s):
    from spikeinfer_amd.kernels import linear_int8, verify_draft_tree
    from spikeinfer_amd.sampler import sampling_probs

    c = s["c"]
    if c["op"] == "linear":
        return linear_int8(s["x"], s["packed"], s["bias"], dtype=DTYPES[c["out"]])
    if c["op"] == "probs":
        return sampling_probs(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return verify_draft_tree(s["tokens"], s["parents"], s["target"], s["draft"], s["uniforms"], s["starts"],
                             c["nodes"], distinct=c["distinct"], out=s["out"])


@torch.no_grad()
def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "probs": _plain_probs, "verify": _plain_verify}[state["c"]["op"]](state)


# -- what a pass cannot do without -----------------------------------------------
def work(case):
    c = case
    size = lambda name: 4 if name == "f32" else 2
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return dict(bytes=M * K * size(c["dtype"]) + N * (K + 4) + M * N * size(c["out"]) +
                    (N * size(c["out"]) if c["bias"] else 0), flops=2 * M * N * K)
    if c["op"] == "probs":
        return dict(bytes=c["rows"] * c["V"] * (size(c["dtype"]) + 4), flops=4 * c["rows"] * c["V"])
    # the two rows of one node a tree, where the path ends (a tree of siblings looks at a few more)
    return dict(bytes=c["n"] * (2 * c["V"] * 4 + c["nodes"] * 32), flops=3 * c["n"] * c["V"])


# -- in 64 bits, on the host but for the products --------------------------------
def _exact_8_bits(x):
    x = x.float().double()
    scale = (x.abs().max(1).values / 127.0).float().double()
    q = (x / scale[:, None]).float().round()  # the quotient as single precision has it
    return torch.where(scale[:, None] > 0, q, 0.0).clamp(-127, 127).double(), scale


def _exact_probs(c, s):
    logits, out = s["logits"].float().cpu().numpy(), np.zeros((c["rows"], c["V"]))
    temp, top_k, top_p, min_p = (s[k].cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p"))
    for r, row in enumerate(logits):
        if temp[r] < 1e-5:
            out[r, int(np.argmax(row))] = 1.0
            continue
        x = (row / temp[r]).astype(np.float64)
        e = np.exp(x - x.max())
        order = np.argsort(-x, kind="stable")
        order = order[e[order] >= float(min_p[r])]
        if top_k[r] >= 1:
            order = order[:top_k[r]]
        if top_p[r] < 1:
            total, cum = e[order].sum(), np.cumsum(e[order])
            order = order[cum - e[order] < float(top_p[r]) * total]
        out[r, order] = e[order] / e[order].sum()
    return torch.from_numpy(out)


@torch.no_grad()
def exact(case, seed):
    """float64 outputs of the products and distributions; a verification answers with whole numbers."""
    c = case
    if c["op"] == "verify":
        return None
    s = prepare(case, seed)
    if c["op"] == "probs":
        return _exact_probs(c, s)
    x, sx = _exact_8_bits(s["x"])
    out = torch.empty((c["M"], c["N"]), dtype=torch.float64, device=DEV)
    for a in range(0, c["N"], 16384):  # columns of the result, the weight's rows
        w = s["wq"][a:a + 16384].double()
        out[:, a:a + 16384] = torch.matmul(x, w.t().contiguous()) * sx[:, None] * s["ws"][a:a + 16384].double()
    return out if s["bias"] is None else out + s["bias"].double()
