"""Plain implementations of the draft-tree and eviction operators in 64 bits, one
sequence, row and head at a time, and inputs for their tests (torch, any device)."""
from __future__ import annotations

import math

import torch

from model_ref import pack_ref


def bits(words, D):
    """[..., W] words -> float64 [..., D] spikes."""
    return ((words.long()[..., None] >> torch.arange(32, device=words.device)) & 1).flatten(-2)[..., :D].double()


def positions(cache, table, length, bs):
    """The words of positions 0..length of a table row, zeros where its block lies
    outside the cache: [T, H, length, W]."""
    pos = torch.arange(length, device=cache.device)
    blk = table.long()[pos // bs] if length else pos
    ok = (blk >= 0) & (blk < cache.shape[2] // bs)
    words = cache[:, :, torch.where(ok, blk, 0) * bs + pos % bs]
    return torch.where(ok[:, None], words, 0)


def tree_ref(q, kw, vw, kc, vc, tables, ctx, starts, masks, max_nodes, D, bs, out):
    """float64 copy of `out` with the rows of every tree."""
    out = out.double().clone()
    hkv = kc.shape[1]
    rep = q.shape[2] // hkv
    starts, ctx = starts.tolist(), ctx.tolist()
    for n in range(len(ctx)):
        a, e = starts[n], min(starts[n + 1], starts[n] + max_nodes)
        if e <= a:
            continue
        m = min(max(ctx[n], 0), tables.shape[1] * bs)
        i = torch.arange(e - a, device=q.device)
        seen = ((masks[a:e][:, i // 64] >> (i % 64)) & 1).bool()
        see = torch.cat([torch.ones((e - a, m), dtype=torch.bool, device=q.device), seen], 1)
        k, v = (torch.cat([bits(positions(c, tables[n], m, bs), D), bits(w[:, a:e], D).transpose(1, 2)], 2)
                for c, w in ((kc, kw), (vc, vw)))
        x = bits(q[:, a:e], D).transpose(1, 2)  # [T, Hq, rows, D]
        s = torch.matmul(x, k.repeat_interleave(rep, 1).transpose(-1, -2).contiguous()) / math.sqrt(D)
        w = torch.exp(s) * see
        o = torch.matmul(w, v.repeat_interleave(rep, 1)) / w.sum(-1, keepdim=True).clamp(min=1e-300)
        out[:, a:e] = o.transpose(1, 2)
    return out


def mass_ref(q, kc, tables, lens, D, bs, starts=None, max_rows=1, cap=None):
    """float64 [N, Hkv, cap]."""
    hkv, N = kc.shape[1], tables.shape[0]
    rep = q.shape[2] // hkv
    cap = tables.shape[1] * bs if cap is None else cap
    out = torch.zeros((N, hkv, cap), dtype=torch.float64, device=q.device)
    starts = list(range(N + 1)) if starts is None else starts.tolist()
    for n in range(N):
        a, e = starts[n], min(starts[n + 1], starts[n] + max_rows)
        m = min(max(int(lens[n]), 0), tables.shape[1] * bs)
        if e <= a or m == 0:
            continue
        k = bits(positions(kc, tables[n], m, bs), D).repeat_interleave(rep, 1)
        s = torch.matmul(bits(q[:, a:e], D).transpose(1, 2), k.transpose(-1, -2).contiguous()) / math.sqrt(D)
        last = torch.arange(m - (e - a), m, device=q.device)
        w = torch.exp(s) * (torch.arange(m, device=q.device) <= last[:, None])
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        w = w.sum((0, 2)).view(hkv, rep, m).sum(1)
        out[n, :, :min(m, cap)] = w[:, :cap]
    return out


def evict_ref(mass, length, budget, sinks, recent):
    """Positions that a list of masses keeps, in order."""
    if length <= budget:
        return list(range(length))
    low = lambda j: (-math.inf, j) if math.isnan(mass[j]) else (mass[j], j)
    rank = sorted(range(sinks, length - recent), key=lambda j: (math.isnan(mass[j]), -low(j)[0], j))
    return sorted([*range(sinks), *rank[:budget - sinks - recent], *range(length - recent, length)])


def accept_ref(tokens, parents, targets):
    """Path of one tree given as lists, and the token after it."""
    if not tokens:
        return [], -1
    path = [0]
    while True:
        child = [i for i in range(path[-1] + 1, len(tokens))
                 if parents[i] == path[-1] and tokens[i] == targets[path[-1]]]
        if not child:
            return path, targets[path[-1]]
        path.append(child[0])


def random_parents(count, g):
    """Parents of a random tree of `count` rows (row 0 the root)."""
    return [-1] + [int(torch.randint(max(0, i - 6), i, (1,), generator=g)) for i in range(1, count)]


def ancestor_masks(parents, words):
    """int64 [rows, words] of one tree's rows."""
    at = []
    for i, p in enumerate(parents):
        at.append((at[p] if 0 <= p < i else 0) | 1 << i)
    sign = lambda x: x - 2**64 if x >= 2**63 else x
    return torch.tensor([[sign((m >> 64 * w) % 2**64) for w in range(words)] for m in at],
                        dtype=torch.int64).view(len(parents), words)


def paged(lens, T, hkv, D, bs, g, dev, density=0.25, width=None, spare=0):
    """Caches of shuffled blocks: (k, v, tables int32 [N, width], blocks left)."""
    need = [-(-int(x) // bs) for x in lens]
    total = sum(need) + spare + 1
    width = width or max(1, max(need, default=1))
    order = torch.randperm(total - 1, generator=g).int()
    tables = torch.full((len(need), width), total - 1, dtype=torch.int32)
    at = 0
    for n, b in enumerate(need):
        tables[n, :b] = order[at:at + b]
        at += b
    spikes = lambda: pack_ref((torch.rand((T, hkv, total * bs, D), generator=g) < density).float())
    return spikes().to(dev), spikes().to(dev), tables.to(dev), order[at:]


def words(shape, D, g, dev, density=0.25):
    return pack_ref((torch.rand((*shape, D), generator=g) < density).float()).to(dev)


def starts_of(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)


def tree_case(T, hq, hkv, D, bs, trees, seed, dev, spare_rows=2, density=0.25, q_density=0.25):
    """Arguments of paged_spike_attn_tree (without max_nodes) for (context, nodes) pairs."""
    g = torch.Generator().manual_seed(seed)
    ctx, counts = zip(*trees)
    k, v, tables, _ = paged(ctx, T, hkv, D, bs, g, dev, density)
    rows = sum(counts) + spare_rows
    M = -(-max(counts) // 64)
    masks = torch.full((rows, M), -1, dtype=torch.int64)
    at = 0
    for c in counts:
        if c:
            masks[at:at + c] = ancestor_masks(random_parents(c, g), M)
        at += c
    w = lambda h, p: words((T, rows, h), D, g, dev, p)
    return dict(q_packed=w(hq, q_density), k_words=w(hkv, density), v_words=w(hkv, density), k_cache=k, v_cache=v,
                block_tables=tables, context_lens=torch.tensor(ctx, dtype=torch.int32).to(dev),
                row_starts=starts_of(counts).to(dev), masks=masks.to(dev), max_nodes=max(counts), head_dim=D,
                block_size=bs)


def tree_want(case, out):
    c = case
    return tree_ref(c["q_packed"], c["k_words"], c["v_words"], c["k_cache"], c["v_cache"], c["block_tables"],
                    c["context_lens"], c["row_starts"], c["masks"], c["max_nodes"], c["head_dim"], c["block_size"], out)
