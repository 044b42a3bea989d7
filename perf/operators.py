"""Operators on the packed spike cache beside plain decoding, as cases that can be
timed: verifying trees of drafted tokens, and keeping a cache within a budget.

  tree    paged_spike_attn_tree: the attention of drafted tokens (each sees the cached
          context and its own ancestors in the tree), one layer
  mass    paged_spike_attn_key_mass: the softmax weight that each cached token gets
          from the last tokens of its sequence, summed over timesteps and query heads
  evict   evict_cache: keeps the tokens of largest weight, and the first and last ones,
          and moves their words together, several layers in one call
  accept  accept_draft_tree: the accepted path of each verified tree, and its words
          from the step's buffers into the cache of every layer

Shapes are those of bench.py and the tests (14 query and 2 kv heads of 64 channels,
T = 4, 16-token blocks, 24 layers) and generic ones around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BS = 16  # tokens per cache block


# -- the cases -----------------------------------------------------------------
def _tree(n, lo, hi, nodes, ragged, dtype="bf16", T=4, hq=14, hkv=2, D=64):
    return dict(op="tree", n=n, lo=lo, hi=hi, nodes=nodes, ragged=ragged, dtype=dtype, T=T, hq=hq, hkv=hkv, D=D)


def _mass(n, lo, hi, rows, ragged=False, T=4, hq=14, hkv=2, D=64):
    return dict(op="mass", n=n, lo=lo, hi=hi, rows=rows, ragged=ragged, T=T, hq=hq, hkv=hkv, D=D)


def _evict(layers, n, lo, hi, budget, sinks=4, recent=32, T=4, hkv=2, D=64):
    return dict(op="evict", layers=layers, n=n, lo=lo, hi=hi, budget=budget, sinks=sinks, recent=recent, T=T,
                hkv=hkv, D=D)


def _accept(layers, n, hi, nodes, T=4, hkv=2, D=64):
    return dict(op="accept", layers=layers, n=n, hi=hi, nodes=nodes, T=T, hkv=hkv, D=D)


def listed():
    return [
        # one user, a short chat, a small draft: latency only
        dict(_tree(1, 128, 128, 8, False), name="tree_one_short"),
        # one user with a long document and a wide draft: few rows, many keys
        dict(_tree(1, 30011, 30011, 61, False), name="tree_one_long"),
        # a chat server verifying drafts of uneven sizes
        dict(_tree(32, 500, 5000, 16, True), name="tree_batch_32"),
        # long contexts and wide drafts, fp32 outputs: bound by arithmetic
        dict(_tree(16, 4096, 16384, 32, False, "f32"), name="tree_long_f32"),
        # heads of 128 channels, an odd number of nodes, fp16 outputs
        dict(_tree(8, 100, 9000, 25, False, "f16", hq=16, hkv=4, D=128), name="tree_head_dim_128"),
        # what one decode step adds to the weights, one user
        dict(_mass(1, 700, 700, 1), name="mass_one_700"),
        # the same for a batch of long contexts: bound by reading the keys
        dict(_mass(64, 4096, 16384, 1), name="mass_decode_64"),
        # an observation window of the last prompt tokens, uneven
        dict(_mass(8, 2000, 8000, 32, True), name="mass_window_32"),
        # one user's cache of one layer cut to a quarter
        dict(_evict(1, 1, 2000, 2000, 512), name="evict_one_layer"),
        # a batch, some sequences within the budget, several layers at once
        dict(_evict(6, 32, 1500, 12000, 2048), name="evict_batch_32"),
        # one user's accepted path, all layers
        dict(_accept(24, 1, 500, 8), name="accept_one"),
        # a full batch with wide drafts, all layers
        dict(_accept(24, 64, 700, 61), name="accept_64"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree"] * 5 + ["mass"] * 3 + ["evict"] * 2 + ["accept"])
    hq, hkv, D = rng.choice([(14, 2, 64)] * 3 + [(8, 8, 64), (16, 4, 128), (16, 2, 128), (6, 3, 32), (8, 2, 96)])
    T = rng.choice([4, 4, 4, 2, 3])
    if op == "tree":
        hi = _log(rng, 32, 32768)
        nodes = _log(rng, 1, 128)
        most = 16 * 16384 * 32 * 4 * 14 * 64  # the largest listed one's (rows, keys, channels)
        n = min(_log(rng, 1, 64), max(1, most // (hi * nodes * T * hq * D)))
        return _tree(n, max(1, hi // rng.choice([1, 2, 8])), hi, nodes, rng.random() < 0.5,
                     rng.choice(["bf16", "bf16", "f16", "f32"]), T, hq, hkv, D)
    if op == "mass":
        hi = _log(rng, 32, 32768)
        rows = rng.choice([1, 1, _log(rng, 2, 64)])
        most = 64 * 16384 * 4 * 14 * 64
        n = min(_log(rng, 1, 64), max(1, most // (hi * rows * T * hq * D)))
        return _mass(n, max(1, hi // rng.choice([1, 2, 8])), hi, min(rows, hi), rows > 1 and rng.random() < 0.5,
                     T, hq, hkv, D)
    if op == "evict":
        hi = _log(rng, 200, 32768)
        layers = _log(rng, 1, 6)
        n = min(_log(rng, 1, 32), max(1, 32 * 12000 * 6 * 4 * 2 * 64 // (hi * layers * T * hkv * D)))
        budget = max(40, int(hi * rng.uniform(0.1, 0.9)))
        return _evict(layers, n, max(1, hi // rng.choice([1, 2, 8])), hi, budget, rng.choice([0, 1, 4]),
                      rng.choice([1, 17, 32]), T, hkv, D)
    return _accept(_log(rng, 2, 24), _log(rng, 1, 64), _log(rng, 16, 700), _log(rng, 2, 61), T, min(hkv, 4), D)


# -- inputs --------------------------------------------------------------------
def _gens(seed):
    return torch.Generator().manual_seed(seed), torch.Generator(device=DEV).manual_seed(seed + 1)


def _words(shape, g):
    """Packed spikes, 3 of 16 bits set."""
    r = [torch.randint(-2**31, 2**31, shape, dtype=torch.int32, device=DEV, generator=g) for _ in range(4)]
    return r[0] & r[1] & (r[2] | r[3])


def _lens(n, lo, hi, g):
    lens = torch.randint(lo, hi + 1, (n,), generator=g, dtype=torch.int32)
    lens[0] = hi  # so that the table's width is the longest sequence's
    return lens


def _tables(lens, width, g, spare=0):
    """Shuffled physical blocks of a pool that holds n full tables and `spare` blocks more
    ([n, width] table padded with the last block, the blocks left, the number of blocks)."""
    need = [-(-int(x) // BS) for x in lens]
    total = len(need) * width + spare + 1
    perm = torch.randperm(total - 1, generator=g).int()
    tables = torch.full((len(need), width), total - 1, dtype=torch.int32)
    at = 0
    for i, nb in enumerate(need):
        tables[i, :nb] = perm[at:at + nb]
        at += nb
    return tables, perm[at:], total


def _row_starts(n, most, ragged, g, limit=None):
    counts = torch.randint(1, most + 1, (n,), generator=g) if ragged else torch.full((n,), most)
    counts[0] = most
    if limit is not None:
        counts = torch.minimum(counts, limit.long())
    return torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).int()


def _parents(n, starts, g):
    """Random trees: node 0 is the root, node i hangs below one of the eight before it."""
    u = torch.rand(int(starts[-1]), generator=g).tolist()
    parents = []
    for s, e in zip(starts[:-1].tolist(), starts[1:].tolist()):
        for i in range(e - s):
            lo = max(0, i - 8)
            parents.append(lo + int(u[s + i] * (i - lo)) if i else -1)
    return parents


def _ancestors(starts, parents, words):
    """Bitmasks int64 [rows, words] of each node's ancestors and itself."""
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
    n, T, hkv, D = c["n"], c["T"], c["hkv"], c["D"]
    W = D // 32
    if c["op"] in ("tree", "mass"):
        lens = _lens(n, c["lo"], c["hi"], gc)
        tables, _, blocks = _tables(lens, -(-c["hi"] // BS), gc)
        kv = (T, hkv, blocks * BS, W)
        s = dict(kc=_words(kv, g), tables=tables.to(DEV), lens=lens.to(DEV))
        if c["op"] == "tree":
            starts = _row_starts(n, c["nodes"], c["ragged"], gc)
            parents = _parents(n, starts, gc)
            rows = n * c["nodes"] + 3  # a buffer is seldom exactly full
            masks = torch.zeros((rows, -(-c["nodes"] // 64)), dtype=torch.int64)
            masks[:int(starts[-1])] = _ancestors(starts, parents, masks.shape[1])
            s.update(vc=_words(kv, g), q=_words((T, rows, c["hq"], W), g), masks=masks.to(DEV),
                     kw=_words((T, rows, hkv, W), g), vw=_words((T, rows, hkv, W), g),
                     starts=starts.to(DEV),
                     out=torch.zeros((T, rows, c["hq"], D), dtype=DTYPES[c["dtype"]], device=DEV))
        else:
            starts = _row_starts(n, c["rows"], c["ragged"], gc, lens)
            s.update(q=_words((T, int(starts[-1]), c["hq"], W), g), starts=starts.to(DEV))
        return dict(c=c, **s)
    if c["op"] == "evict":
        lens = _lens(n, c["lo"], c["hi"], gc)
        width, kept = -(-c["hi"] // BS), -(-c["budget"] // BS)
        tables, spare, blocks = _tables(lens, width, gc, n * kept)
        L = c["layers"]
        # weights as attention leaves them: most tokens little, a few much, exact zeros
        mass = torch.rand((L, n, hkv, c["hi"]), device=DEV, generator=g).pow_(8).mul_(3.0)
        mass *= torch.rand(mass.shape, device=DEV, generator=g) > 0.05
        return dict(c=c, mass=mass, mass_out=torch.empty_like(mass), tables=tables.to(DEV), lens=lens.to(DEV),
                    dst=spare[:n * kept].view(n, kept).to(DEV),
                    layers=[tuple(_words((T, hkv, blocks * BS, W), g) for _ in range(2)) for _ in range(L)])
    lens = _lens(n, max(1, c["hi"] // 4), c["hi"], gc)
    width = -(-(c["hi"] + c["nodes"]) // BS)
    tables, _, blocks = _tables(lens + c["nodes"], width, gc)
    starts = _row_starts(n, c["nodes"], False, gc)
    parents = _parents(n, starts, gc)
    rows = int(starts[-1])
    tokens = torch.randint(0, 50, (rows,), generator=gc)
    targets = torch.randint(0, 50, (rows,), generator=gc)
    hit = torch.rand(rows, generator=gc).tolist()
    at = starts.tolist()
    for i in range(n):  # a drafted token is what the model says three times out of four
        for r in range(at[i + 1] - 1, at[i], -1):
            if hit[r] < 0.75:
                targets[at[i] + parents[r]] = tokens[r]
    masks = _ancestors(starts, parents, -(-c["nodes"] // 64))
    parents = torch.tensor([parents], dtype=torch.int32)[0]
    return dict(c=c, tables=tables.to(DEV), lens=lens.to(DEV), starts=starts.to(DEV), tokens=tokens.to(DEV),
                targets=targets.to(DEV), parents=parents.to(DEV), masks=masks.to(DEV),
                layers=[tuple(_words((T, hkv, blocks * BS, W), g) for _ in range(2)) for _ in range(c["layers"])],
                drafts=[tuple(_words((T, rows, hkv, W), g) for _ in range(2)) for _ in range(c["layers"])])


# -- the plain forms -------------------------------------------------------------
def _bits(words, D):
    shifts = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words[..., None] >> shifts) & 1).flatten(-2)[..., :D].float()


def _slots(tables, pos):
    """Cache slots of positions [n, ...] of each sequence."""
    flat = pos.flatten(1).long()
    return (tables.long().gather(1, flat // BS) * BS + flat % BS).view(pos.shape)


def _cached(cache, tables):
    """Every position that the tables hold: [T, hkv, n, tokens, W]."""
    pos = torch.arange(tables.shape[1] * BS, device=cache.device).expand(tables.shape[0], -1)
    return cache[:, :, _slots(tables, pos)]


def _rows_of(words, starts, most, hkv):
    """Rows of each sequence, padded to `most`: [T, hkv, n, most * heads a kv head, W]."""
    at = (starts[:-1, None].long() + torch.arange(most, device=words.device)).clamp(max=words.shape[1] - 1)
    x = words[:, at]  # [T, n, most, heads, W]
    x = x.unflatten(3, (hkv, -1)).permute(0, 3, 1, 2, 4, 5)
    return x.flatten(3, 4)


def _plain_tree(s):
    c = s["c"]
    T, hq, hkv, D, most = c["T"], c["hq"], c["hkv"], c["D"], c["nodes"]
    dev = s["q"].device
    rep = hq // hkv
    q = _bits(_rows_of(s["q"], s["starts"], most, hkv), D)
    k, v = (torch.cat([_bits(_cached(cache, s["tables"]), D), _bits(_rows_of(w, s["starts"], most, hkv), D)], 3)
            for cache, w in ((s["kc"], s["kw"]), (s["vc"], s["vw"])))
    at = (s["starts"][:-1, None].long() + torch.arange(most, device=dev)).clamp(max=s["masks"].shape[0] - 1)
    bit = torch.arange(most, device=dev)
    seen = (s["masks"][at][:, :, bit // 64] >> (bit % 64)) & 1  # [n, nodes, nodes]
    ctx = torch.arange(s["tables"].shape[1] * BS, device=dev) < s["lens"][:, None]
    see = torch.cat([ctx[:, None].expand(-1, most, -1), seen.bool()], 2).repeat_interleave(rep, 1)
    x = (q @ k.transpose(-1, -2)) / math.sqrt(D)
    x = torch.where(see, x, -1e30)
    e = torch.exp(x - x.amax(-1, keepdim=True)) * see
    o = e @ v / e.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(T, hkv, -1, most, rep, D).permute(0, 2, 3, 1, 4, 5).flatten(3, 4)  # [T, n, most, hq, D]
    row = torch.arange(s["q"].shape[1], device=dev)
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True).clamp(max=c["n"] - 1)
    node = (row - s["starts"].long()[seq]).clamp(max=most - 1)
    live = (row < s["starts"][-1])[:, None, None]
    s["out"].copy_(torch.where(live, o[:, seq, node], s["out"].float()))
    return s["out"]


def _plain_mass(s):
    c = s["c"]
    hkv, D, most = c["hkv"], c["D"], c["rows"]
    dev = s["q"].device
    q = _bits(_rows_of(s["q"], s["starts"], most, hkv), D)
    k = _bits(_cached(s["kc"], s["tables"]), D)
    count = (s["starts"][1:] - s["starts"][:-1])[:, None]
    i = torch.arange(most, device=dev)
    last = torch.where(i < count, s["lens"][:, None] - count + i, -1)  # [n, most]: what each row sees last
    last = last.repeat_interleave(c["hq"] // hkv, 1)
    see = torch.arange(k.shape[3], device=dev) <= last[..., None]
    x = (q @ k.transpose(-1, -2)) / math.sqrt(D)
    x = torch.where(see, x, -1e30)
    e = torch.exp(x - x.amax(-1, keepdim=True)) * see
    w = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return w.sum((0, 3)).permute(1, 0, 2).contiguous()  # [n, hkv, tokens]


def _plain_evict(s):
    c = s["c"]
    budget, hkv = c["budget"], c["hkv"]
    mass, lens = s["mass"], s["lens"][:, None]
    dev = mass.device
    j = torch.arange(c["hi"], device=dev)
    always = ((j < c["sinks"]) | (j >= lens - c["recent"]))[:, None]  # [n, 1, tokens]
    score = torch.where(always, math.inf, mass)
    score = torch.where((j < lens)[:, None], score, -math.inf)
    keep = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :budget].sort(-1).values
    kept = lens[:, 0].clamp(max=budget)
    i = torch.arange(keep.shape[-1], device=dev)
    live = (i < kept[:, None])[:, None]  # [n, 1, budget]
    s["mass_out"].zero_()
    s["mass_out"][..., :keep.shape[-1]] = torch.where(live, mass.gather(-1, keep), 0.0)
    to = _slots(s["dst"], i.expand(c["n"], -1))[:, None].expand(-1, hkv, -1)
    head = torch.arange(hkv, device=dev)[:, None]
    for words, of in zip(s["layers"], keep):
        src = _slots(s["tables"], of)
        for x in words:
            x[:, head, to] = torch.where(live[..., None], x[:, head, src], x[:, head, to])
    return dict(keep=torch.where(live, keep, -1).int(), lens=kept.int(), mass=s["mass_out"], layers=s["layers"])


def _plain_accept(s):
    c = s["c"]
    n, most = c["n"], c["nodes"]
    dev = s["tokens"].device
    i = torch.arange(most, device=dev)
    tokens, targets, parents = (s[k].view(n, most) for k in ("tokens", "targets", "parents"))
    up = parents.long().clamp(min=0)
    hit = (tokens == targets.gather(1, up)) & (i > 0)
    # of siblings with one token the first counts
    twin = (parents[:, :, None] == parents[:, None]) & (tokens[:, :, None] == tokens[:, None]) & (i < i[:, None])
    hit &= ~twin.any(-1)
    seen = ((s["masks"].view(n, most, -1)[:, :, i // 64] >> (i % 64)) & 1).bool()
    ok = (hit | (i == 0))[:, None].logical_or(~seen).all(-1)
    count = ok.sum(1)
    path = torch.where(ok, i, most).sort(1).values
    live = i < count[:, None]
    path = torch.where(live, path, 0)
    after = targets.gather(1, path.gather(1, count[:, None] - 1))[:, 0]
    # entries past the path write the root's words to the root's place again
    to = _slots(s["tables"], s["lens"][:, None] + torch.where(live, i, 0)).view(-1)
    src = (path + i.new_tensor(most) * torch.arange(n, device=dev)[:, None]).view(-1)
    for words, new in zip(s["layers"], s["drafts"]):
        for x, y in zip(words, new):
            x[:, :, to] = y[:, src].transpose(1, 2)
    return dict(path=torch.where(live, path, -1).int(), count=count.int(), next=after, layers=s["layers"])


def _own(s):
    from spikeinfer_amd import kernels

    c = s["c"]
    if c["op"] == "tree":
        return kernels.paged_spike_attn_tree(s["q"], s["kw"], s["vw"], s["kc"], s["vc"], s["tables"], s["lens"],
                                             s["starts"], s["masks"], c["nodes"], c["D"], BS, out=s["out"])
    if c["op"] == "mass":
        return kernels.paged_spike_attn_key_mass(s["q"], s["kc"], s["tables"], s["lens"], c["D"], BS,
                                                 row_starts=s["starts"], max_rows=c["rows"])
    if c["op"] == "evict":
        keep, lens = kernels.evict_cache(s["layers"], s["mass"], s["tables"], s["lens"], c["budget"], BS,
                                         sinks=c["sinks"], recent=c["recent"], dst_tables=s["dst"],
                                         mass_out=s["mass_out"])
        return dict(keep=keep, lens=lens, mass=s["mass_out"], layers=s["layers"])
    path, count, after = kernels.accept_draft_tree(s["tokens"], s["parents"], s["targets"], s["starts"], c["nodes"],
                                                   s["drafts"], s["layers"], s["tables"], s["lens"], BS)
    return dict(path=path, count=count, next=after, layers=s["layers"])


@torch.no_grad()
def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "mass": _plain_mass, "evict": _plain_evict, "accept": _plain_accept}[
        state["c"]["op"]](state)


# -- what a pass cannot do without -----------------------------------------------
def work(case):
    c = case
    T, hkv, W, n = c["T"], c["hkv"], c["D"] // 32, c["n"]
    word = 4 * W * T * hkv  # a token's keys (or values) of one layer
    if c["op"] == "accept":
        rows = c["n"] * 3  # accepted nodes of a tree, about
        return dict(bytes=c["layers"] * rows * 4 * word + n * c["nodes"] * 24, flops=0)
    tokens = n * (c["lo"] + c["hi"]) / 2
    if c["op"] == "evict":
        kept = n * min(c["budget"], (c["lo"] + c["hi"]) / 2)
        return dict(bytes=c["layers"] * (hkv * 4 * (tokens + n * c["hi"] + kept) + 4 * word * kept), flops=0)
    of = c["nodes" if c["op"] == "tree" else "rows"] * (0.5 if c["ragged"] else 1.0)
    rows = n * of
    pairs = T * c["hq"] * of * tokens
    q = 4 * W * T * c["hq"] * rows
    if c["op"] == "mass":
        return dict(bytes=tokens * word + q + n * hkv * c["hi"] * 4, flops=2 * pairs * c["D"])
    size = 4 if c["dtype"] == "f32" else 2
    return dict(bytes=2 * word * (tokens + rows) + q + rows * T * c["hq"] * c["D"] * size,
                flops=4 * (pairs + rows * T * c["hq"] * of / 2) * c["D"])


# -- in 64 bits, one sequence at a time ------------------------------------------
def _dense(words, D):
    x = words.long()
    return torch.stack([(x[..., b // 32] >> (b % 32)) & 1 for b in range(D)], -1).double()


def _exact_kept(c, mass, lens):
    out = np.zeros_like(mass)
    for n, m in enumerate(lens):
        lo, hi = (c["sinks"], m - c["recent"]) if m > c["budget"] else (m, m)
        free = c["budget"] - c["sinks"] - c["recent"]
        for layer, h in np.ndindex(c["layers"], c["hkv"]):
            row = mass[layer, n, h]
            best = np.lexsort((np.arange(lo, hi), -row[lo:hi]))[:free] + lo
            kept = np.sort(np.concatenate([np.arange(lo), best, np.arange(hi, m)]))
            out[layer, n, h, :len(kept)] = row[kept]
    return out


@torch.no_grad()
def exact(case, seed):
    """float64 outputs of the attention cases and the weights that an eviction keeps; the
    rest moves and compares whole numbers."""
    c = case
    if c["op"] == "accept":
        return None
    s = prepare(case, seed)
    if c["op"] == "evict":
        return dict(keep=None, lens=None, mass=_exact_kept(c, s["mass"].double().cpu().numpy(), s["lens"].tolist()),
                    layers=None)
    T, hq, hkv, D = c["T"], c["hq"], c["hkv"], c["D"]
    starts, lens, rep = s["starts"].tolist(), s["lens"].tolist(), hq // hkv
    tree = c["op"] == "tree"
    out = s["out"].double() if tree else torch.zeros((c["n"], hkv, s["tables"].shape[1] * BS), dtype=torch.float64,
                                                      device=DEV)
    for n in range(c["n"]):
        a, e, m = starts[n], starts[n + 1], lens[n]
        rows = e - a
        slots = (s["tables"][n].long()[:, None] * BS + torch.arange(BS, device=DEV)).view(-1)[:m]
        last = torch.arange(m - rows, m, device=DEV)
        for h in range(hkv):
            k = _dense(s["kc"][:, h, slots], D)
            see = torch.ones((rows, m), dtype=torch.bool, device=DEV)
            if tree:
                k = torch.cat([k, _dense(s["kw"][:, a:e, h], D)], 1)
                v = torch.cat([_dense(s["vc"][:, h, slots], D), _dense(s["vw"][:, a:e, h], D)], 1)
                nodes = [[(w >> b) & 1 for w in row for b in range(64)][:rows] for row in s["masks"][a:e].tolist()]
                see = torch.cat([see, torch.tensor(nodes, dtype=torch.bool, device=DEV).view(rows, rows)], 1)
            else:
                see = torch.arange(m, device=DEV) <= last[:, None]
            for g in range(h * rep, (h + 1) * rep):
                p = torch.matmul(_dense(s["q"][:, a:e, g], D), k.transpose(1, 2).contiguous()).div_(math.sqrt(D))
                p = p.masked_fill_(~see, -math.inf).softmax(-1)
                if tree:
                    out[:, a:e, g] = torch.matmul(p, v)
                else:
                    out[n, h, :m] += p.sum((0, 1))
    return out
