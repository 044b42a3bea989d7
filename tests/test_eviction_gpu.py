"""Key weights and eviction on the GPU against plain float64 code.

Key weights: a sum of k positive fp32 terms, each to 2**-22, is off by at most (k + 4) *
2**-24 of itself; no accumulator takes more than a 16th of a sequence's keys in a row, and
a key's own sum has T * heads * rows terms.
"""
from __future__ import annotations

import math

import pytest
import torch

import cache_ops_ref as ref
from spikeinfer_amd.kernels import evict_cache, paged_spike_attn_key_mass

pytestmark = pytest.mark.gpu


def _mass_case(T, hq, hkv, D, bs, lens, rows, seed, dev, density=0.25, q_density=0.25):
    g = torch.Generator().manual_seed(seed)
    k, _, tables, _ = ref.paged(lens, T, hkv, D, bs, g, dev, density)
    starts = None if rows is None else ref.starts_of(rows)
    R = len(lens) if rows is None else sum(rows) + 2
    return dict(q_packed=ref.words((T, R, hq), D, g, dev, q_density), k_cache=k, block_tables=tables,
                seq_lens=torch.tensor(lens, dtype=torch.int32).to(dev), head_dim=D, block_size=bs,
                row_starts=None if starts is None else starts.to(dev), max_rows=1 if rows is None else max(rows))


def _want(c, cap=None):
    return ref.mass_ref(c["q_packed"], c["k_cache"], c["block_tables"], c["seq_lens"], c["head_dim"], c["block_size"],
                        c["row_starts"], c["max_rows"], cap)


def _check(c, got, want):
    T, _, hq, _ = c["q_packed"].shape
    terms = int(c["seq_lens"].max()) / 16 + T * hq / c["k_cache"].shape[1] * c["max_rows"] + 64
    assert ((got.double() - want).abs() <= terms * 2.0**-24 * want).all()


@pytest.mark.parametrize("T,hq,hkv,D,bs,lens,rows", [
    (4, 14, 2, 64, 16, [1, 2, 16, 17, 63, 64, 65, 500], None),
    (4, 14, 2, 64, 16, [4097, 0, 2048, 1023], None),
    (3, 8, 8, 64, 16, [300, 40], None),
    (2, 6, 2, 96, 64, [700, 65], [3, 5]),
    (2, 16, 1, 128, 16, [900, 200, 33], [32, 1, 33]),   # a window as long as its sequence
    (1, 4, 4, 32, 16, [129, 5], [20, 5]),
    (4, 14, 2, 64, 16, [1500, 70, 64, 10], [32, 17, 64, 0]),
    (2, 4, 1, 45, 16, [50], [7]),
    (1, 34, 2, 64, 16, [200, 99], None),
    (5, 14, 2, 64, 1, [333], [40]),
    (1, 2, 2, 64, 16, [1200], [1200]),                  # every row of a prompt
])
def test_matches_float64(gpu, T, hq, hkv, D, bs, lens, rows):
    print(f"mass {T} {hq}/{hkv} {D} {lens} {rows}", flush=True)
    c = _mass_case(T, hq, hkv, D, bs, lens, rows, D + sum(lens), gpu)
    got = paged_spike_attn_key_mass(**c)
    want = _want(c)
    _check(c, got, want)
    used = torch.tensor([rep and n for n, rep in zip(lens, rows or [1] * len(lens))])
    assert torch.allclose(got.sum((1, 2)).cpu().double(),
                          torch.tensor([T * hq * (m if n else 0) for n, m in zip(lens, rows or [1] * len(lens))],
                                       dtype=torch.float64), rtol=1e-4), used


@pytest.mark.parametrize("D", [64, 128])
def test_dense_and_silent_words(gpu, D):
    for qd, kd in ((1.1, 1.1), (1.1, 0.0), (0.0, 1.1), (1.1, 0.5), (1.1, 0.05)):
        c = _mass_case(2, 8, 2, D, 16, [300, 1100], [3, 9], 5, gpu, kd, qd)
        _check(c, paged_spike_attn_key_mass(**c), _want(c))


def test_accumulation_strides_and_capacity(gpu):
    """Adding to a strided slice leaves what lies behind the sequences; without adding it
    becomes 0; a capacity below or above the table's; lengths past the table; bad blocks."""
    c = _mass_case(2, 14, 2, 64, 16, [100, 37], None, 3, gpu)
    want = _want(c)
    big = torch.full((2, 3, 300), 2.0, device=gpu)
    out = big[:, :2, 5:205]
    assert paged_spike_attn_key_mass(**c, out=out, accumulate=True) is out
    _check(c, out[..., :112] - 2.0 * (want == 0), want + 2.0 * (want != 0))
    assert (out[0, :, 100:] == 2).all() and (out[1, :, 37:] == 2).all()
    assert (big[:, 2] == 2).all() and (big[..., :5] == 2).all() and (big[..., 205:] == 2).all()
    paged_spike_attn_key_mass(**c, out=out)
    _check(c, out[..., :112], want)
    assert (out[0, :, 100:] == 0).all() and (out[1, :, 37:] == 0).all() and (big[..., 205:] == 2).all()
    small = torch.full((2, 2, 60), 9.0, device=gpu)
    _check(c, paged_spike_attn_key_mass(**c, out=small), want[..., :60])
    c["block_tables"] = c["block_tables"].clone()
    c["block_tables"][0, 2], c["block_tables"][1, 0] = -1, 10**7
    c["seq_lens"] = torch.tensor([10**9, 37], dtype=torch.int64, device=gpu)
    got = paged_spike_attn_key_mass(**c)
    c["seq_lens"] = torch.tensor([112, 37], device=gpu)
    _check(c, got, _want(c))


def test_mass_does_not_depend_on_the_batch_and_replays(gpu):
    lens, rows = [3000, 70, 0, 1100], [5, 8, 3, 1]
    rows[2] = 0
    c = _mass_case(4, 14, 2, 64, 16, lens, rows, 9, gpu)
    out = paged_spike_attn_key_mass(**c)
    for n in (0, 1, 3):
        a, e = (int(x) for x in c["row_starts"][n:n + 2])
        one = dict(c, q_packed=c["q_packed"][:, a:e], block_tables=c["block_tables"][n:n + 1], max_rows=e - a,
                   seq_lens=c["seq_lens"][n:n + 1], row_starts=torch.tensor([0, e - a], device=gpu))
        assert torch.equal(paged_spike_attn_key_mass(**one)[0], out[n])
    static = {k: v.clone() if torch.is_tensor(v) else v for k, v in c.items()}
    res = torch.empty_like(out)
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_spike_attn_key_mass(**static, out=res)
    for lens2, starts in (([3000, 70, 0, 1100], c["row_starts"]), ([12, 0, 1, 2999], ref.starts_of([3, 0, 1, 8]))):
        static["seq_lens"].copy_(torch.tensor(lens2))
        static["row_starts"].copy_(starts)
        res.fill_(-1.0)
        graph.replay()
        eager = paged_spike_attn_key_mass(**static)
        torch.cuda.synchronize(gpu)
        assert torch.equal(res, eager)
        _check(static, res, _want(static))


def _evict_case(lens, L, T, hkv, D, bs, seed, dev, ties=False, width=None):
    g = torch.Generator().manual_seed(seed)
    caches = []
    for i in range(L):
        k, v, tables, left = ref.paged(lens, T, hkv, D, bs, torch.Generator().manual_seed(seed), dev, width=width,
                                       spare=sum(-(-n // bs) for n in lens) + 3)
        caches.append((k + i, v - 3 * i))
    cap = tables.shape[1] * bs
    mass = torch.rand((L, len(lens), hkv, cap), generator=g) ** 6
    if ties:
        mass = (mass * 4).round() / 4
    return caches, mass.to(dev), tables, torch.tensor(lens, dtype=torch.int32).to(dev), left


def _evict_check(caches, before, mass, tables, lens, dst, keep, new, mass_out, budget, sinks, recent, bs):
    want = [tuple(x.clone() for x in c) for c in before]
    for n, length in enumerate(lens.tolist()):
        assert new[n] == min(length, budget)
        for layer in range(len(before)):
            for h in range(mass.shape[2]):
                row = mass[layer, n, h].tolist()
                kept = ref.evict_ref(row, length, budget, sinks, recent)
                assert keep[layer, n, h].tolist() == kept + [-1] * (budget - len(kept)), (layer, n, h)
                m = mass_out[layer, n, h]
                assert torch.equal(m[:len(kept)], mass[layer, n, h, kept]) or any(map(math.isnan, row))
                assert (m[len(kept):] == 0).all()
                pos = torch.arange(len(kept))
                at = torch.tensor(kept, dtype=torch.long)
                src = (tables[n].cpu()[at // bs] * bs + at % bs).to(mass.device)
                to = (dst[n].cpu()[pos // bs] * bs + pos % bs).to(mass.device)
                for w, b in zip(want[layer], before[layer]):
                    w[:, h, to.long()] = b[:, h, src.long()]
    for got, w in zip(caches, want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("place", ["own", "other"])
@pytest.mark.parametrize("lens,L,T,hkv,D,bs,budget,sinks,recent", [
    ([200, 64, 65, 1, 0, 63], 2, 2, 2, 64, 16, 64, 4, 32),
    ([3000, 1100, 900], 3, 4, 2, 64, 16, 1000, 4, 32),
    ([5000], 1, 1, 4, 32, 32, 4097, 0, 0),
    ([700, 130], 1, 2, 2, 128, 8, 129, 1, 128),        # nothing left to choose
    ([300, 90], 70, 1, 1, 96, 64, 80, 0, 1),           # two launches of layers
    ([40, 500], 1, 3, 2, 45, 1, 1, 1, 0),              # one token, blocks of one
    ([2049, 100], 1, 1, 1, 64, 16, 2, 0, 1),
    ([9000, 8192, 1500], 1, 1, 2, 64, 16, 2000, 4, 32),
    ([33000, 40], 1, 1, 1, 64, 64, 30000, 4, 32),      # masses read again, not kept in registers
])
def test_eviction(gpu, lens, L, T, hkv, D, bs, budget, sinks, recent, place, ties):
    caches, mass, tables, seq, left = _evict_case(lens, L, T, hkv, D, bs, sum(lens) + budget, gpu, ties)
    before, given = [tuple(x.clone() for x in c) for c in caches], mass.clone()
    nb = -(-min(budget, max(lens)) // bs)
    if place == "own":
        keep, new = evict_cache(caches, mass, tables, seq, budget, bs, sinks, recent)
        dst, got = tables, mass
    else:
        dst = torch.full((len(lens), -(-budget // bs)), int(left[0]), dtype=torch.int32)
        at = 1
        for n, x in enumerate(lens):
            need = -(-min(x, budget) // bs)
            dst[n, :need] = left[at:at + need]
            at += need
        assert nb <= dst.shape[1]
        dst = dst.to(gpu)
        got = torch.full_like(mass, -1.0)
        keep, new = evict_cache(caches, mass, tables, seq, budget, bs, sinks, recent, dst_tables=dst, mass_out=got)
        assert torch.equal(mass, given)
    _evict_check(caches, before, given, tables, seq, dst, keep, new, got, budget, sinks, recent, bs)


def test_odd_masses(gpu):
    """NaN last, infinities in order, -0 and +0 equal, negative and subnormal masses."""
    caches, mass, tables, seq, _ = _evict_case([64], 1, 1, 2, 64, 16, 4, gpu)
    odd = [math.nan, math.inf, -math.inf, -0.0, 0.0, 1e-42, -1e-42, 1.0, -1.0, math.nan, 2.0, 0.0, -0.0, 3e38, -3e38]
    mass[0, 0, 0, :60] = torch.tensor(odd * 4)
    mass[0, 0, 1, :] = math.nan
    for budget in (2, 9, 20, 33, 47, 63):
        layers = [tuple(x.clone() for x in c) for c in caches]
        m = mass.clone()
        keep, new = evict_cache(layers, m, tables, seq, budget, 16, 1, 1)
        _evict_check(layers, caches, mass, tables, seq, tables, keep, new, m, budget, 1, 1, 16)


def test_eviction_again_and_again_in_a_graph(gpu):
    """A captured in-place eviction replayed for other lengths and masses."""
    caches, mass, tables, seq, _ = _evict_case([900, 300], 2, 2, 2, 64, 16, 6, gpu)
    first = [tuple(x.clone() for x in c) for c in caches]
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep, new = evict_cache(caches, mass, tables, seq, 128, 16)
    g = torch.Generator().manual_seed(8)
    for lens in ([900, 300], [50, 129], [640, 128]):
        for c, f in zip(caches, first):
            for x, y in zip(c, f):
                x.copy_(y)
        given = torch.rand(mass.shape, generator=g).to(gpu)
        mass.copy_(given)
        seq.copy_(torch.tensor(lens))
        graph.replay()
        torch.cuda.synchronize(gpu)
        _evict_check(caches, first, given, tables, seq, tables, keep, new, mass, 128, 4, 32, 16)
