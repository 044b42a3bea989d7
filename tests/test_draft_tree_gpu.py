"""Draft trees on the GPU against plain float64 code: tree attention, masks, acceptance.

Attention outputs lie in [0, 1].  fp32: weights exact to 2**-23 and sums of at most a
few hundred 32-key partial sums, so 4e-6 as for the prefill kernel; fp16 adds half a step
(2**-12 below 1); bf16 adds half a step (2**-9) and weights of 11 bits: each is off by at
most 2**-11, a quotient of two sums of them by 2**-10.
"""
from __future__ import annotations

import pytest
import torch

import cache_ops_ref as ref
from spikeinfer_amd.kernels import accept_draft_tree, draft_tree_masks, paged_spike_attn_tree

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 4e-6, torch.float16: 4e-6 + 2.0**-12, torch.bfloat16: 4e-6 + 2.0**-9 + 2.0**-10}


def _run(case, dtype=torch.float32, **kw):
    T, R, hq, _ = case["q_packed"].shape
    out = torch.full((T, R, hq, case["head_dim"]), -7.0, dtype=dtype, device=case["masks"].device)
    got = paged_spike_attn_tree(**case, out=out, **kw)
    assert got is out
    return out


def _check(case, out):
    before = torch.full_like(out, -7.0)
    err = (out.double() - ref.tree_want(case, before)).abs().max().item()
    assert err <= TOL[out.dtype], err


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,hq,hkv,D,bs,trees", [
    (4, 14, 2, 64, 16, [(0, 1), (1, 1), (5, 3), (33, 64)]),         # one key, one row, a full mask word
    (4, 14, 2, 64, 16, [(128, 8), (1000, 16), (0, 40), (31, 33), (32, 0), (64, 32)]),
    (2, 14, 2, 64, 32, [(5000, 30), (2047, 5), (2048, 5), (2049, 5)]),  # contexts that are cut
    (1, 4, 4, 32, 16, [(31, 70), (64, 1), (0, 129)]),               # one word, no GQA, three mask words
    (2, 6, 2, 96, 64, [(70, 20), (600, 5)]),
    (2, 16, 1, 128, 16, [(129, 19), (2500, 200)]),
    (2, 16, 4, 128, 8, [(4200, 25), (90, 2)]),
    (2, 4, 1, 45, 16, [(20, 3), (300, 9)]),                         # channels past the head, unaligned rows
    (3, 8, 8, 64, 1, [(300, 7), (64, 50)]),                         # blocks of one token
    (1, 34, 2, 64, 16, [(100, 9)]),                                 # 17 heads a kv head
    (1, 2, 2, 8, 16, [(40, 1024)]),                                 # the widest tree
])
def test_matches_float64(gpu, T, hq, hkv, D, bs, trees, dtype):
    case = ref.tree_case(T, hq, hkv, D, bs, trees, D + sum(n for _, n in trees), gpu)
    print(f"tree {T} {hq}/{hkv} {D} {trees} {dtype}", flush=True)
    _check(case, _run(case, dtype))


@pytest.mark.parametrize("D,hq", [(64, 14), (128, 4)])
def test_dense_and_silent_words(gpu, D, hq):
    """Scores at both ends of the weights' range, for each output type."""
    for qd, kd in ((1.1, 1.1), (1.1, 0.0), (0.0, 1.1), (1.1, 0.5), (1.1, 0.05)):
        case = ref.tree_case(2, hq, 2, D, 16, [(300, 20), (2100, 3)], 5, gpu, density=kd, q_density=qd)
        for dtype in TOL:
            _check(case, _run(case, dtype))


def test_any_mask_and_rows_that_see_nothing(gpu):
    """Random masks (not trees), empty ones with and without context, bits past the
    tree's rows, a self-only mask."""
    case = ref.tree_case(2, 14, 2, 64, 16, [(0, 50), (77, 50), (0, 3)], 11, gpu)
    g = torch.Generator().manual_seed(3)
    m = torch.randint(-2**63, 2**63 - 1, case["masks"].shape, generator=g)
    m[0] = m[7] = m[60] = m[100] = 0
    m[5] = 1 << 5
    m[49] = -1  # bits of rows that the tree does not have
    m[20] = -(1 << 50)  # only such bits
    case["masks"] = m.to(gpu)
    out = _run(case)
    _check(case, out)
    for row in (0, 7, 20, 100):
        assert (out[:, row] == 0).all()
    assert (out[:, 60] != 0).any()


def test_rows_left_out_and_odd_row_starts(gpu):
    """Rows beyond max_nodes, before the first and behind the last sequence keep what
    they hold; row_starts past the buffer end there."""
    case = ref.tree_case(2, 14, 2, 64, 16, [(40, 9), (50, 12), (10, 4)], 7, gpu, spare_rows=6)
    case["max_nodes"] = 10
    out = _run(case)
    _check(case, out)
    assert (out[:, 9 + 10:9 + 12] == -7).all() and (out[:, 25:] == -7).all()
    case["row_starts"] = torch.tensor([3, 9, 9, 2**30], dtype=torch.int32, device=gpu)
    out = _run(case)
    assert (out[:, :3] == -7).all() and (out[:, 19:] == -7).all() and (out[:, 9:19] != -7).all()
    case["row_starts"] = torch.tensor([-5, -2, -1, 0], dtype=torch.int32, device=gpu)
    assert (_run(case) == -7).all()


def test_strides_orders_and_types_of_arguments(gpu):
    """Words and outputs in other orders, int64 index tensors, a table that is a column
    slice, blocks outside the cache (zero spikes, still counted), lengths past the table."""
    case = ref.tree_case(3, 14, 2, 64, 16, [(90, 12), (33, 5)], 13, gpu)
    want = _run(case)
    other = dict(case)
    flip = lambda t: t.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)
    other["q_packed"] = flip(case["q_packed"])
    for name in ("k_words", "v_words", "k_cache", "v_cache"):
        wide = torch.zeros((*case[name].shape[:3], 5), dtype=torch.int32, device=gpu)
        wide[..., 1:3] = case[name]
        other[name] = wide[..., 1:3]
    other["block_tables"] = torch.cat([case["block_tables"]] * 2, 1).long()[:, :6]
    other["context_lens"], other["row_starts"] = case["context_lens"].long(), case["row_starts"].long()
    big = torch.full((14, 3, 70, 19), -7.0, device=gpu)
    out = big[:, :, 1:65].permute(1, 3, 0, 2)  # channels not contiguous
    with pytest.raises(ValueError, match="contiguous channels"):
        paged_spike_attn_tree(**other, out=out)
    big = torch.full((14, 19, 3, 66), -7.0, device=gpu)
    out = big.permute(2, 1, 0, 3)[..., 1:65]
    paged_spike_attn_tree(**other, out=out)
    assert torch.equal(out, want) and (big[..., 0] == -7).all() and (big[..., 65] == -7).all()

    case["block_tables"] = case["block_tables"].clone()
    case["block_tables"][0, 1] = -1
    case["block_tables"][0, 3] = 10**6
    case["block_tables"][1, 0] = 2**31 - 1
    case["context_lens"] = torch.tensor([10**9, -4], dtype=torch.int32, device=gpu)
    _check(case, _run(case))


def test_sequences_do_not_depend_on_their_batch(gpu):
    """Bit-identical alone, in a batch, and with a wider table and max_nodes."""
    trees = [(3000, 16), (70, 9)] + [(17 * i, 1 + i % 7) for i in range(60)] + [(9000, 3)]
    case = ref.tree_case(4, 14, 2, 64, 16, trees, 21, gpu)
    for dtype in TOL:
        out = _run(case, dtype)
        _check(case, out)
        for n in (0, 1, len(trees) - 1):
            a, e = case["row_starts"][n].item(), case["row_starts"][n + 1].item()
            one = {k: (v[:, a:e] if k.endswith(("words", "packed")) else v) for k, v in case.items()}
            one.update(masks=case["masks"][a:e], block_tables=case["block_tables"][n:n + 1],
                       context_lens=case["context_lens"][n:n + 1], max_nodes=max(e - a, 1),
                       row_starts=torch.tensor([0, e - a], dtype=torch.int32, device=gpu))
            assert torch.equal(_run(one, dtype), out[:, a:e]), n
        wide = dict(case, block_tables=torch.nn.functional.pad(case["block_tables"], (0, 500)), max_nodes=64)
        assert torch.equal(_run(wide, dtype), out)


def test_captured_call_takes_other_trees(gpu):
    """One capture, replayed for other lengths, trees and words, each against the eager
    call, with eager work between; and on a stream of its own."""
    base = ref.tree_case(2, 14, 2, 64, 16, [(2500, 12), (100, 12), (60, 12)], 31, gpu)
    static = {k: v.clone() if torch.is_tensor(v) else v for k, v in base.items()}
    out = torch.full((2, 38, 14, 64), -7.0, device=gpu)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        paged_spike_attn_tree(**static, out=out)
    torch.cuda.current_stream(gpu).wait_stream(side)
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_spike_attn_tree(**static, out=out)
    for seed, trees in ((1, [(2500, 12), (100, 12), (60, 12)]), (2, [(0, 1), (2201, 7), (0, 0)]),
                        (3, [(63, 12), (0, 5), (2048, 12)])):
        case = ref.tree_case(2, 14, 2, 64, 16, trees, seed, gpu, spare_rows=38 - sum(n for _, n in trees))
        case["max_nodes"] = 12
        for name in ("q_packed", "k_words", "v_words", "masks", "context_lens", "row_starts"):
            static[name].copy_(case[name])
        for name in ("k_cache", "v_cache"):
            static[name][:, :, :case[name].shape[2]] = case[name]
        static["block_tables"].zero_()
        static["block_tables"][:, :case["block_tables"].shape[1]] = case["block_tables"]
        out.fill_(-7.0)
        graph.replay()
        eager = _run(static)
        torch.cuda.synchronize(gpu)
        assert torch.equal(out, eager)
        _check(static, out)


def test_masks_and_depths(gpu):
    g = torch.Generator().manual_seed(2)
    counts = [1, 64, 0, 65, 200, 3]
    parents = [ref.random_parents(c, g) if c else [] for c in counts]
    want = torch.cat([ref.ancestor_masks(p, 4) for p in parents])
    flat = torch.tensor(sum(parents, []) + [0, 1], dtype=torch.int32, device=gpu)
    starts = ref.starts_of(counts).to(gpu)
    masks, depths = draft_tree_masks(flat, starts, 200)
    assert torch.equal(masks[:-2].cpu(), want) and (masks[-2:] == 0).all()
    bits = sum(((want >> b) & 1).sum(1) for b in range(64))
    assert torch.equal(depths[:-2].cpu(), bits.int() - 1)
    # numbers that are not below the row end its chain; rows of no sequence stay
    odd = torch.tensor([5, 1, -3, 2, 4, 0], dtype=torch.int32, device=gpu)
    m = torch.full((6, 2), 77, dtype=torch.int64, device=gpu)
    d = torch.full((6,), 77, dtype=torch.int32, device=gpu)
    draft_tree_masks(odd, torch.tensor([0, 5], dtype=torch.int32, device=gpu), 100, m, d)
    assert m.tolist() == [[1, 0], [2, 0], [4, 0], [12, 0], [16, 0], [77, 77]]
    assert d.tolist() == [0, 0, 0, 1, 0, 77]


@pytest.mark.parametrize("counts,layers", [([5], 1), ([8, 1, 0, 61, 200], 3), ([30] * 64, 24), ([1024], 70)])
def test_acceptance_and_commit(gpu, counts, layers):
    g = torch.Generator().manual_seed(sum(counts))
    T, hkv, D, bs = 2, 2, 64, 16
    parents = [ref.random_parents(c, g) if c else [] for c in counts]
    R = sum(counts) + 1
    tokens = torch.randint(0, 4, (R,), generator=g)
    targets = torch.randint(0, 4, (R,), generator=g)
    ctx = torch.randint(0, 100, (len(counts),), generator=g)
    k, v, tables, _ = ref.paged(ctx + max(counts), T, hkv, D, bs, g, gpu)
    caches = [(k + 5 * i, v - i) for i in range(layers)]
    new = [tuple(ref.words((T, R, hkv), D, g, gpu) for _ in range(2)) for _ in range(min(layers, 3))]
    new += [tuple(x ^ i for x in new[0]) for i in range(3, layers)]
    want = [tuple(x.clone() for x in c) for c in caches]
    starts = ref.starts_of(counts)
    path, count, after = accept_draft_tree(
        tokens.to(gpu), torch.tensor(sum(parents, []) + [0], dtype=torch.int32, device=gpu), targets.to(gpu),
        starts.to(gpu), max(counts), new, caches, tables, ctx.int().to(gpu), bs)
    for n, c in enumerate(counts):
        a = int(starts[n])
        p, t = ref.accept_ref(tokens[a:a + c].tolist(), parents[n], targets[a:a + c].tolist())
        assert path[n].tolist() == p + [-1] * (max(counts) - len(p))
        assert count[n] == len(p) and after[n] == t
        for i, row in enumerate(p):
            pos = int(ctx[n]) + i
            slot = int(tables[n, pos // bs]) * bs + pos % bs
            for w, x in zip(want, new):
                for dst, src in zip(w, x):
                    dst[:, :, slot] = src[:, a + row]
    for got, w in zip(caches, want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_acceptance_alone_bad_tables_and_replay(gpu):
    """No caches; siblings with one token; steps past the table or the cache are dropped;
    a captured call takes other tokens."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    i64 = lambda *x: torch.tensor(x, device=gpu)
    starts = i32(0, 5)
    parents = i32(-1, 0, 0, 2, 1)
    path, count, after = accept_draft_tree(i64(9, 4, 4, 5, 5), parents, i64(4, 5, 5, 6, 7), starts, 6)
    assert path.tolist() == [[0, 1, 4, -1, -1, -1]] and count.tolist() == [3] and after.tolist() == [7]
    T, hkv, bs = 1, 1, 4
    cache = torch.zeros((T, hkv, 12, 2), dtype=torch.int32, device=gpu)
    new = torch.arange(1, 11, dtype=torch.int32, device=gpu).view(1, 5, 1, 2)
    args = [[(new, new)], [(cache, cache.clone())]]
    accept_draft_tree(i64(9, 4, 4, 5, 5), parents, i64(4, 5, 5, 6, 7), starts, 6, *args,
                      i32(2, 7).view(1, 2), i32(3), bs)
    assert cache[0, 0, 11].tolist() == [1, 2] and cache.sum() == 3  # block 7 lies outside
    accept_draft_tree(i64(9, 4, 4, 5, 5), parents, i64(4, 5, 5, 6, 7), starts, 6, *args, i32(0, 1).view(1, 2),
                      i32(6), bs)
    assert cache[0, 0, 6:8].tolist() == [[1, 2], [3, 4]] and cache[0, 0, :6].sum() == 0  # the table ends at 8

    tok, tgt = i64(9, 4, 4, 5, 5), i64(4, 5, 5, 6, 7)
    out = (torch.empty((1, 6), dtype=torch.int32, device=gpu), i32(0), i64(0))
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        accept_draft_tree(tok, parents, tgt, starts, 6, out=out)
    for values, want in (((4, 5, 5, 6, 7), [0, 1, 4]), ((3, 5, 5, 6, 7), [0]), ((4, 1, 5, 6, 7), [0, 1])):
        tgt.copy_(i64(*values))
        graph.replay()
        torch.cuda.synchronize(gpu)
        assert out[0][0, :out[1].item()].tolist() == want and out[2].item() == values[want[-1]]


def test_empty_calls(gpu):
    case = ref.tree_case(2, 4, 2, 64, 16, [(5, 3)], 1, gpu)
    none = dict(case, block_tables=case["block_tables"][:0], context_lens=case["context_lens"][:0],
                row_starts=case["row_starts"][:1])
    assert (_run(none) == -7).all()
    assert (paged_spike_attn_tree(**none) == 0).all()
    empty = dict(case, q_packed=case["q_packed"][:, :0], k_words=case["k_words"][:, :0],
                 v_words=case["v_words"][:, :0], masks=case["masks"][:0])
    assert paged_spike_attn_tree(**empty).shape == (2, 0, 4, 64)
    z = torch.zeros(0, dtype=torch.int32, device=gpu)
    masks, depths = draft_tree_masks(z, torch.zeros(1, dtype=torch.int32, device=gpu), 8)
    assert masks.shape == (0, 1) and depths.shape == (0,)
    path, count, after = accept_draft_tree(z.long(), z, z.long(), torch.zeros(3, dtype=torch.int32, device=gpu), 4)
    assert (path == -1).all() and count.tolist() == [0, 0] and after.tolist() == [-1, -1]
