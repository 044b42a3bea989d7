"""The draft-tree and eviction operators together: large strides, streams, shared scratch,
sequences that meet different kernels, and arguments that are refused."""
from __future__ import annotations

import pytest
import torch

import cache_ops_ref as ref
from spikeinfer_amd.kernels import (
    accept_draft_tree,
    draft_tree_masks,
    evict_cache,
    key_mass_workspace_bytes,
    paged_spike_attn_key_mass,
    paged_spike_attn_tree,
    tree_attn_workspace_bytes,
)
from test_eviction_gpu import _check, _mass_case, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,hq,hkv,D,bs,lens,rows", [
    (4, 16, 4, 128, 16, [1500, 40], None),           # four timestep groups of one
    (3, 4, 1, 128, 8, [70, 1030], None),             # blocks smaller than a key tile
    (8, 8, 2, 64, 16, [2100, 5], None),
    (4, 8, 8, 32, 2, [1025, 3], None),               # one group of four timesteps
    (6, 4, 4, 128, 16, [1100, 17], None),            # more groups than a wave holds
    (4, 14, 2, 64, 4, [1300, 70], [20, 3]),
    (2, 4, 2, 96, 8, [40, 2050], [9, 40]),
    (4, 14, 2, 64, 2048, [2500, 100], [1, 70]),      # blocks larger than a part
])
def test_key_mass_kernels(gpu, T, hq, hkv, D, bs, lens, rows):
    print(f"mass {T} {hq}/{hkv} {D} {bs} {lens} {rows}", flush=True)
    c = _mass_case(T, hq, hkv, D, bs, lens, rows, D + sum(lens), gpu)
    _check(c, paged_spike_attn_key_mass(**c), _want(c))


@pytest.mark.parametrize("T,D,bs", [(4, 64, 16), (4, 128, 16), (3, 128, 4), (8, 64, 16), (1, 32, 16)])
def test_key_mass_is_the_same_from_every_kernel(gpu, T, D, bs):
    """A sequence's one row alone, under a longer table, and beside a sequence of many rows."""
    lens = [900, 1500]
    c = _mass_case(T, 8, 2, D, bs, lens, [1, 60], 3, gpu)
    both = paged_spike_attn_key_mass(**c)
    used = -(-lens[0] // bs)
    one = dict(c, q_packed=c["q_packed"][:, :1], seq_lens=c["seq_lens"][:1], row_starts=None, max_rows=1)
    for tables in (c["block_tables"][:1, :used], c["block_tables"][:1],
                   torch.nn.functional.pad(c["block_tables"][:1], (0, 5000))):
        got = paged_spike_attn_key_mass(**dict(one, block_tables=tables.contiguous()))
        assert torch.equal(got[0, :, :lens[0]], both[0, :, :lens[0]])
        assert (got[..., lens[0]:] == 0).all()


def _far(cache):
    """The same words in planes of 2**33 bytes."""
    T, H, slots, W = cache.shape
    big = torch.empty((T, H, slots, 2**31 // slots + 7), dtype=torch.int32, device=cache.device)
    far = big[..., :W]
    far.copy_(cache)
    assert far.stride(1) * 4 > 2**32
    return far


def test_offsets_past_32_bits(gpu):
    """Caches whose planes pass 2**32 bytes give what compact ones give."""
    T, hq, D, bs, lens = 2, 4, 64, 16, [3900, 60]
    case = ref.tree_case(T, hq, 1, D, bs, [(n, k) for n, k in zip(lens, (30, 5))], 4, gpu)
    near = (case["k_cache"], case["v_cache"])
    far = tuple(_far(x) for x in near)
    assert int(case["block_tables"].max()) * bs * far[0].stride(2) > 2**30
    for dtype in (torch.float32, torch.bfloat16):
        a = paged_spike_attn_tree(**case, dtype=dtype)
        b = paged_spike_attn_tree(**dict(case, k_cache=far[0], v_cache=far[1]), dtype=dtype)
        assert torch.equal(a, b)
    for starts, most in ((None, 1), (ref.starts_of([30, 5]).to(gpu), 30)):
        m = dict(q_packed=case["q_packed"], block_tables=case["block_tables"], seq_lens=case["context_lens"], head_dim=D,
                 block_size=bs, row_starts=starts, max_rows=most)
        mass = paged_spike_attn_key_mass(k_cache=near[0], **m)
        assert torch.equal(mass, paged_spike_attn_key_mass(k_cache=far[0], **m))
    rows = case["q_packed"].shape[1]
    tokens = torch.zeros(rows, dtype=torch.int64, device=gpu)
    parents = torch.tensor([-1, *range(29), -1, *range(4), -1, -1], dtype=torch.int32, device=gpu)
    lens_short = case["context_lens"] - 40
    words = [(case["k_words"], case["v_words"])]
    for layer in (near, far):
        accept_draft_tree(tokens, parents, tokens, case["row_starts"], 30, words, [layer], case["block_tables"],
                          lens_short, bs)
    for x, y in zip(near, far):
        assert torch.equal(x, y)
    old = near[0].clone()
    kept = [evict_cache([layer], mass[None].clone(), case["block_tables"], case["context_lens"], 500, bs)
            for layer in (near, far)]
    assert torch.equal(kept[0][0], kept[1][0]) and not torch.equal(near[0], old)
    for x, y in zip(near, far):
        assert torch.equal(x, y)


def test_on_another_stream(gpu):
    """Every operator behind work of its own stream, arguments of the usual and of other forms."""
    case = ref.tree_case(2, 14, 2, 64, 16, [(3000, 12), (50, 3)], 2, gpu)
    starts = case["row_starts"]
    parents = torch.tensor([-1, *range(11), -1, 0, 1, -1, -1], dtype=torch.int32, device=gpu)
    tokens = torch.zeros(parents.numel(), dtype=torch.int64, device=gpu)
    layer = (case["k_cache"], case["v_cache"])

    def run(lens):
        masks, depths = draft_tree_masks(parents, starts, 12)
        out = paged_spike_attn_tree(**dict(case, masks=masks, context_lens=lens))
        mass = paged_spike_attn_key_mass(case["q_packed"], case["k_cache"], case["block_tables"], lens, 64, 16, starts, 12)
        caches = [tuple(x.clone() for x in layer)]
        path = accept_draft_tree(tokens, parents, tokens, starts, 12, [(case["k_words"], case["v_words"])], caches,
                                 case["block_tables"], lens - 20, 16)
        keep = evict_cache(caches, mass[None], case["block_tables"], lens, 128, 16)
        return [masks, depths, out, mass, *path, *keep, *caches[0]]

    want = run(case["context_lens"])
    torch.cuda.synchronize(gpu)
    for form in (torch.int32, torch.int64):
        stream = torch.cuda.Stream(gpu)
        with torch.cuda.stream(stream):
            x = torch.zeros((4096, 4096), device=gpu)
            for _ in range(20):  # the lengths come late
                x = x @ x
            lens = (case["context_lens"] + x[0, 0].int()).to(form)
            got = run(lens)
        stream.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_graphs_that_share_their_scratch(gpu):
    cases = [ref.tree_case(2, 14, 2, 64, 16, trees, 7 + i, gpu) for i, trees in
             enumerate(([(5000, 20), (70, 3)], [(2500, 9), (4100, 20)]))]
    need = max(tree_attn_workspace_bytes(2, 2, 14, 2, 64, c["max_nodes"], 16, c["block_tables"].shape[1]) for c in cases)
    need = max([need] + [key_mass_workspace_bytes(2, 2, 14, 2, 64, 20, 16, c["block_tables"].shape[1]) for c in cases])
    scratch = torch.empty(need, dtype=torch.uint8, device=gpu)

    def run(c, ws, out, mass):
        paged_spike_attn_tree(**c, out=out, workspace=ws)
        paged_spike_attn_key_mass(c["q_packed"], c["k_cache"], c["block_tables"], c["context_lens"], 64, 16,
                                  c["row_starts"], 20, out=mass, workspace=ws)

    graphs, outs = [], []
    for c in cases:
        outs.append([torch.zeros((*c["q_packed"].shape[:3], 64), device=gpu),
                     torch.zeros((2, 2, c["block_tables"].shape[1] * 16), device=gpu)])
        run(c, None, *outs[-1])
    want = [[x.clone() for x in o] for o in outs]
    torch.cuda.synchronize(gpu)
    for c, o in zip(cases, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(c, scratch, *o)
    for turn in (0, 1, 1, 0, 0, 1):
        for x in outs[turn]:
            x.fill_(-1.0)
        outs[turn][0][:, -2:] = 0  # rows of no tree
        graphs[turn].replay()
        torch.cuda.synchronize(gpu)
        for a, b in zip(outs[turn], want[turn]):
            assert torch.equal(a, b)


def test_refused_arguments(gpu):
    """Wrong types, shapes and devices name their argument; nothing is launched."""
    c = ref.tree_case(2, 14, 2, 64, 16, [(40, 5), (9, 3)], 1, gpu)
    R = c["q_packed"].shape[1]
    f = lambda *shape: torch.zeros(shape, device=gpu)
    for kw in (dict(head_dim=32), dict(max_nodes=0), dict(max_nodes=2000), dict(max_nodes=65), dict(block_size=12),
               dict(q_packed=c["q_packed"].float()), dict(q_packed=c["q_packed"][:, :, :13]),
               dict(k_words=c["k_words"][:, :-1]), dict(v_words=c["v_words"][:, :, :1]),
               dict(v_cache=c["v_cache"][:, :, 16:]), dict(k_cache=c["k_cache"][:1], v_cache=c["v_cache"][:1]),
               dict(block_tables=c["block_tables"][0]), dict(context_lens=c["context_lens"][:1]),
               dict(row_starts=c["row_starts"][:2]), dict(masks=c["masks"].int()), dict(masks=c["masks"][1:]),
               dict(context_lens=c["context_lens"].cpu()), dict(masks=c["masks"].cpu()),
               dict(out=f(2, R, 14, 32)), dict(out=f(2, R, 14, 64).int()), dict(out=f(1, R, 14, 64).expand(2, R, 14, 64)),
               dict(block_tables=torch.zeros((2, 400), dtype=torch.int32, device=gpu),
                    workspace=torch.zeros(16, dtype=torch.uint8, device=gpu))):
        with pytest.raises(ValueError):
            paged_spike_attn_tree(**dict(c, **kw))
            raise AssertionError(kw)
    m = dict(q_packed=c["q_packed"], k_cache=c["k_cache"], block_tables=c["block_tables"], seq_lens=c["context_lens"],
             head_dim=64, block_size=16)
    for kw in (dict(head_dim=96), dict(block_size=0), dict(q_packed=c["q_packed"][:, :1]), dict(q_packed=c["q_packed"][:1]),
               dict(k_cache=c["k_cache"].float()), dict(seq_lens=c["context_lens"][:1]), dict(accumulate=True),
               dict(row_starts=c["row_starts"], max_rows=0), dict(row_starts=c["row_starts"][:2], max_rows=5),
               dict(out=f(2, 2, 48).half()), dict(out=f(2, 1, 48)), dict(out=f(1, 2, 48).expand(2, 2, 48)),
               dict(seq_lens=c["context_lens"].cpu()), dict(workspace=torch.zeros(8, dtype=torch.uint8, device=gpu))):
        with pytest.raises(ValueError):
            paged_spike_attn_key_mass(**dict(m, **kw))
            raise AssertionError(kw)
    layer, words = (c["k_cache"], c["v_cache"]), (c["k_words"], c["v_words"])
    ids, par = torch.zeros(R, dtype=torch.int64, device=gpu), torch.full((R,), -1, dtype=torch.int32, device=gpu)
    a = dict(tokens=ids, parents=par, targets=ids, row_starts=c["row_starts"], max_nodes=5, drafts=[words], layers=[layer],
             block_tables=c["block_tables"], context_lens=c["context_lens"], block_size=16)
    for kw in (dict(tokens=ids.int()), dict(targets=ids[1:]), dict(parents=par[1:]), dict(drafts=[]),
               dict(drafts=[words] * 2, layers=[layer] * 2), dict(drafts=[tuple(w[:, 1:] for w in words)]),
               dict(block_tables=None), dict(block_tables=c["block_tables"][:1]), dict(block_size=5), dict(max_nodes=1025),
               dict(context_lens=c["context_lens"].cpu()), dict(layers=[(layer[0], layer[1].cpu())]),
               dict(out=(ids.int(), ids.int(), ids))):
        with pytest.raises(ValueError):
            accept_draft_tree(**dict(a, **kw))
            raise AssertionError(kw)
    e = dict(layers=[layer], mass=f(1, 2, 2, 48), block_tables=c["block_tables"], seq_lens=c["context_lens"], budget=40,
             block_size=16)
    for kw in (dict(layers=[]), dict(layers=[layer] * 2, mass=f(2, 2, 2, 48)), dict(mass=f(1, 2, 1, 48)),
               dict(mass=f(1, 2, 2, 48).double()), dict(mass=f(1, 1, 1, 48).expand(1, 2, 2, 48)), dict(budget=20),
               dict(budget=0), dict(sinks=-1), dict(mass_out=f(1, 2, 2, 47)), dict(block_size=3),
               dict(dst_tables=c["block_tables"][:1]), dict(dst_tables=c["block_tables"][:, :1].contiguous()),
               dict(seq_lens=c["context_lens"][:1]), dict(mass=f(1, 2, 2, 48).cpu())):
        with pytest.raises(ValueError):
            evict_cache(**dict(e, **kw))
            raise AssertionError(kw)
