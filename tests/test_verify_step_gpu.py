"""The cache operators together, as a decoder uses them: a step that verifies drafted
trees (forward over the rows, tokens, acceptance, commit), eager and captured, and decoding
with accumulated weights and evictions between the steps."""
from __future__ import annotations

import math
from dataclasses import replace

import pytest
import torch

import cache_ops_ref as ref
from spikeinfer_amd.attention import AttentionMetadata, DraftTrees
from spikeinfer_amd.kernels import (accept_draft_tree, draft_tree_masks, paged_spike_attn_decode,
                                    paged_spike_attn_key_mass)
from spikeinfer_amd.model import SpikingDecoder, SpikingQwenConfig
from spikeinfer_amd.sampler import sample_tokens
from spikeinfer_amd.spike_cache import PagedSpikeCache

pytestmark = pytest.mark.gpu
BS = 16


def _model(gpu, layers=2, vocab=512):
    return SpikingDecoder(SpikingQwenConfig(vocab_size=vocab, hidden_size=512, intermediate_size=1024,
                                            num_hidden_layers=layers, num_attention_heads=8, num_key_value_heads=2,
                                            max_position_embeddings=512), device=gpu, seed=3, init_std=0.05)


def _prefill(model, cache, prompts, tables, gpu):
    ids, pos, slots, starts = [], [], [], []
    for p, tab in zip(prompts, tables.tolist()):
        starts.append(len(ids))
        ids += p
        pos += range(len(p))
        slots += [tab[i // BS] * BS + i % BS for i in range(len(p))]
    meta = AttentionMetadata(slot_mapping=torch.tensor(slots, device=gpu), block_size=BS, prefill_query_starts=starts,
                             prefill_query_lens=[len(p) for p in prompts], prefill_context_lens=[0] * len(prompts),
                             prefill_block_tables=[t.to(gpu) for t in tables])
    model.forward_paged(torch.tensor(ids, device=gpu), torch.tensor(pos, device=gpu), cache.layers, meta)


def _decode(model, cache, ids, lens, tables, key_mass=None, positions=None):
    """One decode step behind `lens` cached tokens: logits [N, vocab]."""
    slots = tables.long().gather(1, (lens.long() // BS)[:, None])[:, 0] * BS + lens.long() % BS
    meta = AttentionMetadata(slot_mapping=slots, block_size=BS, num_decode_tokens=len(ids), block_tables=tables,
                             seq_lens=(lens + 1).int(), key_mass=key_mass)
    pos = lens.long() if positions is None else positions
    return model.compute_logits(model.forward_paged(ids, pos, cache.layers, meta))


def _trees(gpu, counts, seed, vocab, chains):
    """Row starts, parents and tokens of random trees whose first rows are the given chains."""
    g = torch.Generator().manual_seed(seed)
    parents, tokens = [], []
    for c, chain in zip(counts, chains):
        p = ref.random_parents(c, g)
        p[1:len(chain)] = range(len(chain) - 1)
        t = torch.randint(0, vocab, (c,), generator=g).tolist()
        t[:len(chain)] = chain
        parents += p
        tokens += t
    return (ref.starts_of(counts).to(gpu), torch.tensor(parents, dtype=torch.int32, device=gpu),
            torch.tensor(tokens, device=gpu))


@pytest.mark.parametrize("layers", [1, 2])
def test_verifying_trees_against_decoding(gpu, layers):
    """Rows of a chain of the tokens that decoding gives: the first layer's words are
    decoding's bit for bit, every layer's cache gets the accepted rows' words, and the path is
    the one that the targets give.  One layer's logits are decoding's up to MLP spikes that a
    rounding of the attention turns (a layer adds less than it is given, and few spikes turn:
    under 5 % in the 2-norm); behind it keys differ by whole spikes, and nothing bounds that."""
    model, vocab = _model(gpu, layers), 512
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (37, 5, 90)]
    tables = torch.randperm(24, generator=g).int().view(3, 8)
    depth = 4
    plain, cache = (PagedSpikeCache(layers, 4, 2, 64, 25, BS, device=gpu) for _ in range(2))
    dev_tables = tables.to(gpu)
    for c in (plain, cache):
        _prefill(model, c, [p[:-1] for p in prompts], tables, gpu)
    lens = torch.tensor([len(p) - 1 for p in prompts], device=gpu)
    ids = torch.tensor([p[-1] for p in prompts], device=gpu)
    chain, want = [ids], []
    for i in range(depth):
        want.append(_decode(model, plain, chain[-1], lens + i, dev_tables))
        chain.append(want[-1].argmax(-1))
    counts = [depth + 9, depth, depth + 3]
    starts, parents, tokens = _trees(gpu, counts, 5, vocab, torch.stack(chain[:depth], 1).tolist())
    masks, depths = draft_tree_masks(parents, starts, max(counts))
    seq = torch.repeat_interleave(torch.arange(3, device=gpu), torch.tensor(counts, device=gpu))
    trees = DraftTrees(starts, masks, max(counts), lens.int(), dev_tables)
    meta = AttentionMetadata(slot_mapping=torch.full((len(seq),), -1, device=gpu), block_size=BS, draft=trees)
    before = [tuple(x.clone() for x in c) for c in cache.layers]
    logits = model.compute_logits(model.forward_paged(tokens, lens[seq] + depths, cache.layers, meta))
    for old, new in zip(before, cache.layers):  # nothing of the step is in the cache
        assert torch.equal(old[0], new[0]) and torch.equal(old[1], new[1])
    for i in range(depth if layers == 1 else 0):
        got = logits[(starts[:-1] + i).long()].float()
        assert (got - want[i].float()).norm() / want[i].float().norm() <= 0.05, i
    # greedy tokens of every row, and the walk
    targets = sample_tokens(logits, torch.zeros(len(seq), device=gpu))
    assert torch.equal(targets, logits.float().argmax(-1))
    path, count, after = accept_draft_tree(tokens, parents, targets, starts, max(counts), trees.words, cache.layers,
                                           dev_tables, lens.int(), BS)
    at = starts.tolist()
    for n in range(3):
        rows = slice(at[n], at[n + 1])
        p, t = ref.accept_ref(tokens[rows].tolist(), parents[rows].tolist(), targets[rows].tolist())
        assert path[n, :count[n]].tolist() == p and after[n] == t
        for i, row in enumerate(p):
            pos = int(lens[n]) + i
            slot = int(tables[n, pos // BS]) * BS + pos % BS
            for new, committed in zip(trees.words, cache.layers):
                for x, y in zip(new, committed):
                    assert torch.equal(x[:, at[n] + row], y[:, :, slot])
        agree = 0
        while agree < len(p) and p[agree] == agree and agree < depth:
            agree += 1
        assert agree >= 1
        for i in range(agree):  # as far as the path is the chain, the first layer's words are decoding's
            pos = int(lens[n]) + i
            slot = int(tables[n, pos // BS]) * BS + pos % BS
            for x, y in zip(cache.layers[0], plain.layers[0]):
                assert torch.equal(x[:, :, slot], y[:, :, slot]), (n, i)
    assert torch.isfinite(logits).all()


def test_captured_verification_replays(gpu):
    """Masks, forward, tokens, acceptance and commit in one graph, replayed for other trees
    and lengths, each time against the eager step on a copy of the cache."""
    model, vocab, N, M = _model(gpu, 1), 512, 4, 12
    g = torch.Generator().manual_seed(9)
    tables = torch.randperm(32, generator=g).int().view(4, 8).to(gpu)
    cache = PagedSpikeCache(1, 4, 2, 64, 33, BS, device=gpu)
    for x in cache.layers[0]:
        x.copy_(ref.words(x.shape[:3], 64, g, gpu))
    R = N * M
    static = dict(tokens=torch.zeros(R, dtype=torch.int64, device=gpu), lens=torch.ones(N, dtype=torch.int32, device=gpu),
                  parents=torch.full((R,), -1, dtype=torch.int32, device=gpu),
                  starts=torch.arange(N + 1, dtype=torch.int32, device=gpu))
    zero = torch.zeros(R, device=gpu)
    row = torch.arange(R, device=gpu)

    def step():
        s = static
        seq = torch.searchsorted(s["starts"][1:].contiguous(), row.int(), right=True).clamp(max=N - 1)
        masks, depths = draft_tree_masks(s["parents"], s["starts"], M)
        trees = DraftTrees(s["starts"], masks, M, s["lens"], tables)
        meta = AttentionMetadata(slot_mapping=torch.full((R,), -1, device=gpu), block_size=BS, draft=trees)
        out = model.forward_paged(s["tokens"], s["lens"].long()[seq] + depths, cache.layers, meta,
                                  dict(attn=torch.zeros((4, R, 8, 64), dtype=torch.bfloat16, device=gpu)))
        logits = model.compute_logits(out)
        targets = sample_tokens(logits, zero)
        return logits, *accept_draft_tree(s["tokens"], s["parents"], targets, s["starts"], M, trees.words, cache.layers,
                                          tables, s["lens"], BS)

    def fill(seed):
        h = torch.Generator().manual_seed(seed)
        counts = torch.randint(1, M + 1, (N,), generator=h).tolist()
        parents = sum([ref.random_parents(c, h) for c in counts], [])
        static["starts"].copy_(ref.starts_of(counts))
        static["parents"].fill_(-1)
        static["parents"][:len(parents)] = torch.tensor(parents, dtype=torch.int32)
        static["tokens"].copy_(torch.randint(0, vocab, (R,), generator=h))
        static["lens"].copy_(torch.randint(0, 100, (N,), generator=h))
        return sum(counts)

    with torch.no_grad():
        fill(0)
        side = torch.cuda.Stream(gpu)
        side.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream(gpu).wait_stream(side)
        torch.cuda.synchronize(gpu)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for seed in (1, 2, 3):
            live = fill(seed)
            old = [x.clone() for x in cache.layers[0]]
            eager = step()
            eager_cache = [x.clone() for x in cache.layers[0]]
            for x, y in zip(cache.layers[0], old):
                x.copy_(y)
            graph.replay()
            torch.cuda.synchronize(gpu)
            assert torch.equal(captured[0][:live], eager[0][:live])
            for x, y in zip(captured[1:], eager[1:]):
                assert torch.equal(x, y)
            for x, y in zip(cache.layers[0], eager_cache):
                assert torch.equal(x, y)
            assert not all(torch.equal(x, y) for x, y in zip(cache.layers[0], old))


def test_decoding_with_weights_and_evictions(gpu):
    """Weights accumulate as the separate operator gives them, without changing the step;
    after an eviction the attention is that over the kept tokens, and decoding goes on at
    the sequence's own positions."""
    model, layers = _model(gpu, 2), 2
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (100, 33, 70)]
    tables = torch.randperm(24, generator=g).int().view(3, 8)
    dev_tables = tables.to(gpu)
    cache, other = (PagedSpikeCache(layers, 4, 2, 64, 25, BS, device=gpu) for _ in range(2))
    for c in (cache, other):
        _prefill(model, c, prompts, tables, gpu)
    lens = torch.tensor([len(p) for p in prompts], device=gpu)
    pos = lens.clone()
    ids = torch.tensor([1, 2, 3], device=gpu)
    mass = torch.zeros((layers, 3, 2, 128), device=gpu)
    for i in range(3):
        logits = _decode(model, cache, ids, lens + i, dev_tables, list(mass))
        model.fused_attention = False
        plain = _decode(model, other, ids, lens + i, dev_tables)
        model.fused_attention = True
        assert torch.equal(logits, plain)
        ids = logits.argmax(-1)
    lens, pos = lens + 3, pos + 3
    for n in range(3):  # a step gives each timestep's four heads one weight in all
        assert torch.allclose(mass[:, n].sum(-1), torch.full((layers, 2), 3.0 * 4 * 4, device=gpu), rtol=1e-4)
        assert (mass[:, n, :, int(lens[n]):] == 0).all()

    old = [tuple(x.clone() for x in c) for c in cache.layers]
    given = mass.clone()
    keep, kept = cache.evict(mass, dev_tables, lens.int(), 40, sinks=2, recent=8)
    assert kept.tolist() == [40, 36, 40]
    q = ref.words((4, 3, 8), 64, g, gpu)
    for layer in range(layers):
        k, v = cache.layers[layer]
        out = paged_spike_attn_decode(q, k, v, dev_tables, kept, 64, BS, 8, 2)
        for n in range(3):
            for h in range(2):
                rows = ref.evict_ref(given[layer, n, h].tolist(), int(lens[n]), 40, 2, 8)
                assert keep[layer, n, h, :len(rows)].tolist() == rows
                kk, vv = (ref.bits(ref.positions(x, dev_tables[n], int(lens[n]), BS)[:, h, rows], 64) for x in old[layer])
                x = ref.bits(q[:, n, 4 * h:4 * h + 4], 64)
                w = torch.softmax(torch.matmul(x, kk.transpose(1, 2).contiguous()) / 8.0, -1)
                assert (out[:, n, 4 * h:4 * h + 4].double() - torch.matmul(w, vv)).abs().max() <= 1e-5
    logits = _decode(model, cache, ids, kept.long(), dev_tables, list(mass), positions=pos)
    assert torch.isfinite(logits).all()
    got = paged_spike_attn_key_mass(q, cache.layers[0][0], dev_tables, (kept + 1).int(), 64, BS)
    assert math.isclose(got.sum().item(), 3 * 4 * 8, rel_tol=1e-4)


def test_a_step_of_trees_takes_no_other_tokens(gpu):
    model = _model(gpu, 1)
    cache = PagedSpikeCache(1, 4, 2, 64, 3, BS, device=gpu)
    z = torch.zeros(2, dtype=torch.int32, device=gpu)
    trees = DraftTrees(z, torch.zeros((1, 1), dtype=torch.int64, device=gpu), 1, z[:1], z.view(1, 2))
    meta = AttentionMetadata(slot_mapping=torch.full((1,), -1, device=gpu), block_size=BS, num_decode_tokens=1, draft=trees)
    with pytest.raises(ValueError, match="drafted trees"):
        model.forward_paged(z[:1].long(), z[:1].long(), cache.layers, meta)


def test_metadata_of_another_model_is_refused(gpu):
    model = _model(gpu, 2)
    cache = PagedSpikeCache(2, 4, 2, 64, 3, BS, device=gpu)
    z = torch.zeros(2, dtype=torch.int32, device=gpu)
    word = torch.zeros((4, 1, 2, 2), dtype=torch.int32, device=gpu)
    trees = DraftTrees(z, torch.zeros((1, 1), dtype=torch.int64, device=gpu), 1, z[:1], z[:1].view(1, 1),
                       words=[(word, word.clone())])
    slots, mass = torch.full((1,), -1, device=gpu), torch.zeros((1, 2, BS), device=gpu)
    for meta, match in ((AttentionMetadata(slots, BS, draft=trees), "draft.words has 1 layers"),
                        (AttentionMetadata(slots, BS, draft=replace(trees, words=None), key_mass=[mass] * 2), "decode tokens"),
                        (AttentionMetadata(slots, BS, 1, z[:1].view(1, 1), z[:1], key_mass=[mass]), "key_mass has 1 layers")):
        with pytest.raises(ValueError, match=match):
            model.forward_paged(z[:1].long(), z[:1].long(), cache.layers, meta)
