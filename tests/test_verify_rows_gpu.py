"""The attention of a verification step inside a decoder, every layer: rows against float64
code on the step's own words, and rows of a chain against decoding over the committed words.

A bf16 row is off by its half step and 4e-6 (32-bit weights and sums); so is decoding's, so
the two may differ only where the exact value lies within that of the middle between two
neighbours."""
from __future__ import annotations

import pytest
import torch

import cache_ops_ref as ref
import spikeinfer_amd.model as model_module
from spikeinfer_amd.attention import AttentionMetadata, DraftTrees
from spikeinfer_amd.kernels import accept_draft_tree, draft_tree_masks, paged_spike_attn_decode
from spikeinfer_amd.spike_cache import PagedSpikeCache
from test_tree_attn_rounding_gpu import _half_step
from test_verify_step_gpu import BS, _model, _prefill, _trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers", [1, 3])
def test_rows_of_every_layer(gpu, layers, monkeypatch):
    model, vocab, depth = _model(gpu, layers), 512, 5
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (60, 7, 101)]
    tables = torch.randperm(24, generator=g).int().view(3, 8)
    dev_tables = tables.to(gpu)
    cache = PagedSpikeCache(layers, 4, 2, 64, 25, BS, device=gpu)
    _prefill(model, cache, prompts, tables, gpu)
    lens = torch.tensor([len(p) for p in prompts], device=gpu)
    counts = [depth + 4, depth, depth + 11]
    chains = torch.randint(0, vocab, (3, depth), generator=g).tolist()
    starts, parents, tokens = _trees(gpu, counts, 5, vocab, chains)
    masks, depths = draft_tree_masks(parents, starts, max(counts))
    seq = torch.repeat_interleave(torch.arange(3, device=gpu), torch.tensor(counts, device=gpu))
    trees = DraftTrees(starts, masks, max(counts), lens.int(), dev_tables)
    meta = AttentionMetadata(slot_mapping=torch.full((len(seq),), -1, device=gpu), block_size=BS, draft=trees)
    calls, real = [], model_module.paged_spike_attn_tree

    def recorded(q, *args, out):
        real(q, *args, out=out)
        calls.append((q.clone(), out.clone()))
        return out

    monkeypatch.setattr(model_module, "paged_spike_attn_tree", recorded)
    model.forward_paged(tokens, lens[seq] + depths, cache.layers, meta)
    assert len(calls) == layers
    wants = []
    for (q, out), (kw, vw), (k, v) in zip(calls, trees.words, cache.layers):
        want = ref.tree_ref(q, kw, vw, k, v, dev_tables, lens, starts, masks, max(counts), 64, BS, torch.zeros_like(out))
        wants.append(want)
        assert ((out.double() - want).abs() <= _half_step(want, out.dtype) + 4e-6).all()
    # the chains are accepted: targets that name the next of each
    targets = torch.full((len(seq),), -1, dtype=torch.int64, device=gpu)
    at = starts.tolist()
    for n in range(3):
        targets[at[n]:at[n] + depth - 1] = tokens[at[n] + 1:at[n] + depth]
    path, count, _ = accept_draft_tree(tokens, parents, targets, starts, max(counts), trees.words, cache.layers,
                                       dev_tables, lens.int(), BS)
    assert count.tolist() == [depth] * 3 and path[:, :depth].tolist() == [list(range(depth))] * 3
    for (q, out), want, (k, v) in zip(calls, wants, cache.layers):
        for i in range(depth):
            rows = (starts[:-1] + i).long()
            got = paged_spike_attn_decode(q[:, rows].contiguous(), k, v, dev_tables, (lens + i + 1).int(), 64, BS, 8, 2,
                                          out=torch.empty_like(out[:, rows]))
            x = want[:, rows]
            assert ((got.double() - x).abs() <= _half_step(x, out.dtype) + 4e-6).all()
            differ = got != out[:, rows]
            middle = (got.double() + out[:, rows].double()) / 2
            assert (~differ | ((x - middle).abs() <= 4e-6)).all()
