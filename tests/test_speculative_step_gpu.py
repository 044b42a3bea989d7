"""Speculative decoding as a decoder does it: an 8-bit copy of the model drafts by sampling,
the model's step over the drafted rows, both distributions, verification by random numbers,
acceptance; and the copy's products one by one."""
from __future__ import annotations

import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd import model as model_mod
from spikeinfer_amd.attention import AttentionMetadata, DraftTrees
from spikeinfer_amd.kernels import accept_draft_tree, draft_tree_masks, verify_draft_tree, verify_workspace_bytes
from spikeinfer_amd.runner import DecodeRunner
from spikeinfer_amd.sampler import SamplingParams, sample_tokens, sampling_probs, sampling_probs_workspace_bytes
from spikeinfer_amd.spike_cache import PagedSpikeCache
from test_verify_step_gpu import BS, _decode, _model, _prefill

pytestmark = pytest.mark.gpu


def test_the_copys_products(gpu, monkeypatch):
    """Every linear layer of a prefill, a decode step and the head is an 8-bit product of the
    layer's own weight and input."""
    model = _model(gpu)
    drafter = model.int8_copy()
    assert model.lm_head_int8 is None and all(L.int8 is None for L in model.layers)
    assert drafter.embed is model.embed and drafter.weight_bytes < 0.6 * model.weight_bytes
    originals = {id(w8): (name, getattr(L, name)) for L in drafter.layers for name, w8 in L.int8.items()}
    originals[id(drafter.lm_head_int8)] = ("lm_head", drafter.lm_head)
    seen = []

    def recorded(x, w8, bias=None, out=None):
        y = model_mod_linear(x, w8, bias, out)
        seen.append((x.clone(), w8, bias, y.clone()))
        return y

    model_mod_linear = model_mod.linear_int8
    monkeypatch.setattr(model_mod, "linear_int8", recorded)
    cache = PagedSpikeCache(2, 4, 2, 64, 25, BS, device=gpu)
    tables = torch.randperm(24, generator=torch.Generator().manual_seed(0)).int().view(3, 8)
    _prefill(drafter, cache, [[5, 6, 7] * 9, [1], [2] * 40], tables, gpu)
    lens = torch.tensor([27, 1, 40], device=gpu).int()
    logits = _decode(drafter, cache, torch.tensor([1, 2, 3], device=gpu), lens, tables.to(gpu))
    assert logits.isfinite().all()
    names = [originals[id(w8)][0] for _, w8, _, _ in seen]
    assert names == ["w_qkv", "w_o", "w_gu", "w_down"] * 4 + ["lm_head"]
    for x, w8, bias, y in seen:
        want, off = ref.linear(x.reshape(-1, x.shape[-1]), originals[id(w8)][1], bias)
        tol = off + (want.abs() + off) * torch.finfo(y.dtype).eps / 2
        assert ((y.cpu().double().reshape(want.shape) - want).abs() <= tol).all()


def test_a_runner_on_the_copy(gpu):
    """The copy under the runner: a captured step gives the tokens of eager ones."""
    drafter = _model(gpu).int8_copy()
    prompts, n = [[3, 4, 5, 6], [9] * 20], 6
    runner = DecodeRunner(drafter, PagedSpikeCache(2, 4, 2, 64, 64, BS, device=gpu), 2, 128)
    got = runner.generate(prompts, [SamplingParams(temperature=0.0)] * 2, n)
    cache = PagedSpikeCache(2, 4, 2, 64, 64, BS, device=gpu)
    tables = torch.arange(16).int().view(2, 8)
    want = []
    for i, p in enumerate(prompts):  # (one prompt at a time, as the runner prefills)
        _prefill(drafter, cache, [p[:-1]], tables[i:i + 1], gpu)
    ids = torch.tensor([p[-1] for p in prompts], device=gpu)
    lens = torch.tensor([len(p) - 1 for p in prompts], device=gpu).int()
    for _ in range(n):
        ids = _decode(drafter, cache, ids, lens, tables.to(gpu)).float().argmax(-1)
        want.append(ids)
        lens = lens + 1
    assert [list(map(int, t)) for t in got] == torch.stack(want, 1).tolist()


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_drafting_and_verifying(gpu, temperature):
    """Steps of three sequences: the drafter samples a chain of three tokens each, the model
    verifies.  The tokens are those that plain code accepts from the same distributions, and both
    caches go on from the accepted rows."""
    model = _model(gpu)
    drafter = model.int8_copy()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (37, 5, 90)]
    n, depth, V = 3, 3, 512
    tables = torch.randperm(24, generator=g).int().view(n, 8)
    caches = [PagedSpikeCache(2, 4, 2, 64, 25, BS, device=gpu) for _ in range(2)]
    for m, cache in zip((model, drafter), caches):
        _prefill(m, cache, [p[:-1] for p in prompts], tables, gpu)
    tables = tables.to(gpu)
    lens = torch.tensor([len(p) - 1 for p in prompts], device=gpu).int()
    last = torch.tensor([p[-1] for p in prompts], device=gpu)
    rows = n * (depth + 1)
    starts = torch.arange(0, rows + 1, depth + 1, device=gpu).int()
    parents = (torch.arange(rows, device=gpu) % (depth + 1) - 1).int()
    masks, depths = draft_tree_masks(parents, starts, depth + 1)
    full = lambda v, k, dt=torch.float32: torch.full((k,), v, dtype=dt, device=gpu)
    settings = lambda k: (full(temperature, k), full(40, k, torch.int32), full(0.95, k))
    kept = 0
    for step in range(4):
        # ---- the drafter's chain: its last call caches the last drafted token ----
        tokens, draft = [last], []
        for d in range(depth + 1):
            logits = _decode(drafter, caches[1], tokens[-1], lens + d, tables)
            draft.append(sampling_probs(logits, *settings(n)))
            if d < depth:
                u = torch.rand(n, generator=g).to(gpu)
                tokens.append(sample_tokens(logits, *settings(n), uniforms=u))
        tokens, draft = torch.stack(tokens, 1).flatten(), torch.stack(draft, 1).flatten(0, 1)
        # ---- the model's step ----
        trees = DraftTrees(starts, masks, depth + 1, lens, tables)
        meta = AttentionMetadata(slot_mapping=torch.full((rows,), -1, device=gpu), block_size=BS, draft=trees)
        positions = lens.long().repeat_interleave(depth + 1) + depths
        hidden = model.forward_paged(tokens, positions, caches[0].layers, meta)
        target = sampling_probs(model.compute_logits(hidden), *settings(rows))
        u = torch.rand(rows, generator=g)
        targets = verify_draft_tree(tokens, parents, target, draft, u.to(gpu), starts, depth + 1)
        path, count, after = accept_draft_tree(tokens, parents, targets, starts, depth + 1, trees.words,
                                               caches[0].layers, tables, lens, BS)
        want = ref.verify(tokens.cpu(), parents.cpu(), target, draft, u, starts.cpu(), depth + 1)
        assert targets.tolist() == want
        for i in range(n):
            c = int(count[i])
            assert path[i, :c].tolist() == list(range(c))
            assert want[4 * i:4 * i + c - 1] == tokens[4 * i + 1:4 * i + c].tolist() and int(after[i]) == want[4 * i + c - 1]
            if temperature == 0.0:  # the path goes as far as both agree
                assert want[4 * i:4 * i + c] == target[4 * i:4 * i + c].argmax(1).tolist()
        kept += int(count.sum()) - n
        lens = lens + count
        last = after
    assert kept > 0  # (a random model's 8-bit copy agrees with it now and then)


def test_captured_steps_share_a_workspace(gpu):
    """Distributions of both models, verification and acceptance as one captured step; two such
    steps of other sizes, whose graphs share their scratch, replayed in turn with eager work
    between them."""
    V, g = 5003, torch.Generator().manual_seed(3)
    scratch = torch.empty(1 << 22, dtype=torch.uint8, device=gpu)
    steps = []
    for counts, dtype in (([5, 5, 5], torch.bfloat16), ([17, 2, 9, 1, 12], torch.float32)):
        case = ref.draft_case(counts, V, sum(counts), 3)
        rows, n = len(case["tokens"]), len(counts)
        s = {k: v.to(gpu) for k, v in case.items() if isinstance(v, torch.Tensor) and not k.endswith("probs")}
        s.update(logits=torch.zeros((2, rows, V), dtype=dtype, device=gpu), probs=torch.zeros((2, rows, V), device=gpu),
                 temp=torch.full((rows,), 0.8, device=gpu), top_p=torch.full((rows,), 0.9, device=gpu),
                 out=torch.full((rows,), -1, device=gpu), most=case["max_nodes"],)
        assert max(sampling_probs_workspace_bytes(rows, V), verify_workspace_bytes(n, V)) <= scratch.numel()
        steps.append(s)

    def run(s, probs, out, workspace):
        for i in range(2):
            sampling_probs(s["logits"][i], s["temp"], None, s["top_p"], out=probs[i], workspace=workspace)
        verify_draft_tree(s["tokens"], s["parents"], probs[0], probs[1], s["uniforms"], s["row_starts"], s["most"],
                          out=out, workspace=workspace)
        return accept_draft_tree(s["tokens"], s["parents"], out, s["row_starts"], s["most"])

    graphs = []
    for s in steps:
        run(s, s["probs"], s["out"], scratch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s["accepted"] = run(s, s["probs"], s["out"], scratch)
        graphs.append(graph)
    for turn in range(4):
        for s in steps:
            x = torch.randn(s["logits"].shape[1:], generator=g) * 3
            s["logits"].copy_(torch.stack([x, x + torch.randn(x.shape, generator=g)]))
            s["uniforms"].copy_(torch.rand(len(s["uniforms"]), generator=g))
            starts = s["row_starts"].tolist()
            for a, e in zip(starts[:-1], starts[1:]):  # drafts that the drafter favours
                s["tokens"][a + 1:e] = s["logits"][1][a + s["parents"][a + 1:e].long()].argmax(1)
        for graph in graphs[::1 if turn % 2 else -1]:
            graph.replay()
        for s in steps:
            probs, out = torch.zeros_like(s["probs"]), torch.full_like(s["out"], -1)
            path, count, after = run(s, probs, out, None)
            assert torch.equal(probs, s["probs"]) and torch.equal(out, s["out"])
            assert out.tolist() == ref.verify(s["tokens"].cpu(), s["parents"].cpu(), probs[0], probs[1], s["uniforms"].cpu(),
                                              s["row_starts"].cpu(), s["most"])
            assert torch.equal(count, s["accepted"][1]) and torch.equal(after, s["accepted"][2])
            for i, c in enumerate(count.tolist()):
                assert torch.equal(path[i, :c], s["accepted"][0][i, :c])
