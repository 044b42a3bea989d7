"""sampling_probs on the GPU against 64-bit code.

A probability is an exponential, a product and a quotient in fp32 or better: the exponential
of a difference of up to 104 (below, the result is 0 in fp32) rounded to fp32 is off by 2^-24 of
that difference, and each step adds a few of its own: 2^-24 (104 + 8), relative; below the
normal range 2^-149 more.  What a cut leaves out is 0 exactly."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd.sampler import (BatchSampler, SamplingParams, sample_tokens, sampling_probs,
                                    sampling_probs_workspace_bytes)

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
REL = 2.0**-24 * 112


def _rows(logits, temp, k, p, m):
    x = logits.float().cpu().numpy()
    return torch.from_numpy(np.stack([ref.probs(x[r], temp[r], k[r], p[r], m[r]) for r in range(len(x))]))


def _assert_close(got, want):
    got = got.cpu().double()
    tiny = want < 2.0**-126  # a weight of that size may be rounded away
    assert torch.equal(got > 0, (want > 0) & ~tiny | (got > 0) & tiny)
    assert ((got - want).abs() <= want * REL + 2.0**-149).all()


def _params(rows, gpu, seed, temps=(1.0,), ks=(-1,), ps=(1.0,), ms=(0.0,)):
    """Every combination in turn."""
    combos = [(t, k, p, m) for t in temps for k in ks for p in ps for m in ms]
    cols = list(zip(*(combos[r % len(combos)] for r in range(rows))))
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=gpu)
    return cols, (f(cols[0]), torch.tensor(cols[1], dtype=torch.int32, device=gpu), f(cols[2]), f(cols[3]))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,scale", [(1, 1.0), (2, 1.0), (63, 2.0), (1000, 0.1), (1025, 4.0), (32003, 1.0), (50257, 6.0),
                                     (151936, 3.0), (262144, 0.5)])
def test_matches_64_bits(gpu, V, scale, dtype):
    print(f"probs {V} {scale} {dtype}", flush=True)
    rows = 26
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn((rows, V), generator=g) * scale + 1.5).to(DTYPES[dtype])
    cols, args = _params(rows, gpu, V, (0.7, 1.3), (-1, 1, 50, 1000), (1.0, 0.9, 0.3), (0.0, 0.05))
    args[0][3::11] = 0.0  # greedy
    temp = args[0].tolist()
    _assert_close(sampling_probs(logits.to(gpu), *args), _rows(logits, temp, *cols[1:]))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [0.3, 1.0, 2.7])
def test_cuts_that_keep_many(gpu, scale, dtype):
    """Rows whose cuts lie far down: nearly flat ones by top_p, large top_k, small min_p."""
    V = 151936
    combos = [(1.0, -1, 0.5, 0.0), (1.0, -1, 0.97, 0.0), (1.0, 2049, 1.0, 0.0), (0.7, 5000, 0.9, 0.0), (1.3, 100000, 1.0, 0.0),
              (1.0, -1, 1.0, 0.01), (1.0, -1, 0.8, 1e-4), (1.0, 20000, 0.99, 1e-5), (5.0, -1, 0.3, 0.0), (1.0, 2048, 0.999, 0.0)]
    g = torch.Generator().manual_seed(int(10 * scale))
    logits = (torch.randn((len(combos), V), generator=g) * scale).to(DTYPES[dtype])
    logits[::2, ::7] = -torch.inf
    cols = list(zip(*combos))
    args = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device=gpu) for i, c in enumerate(cols)]
    _assert_close(sampling_probs(logits.to(gpu), *args), _rows(logits, *cols))


def test_parameters_out_of_range(gpu):
    """A top_p of 0 or less and a min_p above 1 leave the first token (those equal to it); a
    temperature that is no number, or negative, is greedy; cuts that are none of a number's
    order are off; an infinite temperature makes all equal."""
    inf, nan = float("inf"), float("nan")
    V = 3000
    logits = torch.randn((9, V), generator=torch.Generator().manual_seed(11))
    given = [(1.0, -1, 0.0, 0.0), (1.0, -1, -3.0, 0.0), (1.0, -1, 1.0, 1.5), (nan, 5, 0.5, 0.1), (-1.0, -1, 1.0, 0.0),
             (1.0, -1, nan, nan), (1.0, 0, 2.0, -1.0), (inf, 7, 1.0, 0.0), (1.0, 2**31 - 1, inf, 0.0)]
    same = [(1.0, 1, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (0.0, -1, 1.0, 0.0), (0.0, -1, 1.0, 0.0),
            (1.0, -1, 1.0, 0.0), (1.0, -1, 1.0, 0.0), (inf, 7, 1.0, 0.0), (1.0, -1, 1.0, 0.0)]
    cols = list(zip(*given))
    args = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device=gpu) for i, c in enumerate(cols)]
    _assert_close(sampling_probs(logits.to(gpu), *args), _rows(logits, *zip(*same)))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equal_logits(gpu, dtype):
    """A cut within equal logits keeps the lowest indices; whole rows of one value, of two,
    values that become equal by the temperature, zeros of both signs."""
    V = 5000
    g = torch.Generator().manual_seed(0)
    base = torch.stack([torch.zeros(V), torch.full((V,), -3.25), torch.randint(0, 2, (V,), generator=g).float(),
                        torch.randint(0, 5, (V,), generator=g) * 0.5, torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0),
                        torch.arange(V) * 2.0**-24 + 1.0])
    combos = [(1.0, 7, 1.0, 0.0), (1.0, -1, 0.333, 0.0), (0.9, 2500, 0.5, 0.0), (1e4, 600, 0.9, 0.5), (1.0, 4999, 1.0, 1.0),
              (0.7, 5000, 0.999, 0.0)]
    logits = base.repeat_interleave(len(combos), 0).to(DTYPES[dtype])
    cols = list(zip(*(combos * len(base))))
    args = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device=gpu) for i, c in enumerate(cols)]
    _assert_close(sampling_probs(logits.to(gpu), *args), _rows(logits, *cols))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masked_infinite_and_nan_logits(gpu, dtype):
    """Masks of -infinity and of the type's lowest value, rows with one token left, with none,
    infinities, NaN at the first, last and largest place."""
    V, dt = 3001, DTYPES[dtype]
    low = torch.finfo(dt).min
    g = torch.Generator().manual_seed(1)
    rows = torch.randn((12, V), generator=g).to(dt)
    rows[0, 1:] = -torch.inf
    rows[1, :] = -torch.inf
    rows[2, :] = torch.nan
    rows[3, :2000] = low
    rows[4, :] = low
    rows[5, 17] = rows[5, 2222] = torch.inf
    rows[6, [0, 3000]] = torch.nan
    rows[7, ::3] = -torch.inf
    rows[8, :] = torch.where(torch.arange(V) % 2 == 0, torch.nan, -torch.inf)
    rows[9, :3000] = -torch.inf
    rows[10, 5] = torch.finfo(dt).max
    rows[11, ::2] = torch.nan
    combos = [(1.0, -1, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (0.8, -1, 0.9, 0.1), (0.0, -1, 1.0, 0.0), (2.0, 2999, 0.5, 0.0)]
    logits = rows.repeat_interleave(len(combos), 0)
    cols = list(zip(*(combos * len(rows))))
    args = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device=gpu) for i, c in enumerate(cols)]
    got = sampling_probs(logits.to(gpu), *args)
    _assert_close(got, _rows(logits, *cols))
    assert not got[5:10].any() and not got[10:15].any()


def test_strides_out_and_defaults(gpu):
    g = torch.Generator().manual_seed(2)
    for dt, lead, V in ((torch.bfloat16, 1, 999), (torch.float32, 3, 1000), (torch.float16, 0, 1001), (torch.bfloat16, 8, 4096)):
        wide = (torch.randn((9, V + 11), generator=g) * 3).to(dt)
        view = wide[:, lead:lead + V]
        big = torch.full((9, V + 5), -7.0, device=gpu)
        out = big[:, 2:2 + V]
        one = torch.ones(12, device=gpu)
        assert sampling_probs(wide.to(gpu)[:, lead:lead + V], one, out=out) is out
        _assert_close(out, _rows(view, [1.0] * 9, [-1] * 9, [1.0] * 9, [0.0] * 9))
        assert (big[:, :2] == -7).all() and (big[:, 2 + V:] == -7).all()
        got = sampling_probs(wide.to(gpu)[::2, lead:lead + V], one, top_p=one * 0.8)
        _assert_close(got, _rows(view[::2], [1.0] * 9, [-1] * 9, [0.8] * 9, [0.0] * 9))
        repeated = sampling_probs(wide.to(gpu)[:1, lead:lead + V].expand(4, V), one, top_p=one * 0.8)
        assert torch.equal(repeated, got[:1].expand(4, V))
    assert sampling_probs(torch.zeros((0, 5), device=gpu), torch.zeros(0, device=gpu)).shape == (0, 5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows_keep_their_counts(gpu, dtype):
    """Thousands of rows whose top_k is decided among hundreds of candidates, all at once: each
    keeps the first k of its order, every call."""
    rows, V, k = 3000, 32003, 200
    logits = (torch.randn((rows, V), generator=torch.Generator().manual_seed(13)) * 2).to(DTYPES[dtype]).to(gpu)
    one, ks = torch.ones(rows, device=gpu), torch.full((rows,), k, dtype=torch.int32, device=gpu)
    order = logits.float().sort(dim=1, descending=True, stable=True).indices[:, :k]
    want = torch.zeros((rows, V), dtype=torch.bool, device=gpu).scatter_(1, order, True)
    first = sampling_probs(logits, one, ks)
    assert torch.equal(first > 0, want)
    for _ in range(4):
        assert torch.equal(sampling_probs(logits, one, ks), first)


def test_rows_between_the_logits(gpu):
    """Logits and probabilities in turn in one tensor; on one another they are refused."""
    both = torch.randn((6, 2, 700), generator=torch.Generator().manual_seed(12)).to(gpu) * 3
    logits, one = both[:, 0].clone(), torch.ones(6, device=gpu)
    out = sampling_probs(both[:, 0], one, top_p=one * 0.8, out=both[:, 1])
    assert torch.equal(both[:, 0], logits) and torch.equal(out, sampling_probs(logits, one, top_p=one * 0.8))
    for bad in (both[:, 0], both.view(-1)[1:1 + 6 * 700].view(6, 700)):
        with pytest.raises(ValueError, match="lies on the logits"):
            sampling_probs(both[:, 0], one, out=bad)


def test_offsets_past_32_bits(gpu):
    """A batch of more than 2^32 bytes of logits and of probabilities."""
    rows, V = 9000, 262144
    logits = torch.zeros((rows, V), dtype=torch.bfloat16, device=gpu)
    g = torch.Generator().manual_seed(3)
    some = torch.tensor([0, 4096, 8191, 8999])
    values = (torch.randn((4, V), generator=g) * 2).bfloat16()
    logits[some.to(gpu)] = values.to(gpu)
    temp, k = torch.ones(rows, device=gpu), torch.full((rows,), 40, dtype=torch.int32, device=gpu)
    got = sampling_probs(logits, temp, k)
    _assert_close(got[some.to(gpu)], _rows(values, [1.0] * 4, [40] * 4, [1.0] * 4, [0.0] * 4))
    rest = torch.ones(rows, dtype=torch.bool)
    rest[some] = False
    other = got[rest.to(gpu)]
    assert torch.equal(other[:, :40], torch.full_like(other[:, :40], 1 / 40)) and not other[:, 40:].any()


def test_rows_do_not_depend_on_the_batch(gpu):
    g = torch.Generator().manual_seed(4)
    logits = (torch.randn((300, 40000), generator=g) * 3).bfloat16().to(gpu)
    _, args = _params(300, gpu, 0, (0.7, 1.0), (-1, 30), (1.0, 0.9), (0.0, 0.02))
    whole = sampling_probs(logits, *args)
    for a, e in ((0, 1), (7, 9), (100, 133), (0, 300), (250, 300)):
        assert torch.equal(sampling_probs(logits[a:e], *(t[a:e] for t in args)), whole[a:e]), (a, e)


def test_captured_call_takes_other_inputs(gpu):
    rows, V = 6, 20000
    g = torch.Generator().manual_seed(5)
    batches = [(torch.randn((rows, V), generator=g) * 3).bfloat16().to(gpu) for _ in range(3)]
    _, args = _params(rows, gpu, 0, (0.8,), (-1, 40), (1.0, 0.9), (0.0,))
    static, out = batches[0].clone(), torch.empty((rows, V), device=gpu)
    ws = torch.empty(max(1, sampling_probs_workspace_bytes(rows, V)), dtype=torch.uint8, device=gpu)
    sampling_probs(static, *args, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling_probs(static, *args, out=out, workspace=ws)
    for i, batch in enumerate(batches + batches):
        static.copy_(batch)
        args[0].fill_(0.5 + 0.1 * i)
        graph.replay()
        eager = sampling_probs(batch, *args)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_the_sampler_draws_from_it(gpu):
    """The tokens of sample_tokens at a grid of uniforms: each has weight, and the uniforms at
    which it is drawn make up its probability.  The sampler takes tokens by value descending,
    so a token's uniforms are an interval: over a grid of n its share is off by 1 / n, and by
    what fp32 weights are off."""
    V, n = 1000, 4096
    g = torch.Generator().manual_seed(6)
    logits = (torch.randn((1, V), generator=g) * 3).bfloat16().to(gpu)
    for k, p, m in ((-1, 1.0, 0.0), (50, 0.9, 0.0), (-1, 0.8, 0.02), (7, 1.0, 0.1)):
        full = lambda v, dt=torch.float32, r=n: torch.full((r,), v, dtype=dt, device=gpu)
        want = sampling_probs(logits, full(0.9, r=1), full(k, torch.int32, 1), full(p, r=1), full(m, r=1))[0].double()
        u = (torch.arange(n, device=gpu) + 0.5) / n
        tokens = sample_tokens(logits.expand(n, V).contiguous(), full(0.9), full(k, torch.int32), full(p), full(m), uniforms=u)
        share = torch.bincount(tokens, minlength=V).double() / n
        assert (want[tokens] > 0).all()
        assert (share - want).abs().max().item() <= 1.0 / n + 1e-5


def test_a_batch_samplers_distributions(gpu):
    g = torch.Generator().manual_seed(7)
    logits = (torch.randn((3, 500), generator=g) * 3).to(gpu)
    s = BatchSampler(4, gpu)
    s.set_params([SamplingParams(temperature=0.7, top_k=20), SamplingParams(temperature=0.0), SamplingParams(top_p=0.5)])
    _assert_close(s.probs(logits), _rows(logits.cpu(), [0.7, 0.0, 1.0], [20, -1, -1], [1.0, 1.0, 0.5], [0.0] * 3))
    biased = [SamplingParams(logit_bias={3: 2.0})] * 3
    s.set_params(biased)
    want = logits.cpu().clone()
    want[:, 3] += 2.0
    _assert_close(s.probs(logits), _rows(want, [1.0] * 3, [-1] * 3, [1.0] * 3, [0.0] * 3))
    s.set_params([SamplingParams(presence_penalty=0.5)] * 3)
    with pytest.raises(ValueError, match="penalties"):
        s.probs(logits)
