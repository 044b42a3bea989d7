"""Rounding of the draft-tree attention, against plain float64 code.

Outputs lie in [0, 1].  Weights and sums hold 32 bits (4e-6, as for the prefill kernel);
a 16-bit output adds the half step of its own rounding and nothing else.
"""
from __future__ import annotations

import pytest
import torch

import cache_ops_ref as ref
from spikeinfer_amd.kernels import paged_spike_attn_tree

pytestmark = pytest.mark.gpu


def _half_step(x, dtype):
    """Half the distance of `dtype`'s numbers around x (float64)."""
    if dtype == torch.float32:
        return torch.zeros_like(x)
    return torch.ldexp(torch.full_like(x, torch.finfo(dtype).eps / 2), torch.frexp(x)[1] - 1)


@pytest.mark.parametrize("T,hq,hkv,D,trees", [
    (4, 14, 2, 64, [(5, 3), (40, 4)]),                   # one row tile: all waves share it
    (4, 14, 2, 64, [(700, 8), (3000, 16), (65, 40)]),    # two, four and more, a context in parts
    (2, 16, 4, 128, [(900, 25), (33, 2)]),
    (1, 4, 4, 32, [(300, 70)]),
])
def test_16_bit_outputs_are_off_by_their_own_rounding(gpu, T, hq, hkv, D, trees):
    case = ref.tree_case(T, hq, hkv, D, 16, trees, 3 * D + len(trees), gpu)
    rows = int(case["row_starts"][-1])
    want = ref.tree_want(case, torch.zeros((T, case["q_packed"].shape[1], hq, D), device=gpu))[:, :rows]
    for dtype in (torch.bfloat16, torch.float16):
        err = (paged_spike_attn_tree(**case, dtype=dtype)[:, :rows].double() - want).abs()
        assert (err <= _half_step(want, dtype) + 4e-6).all(), (dtype, (err - _half_step(want, dtype)).max().item())


@pytest.mark.parametrize("T,hq,hkv,D,trees", [
    (1, 14, 2, 64, [(20011, 5), (16385, 40)]),   # more parts than a join has on their way at once
    (1, 2, 1, 128, [(33000, 40)]),
    (1, 2, 1, 64, [(65537, 3), (70001, 200)]),   # parts longer than usual
    (1, 1, 1, 64, [(300007, 140)]),
])
def test_long_contexts(gpu, T, hq, hkv, D, trees):
    case = ref.tree_case(T, hq, hkv, D, 16, trees, len(trees) + D, gpu)
    rows = int(case["row_starts"][-1])
    want = ref.tree_want(case, torch.zeros((T, case["q_packed"].shape[1], hq, D), device=gpu))[:, :rows]
    for dtype in (torch.float32, torch.bfloat16):
        err = (paged_spike_attn_tree(**case, dtype=dtype)[:, :rows].double() - want).abs() - _half_step(want, dtype)
        assert (err <= 4e-6).all(), (dtype, err.max().item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_long_context_does_not_depend_on_its_batch(gpu, dtype):
    """Nor on its table's width: parts of several turns are another kernel's."""
    case = ref.tree_case(1, 2, 1, 64, 16, [(140000, 70), (90, 9), (66000, 20)], 3, gpu)
    out = paged_spike_attn_tree(**case, dtype=dtype)
    for n in range(3):
        a, e = case["row_starts"][n].item(), case["row_starts"][n + 1].item()
        one = {k: (v[:, a:e] if k.endswith(("words", "packed")) else v) for k, v in case.items()}
        one.update(masks=case["masks"][a:e], block_tables=case["block_tables"][n:n + 1], max_nodes=e - a,
                   context_lens=case["context_lens"][n:n + 1],
                   row_starts=torch.tensor([0, e - a], dtype=torch.int32, device=gpu))
        for blocks in (None, -(-int(case["context_lens"][n]) // 16)):
            one["block_tables"] = case["block_tables"][n:n + 1, :blocks]
            assert torch.equal(paged_spike_attn_tree(**one, dtype=dtype), out[:, a:e])


@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_sums_of_three_equal_weights(gpu, D):
    """Three keys of one score, w = hi + lo, whose values are all ones: outputs are 1 up to
    roundings of 2**-24 each.  The sums of three hi and of three lo fit fp32, adding the two is
    off by one rounding.  The numerator has three rounded additions, to 2w, 3w and 3w, each off
    by a step at most: 16/3 * 2**-24.  A reciprocal and a product add two: below 9."""
    W = -(-D // 32)
    full = [(1 << min(32, D - 32 * w)) - 1 for w in range(W)]
    word = lambda m: m - 2**32 if m >= 2**31 else m
    tokens = [0, 2, 8]  # the same lane's keys
    q = torch.tensor([word(x) for x in full], dtype=torch.int32, device=gpu).expand(1, 11, 1, W).contiguous()
    masks = torch.full((11, 1), sum(1 << i for i in tokens), dtype=torch.int64, device=gpu)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    cache = torch.zeros((1, 1, 16, W), dtype=torch.int32, device=gpu)
    for score in range(D + 1):
        bits = (1 << score) - 1
        k = i32(*[word(bits >> (32 * w) & 0xffffffff) for w in range(W)]).expand(1, 11, 1, W).contiguous()
        out = paged_spike_attn_tree(q, k, q, cache, cache, i32(0).view(1, 1), i32(0), i32(0, 11), masks, 11, D, 16)
        assert ((out.double() - 1).abs() <= 9 * 2.0**-24).all(), (score, (out.double() - 1).abs().max().item() * 2**24)


@pytest.mark.parametrize("D,tokens", [(64, 1 << 20), (128, 1 << 20), (64, 1 << 22)])
def test_the_error_does_not_grow_with_the_length(gpu, D, tokens):
    """Keys of one score whose values are all ones: outputs are 1.  Counted in 2**-24: at most 64
    tiles go into one accumulator, 4 additions each, the i-th off by a step (2) of i / 256 of the
    sum: 256.  A denominator's sums take as many, each off by half a step: 128.  Beyond 65,536
    tokens each of 32 parts has tokens / 65536 such sums: that many additions and 32, each off
    by half a step of half the sum on average, above and below the line; a few roundings at
    the end."""
    W, rows = D // 32, 140
    word = lambda m: m - 2**32 if m >= 2**31 else m
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)
    q = torch.full((1, rows, 1, W), -1, dtype=torch.int32, device=gpu)
    masks = torch.zeros((rows, 3), dtype=torch.int64, device=gpu)
    tables = torch.arange(tokens // 16, dtype=torch.int32, device=gpu).view(1, -1)
    bound = (256 + 128 + tokens / 65536 + 32 + 8) * 2.0**-24
    for score in (0, 1, D // 5, D // 3, D // 2, D):
        bits = (1 << score) - 1
        key = i32(*[word(bits >> (32 * w) & 0xffffffff) for w in range(W)])
        k = key.expand(1, 1, tokens, W).contiguous()
        out = paged_spike_attn_tree(q, key.expand(1, rows, 1, W).contiguous(), q, k, torch.full_like(k, -1), tables,
                                    i32(tokens), i32(0, rows), masks, rows, D, 16)
        err = (out.double() - 1).abs().max().item()
        print(f"{D} {tokens} {score}: {err:.2e}", flush=True)
        assert err <= bound, (score, err, bound)
