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
