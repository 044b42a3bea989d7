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
