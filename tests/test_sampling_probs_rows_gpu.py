"""sampling_probs on rows that cuts treat otherwise than logits in random order over one slice:
masks that leave few tokens of a real vocabulary, likely tokens side by side.  Tolerances as derived in test_sampling_probs_gpu."""
from __future__ import annotations

import pytest
import torch

from spikeinfer_amd.sampler import sampling_probs
from test_sampling_probs_gpu import DTYPES, _assert_close, _rows

pytestmark = pytest.mark.gpu
V = 151936
INF = float("inf")


def check(gpu, rows, combos):
    """Every row with every combination of (temperature, top_k, top_p, min_p)."""
    logits = rows.repeat_interleave(len(combos), 0)
    cols = list(zip(*(combos * len(rows))))
    args = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device=gpu) for i, c in enumerate(cols)]
    got = sampling_probs(logits.to(gpu), *args)
    _assert_close(got, _rows(logits, *cols))
    return got


CUTS = [(0.8, -1, 0.9, 0.0), (0.8, 50, 1.0, 0.0), (0.8, 50, 0.9, 0.0), (1.0, -1, 1.0, 0.05), (1.0, -1, 1.0, 0.0), (1.2, 1000, 0.95, 0.0)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mask", ["infinity", "lowest"])
def test_masks_that_leave_few_tokens(gpu, mask, dtype):
    """20, 200 and 2,000 tokens left anywhere, 30 within one slice, one token, and two rows' ends."""
    print(f"masks {mask} {dtype}", flush=True)
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(0)
    left = torch.zeros((7, V), dtype=torch.bool)
    for r, n in enumerate((20, 200, 2000)):
        left[r, torch.randperm(V, generator=g)[:n]] = True
    left[3, 40000:40030] = True
    left[4, 77777] = True
    left[5, [0, V - 1]] = True
    left[6, :30000] = True
    rows = (torch.randn((7, V), generator=g) * 3).to(dt)
    rows = torch.where(left, rows, torch.tensor(-INF if mask == "infinity" else torch.finfo(dt).min, dtype=dt))
    got = check(gpu, rows, CUTS)
    assert not got.cpu()[~left.repeat_interleave(len(CUTS), 0)].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_likely_tokens_side_by_side(gpu, dtype):
    """Rows in descending and ascending order, the likely ones in one slice, in its last tokens
    and across a border, a flat head above a steep tail."""
    print(f"side by side {dtype}", flush=True)
    g = torch.Generator().manual_seed(1)
    base = torch.randn(V, generator=g) * 3
    ordered = base.sort(descending=True).values
    slices, border, head = base.clone(), base.clone(), base.clone()
    slices[:12000] += 9.0
    border[20000:21000] += 12.0
    head[:3000] = 15.0 + 0.01 * torch.randn(3000, generator=g)
    rows = torch.stack([ordered, ordered.flip(0), slices, border, head]).to(DTYPES[dtype])
    check(gpu, rows, CUTS + [(1.0, 300, 1.0, 0.0), (1.0, 2048, 0.99, 0.0), (1.0, 2049, 1.0, 0.0), (0.7, -1, 0.5, 0.001)])
