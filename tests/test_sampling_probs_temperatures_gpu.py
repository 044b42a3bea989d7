"""sampling_probs at temperatures at the ends of their range, the infinite one among them.
Tolerances as derived in test_sampling_probs_gpu."""
from __future__ import annotations

import pytest
import torch

from spikeinfer_amd.sampler import sampling_probs
from test_sampling_probs_gpu import DTYPES, _assert_close, _rows

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _check(gpu, rows, combos):
    """Every row with every combination of (temperature, top_k, top_p, min_p)."""
    logits = rows.repeat_interleave(len(combos), 0)
    cols = list(zip(*(combos * len(rows))))
    args = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device=gpu) for i, c in enumerate(cols)]
    got = sampling_probs(logits.to(gpu), *args)
    # min_p = 1 keeps what equals the largest (exp(-d) < 1 for every d > 0, which the plain code's
    # fp64 rounds to 1 below 2^-54): the others masked say the same without an exponential
    plain = logits.float()
    for r, (temp, _, _, m) in enumerate(zip(*cols)):
        if m == 1.0:
            x = torch.where(plain[r].isfinite(), plain[r] / temp, plain[r])
            plain[r, x < x[~x.isnan()].max()] = -INF
    _assert_close(got, _rows(plain, *cols))
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_temperatures_at_the_ends(gpu, dtype):
    """An infinite temperature makes all finite logits equal, with cuts and without; of infinite
    logits and NaN the rows are as at any temperature."""
    n = 3000
    rows = (torch.randn((6, n), generator=torch.Generator().manual_seed(2)) * 3).to(DTYPES[dtype])
    rows[1, ::5] = -INF
    rows[2, 7] = INF
    rows[3, [0, 2999]] = NAN
    rows[4, 9:2990] = torch.finfo(DTYPES[dtype]).min
    rows[5, :2999] = -INF
    cuts = [(-1, 1.0, 0.0), (7, 1.0, 0.0), (-1, 0.5, 0.0), (-1, 1.0, 1.0), (-1, 1.0, 0.3), (9, 0.5, 1.0)]
    temps = [INF, 3.4e38, 1e30, 1e5, 1e-3, 1.0001e-5]
    _check(gpu, rows, [(t, *c) for t in temps for c in cuts])
