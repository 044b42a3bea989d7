"""verify_draft_tree where a draw's number lies on a border between two sums."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from spikeinfer_amd.kernels import verify_draft_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("apart", [4, 4096])
def test_a_draw_on_a_border(gpu, apart):
    """Half of the sum is exactly what stands before the third token with weight: the draw is that
    token.  The sums on either side of the border are rounded differently (of 1 + 3 e, 1 and 3 e,
    e a step of fp64 at 1, the first two add to 2 + 4 e, and 2 + 4 e - 1 is above 1 + 3 e), in
    neighbouring threads and in neighbouring slices."""
    e = 2.0**-52
    V = 3 * apart
    P = np.zeros((1, V))
    P[0, 0], P[0, 1], P[0, apart], P[0, 2 * apart] = 0.5, 1.5 * e, 0.5, 1.5 * e
    assert 1.0 + (1.0 + 3 * e) == 2.0 + 4 * e and 2.0 + 4 * e - 1.0 > 1.0 + 3 * e
    P = torch.from_numpy(P).float()
    assert math.fsum(P[0].tolist()) == 1.0 + 3 * e
    for u, want in ((0.5, apart), (0.5 - 2.0**-24, 0), (0.5 + 2.0**-24, apart)):
        got = verify_draft_tree(torch.zeros(1, dtype=torch.int64, device=gpu),
                                torch.full((1,), -1, dtype=torch.int32, device=gpu), P.to(gpu), P.to(gpu),
                                torch.full((1,), u, device=gpu), torch.tensor([0, 1], dtype=torch.int32, device=gpu), 1)
        assert got.tolist() == [want], u
