"""Outputs on the memory of other arguments: refused, or as anywhere else."""
from __future__ import annotations

import pytest
import torch

from spikeinfer_amd.kernels import linear_int8, pack_linear_int8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,K", [(70, 64), (1152, 896), (33001, 128)])
def test_one_row_in_place_of_its_bias(gpu, N, K):
    """h += W x, with h as the bias and the result; of more rows the first may not be it."""
    g = torch.Generator().manual_seed(N)
    x, w8 = torch.randn((2, K), generator=g).to(gpu), pack_linear_int8(torch.randn((N, K), generator=g).to(gpu))
    for dtype in (torch.bfloat16, torch.float32):
        h = torch.randn(N, generator=g).to(dtype).to(gpu)
        want = linear_int8(x[:1], w8, h, dtype=dtype)
        kept = h.clone()
        assert torch.equal(linear_int8(x[:1], w8, h, out=h[None]), want)
        both = torch.stack([kept, kept])
        with pytest.raises(ValueError, match="y lies on bias"):
            linear_int8(x, w8, both[0], out=both)
        assert torch.equal(both[0], kept)
        rows = torch.zeros((2, 2, N), dtype=dtype, device=gpu)  # a bias between two rows
        rows[0, 1] = kept
        got = linear_int8(x, w8, rows[0, 1], out=rows[:, 0])
        assert torch.equal(got, linear_int8(x, w8, kept, dtype=dtype)) and torch.equal(rows[0, 1], kept)
