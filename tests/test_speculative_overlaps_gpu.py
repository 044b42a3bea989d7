"""Outputs on the memory of other arguments: refused, or as anywhere else."""
from __future__ import annotations

import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd.kernels import linear_int8, pack_linear_int8, verify_draft_tree

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


def test_targets_in_place_of_the_tokens(gpu):
    """Hundreds of trees, each reading its own tokens only; shifted they are refused."""
    case = ref.draft_case([7, 3, 12] * 200, 600, 5, 3)
    d = {k: v.to(gpu) if isinstance(v, torch.Tensor) else v for k, v in case.items()}
    rows, used = len(case["tokens"]), int(case["row_starts"][-1])
    want = verify_draft_tree(**d)
    buffer = torch.zeros(rows + 5, dtype=torch.int64, device=gpu)
    tokens = buffer[:rows]
    tokens.copy_(d["tokens"])
    with pytest.raises(ValueError, match="targets lie on"):
        verify_draft_tree(**{**d, "tokens": tokens}, out=buffer[5:])
    assert torch.equal(tokens, d["tokens"])
    out = verify_draft_tree(**{**d, "tokens": tokens}, out=tokens)
    assert torch.equal(out[:used], want[:used]) and torch.equal(out[used:], d["tokens"][used:])
