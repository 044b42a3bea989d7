"""BatchSampler's filters before a draw, on the host."""
from __future__ import annotations

import pytest
import torch

from spikeinfer_amd.sampler import BatchSampler, SamplingParams


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_filters_leave_the_callers_logits(dtype):
    """Bias and min_tokens go into a copy, also where the logits are fp32 already: a second call
    finds what the first found."""
    s = BatchSampler(2, torch.device("cpu"), eos_token_id=4)
    s.set_params([SamplingParams(logit_bias={1: 2.0, 3: -1.0}), SamplingParams(min_tokens=2, stop_token_ids=[0])])
    logits = torch.arange(12.0).reshape(2, 6).to(dtype)
    before = logits.clone()
    want = before.clone().float()
    want[0, 1] += 2.0
    want[0, 3] -= 1.0
    want[1, 0] = want[1, 4] = -torch.inf
    for _ in range(2):
        assert torch.equal(s._pre_filter(logits, 2), want)
        assert torch.equal(logits, before)
    s.set_params([SamplingParams()] * 2)
    assert s._pre_filter(logits, 2) is logits
