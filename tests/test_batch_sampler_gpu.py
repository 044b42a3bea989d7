"""BatchSampler: the distributions it gives are those that it draws from."""
from __future__ import annotations

import pytest
import torch

from spikeinfer_amd.sampler import BatchSampler, SamplingParams, sampling_probs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distributions_then_a_draw(gpu, dtype):
    """probs and sample in turn on the same logits, whose bias and blocked tokens count once:
    both take them as a row without them would take the changed logits."""
    n, V = 3, 700
    logits = torch.randn((n, V), generator=torch.Generator().manual_seed(0)).to(dtype).to(gpu)
    before = logits.clone()
    changed = before.clone().float()
    changed[0, 5] += 6.0
    changed[1, 7] = -torch.inf
    changed[1, 9] = -torch.inf
    s, plain = BatchSampler(n, gpu, eos_token_id=9), BatchSampler(n, gpu)
    s.set_params([SamplingParams(logit_bias={5: 6.0}), SamplingParams(min_tokens=3, stop_token_ids=[7]),
                  SamplingParams(top_k=20)])
    plain.set_params([SamplingParams(), SamplingParams(), SamplingParams(top_k=20)])
    want = sampling_probs(changed, *(getattr(plain, k)[:n] for k in ("temperature", "top_k", "top_p", "min_p")))
    for u in (0.05, 0.35, 0.65, 0.95):
        s.uniforms.fill_(u)
        plain.uniforms.fill_(u)
        for _ in range(2):
            assert torch.equal(s.probs(logits), want)
            assert torch.equal(s.sample(logits, record=False), plain.sample(changed, record=False))
            assert torch.equal(logits, before)
