"""Evictions of lengths that each selection kernel takes, and masses that move bit for bit."""
from __future__ import annotations

import math

import pytest
import torch

from spikeinfer_amd.kernels import evict_cache
from test_eviction_gpu import _evict_case, _evict_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("place", ["own", "other"])
@pytest.mark.parametrize("lens,budget", [
    ([16385, 100], 9000),
    ([20011, 16384, 3000], 2048),
    ([32768, 32767], 20000),
    ([32769], 300),
])
def test_long_sequences(gpu, lens, budget, place):
    """Ties among them, in place and elsewhere."""
    caches, mass, tables, seq, left = _evict_case(lens, 1, 1, 1, 32, 64, sum(lens), gpu, ties=place == "own")
    before, given = [tuple(x.clone() for x in c) for c in caches], mass.clone()
    if place == "own":
        dst, out = tables, mass
        keep, new = evict_cache(caches, mass, tables, seq, budget, 64, 4, 32)
    else:
        blocks = -(-budget // 64)
        dst = torch.full((len(lens), blocks), int(left[0]), dtype=torch.int32)
        at = 1
        for n, x in enumerate(lens):
            need = -(-min(x, budget) // 64)
            dst[n, :need] = left[at:at + need]
            at += need
        dst, out = dst.to(gpu), torch.full_like(mass, -1.0)
        keep, new = evict_cache(caches, mass, tables, seq, budget, 64, 4, 32, dst_tables=dst, mass_out=out)
    _evict_check(caches, before, given, tables, seq, dst, keep, new, out, budget, 4, 32, 64)


@pytest.mark.parametrize("length", [64, 3000, 9000, 20000, 33000])
def test_masses_move_bit_for_bit(gpu, length):
    """NaN with payloads, infinities, -0 and subnormal masses too."""
    caches, mass, tables, seq, _ = _evict_case([length], 1, 1, 2, 32, 64, 4, gpu)
    odd = torch.tensor([math.inf, -math.inf, -0.0, 0.0, 1e-42, -1e-42, 1.0, 3e38])
    mass[0, 0, 0, :length] = odd.repeat(-(-length // 8))[:length].to(gpu)
    words = mass.view(torch.int32)
    words[0, 0, :, 5:length:9] = 0x7fc01234
    words[0, 0, 1, 7:length:11] = -0x3fedcc  # a negative NaN
    given = words.clone()
    budget = length * 3 // 4
    keep, new = evict_cache(caches, mass, tables, seq, budget, 64, 2, 3)
    assert new.tolist() == [budget]
    for h in range(2):
        kept = keep[0, 0, h].long()
        assert torch.equal(words[0, 0, h, :budget], given[0, 0, h, kept])
        assert (words[0, 0, h, budget:] == 0).all()
