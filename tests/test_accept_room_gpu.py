"""Acceptance where the block table or the cache ends inside the path: the path ends with
the last row whose words are in the cache."""
from __future__ import annotations

import pytest
import torch

from spikeinfer_amd.kernels import accept_draft_tree

pytestmark = pytest.mark.gpu
BS = 4


@pytest.mark.parametrize("layers", [1, 70])
def test_a_path_ends_where_its_words_have_no_place(gpu, layers):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    depth, ctx = 9, [3, 0, 8, 12, 11, 5]
    # a table that goes on, one with a block outside the cache, ones that end, a full one
    tables = [[0, 1, 2, 3], [4, 99, 5, 6], [7, 8, -1, 9], [10, 11, 12, -1], [13, 14, 15, 16], [17, -1, 18, 19]]
    room = [9, 4, 0, 0, 5, 0]
    N, R = len(ctx), len(ctx) * depth
    starts = i32([depth * n for n in range(N + 1)])
    parents = i32([i - 1 for i in range(depth)] * N)
    tokens = torch.arange(R, device=gpu)
    targets = tokens + 1  # a chain, all of it accepted
    new = torch.arange(1, R + 1, dtype=torch.int32, device=gpu).view(1, R, 1, 1)
    caches = [tuple(torch.zeros((1, 1, 20 * BS, 1), dtype=torch.int32, device=gpu) for _ in range(2))
              for _ in range(layers)]
    path, count, after = accept_draft_tree(tokens, parents, targets, starts, depth, [(new, new + 1000)] * layers, caches,
                                           i32(tables), i32(ctx), BS)
    assert count.tolist() == room
    want = torch.zeros(20 * BS, dtype=torch.int32)
    for n, m in enumerate(room):
        assert path[n].tolist() == list(range(m)) + [-1] * (depth - m)
        assert after[n] == (n * depth + m if m else -1)
        for i in range(m):
            pos = ctx[n] + i
            want[tables[n][pos // BS] * BS + pos % BS] = n * depth + i + 1
    for k, v in caches:
        assert torch.equal(k[0, 0, :, 0].cpu(), want)
        assert torch.equal(v[0, 0, :, 0].cpu(), want + 1000 * (want != 0))
