"""Key weights of windows whose rows are not all taken, against float64 code written from
the definition: row i of a sequence's m rows is the token at position len - m + i; of more
than max_rows rows the last max_rows count, and rows that the buffer does not have never do."""
from __future__ import annotations

import math

import pytest
import torch

import cache_ops_ref as ref
from spikeinfer_amd.kernels import paged_spike_attn_key_mass
from test_eviction_gpu import _check, _mass_case, _want

pytestmark = pytest.mark.gpu


def _window(c):
    q, kc, tables, bs, D = c["q_packed"], c["k_cache"], c["block_tables"], c["block_size"], c["head_dim"]
    T, R, hq, _ = q.shape
    hkv = kc.shape[1]
    out = torch.zeros((tables.shape[0], hkv, tables.shape[1] * bs), dtype=torch.float64, device=q.device)
    starts = c["row_starts"].tolist()
    for n in range(tables.shape[0]):
        length, m = int(c["seq_lens"][n]), max(starts[n + 1] - starts[n], 0)
        k = ref.bits(ref.positions(kc, tables[n], length, bs), D)
        for i in range(max(0, m - c["max_rows"], -starts[n]), m):
            row, seen = starts[n] + i, length - m + i + 1
            if row >= R:
                break
            if seen <= 0:
                continue
            x = ref.bits(q[:, row], D).view(T, hkv, hq // hkv, D)
            s = torch.matmul(x, k[:, :, :seen].transpose(-1, -2).contiguous()) / math.sqrt(D)
            out[n, :, :seen] += torch.softmax(s, -1).sum((0, 2))
    return out


@pytest.mark.parametrize("T,hq,hkv,D,lens,rows,max_rows", [
    (4, 14, 2, 64, [70, 1100, 33], [3, 1, 2], 1),        # a decode step's kernels
    (4, 14, 2, 64, [700, 90], [12, 20], 8),
    (2, 16, 4, 128, [300, 2100], [40, 33], 32),
    (1, 4, 4, 32, [129, 5], [20, 9], 6),                 # rows before the sequence's first token
])
def test_of_too_many_rows_the_last_count(gpu, T, hq, hkv, D, lens, rows, max_rows):
    c = _mass_case(T, hq, hkv, D, 16, lens, rows, D + sum(lens), gpu)
    c["max_rows"] = max_rows
    _check(c, paged_spike_attn_key_mass(**c), _window(c))


@pytest.mark.parametrize("starts", [[2, 9, 22], [-3, 4, 30], [0, 5, 2**30], [6, 6, 13]])
@pytest.mark.parametrize("max_rows", [1, 7, 40])
def test_rows_that_the_buffer_does_not_have(gpu, starts, max_rows):
    c = _mass_case(2, 6, 2, 64, 16, [90, 1200], [5, 7], 8, gpu)  # 14 rows
    c["row_starts"] = torch.tensor(starts, dtype=torch.int32, device=gpu)
    c["max_rows"] = max_rows
    _check(c, paged_spike_attn_key_mass(**c), _window(c))


def test_a_replay_with_longer_windows(gpu):
    c = _mass_case(2, 14, 2, 64, 16, [400, 90], [8, 8], 5, gpu)
    starts = c["row_starts"]
    out = torch.zeros((2, 2, c["block_tables"].shape[1] * 16), device=gpu)
    torch.cuda.synchronize(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_spike_attn_key_mass(**c, out=out)
    for new in ([0, 8, 16], [0, 14, 18], [1, 3, 16]):
        starts.copy_(torch.tensor(new))
        graph.replay()
        torch.cuda.synchronize(gpu)
        _check(c, out, _window(c))
        assert torch.equal(out, paged_spike_attn_key_mass(**c))


@pytest.mark.parametrize("T,hq,hkv,D,lens,rows", [
    (2, 14, 2, 64, [8193, 20011], None),          # more parts than are on their way at once
    (1, 6, 2, 64, [9000, 17000, 70], [9, 20, 70]),
    (1, 2, 1, 128, [66000], [3]),
])
def test_long_sequences(gpu, T, hq, hkv, D, lens, rows):
    c = _mass_case(T, hq, hkv, D, 16, lens, rows, D + sum(lens), gpu)
    want = _want(c) if rows is None else _window(c)
    _check(c, paged_spike_attn_key_mass(**c), want)
