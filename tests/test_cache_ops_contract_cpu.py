"""Calls of the draft-tree and eviction operators that are refused on the host: nothing is
launched, and no pointer is read."""
from __future__ import annotations

import pytest
import torch

from spikeinfer_amd import _lib, kernels
from spikeinfer_amd.attention import AttentionMetadata, DraftTrees, paged_attention, paged_attention_fused
from test_cache_ops_cpu import P, _i64, _tree


def _mass(lib, hq=14, hkv=2, most=1, T=1, mb=8):
    s = _i64(1, 1, 1)
    return lib.spk_key_mass(P, s, P, s, 100, P, 8, 1, P, P, P, _i64(1, 1), 100, 0, 2, 1, most, T, hq, hkv, 64, 16, mb,
                            0.125, P, 1 << 60, None)


def test_head_ratios_that_the_row_division_does_not_hold():
    """Rows are divided by the heads a kv head with one multiplication, r * ceil(2^32 / n) >> 32.
    A ratio for which that names a wrong head for some row of the call is refused."""
    def wrong(n, rows):  # the first row that the multiplication gets wrong
        m = -(-2**32 // n)
        over = m * n - 2**32
        r = -(-2**32 // over) if over else rows
        r += (n - 1 - r) % n  # (the last of a quotient's)
        return r if r < rows else None

    for n, rows in ((257, 65280 * 257), (4097, 1024 * 4097)):
        r = wrong(n, rows)
        if r is not None:
            assert r * -(-2**32 // n) >> 32 != r // n
    lib = _lib.load()
    bad = [n for n in range(2049, 16384, 7) if wrong(n, 1024 * n) is not None]
    good = [n for n in (7, 17, 256, 1024, 2048) if wrong(n, 1024 * n) is None]
    assert len(bad) > 100 and len(good) == 5
    for n in bad[:3] + bad[-3:]:
        assert _tree(lib, T=1, hq=n, hkv=1, max_nodes=1024, mask_words=16, mb=1) == _lib.SPK_EUNSUPPORTED, n
        assert b"heads" in lib.spk_last_error()
    most = lambda n: (1 << 24) // n
    bad = [n for n in range(257, 5000, 3) if wrong(n, most(n) * n) is not None]
    assert len(bad) > 100
    for n in bad[:3] + bad[-3:]:
        assert _mass(lib, hq=n, hkv=1, most=most(n), mb=1) == _lib.SPK_EUNSUPPORTED, n
        assert b"heads" in lib.spk_last_error()


@pytest.mark.parametrize("what", ["draft", "key_mass"])
def test_metadata_that_one_layer_cannot_honour(what):
    """Neither drops the weights that a step asks for, nor takes drafted rows for tokens."""
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    given = dict(draft=DraftTrees(i32(2), torch.zeros((3, 1), dtype=torch.int64), 3, i32(1), i32(1, 4)),
                 key_mass=[torch.zeros((1, 2, 64))])[what]
    meta = AttentionMetadata(slot_mapping=torch.full((3,), -1), block_size=16, num_decode_tokens=0 if what == "draft" else 3,
                             block_tables=i32(3, 4), seq_lens=i32(3), **{what: given})
    cache = i32(2, 2, 64, 2)
    spikes = lambda h: torch.zeros((2, 1, h, 3, 64))
    with pytest.raises(ValueError, match=f"{what} is for SpikingDecoder.forward_paged"):
        paged_attention(spikes(4), spikes(2), spikes(2), cache, cache.clone(), meta, 4, 2, 64)
    cur, lif = lambda h: torch.zeros((2, 3, h, 64)), (torch.full((64,), 0.9), torch.ones(64))
    with pytest.raises(ValueError, match=f"{what} is for SpikingDecoder.forward_paged"):
        paged_attention_fused(cur(4), cur(2), cur(2), lif, lif, lif, cache, cache.clone(), meta, 4, 2, 64)


def test_layers_and_outputs_that_are_no_pairs_and_triples(monkeypatch):
    """The addresses of every layer go to the host entry as pairs: one tensor less and it
    would read behind them."""
    def launched(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "native", lambda: None)
    monkeypatch.setattr(_lib, "launch", launched)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    k, w, ids = i32(2, 2, 64, 2), i32(2, 3, 2, 2), torch.zeros(3, dtype=torch.int64)
    for layer in ((k,), (k, k.clone(), k.clone()), ()):
        for layers in ([layer], [(k, k.clone()), layer], [layer, (k, k.clone())]):
            with pytest.raises(ValueError, match="layers: .* pair"):
                kernels.evict_cache(layers, torch.zeros(len(layers), 1, 2, 64), i32(1, 4), i32(1), 40, 16)
            good = [(w, w.clone())] * len(layers)
            with pytest.raises(ValueError, match="layers: .* pair"):
                kernels.accept_draft_tree(ids, i32(3), ids, i32(2), 3, good, layers, i32(1, 4), i32(1), 16)
    for draft in ((w,), (w, w, w), ()):
        with pytest.raises(ValueError, match="drafts: .* pair"):
            kernels.accept_draft_tree(ids, i32(3), ids, i32(2), 3, [draft], [(k, k.clone())], i32(1, 4), i32(1), 16)
    path, count, after = i32(1, 3), i32(1), torch.zeros(1, dtype=torch.int64)
    for out in ((path, count), (path, count, after, after), ()):
        with pytest.raises(ValueError, match="path, count, next"):
            kernels.accept_draft_tree(ids, i32(3), ids, i32(2), 3, out=out)


def test_one_cache_as_keys_and_values():
    """Its words would be written by several threads at once, whichever places name it."""
    lib = _lib.load()
    s = _i64(1, 1, 1)
    words = lambda *p: b"".join((x * P).to_bytes(8, "little") for x in p)

    def accept(layers):
        return lib.spk_accept_tree(P, P, P, P, 10, 2, 8, P, P, P, layers, len(layers) // 32, s, s, 100, P, 8, 1, P, 4, 2,
                                   64, 16, 8, None)

    def evict(layers):
        return lib.spk_evict(layers, len(layers) // 16, s, 100, P, s, P, s, 128, P, 8, 1, 8, None, 0, 0, 0, P, P, P, 64, 4,
                             32, 4, 2, 2, 64, 16, None)

    for pairs in ([(5, 5)], [(1, 2), (3, 1)], [(1, 2), (2, 3)], [(1, 2), (3, 4), (5, 6), (7, 3)], [(1, 2), (4, 4)]):
        assert accept(b"".join(words(98, 99, *kv) for kv in pairs)) == _lib.SPK_EINVAL, pairs
        assert b"one cache" in lib.spk_last_error()
        assert evict(b"".join(words(*kv) for kv in pairs)) == _lib.SPK_EINVAL, pairs
        assert b"one cache" in lib.spk_last_error()


def test_metadata_moved_to_the_current_device(monkeypatch):
    """A device without a number is the current one, whichever that is."""
    from types import SimpleNamespace

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    on = lambda i: [SimpleNamespace(device=torch.device("cuda", i))]
    slots = SimpleNamespace(device=torch.device("cpu"), to=lambda device, non_blocking: None)
    meta = lambda mass: AttentionMetadata(slot_mapping=slots, block_size=16, key_mass=mass)
    for device in ("cuda", torch.device("cuda"), "cuda:1"):
        assert meta(on(1)).on(device).key_mass[0].device.index == 1
        with pytest.raises(ValueError, match="must be on cuda"):
            meta(on(0)).on(device)
    assert meta(on(0)).on("cuda:0").key_mass[0].device.index == 0
