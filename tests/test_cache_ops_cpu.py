"""Refusals of the draft-tree and eviction operators, on the host (no kernel is
launched), and the plain code that their GPU tests compare with."""
from __future__ import annotations

import ctypes

import pytest
import torch

import cache_ops_ref as ref
from spikeinfer_amd import _lib, kernels

P = 0x10000  # a pointer that nothing reads


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _tree(lib, **kw):
    a = dict(mask_words=1, dt=0, rows=10, N=2, max_nodes=8, T=4, hq=14, hkv=2, D=64, bs=16, mb=8, scale=0.125, q=P,
             slots=100, ws=None, wsb=0)
    a.update(kw)
    s = _i64(1, 1, 1)
    return lib.spk_tree_attn(a["q"], s, P, P, s, P, P, s, a["slots"], P, 8, 1, P, P, P, a["mask_words"], P, a["dt"], s,
                             a["rows"], a["N"], a["max_nodes"], a["T"], a["hq"], a["hkv"], a["D"], a["bs"], a["mb"],
                             a["scale"], a["ws"], a["wsb"], None)


def test_tree_attention_refusals():
    lib = _lib.load()
    for kw, rc in ((dict(hq=13), 1), (dict(T=0), 1), (dict(D=160), 2), (dict(max_nodes=1025, mask_words=17), 2),
                   (dict(max_nodes=65), 1), (dict(dt=_lib.SPK_I32), 1), (dict(bs=24), 1), (dict(scale=0.5), 1),
                   (dict(scale=0.0), 1), (dict(mb=1 << 27), 2), (dict(q=None), 1), (dict(rows=-1), 1),
                   (dict(max_nodes=0), 1), (dict(slots=-1), 1), (dict(N=1 << 16), 2)):
        assert _tree(lib, **kw) == rc, kw
    assert _tree(lib, N=0) == _tree(lib, rows=0) == _lib.SPK_OK


def test_mask_and_acceptance_refusals():
    lib = _lib.load()
    assert lib.spk_tree_masks(P, P, 10, 2, 65, P, 1, P, None) == _lib.SPK_EINVAL
    assert lib.spk_tree_masks(P, P, -1, 2, 8, P, 1, P, None) == _lib.SPK_EINVAL
    assert lib.spk_tree_masks(None, P, 10, 2, 8, P, 1, P, None) == _lib.SPK_EINVAL
    assert lib.spk_tree_masks(P, P, 1 << 31, 2, 8, P, 1, P, None) == _lib.SPK_EUNSUPPORTED
    assert lib.spk_tree_masks(P, P, 0, 2, 8, P, 1, P, None) == _lib.SPK_OK
    s = _i64(1, 1, 1)

    def accept(rows=10, N=2, nodes=8, layers=b"", n=0, T=4, D=64, bs=16, bt=P, tokens=P):
        return lib.spk_accept_tree(tokens, P, P, P, rows, N, nodes, P, P, P, layers, n, s, s, 100, bt, 8, 1, P, T, 2, D,
                                   bs, 8, None)

    four = lambda *p: b"".join(x.to_bytes(8, "little") for x in p)
    assert accept(nodes=1025) == _lib.SPK_EUNSUPPORTED
    assert accept(nodes=0) == accept(rows=-1) == accept(tokens=None) == _lib.SPK_EINVAL
    assert accept(layers=four(P, P, P, 0), n=1) == _lib.SPK_EINVAL
    assert accept(layers=four(P, P, P, P), n=1, bs=3) == _lib.SPK_EINVAL
    assert accept(layers=four(P, P, P, P), n=1, bt=None) == _lib.SPK_EINVAL
    assert accept(layers=four(P, P, P, P), n=1, D=1024) == _lib.SPK_EUNSUPPORTED
    assert accept(N=0) == _lib.SPK_OK
    assert len(four(P, P, P, P)) == 32


def test_key_mass_and_eviction_refusals():
    lib = _lib.load()
    s, m = _i64(1, 1, 1), _i64(1, 1)

    def mass(rows=2, N=2, most=1, hq=14, D=64, bs=16, mb=8, scale=0.125, cap=100, ws=P, wsb=1 << 20, q=P):
        return lib.spk_key_mass(q, s, P, s, 100, P, 8, 1, P, None, P, m, cap, 0, rows, N, most, 4, hq, 2, D, bs, mb,
                                scale, ws, wsb, None)

    for kw, rc in ((dict(hq=13), 1), (dict(D=160), 2), (dict(bs=5), 1), (dict(scale=1.0), 1), (dict(most=0), 1),
                   (dict(cap=-1), 1), (dict(ws=None), 1), (dict(wsb=8), 1), (dict(q=None), 1), (dict(mb=1 << 27), 2),
                   (dict(N=1 << 20), 2)):
        assert mass(**kw) == rc, kw
    assert mass(N=0) == mass(cap=0) == _lib.SPK_OK

    def evict(budget=64, sinks=4, recent=32, D=64, bs=16, mb=8, dt=None, db=0, n=1, mass=P, layers=None, N=2, T=4):
        layers = layers or (P).to_bytes(8, "little") * 2 * n
        return lib.spk_evict(layers, n, s, 100, mass, s, P, s, 128, P, 8, 1, mb, dt, 4, 1, db, P, P, P, budget, sinks,
                             recent, T, N, 2, D, bs, None)

    for kw, rc in ((dict(budget=0), 1), (dict(budget=35), 1), (dict(sinks=-1), 1), (dict(D=160), 2), (dict(bs=12), 1),
                   (dict(dt=P, db=3), 1), (dict(mass=None), 1), (dict(layers=bytes(16)), 1), (dict(mb=1 << 27), 2),
                   (dict(recent=2**31 - 1), 1), (dict(N=1 << 16), 2), (dict(T=0), 1)):
        assert evict(**kw) == rc, kw
    assert evict(N=0) == evict(n=0) == _lib.SPK_OK


def test_python_refusals():
    """Shapes and types are looked at before anything is launched; CPU tensors are refused."""
    case = ref.tree_case(2, 4, 2, 64, 16, [(20, 5), (3, 2)], 1, "cpu")
    with pytest.raises(ValueError, match="GPU"):
        kernels.paged_spike_attn_tree(**case)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        kernels.draft_tree_masks(i32, i32, 4)
    with pytest.raises(ValueError, match="GPU"):
        kernels.accept_draft_tree(i32.long(), i32, i32.long(), i32, 4)
    with pytest.raises(ValueError, match="GPU"):
        kernels.paged_spike_attn_key_mass(case["q_packed"], case["k_cache"], case["block_tables"],
                                          case["context_lens"], 64, 16)
    with pytest.raises(ValueError, match="GPU"):
        kernels.evict_cache([(case["k_cache"], case["v_cache"])], torch.zeros(1, 2, 2, 32), case["block_tables"],
                            case["context_lens"], 10, 16)


def test_plain_code():
    """Hand-made cases of what the GPU results are compared with."""
    assert ref.evict_ref([5.0, 1.0, 3.0, 3.0, 0.0, 2.0], 6, 4, 1, 1) == [0, 2, 3, 5]
    assert ref.evict_ref([0.0, 2.0, 2.0, 2.0], 4, 2, 0, 0) == [1, 2]
    assert ref.evict_ref([float("nan"), -1.0, float("-inf")], 3, 2, 0, 0) == [1, 2]
    assert ref.evict_ref([1.0], 1, 4, 2, 2) == [0]
    assert ref.accept_ref([9, 4, 4, 5, 5], [-1, 0, 0, 2, 1], [4, 5, 5, 6, 7]) == ([0, 1, 4], 7)
    assert ref.ancestor_masks([-1, 0, 0, 2], 1)[:, 0].tolist() == [1, 3, 5, 13]
    case = ref.tree_case(1, 1, 1, 32, 16, [(2, 1)], 1, "cpu")
    out = ref.tree_want(case, torch.zeros(1, 3, 1, 32))
    q, k = int(case["q_packed"][0, 0, 0, 0]), [int(x) for x in ref.positions(case["k_cache"], case["block_tables"][0],
                                                                              2, 16)[0, 0, :, 0]]
    k.append(int(case["k_words"][0, 0, 0, 0]))
    w = torch.tensor([bin(q & x & 0xffffffff).count("1") / 32**0.5 for x in k], dtype=torch.float64).softmax(0)
    v = torch.cat([ref.bits(ref.positions(case["v_cache"], case["block_tables"][0], 2, 16), 32)[0, 0],
                   ref.bits(case["v_words"], 32)[0, :1, 0]])
    assert torch.allclose(out[0, 0, 0], w @ v)


def test_outputs_that_lie_on_one_another_are_refused():
    """Broadcast outputs and a cache given as two layers would be written by several
    workgroups at once."""
    lib = _lib.load()
    s, flat = _i64(1, 1, 1), _i64(0, 1, 1)

    def tree(out_strides, T=4, hq=14, rows=10):
        return lib.spk_tree_attn(P, s, P, P, s, P, P, s, 100, P, 8, 1, P, P, P, 1, P, 0, out_strides, rows, 2, 8, T, hq,
                                 2, 64, 16, 1 << 10, 0.125, None, 0, None)

    for i in range(3):
        assert tree(_i64(*(int(i != j) for j in range(3)))) == _lib.SPK_EINVAL
        assert b"one another" in lib.spk_last_error()

    def mass(strides):
        return lib.spk_key_mass(P, s, P, s, 100, P, 8, 1, P, None, P, strides, 100, 0, 2, 2, 1, 4, 14, 2, 64, 16, 8,
                                0.125, P, 1 << 20, None)

    for strides in (_i64(0, 1), _i64(1, 0)):
        assert mass(strides) == _lib.SPK_EINVAL and b"one another" in lib.spk_last_error()

    words = lambda *p: b"".join(x.to_bytes(8, "little") for x in p)

    def accept(layers, strides):
        return lib.spk_accept_tree(P, P, P, P, 10, 2, 8, P, P, P, layers, len(layers) // 32, s, strides, 100, P, 8, 1, P,
                                   4, 2, 64, 16, 8, None)

    def evict(layers, strides=s, to=s):
        return lib.spk_evict(layers, len(layers) // 16, strides, 100, P, s, P, to, 128, P, 8, 1, 8, None, 0, 0, 0, P, P,
                             P, 64, 4, 32, 4, 2, 2, 64, 16, None)

    four, two = words(P, P, P, 2 * P), words(P, 2 * P)
    for i in range(3):
        strides = _i64(*(int(i != j) for j in range(3)))
        assert accept(four, strides) == evict(two, strides) == evict(two + words(3 * P, 4 * P), s, strides) == \
            _lib.SPK_EINVAL
        assert b"one another" in lib.spk_last_error()
    for last in (words(P, 5 * P), words(5 * P, 2 * P)):
        assert accept(four + words(P, P) + last, s) == _lib.SPK_EINVAL and b"one cache" in lib.spk_last_error()
        assert evict(two + last) == _lib.SPK_EINVAL and b"one cache" in lib.spk_last_error()


def test_metadata_moved_to_a_device_keeps_what_the_step_writes():
    """A copy on another device shares the list that the step's words come into, and
    refuses tensors that the caller would wait for in vain."""
    from dataclasses import replace

    from spikeinfer_amd.attention import AttentionMetadata, DraftTrees

    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    trees = DraftTrees(i32(2), torch.zeros((3, 1), dtype=torch.int64), 3, i32(1), i32(1, 4))
    meta = AttentionMetadata(slot_mapping=torch.full((3,), -1), block_size=16, draft=trees)
    copy = meta.on("meta")
    assert copy.draft.masks.device.type == "meta" and trees.masks.device.type == "cpu"
    assert copy.draft.words is trees.words and trees.words == []
    assert meta.on("cpu").draft is trees
    for bad in (replace(meta, draft=replace(trees, words=[(i32(1), i32(1))]), _copies={}),
                replace(meta, draft=None, key_mass=[torch.zeros(1, 1, 8)], _copies={})):
        with pytest.raises(ValueError, match="must be on meta"):
            bad.on("meta")


def test_sizes_beyond_a_launch_are_refused():
    lib = _lib.load()
    assert _tree(lib, T=1 << 12, hq=1 << 12, hkv=1 << 12, max_nodes=1024, mask_words=16) == _lib.SPK_EUNSUPPORTED
    assert _tree(lib, T=1 << 10, hq=1 << 10, hkv=1 << 10, mb=1 << 20, ws=P, wsb=1 << 60) == _lib.SPK_EUNSUPPORTED
    s, m = _i64(1, 1, 1), _i64(1, 1)

    def mass(most=1, mb=8, cap=100, T=4):
        return lib.spk_key_mass(P, s, P, s, 100, P, 8, 1, P, P, P, m, cap, 0, 2, 2, most, T, 14, 2, 64, 16, mb, 0.125, P,
                                1 << 60, None)

    assert mass(cap=(1 << 29) + 1) == mass(most=1 << 20, mb=1 << 17) == mass(T=1 << 20, mb=1 << 10) == \
        _lib.SPK_EUNSUPPORTED
