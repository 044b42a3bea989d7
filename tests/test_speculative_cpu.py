"""8-bit products, sampling distributions and verification: refusals on the host (nothing is
launched and no pointer read), and the plain code that the GPU tests compare with."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd import _lib, kernels, sampler

P = 0x10000  # a pointer that nothing reads


def test_linear_refusals():
    lib = _lib.load()

    def pack(w=P, dt=2, N=16, K=64, packed=P, scales=P):
        return lib.spk_linear_int8_pack(w, dt, K, N, K, packed, scales, None)

    for kw, rc in ((dict(w=None), 1), (dict(dt=4), 1), (dict(K=0), 1), (dict(N=-1), 1), (dict(K=131073), 2),
                   (dict(packed=None), 1), (dict(packed=P + 8), 1), (dict(scales=None), 1)):
        assert pack(**kw) == rc, kw
    assert pack(N=0) == _lib.SPK_OK

    def linear(x=P, xdt=2, packed=P, scales=P, bias=None, bdt=0, y=P, ydt=2, ys=48, M=5, N=48, K=64, ws=P, wsb=1 << 40):
        return lib.spk_linear_int8(x, xdt, K, packed, scales, bias, bdt, y, ydt, ys, M, N, K, ws, wsb, None)

    for kw, rc in ((dict(x=None), 1), (dict(xdt=3), 1), (dict(ydt=9), 1), (dict(bias=P, bdt=4), 1), (dict(N=0), 1),
                   (dict(K=0), 1), (dict(M=-1), 1), (dict(K=131073), 2), (dict(M=(1 << 30) + 1), 2), (dict(N=(1 << 30) + 1, ys=1 << 31), 2), (dict(ys=47), 1),
                   (dict(ys=0), 1), (dict(packed=None), 1), (dict(scales=None), 1), (dict(y=None), 1),
                   (dict(ws=None), 1), (dict(wsb=16), 1), (dict(ws=P + 4), 1), (dict(packed=P + 1), 1)):
        assert linear(**kw) == rc, kw
    assert linear(M=0) == _lib.SPK_OK
    for kw in (dict(y=P), dict(y=P + 4 * 64 * 2), dict(y=P - 2 * 48 * 4), dict(x=P + 2 * 48 * 4, y=P)):
        assert linear(**kw) == 1 and b"y lies on x" in lib.spk_last_error(), kw
    # more threads than a launch has
    assert linear(M=1 << 30, N=1 << 20, ys=1 << 20, wsb=1 << 62) == _lib.SPK_EUNSUPPORTED
    assert linear(M=1 << 30, K=4096, wsb=1 << 62) == _lib.SPK_EUNSUPPORTED and b"launch" in lib.spk_last_error()
    assert lib.spk_linear_int8_packed_bytes(17, 65) == 4 * 2 * 1024
    assert lib.spk_linear_int8_packed_bytes(0, 65) == lib.spk_linear_int8_packed_bytes(4, -1) == 0
    # offsets in 64 bits
    assert lib.spk_linear_int8_packed_bytes(2**31 - 1, 131072) == 2**31 * 131072
    assert lib.spk_linear_int8_workspace_bytes(1 << 30, 16, 131072) >= 2**30 * 131072


def test_distribution_refusals():
    lib = _lib.load()

    def probs(x=P, dt=0, rows=2, V=100, temp=P, out=P, os=100, ws=P, wsb=1 << 40):
        return lib.spk_sample_probs(x, dt, V, rows, V, temp, None, None, None, out, os, ws, wsb, None)

    for kw, rc in ((dict(x=None), 1), (dict(dt=4), 1), (dict(rows=-1), 1), (dict(V=0), 1), (dict(V=262145), 1),
                   (dict(temp=None), 1), (dict(out=None), 1), (dict(os=99), 1), (dict(os=0), 1),
                   (dict(rows=1 << 23, V=10, os=10, wsb=1 << 62), 2), (dict(ws=None), 1), (dict(wsb=64), 1),
                   (dict(ws=P + 8), 1)):
        assert probs(**kw) == rc, kw
    assert probs(rows=0) == _lib.SPK_OK


def test_distributions_on_their_logits_are_refused():
    """Whole, in part, at either end, rows of one between rows of the other."""
    lib = _lib.load()
    V, rows = 100, 3

    def probs(out, os, dt=0, row_stride=V):
        rc = lib.spk_sample_probs(1 << 20, dt, row_stride, rows, V, P, None, None, None, out, os, P, 1 << 40, None)
        return rc, lib.spk_last_error()

    base = 1 << 20
    for out, os, dt, stride in ((base, V, 0, V), (base + 4, V, 0, V), (base + 4 * (rows * V - 1), V, 0, V),
                                (base - 4 * (rows * V - 1), V, 0, V), (base, 2 * V, 0, V), (base + 2 * V, 2 * V, 2, V),
                                (base + 4 * (V - 1), 2 * V, 0, 2 * V), (base + 4 * (V + 1), 2 * V, 0, 2 * V),
                                (base, V, 0, 0), (base - 4 * V, 2 * V, 0, 0)):
        rc, why = probs(out, os, dt, stride)
        assert rc == 1 and b"lies on the logits" in why, (out - base, os, dt, stride)


def test_verification_refusals():
    lib = _lib.load()

    def verify(tokens=P, p=P, q=P, u=P, starts=P, rows=10, N=2, nodes=8, V=100, out=P, ws=P, wsb=1 << 40):
        return lib.spk_verify_tree(tokens, P, p, V, q, V, u, starts, rows, N, nodes, V, 0, out, ws, wsb, None)

    for kw, rc in ((dict(tokens=None), 1), (dict(p=None), 1), (dict(q=None), 1), (dict(u=None), 1), (dict(starts=None), 1),
                   (dict(rows=-1), 1), (dict(N=-1), 1), (dict(nodes=0), 1), (dict(V=0), 1), (dict(nodes=1025), 2),
                   (dict(N=65536), 2), (dict(out=None), 1), (dict(ws=None), 1), (dict(wsb=1), 1), (dict(ws=P + 4), 1)):
        assert verify(**kw) == rc, kw
    assert verify(N=0) == verify(rows=0) == _lib.SPK_OK


def test_python_refuses_cpu_tensors():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    with pytest.raises(ValueError, match="GPU"):
        kernels.pack_linear_int8(w)
    with pytest.raises(ValueError, match="GPU"):
        kernels.linear_int8(x, kernels.Int8Weight(torch.zeros(1024, dtype=torch.uint8), torch.zeros(16), 4, 8))
    with pytest.raises(ValueError, match="GPU"):
        sampler.sampling_probs(x, torch.ones(2))
    with pytest.raises(ValueError, match="GPU"):
        kernels.verify_draft_tree(**ref.draft_case([3], 8, 0))


@pytest.fixture
def no_launch(monkeypatch):
    """The wrappers' own checks on CPU tensors; a launch fails the test."""
    def launched(*_):
        raise AssertionError("launched")

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "native", lambda: None)
    monkeypatch.setattr(_lib, "launch", launched)


def test_linear_arguments(no_launch):
    w8 = kernels.Int8Weight(torch.zeros(1024, dtype=torch.uint8), torch.zeros(16), 4, 8)
    x, f = torch.zeros(2, 8), torch.zeros
    for bad in (f(2, 9), f(8, dtype=torch.int32), torch.tensor(1.0)):
        with pytest.raises(ValueError, match="x must be"):
            kernels.linear_int8(bad, w8)
    for bad in (f(5), f(4, 1), f(4, dtype=torch.int64)):
        with pytest.raises(ValueError, match="bias must be"):
            kernels.linear_int8(x, w8, bad)
    for bad in (f(2, 5), f(3, 4), f(2, 1, 4), f(2, 4, dtype=torch.int32), f(4, 2).t(), f(2, 8)[:, ::2]):
        with pytest.raises(ValueError, match="out"):
            kernels.linear_int8(x, w8, out=bad)
    with pytest.raises(ValueError, match="out must be"):
        kernels.linear_int8(x, w8, out=f(2, 4), dtype=torch.float16)
    with pytest.raises(ValueError, match="one distance"):
        kernels.linear_int8(f(2, 3, 8), w8, out=f(2, 4, 4)[:, :3])
    with pytest.raises(ValueError, match="float type"):
        kernels.linear_int8(x, w8, dtype=torch.int8)
    for bad in (f(8, dtype=torch.uint8), f(1 << 16, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            kernels.linear_int8(x, w8, workspace=bad)
    assert kernels.linear_int8(f(0, 8), w8).shape == (0, 4)
    for bad in (f(4), f(0, 8), f(4, 0), f(4, 8, dtype=torch.int8)):
        with pytest.raises(ValueError, match="w must be"):
            kernels.pack_linear_int8(bad)


def test_distribution_arguments(no_launch):
    f, one = torch.zeros, torch.ones(3)
    for bad in (f(8), f(2, 3, 4), f(8, 3).t()):
        with pytest.raises(ValueError, match="logits must be"):
            sampler.sampling_probs(bad, one)
    for kw in (dict(temperature=f(2)), dict(temperature=one.double()), dict(top_k=f(3)), dict(top_p=f(6)[::2]),
               dict(min_p=f(2))):
        with pytest.raises(ValueError, match=f"{next(iter(kw))} must be"):
            sampler.sampling_probs(f(3, 8), **{"temperature": one, **kw})
    for bad in (f(3, 9), f(3, 8, dtype=torch.float16), f(8, 3).t()):
        with pytest.raises(ValueError, match="out must be"):
            sampler.sampling_probs(f(3, 8), one, out=bad)


def test_verification_arguments(no_launch):
    case = ref.draft_case([3, 2], 8, 0)
    bad = dict(tokens=case["tokens"].int(), parents=case["parents"][:-1], uniforms=case["uniforms"].double(),
               target_probs=case["target_probs"].half(), draft_probs=case["draft_probs"][:2], max_nodes=1025,
               out=torch.zeros(3, dtype=torch.int64), workspace=torch.zeros(1, dtype=torch.uint8))
    for name, value in bad.items():
        with pytest.raises(ValueError, match=name):
            kernels.verify_draft_tree(**{**case, name: value})
    with pytest.raises(ValueError, match="draft_probs have 7 tokens"):
        kernels.verify_draft_tree(**{**case, "draft_probs": case["draft_probs"][:, :7]})
    with pytest.raises(ValueError, match="vocab axis"):
        kernels.verify_draft_tree(**{**case, "target_probs": case["target_probs"].t().contiguous().t()})
    with pytest.raises(ValueError, match=r"\[N \+ 1\]"):
        kernels.verify_draft_tree(**{**case, "row_starts": case["row_starts"][:0]})
    empty = kernels.verify_draft_tree(**{**case, "row_starts": case["row_starts"][:1]})
    assert empty.tolist() == [-1] * 8


# -- the plain code ---------------------------------------------------------------
def test_plain_8_bits():
    q, s = ref.rows_to_8_bits(torch.tensor([[127.0, -127.0, 0.5, 1.5, 2.5, -0.5], [0.0] * 6, [1e-45] + [0.0] * 5,
                                            [float("inf")] + [1.0] * 5]))
    assert q[0].tolist() == [127, -127, 0, 2, 2, 0] and s[0] == 1
    assert not q[1:].any() and s[1] == 0 and s[2] == 0 and s[3].isnan()


def test_plain_distributions():
    row = np.log(np.array([0.1, 0.4, 0.2, 0.2, 0.1], np.float32))
    got = lambda **kw: ref.probs(row, 1.0, **kw).round(5).tolist()
    assert got() == [0.1, 0.4, 0.2, 0.2, 0.1]
    assert got(top_k=2) == [0, round(2 / 3, 5), round(1 / 3, 5), 0, 0]
    assert got(top_p=0.65) == [0, 0.5, 0.25, 0.25, 0]
    assert got(top_k=3, top_p=0.6) == [0, round(2 / 3, 5), round(1 / 3, 5), 0, 0]
    assert got(min_p=0.3) == [0, 0.5, 0.25, 0.25, 0]
    assert ref.probs(row, 0.0).tolist() == [0, 1, 0, 0, 0]
    assert not ref.probs(np.full(3, -np.inf, np.float32), 1.0).any()
    assert ref.probs(np.array([np.nan, np.inf, 0, np.inf], np.float32), 1.0).tolist() == [0, 0.5, 0, 0.5]


@pytest.mark.parametrize("distinct", [False, True])
def test_plain_verification_keeps_the_targets_distribution(distinct):
    """Two levels of siblings over five tokens: the first two tokens that come out are
    distributed as the target's, whatever the drafter's distribution.  Summed exactly over the
    drafts, and over a grid of the random numbers."""
    g = np.random.default_rng(0)
    V, grid = 4, 24
    P, Q = (g.dirichlet(np.ones(V), 4) for _ in range(2))
    mids = (np.arange(grid) + 0.5) / grid
    want, got = P[0], np.zeros(V)
    for a in range(V):
        for b in range(V):
            if distinct and a == b:
                continue
            weight = Q[0, a] * (Q[0, b] / (1 - Q[0, a]) if distinct else Q[0, b])
            for ua in mids:
                for ub in mids:
                    for u0 in mids:
                        out = ref.verify_tree([0, a, b], [-1, 0, 0], P, Q, [u0, ua, ub], distinct)
                        got[out[0]] += weight / grid**3
    # the midpoint rule: each of three numbers decides borders within half a cell
    assert np.abs(got - want).max() < 1.5 / grid


def test_plain_verification_by_hand():
    P = np.array([[0.5, 0.25, 0.25], [0.0, 1.0, 0.0], [0.2, 0.3, 0.5]])
    Q = np.array([[0.25, 0.75, 0.0], [0.5, 0.5, 0.0], [1.0, 0.0, 0.0]])
    # 0.25 / 0.75 of token 1 stay; then row 1's distribution, whose draft 0 never does
    assert ref.verify_tree([9, 1, 0], [-1, 0, 1], P, Q, [0.1, 0.3, 0.0]) == [1, 1, -1]
    # it does not: w = (0.25, 0, 0.25), and u = 0.5 draws token 2
    assert ref.verify_tree([9, 1, 0], [-1, 0, 1], P, Q, [0.5, 0.4, 0.0]) == [2, -1, -1]
    # the second sibling takes what the first left: 0.25 of token 0 against 0.5 * 0.25
    assert ref.verify_tree([9, 1, 0], [-1, 0, 0], P, Q, [0.9, 0.4, 0.99]) == [0, -1, 2]
    assert ref.verify_tree([9], [-1], P * 0, Q, [0.5]) == [-1]
