"""The plain verification that the GPU tests compare with keeps the target's distribution,
summed exactly over the drafts and over the intervals of the random numbers; and the sum sees the
mistakes that such code can hold.

A test's or draw's outcome changes once as its random number grows, so bisection finds the
border to 2^-50; a sum over at most 60 drafts of products of at most four such numbers is off by
less than 1e-12, and the mistakes change it by more than 1e-3."""
from __future__ import annotations

import inspect
import itertools

import numpy as np
import pytest

import speculative_ref as ref

V = 4
LAST = 1.0 - 2.0**-40  # a child that may be rejected is


def _case(seed=3):
    g = np.random.default_rng(seed)
    P, Q = g.dirichlet(np.ones(V), 5), g.dirichlet(np.ones(V), 5)
    return P, Q


def _border(holds) -> float:
    """Where the numbers from 0 on for which `holds` end."""
    if not holds(0.0):
        return 0.0
    if holds(LAST):
        return 1.0
    lo, hi = 0.0, LAST
    for _ in range(50):
        mid = 0.5 * (lo + hi)
        lo, hi = (mid, hi) if holds(mid) else (lo, mid)
    return hi


def _draws(out_of) -> np.ndarray:
    """How the token out_of(u), which does not decrease in u, is distributed."""
    ends = [_border(lambda u: out_of(u) <= x) for x in range(V)]
    return np.diff([0.0, *ends])


def _first_tokens(verify, P, Q, siblings, distinct, told):
    """(what comes out after row 0; after row 1, given that its token stays; its weight), where
    row 0 has `siblings` children and the first of them one.  `told`: what verify is told of them."""
    parents = [-1] + [0] * siblings + [1]
    first, second, reach = np.zeros(V), np.zeros(V), 0.0
    for drafts in itertools.product(range(V), repeat=siblings):
        if distinct and len(set(drafts)) < siblings:
            continue
        weight, left = 1.0, 1.0
        for x in drafts:
            weight *= Q[0, x] / left
            left -= Q[0, x] if distinct else 0.0
        for below in range(V):
            tokens = [0, *drafts, below]

            def out(us, u0, at=0):
                return verify(tokens, parents, P, Q, [u0, *us], told)[at]

            w = weight * Q[1, below]
            rest = w
            for k in range(siblings):  # child k stays, those before it did not
                stays = lambda u: verify(tokens, parents, P, Q, [0.0, *[LAST] * k, u, *[LAST] * (siblings - k)],
                                         told)[1 + k] >= 0
                share = _border(stays)
                first[drafts[k]] += rest * share
                if k == 0 and share > 0.0:  # the path is at row 1: its child, then the draw
                    reach += w * share
                    more = [0.0] * siblings
                    kept = _border(lambda u: out([*more, u], 0.0, siblings + 1) >= 0)
                    second[below] += w * share * kept
                    if kept < 1.0:
                        second += w * share * (1.0 - kept) * _draws(lambda u0: out([*more, LAST], u0, 1))
                rest *= 1.0 - share
            if rest > 0.0:
                first += rest * _draws(lambda u0: out([LAST] * (siblings + 1), u0))
    return first, second, reach


def _left(p, q, c):
    w = np.maximum(p - c * q, 0.0)
    return w, w.sum()


@pytest.mark.parametrize("distinct", [False, True])
@pytest.mark.parametrize("siblings", [1, 2, 3])
def test_the_targets_distribution_is_kept(siblings, distinct):
    P, Q = _case()
    first, second, reach = _first_tokens(ref.verify_tree, P, Q, siblings, distinct, distinct)
    assert np.abs(first - P[0]).max() < 1e-12
    assert reach > 0.01 and np.abs(second / reach - P[1]).max() < 1e-11


def test_the_case_can_tell():
    """After the first rejection, and after the second, two tokens or more have weight left."""
    P, Q = _case()
    w, c = _left(P[0], Q[0], 1.0)
    assert (w > 0).sum() >= 2
    w, _ = _left(P[0], Q[0], 1.0 + c)
    assert (w > 0).sum() >= 2


@pytest.mark.parametrize("siblings", [2, 3])
def test_mistakes_show(siblings):
    """Told the wrong kind of siblings, or with the sum that a rejection leaves taken as 1."""
    P, Q = _case()
    for distinct in (False, True):
        first, _, _ = _first_tokens(ref.verify_tree, P, Q, siblings, distinct, not distinct)
        assert np.abs(first - P[0]).max() > 1e-3
    source = inspect.getsource(ref.verify_tree)
    line = "c = np.maximum(P[at] - A * Q[at], 0.0).sum()"
    assert source.count(line) == 1
    scope = {"np": np}
    exec(source.replace(line, "c = 1.0"), scope)
    first, _, _ = _first_tokens(scope["verify_tree"], P, Q, siblings, False, False)
    assert np.abs(first - P[0]).max() > 1e-3
