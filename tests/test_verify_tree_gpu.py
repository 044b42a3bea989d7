"""verify_draft_tree on the GPU against plain float64 code: the tokens are the same."""
from __future__ import annotations

import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd.kernels import accept_draft_tree, verify_draft_tree, verify_workspace_bytes

pytestmark = pytest.mark.gpu


def _on(case, gpu):
    return {k: v.to(gpu) if isinstance(v, torch.Tensor) else v for k, v in case.items()}


def _want(case, distinct=False, before=-1):
    return ref.verify(case["tokens"], case["parents"], case["target_probs"], case["draft_probs"], case["uniforms"],
                      case["row_starts"], case["max_nodes"], distinct, before)


@pytest.mark.parametrize("distinct", [False, True])
@pytest.mark.parametrize("counts,V,width,near,keep", [
    ([1], 1, 1, 0.5, None),                                    # one token there is
    ([2, 1, 3], 2, 2, 0.5, None),
    ([1, 1, 1], 1000, 1, 0.5, None),                           # nothing drafted
    ([5], 151936, 1, 0.5, None),
    ([5, 1, 9, 3], 777, 1, 0.5, None),                         # chains
    ([8] * 40, 4097, 1, 0.2, None),
    ([25, 13, 2, 40], 5003, 3, 0.5, None),                     # trees
    ([30, 30, 30], 50, 5, 1.5, None),                          # a poor drafter, siblings alike
    ([25] * 6, 32003, 4, 1.5, 20),                             # distributions of 20 tokens
    ([70, 129], 300, 2, 0.1, None),                            # a good one, long paths
    ([6, 6], 262144, 2, 0.5, 1000),
    ([1024], 64, 3, 0.3, None),                                # the widest tree
    ([12] * 5, 30, 6, 0.5, 3),                                 # more siblings than tokens with weight
])
def test_matches_float64(gpu, counts, V, width, near, keep, distinct):
    print(f"verify {counts[:6]} {V} {width} {distinct}", flush=True)
    case = ref.draft_case(counts, V, sum(counts) + V, width, distinct, near, keep=keep)
    for seed in range(4):
        case["uniforms"] = torch.rand(len(case["tokens"]), generator=torch.Generator().manual_seed(seed))
        got = verify_draft_tree(**_on(case, gpu), distinct=distinct)
        assert got.tolist() == _want(case, distinct)


def test_ends_of_the_random_numbers(gpu):
    """0 keeps every token that the target gives any weight, the largest number below 1
    draws the last token with weight."""
    case = ref.draft_case([9, 5, 16], 901, 3, 2)
    for u in (0.0, 1.0 - 2.0**-24, 0.5):
        case["uniforms"].fill_(u)
        assert verify_draft_tree(**_on(case, gpu)).tolist() == _want(case)
    case = ref.draft_case([3], 901, 4, keep=30)
    case["uniforms"][:] = torch.tensor([1.0 - 2.0**-24, 1.0, 1.0] + [0.0] * 3)
    out = verify_draft_tree(**_on(case, gpu)).tolist()
    assert out == _want(case)


def test_rows_left_out(gpu):
    """Trees without rows, rows of no sequence, more rows than max_nodes, starts past the rows
    and below zero: what is no tree's stays."""
    case = ref.draft_case([4, 6, 3, 8], 500, 6, 2, spare=9)
    R = len(case["tokens"])
    for starts, most in (([0, 4, 4, 10, 13], 6), ([4, 10, 21, 30], 8), ([-3, 4, 10], 6), ([0, 4, 10, 13, 21], 3),
                         ([0, 0, 0], 8), ([R, R + 5], 4)):
        c = {**case, "row_starts": torch.tensor(starts, dtype=torch.int32), "max_nodes": most}
        out = torch.full((R,), -7, dtype=torch.int64, device=gpu)
        assert verify_draft_tree(**_on(c, gpu), out=out) is out
        want = [-7] * R
        for a, e in zip(starts[:-1], starts[1:]):
            a = min(max(a, 0), R)
            e = min(max(min(e, R), a), a + most)
            if e > a:
                want[a:e] = ref.verify_tree(c["tokens"][a:e].tolist(), c["parents"][a:e].tolist(),
                                            c["target_probs"][a:e].double().numpy(),
                                            c["draft_probs"][a:e].double().numpy(), c["uniforms"][a:e].tolist())
        assert out.tolist() == want, starts


def test_tokens_and_distributions_without_sense(gpu):
    """Tokens outside the vocabulary do not stay; a target without weight gives no token; a row
    whose rejected draft takes all of p draws from p; NaN has no weight; parents that are not
    below their row belong to no one."""
    case = ref.draft_case([6, 6, 6], 400, 8, 2)
    case["tokens"][1], case["tokens"][7], case["tokens"][13] = -5, 400, 2**62
    assert verify_draft_tree(**_on(case, gpu)).tolist() == _want(case)
    case = ref.draft_case([3, 3], 64, 9)
    case["target_probs"][0] = 0.0
    case["target_probs"][3] = case["draft_probs"][3]  # equal: a token that q lacks is drafted
    case["target_probs"][3, 5] = case["draft_probs"][3, 5] = 0.0
    case["tokens"][4] = 5
    got = verify_draft_tree(**_on(case, gpu)).tolist()
    assert got == _want(case) and got[:3] == [-1] * 3 and got[3] >= 0
    case = ref.draft_case([2], 64, 10)
    case["target_probs"][0, 10:20] = torch.nan
    case["tokens"][1] = 12
    assert verify_draft_tree(**_on(case, gpu)).tolist()[0] not in (-1, *range(10, 20))
    case["target_probs"][:] = torch.nan
    assert verify_draft_tree(**_on(case, gpu)).tolist() == [-1] * 5
    case = ref.draft_case([5], 64, 11)
    case["parents"][1:5] = torch.tensor([4, 2, -3, 7], dtype=torch.int32)
    assert verify_draft_tree(**_on(case, gpu)).tolist() == _want(case)


def test_types_and_strides(gpu):
    """int64 parents and starts, distributions whose rows lie apart or are shared."""
    case = ref.draft_case([5, 7], 1003, 12, 2)
    want = _want(case)
    d = _on(case, gpu)
    R, V = case["target_probs"].shape
    for pad, at in ((1, 0), (5, 3), (8, 4)):
        wide = torch.zeros((2, R, V + pad), device=gpu)
        wide[0, :, at:at + V], wide[1, :, at:at + V] = d["target_probs"], d["draft_probs"]
        args = {**d, "target_probs": wide[0, :, at:at + V], "draft_probs": wide[1, :, at:at + V],
                "parents": d["parents"].long(), "row_starts": d["row_starts"].long()}
        assert verify_draft_tree(**args).tolist() == want
        args["draft_probs"] = d["draft_probs"]  # the two differ in their alignment
        assert verify_draft_tree(**args).tolist() == want
    one = {**case, "target_probs": case["target_probs"][:1].expand(R, V), "draft_probs": case["draft_probs"][:1].expand(R, V)}
    got = verify_draft_tree(**{**d, "target_probs": d["target_probs"][:1].expand(R, V),
                               "draft_probs": d["draft_probs"][:1].expand(R, V)})
    assert got.tolist() == _want(one)


def test_offsets_past_32_bits(gpu):
    rows, V = 9000, 150001
    P = torch.zeros((rows, V), device=gpu)
    Q = P[:1].expand(rows, V)
    small = ref.draft_case([4], V, 13)
    first = rows - 7
    P[first:] = small["target_probs"][:7].to(gpu)
    Q = torch.zeros((rows, V), device=gpu)
    Q[first:] = small["draft_probs"][:7].to(gpu)
    long = lambda t, fill: torch.cat([torch.full((first,), fill, dtype=t.dtype), t]).to(gpu)
    for u in (0.1, 0.5, 0.9):
        small["uniforms"].fill_(u)
        got = verify_draft_tree(long(small["tokens"], 0), long(small["parents"], -1), P, Q, long(small["uniforms"], 0.0),
                                torch.tensor([first, first + 4], dtype=torch.int32, device=gpu), 4)
        assert got[first:].tolist() == _want(small)


def test_trees_do_not_depend_on_their_batch(gpu):
    case = ref.draft_case([9, 4, 16, 7] * 20, 2000, 14, 3)
    d = _on(case, gpu)
    whole = verify_draft_tree(**d)
    starts = case["row_starts"].tolist()
    for n in (0, 5, 42, 79):
        a, e = starts[n], starts[n + 1]
        part = {k: v[a:e] if isinstance(v, torch.Tensor) else v for k, v in d.items()}
        part["row_starts"] = torch.tensor([0, e - a], dtype=torch.int32, device=gpu)
        assert torch.equal(verify_draft_tree(**part), whole[a:e])


def test_captured_call_takes_other_trees(gpu):
    cases = [ref.draft_case([6, 9, 4], 3000, s, 2, spare=2) for s in (20, 21, 22)]
    static = _on(cases[0], gpu)
    out = torch.full((len(cases[0]["tokens"]),), -7, dtype=torch.int64, device=gpu)
    ws = torch.empty(verify_workspace_bytes(3, 3000), dtype=torch.uint8, device=gpu)
    verify_draft_tree(**static, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        verify_draft_tree(**static, out=out, workspace=ws)
    for case in cases + cases[::-1]:
        for k, v in case.items():
            if isinstance(v, torch.Tensor):
                static[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert out.tolist() == _want(case, before=-7)


def test_accepted_paths(gpu):
    """accept_draft_tree goes the way that the targets give, to the token behind it."""
    for distinct in (False, True):
        case = ref.draft_case([12, 5, 1, 20], 700, 30, 3, distinct, 0.3)
        d = _on(case, gpu)
        targets = verify_draft_tree(**d, distinct=distinct)
        path, count, after = accept_draft_tree(d["tokens"], d["parents"], targets, d["row_starts"], d["max_nodes"])
        starts, t = case["row_starts"].tolist(), targets.tolist()
        assert int(count.sum()) > 4
        for n, a in enumerate(starts[:-1]):
            rows = path[n][:int(count[n])].tolist()
            assert [a + r for r in rows] == [r for r in range(a, starts[n + 1]) if t[r] >= 0]
            assert int(after[n]) == t[a + rows[-1]]
