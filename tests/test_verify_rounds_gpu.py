"""verify_draft_tree where several launches of sums precede the draw (more than 8 rows a tree and
65,536 tokens or more)."""
from __future__ import annotations

import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd.kernels import verify_draft_tree, verify_workspace_bytes

pytestmark = pytest.mark.gpu
LAUNCHES = 4  # of sums, before the last one


def _on(case, gpu):
    return {k: v.to(gpu) if isinstance(v, torch.Tensor) else v for k, v in case.items()}


def _want(case, distinct=False, before=-1):
    return ref.verify(case["tokens"], case["parents"], case["target_probs"], case["draft_probs"], case["uniforms"],
                      case["row_starts"], case["max_nodes"], distinct, before)


def _sums(case, targets) -> list[int]:
    """How many sums over the vocabulary each tree's walk took: one a rejected child (those before
    the child that stayed, all where none did), and one for a draw without any."""
    counts = []
    starts, parents, tokens = (case[k].tolist() for k in ("row_starts", "parents", "tokens"))
    for a, e in zip(starts[:-1], starts[1:]):
        at, n = 0, 0
        while e > a:
            kids = [i for i in range(at + 1, e - a) if parents[a + i] == at]
            stays = [i for i in kids if tokens[a + i] == targets[a + at]]
            if not stays:
                n += max(len(kids), 1)
                break
            n += kids.index(stays[0])
            at = stays[0]
        counts.append(n)
    return counts


@pytest.mark.parametrize("distinct", [False, True])
@pytest.mark.parametrize("V,counts,width,near,keep", [
    (65536, [25] * 4, 3, 1.5, None),
    (65536, [9, 12, 0, 16, 1, 10], 8, 4.0, None),     # an empty tree, one of a row; a poor drafter
    (151936, [25] * 4, 5, 1.5, None),
    (151936, [30, 3, 0, 17], 4, 0.3, 40),             # 40 tokens with weight
    (65537, [64, 20], 1, 0.1, None),                  # chains, mostly accepted
    (65536, [9] * 70, 6, 6.0, None),                  # more trees than slices each
])
def test_matches_float64(gpu, V, counts, width, near, keep, distinct):
    print(f"verify {counts[:6]} {V} {width} {distinct}", flush=True)
    case = ref.draft_case(counts, V, V + width, width, distinct, near, keep=keep)
    d = _on(case, gpu)
    rows = len(case["tokens"])
    ws = torch.full((verify_workspace_bytes(len(counts), V),), 0xff, dtype=torch.uint8, device=gpu)  # (NaN, and -1 launches)
    seen = set()
    for seed in range(3):
        case["uniforms"] = torch.rand(rows, generator=torch.Generator().manual_seed(seed))
        if seed == 2:  # (large numbers reject)
            case["uniforms"] = 1.0 - 0.1 * case["uniforms"]
        d["uniforms"] = case["uniforms"].to(gpu)
        out = torch.full((rows,), -7, dtype=torch.int64, device=gpu)
        want = _want(case, distinct, -7)
        assert verify_draft_tree(**d, distinct=distinct, out=out, workspace=ws).tolist() == want
        seen |= set(_sums(case, want))
    assert seen == {1} if width == 1 else len(seen) > 2  # (a chain's sum is its one rejection's, or the draw's)
    if near >= 4.0:
        assert max(seen) >= LAUNCHES


def test_trees_that_need_any_number_of_sums(gpu):
    """Row 0 and k siblings that the target gives no weight, then a chain that it likes: from
    one sum to twice as many as the launches make, each tree alone and all at once."""
    V = 65536
    cases = []
    for k in range(8):
        c = ref.draft_case([10], V, k, 1, near=0.1, spare=0)
        c["parents"][1:] = torch.tensor([0] * k + [0] + list(range(k + 1, 9)), dtype=torch.int32)
        c["tokens"][1:k + 1] = 11 * torch.arange(1, k + 1)
        c["target_probs"][0, 11:100:11] = 0.0
        c["draft_probs"][0] = 0.0
        c["draft_probs"][0, 11:100:11] = 1 / 9
        cases.append(c)
    whole = {k: torch.cat([c[k] for c in cases]) for k in ("tokens", "parents", "target_probs", "draft_probs", "uniforms")}
    whole.update(row_starts=torch.arange(0, 81, 10).int(), max_nodes=10)
    want = _want(whole)
    assert _sums(whole, want) == [1, 2, 3, 4, 5, 6, 7, 8]
    assert verify_draft_tree(**_on(whole, gpu)).tolist() == want
    for i, c in enumerate(cases):
        assert verify_draft_tree(**_on(c, gpu)).tolist() == want[10 * i:10 * i + 10]


def test_replays_that_need_other_numbers_of_sums(gpu):
    """A captured call whose workspace holds another step's sums."""
    V, counts = 65536, [9, 25, 12]
    cases = [ref.draft_case(counts, V, s, w, near=near) for s, w, near in ((1, 1, 0.1), (2, 8, 5.0), (3, 3, 1.5), (4, 2, 0.5))]
    static = _on(cases[0], gpu)
    out = torch.full((len(cases[0]["tokens"]),), -7, dtype=torch.int64, device=gpu)
    ws = torch.empty(verify_workspace_bytes(len(counts), V), dtype=torch.uint8, device=gpu)
    verify_draft_tree(**static, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        verify_draft_tree(**static, out=out, workspace=ws)
    sums = []
    for case in cases + cases[::-1]:
        for k, v in case.items():
            if isinstance(v, torch.Tensor):
                static[k].copy_(v)
        graph.replay()
        eager = verify_draft_tree(**_on(case, gpu))
        torch.cuda.synchronize()
        want = _want(case, before=-7)
        assert out.tolist() == want
        assert eager.tolist() == [-1 if t == -7 else t for t in want]
        sums.append(tuple(_sums(case, want)))
    assert len(set(sums)) == len(cases)
