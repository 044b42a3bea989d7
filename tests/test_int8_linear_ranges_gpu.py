"""linear_int8 over the range of fp32: scales whose product alone has no value there.

Tolerance: what ref.linear derives for the fp32 steps and half a step of y's type, with steps of
2^-149 (fp32), 2^-133 (bf16) and 2^-24 (fp16) below the normal range for each of the two last."""
from __future__ import annotations

import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd.kernels import linear_int8, pack_linear_int8

pytestmark = pytest.mark.gpu
STEP = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24}
MOST = {t: float(torch.finfo(t).max) for t in STEP}


@pytest.mark.parametrize("out", list(STEP))
@pytest.mark.parametrize("M,N", [(4, 70), (40, 70), (300, 70), (600, 700), (16, 32800)])
def test_scales_of_any_size(gpu, M, N, out):
    """Rows of x times rows of W: large by large (0 where the sum is 0, infinite beyond the type),
    small by small, and large by small, whose products are ordinary numbers."""
    print(f"scales {M} {N} {out}", flush=True)
    K = 128
    g = torch.Generator().manual_seed(M)
    x, w = torch.randn((M, K), generator=g), torch.randn((N, K), generator=g)
    # powers of two change no quotient
    ex = torch.tensor([-120.0, 120.0, -60.0, 0.0, 60.0, 100.0, -100.0])
    x, w = x.clamp(-4, 4), w.clamp(-4, 4)
    x *= 2.0 ** ex[torch.arange(M) % 7][:, None]
    w *= 2.0 ** ex[torch.arange(N) // 2 % 7][:, None]
    x[1, K // 2:] = 0.0  # sums of 0 in every column whose first half is
    w[::3, :K // 2] = 0.0
    x[2] = 0.0
    w[4] = 0.0
    bias = torch.randn(N, generator=g)
    want, off = ref.linear(x, w)
    assert (want[1, ::3] == 0).all() and (want[3].abs() > MOST[torch.float32]).sum() == 0
    w8 = pack_linear_int8(w.to(gpu))
    for b in (None, bias):
        exact, off = ref.linear(x, w, b)
        got = linear_int8(x.to(gpu), w8, None if b is None else b.to(gpu), dtype=out).cpu().double()
        assert not got.isnan().any()
        tol = off + (exact.abs() + off) * torch.finfo(out).eps / 2 + STEP[torch.float32] + STEP[out]
        large = exact.abs() + tol > MOST[out]  # may round to infinity, and does well above
        assert torch.equal(got[large].sign(), exact[large].sign())
        assert got[exact.abs() - tol > MOST[out] * (1 + torch.finfo(out).eps)].isinf().all()
        assert ((got - exact).abs() <= tol)[~large].all()
