"""linear_int8 on the GPU against 64-bit code: exact sums, scales in fp32, one rounding.

Tolerance: what ref.linear derives for the fp32 steps, and half a step of y's type."""
from __future__ import annotations

import pytest
import torch

import speculative_ref as ref
from spikeinfer_amd.kernels import linear_int8, linear_int8_workspace_bytes, pack_linear_int8

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
# fp16 below 2^-14 has steps of 2^-24
FLOOR = {F32: 0.0, F16: 2.0**-25, BF16: 0.0}


def _assert_close(out, x, w, bias=None):
    want, off = ref.linear(x.reshape(-1, x.shape[-1]), w, bias)
    got = out.detach().cpu().double().reshape(want.shape)
    assert torch.equal(got.isnan(), want.isnan())
    want, off, got = (torch.where(want.isnan(), 0.0, t) for t in (want, off, got))
    tol = off + (want.abs() + off) * torch.finfo(out.dtype).eps / 2 + FLOOR[out.dtype]
    bad = (got - want).abs() - tol
    assert bad.max().item() <= 0, (bad.max().item(), int((bad > 0).sum()))


def _data(M, N, K, seed, dtype=BF16, wdtype=BF16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((M, K), generator=g) * torch.exp(0.5 * torch.randn((M, 1), generator=g))
    w = torch.randn((N, K), generator=g) * 0.02
    return x.to(dtype), w.to(wdtype)


SIZES = [(1, 1, 1), (3, 5, 7), (16, 16, 64), (17, 33, 65), (4, 1152, 896), (64, 200, 896), (65, 130, 129),
         (130, 257, 777), (300, 96, 4864), (257, 512, 200), (1, 5000, 64), (1000, 16, 16), (33, 64, 9000),
         (512, 300, 128), (129, 1153, 320)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_matches_64_bits(gpu, M, N, K):
    print(f"linear {M} {N} {K}", flush=True)
    x, w = _data(M, N, K, M + N + K)
    w8 = pack_linear_int8(w.to(gpu))
    _assert_close(linear_int8(x.to(gpu), w8), x, w)


@pytest.mark.parametrize("M,N,K", [
    (1, 32769, 64), (17, 32770, 200), (33, 32800, 65), (64, 32769, 1024), (64, 32769, 1030), (16, 32769, 1030),  # many columns
    (16, 70, 1025), (9, 70, 5121), (2, 8, 5120), (16, 1000, 9000),                                               # few rows
    (4096, 1100, 64), (4100, 300, 65), (300, 9000, 192), (2049, 1025, 130), (129, 20000, 64)])                   # many of both
def test_sizes_of_every_kernel(gpu, M, N, K):
    """Around the sizes from which another kernel takes the call: what fits LDS or is kept in
    registers, odd and even numbers of steps, tiles that end inside."""
    print(f"linear {M} {N} {K}", flush=True)
    x, w = _data(M, N, K, M + N + K)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(K))
    _assert_close(linear_int8(x.to(gpu), pack_linear_int8(w.to(gpu)), bias.to(gpu)), x, w, bias)


@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_types_and_bias(gpu, dtype, out):
    for M, N, K in ((5, 40, 100), (150, 200, 256), (80, 1000, 96)):
        x, w = _data(M, N, K, M, dtype, dtype)
        g = torch.Generator().manual_seed(1)
        w8 = pack_linear_int8(w.to(gpu))
        for bdt in (F32, F16, BF16):
            bias = torch.randn(N, generator=g).to(bdt)
            y = linear_int8(x.to(gpu), w8, bias.to(gpu), dtype=out)
            assert y.dtype == out
            _assert_close(y, x, w, bias)


@pytest.mark.parametrize("M", [3, 70, 400])
def test_strides_and_shapes(gpu, M):
    """Rows at any distance (odd ones too), transposed inputs, leading axes, outputs within a
    larger tensor, whose other columns stay."""
    K, N = 96, 80
    x, w = _data(M, N, 3 * K + 1, M)
    xd = x.to(gpu)
    w = w[:, 1:K + 1]
    w8 = pack_linear_int8(w.to(gpu))
    for view in (x[:, :K], x[:, 1:K + 1], x[:, 3:3 + 3 * K:3]):
        d = xd.as_strided(view.shape, view.stride(), view.storage_offset())
        _assert_close(linear_int8(d, w8), view, w)
    t = x[:, :K].t().contiguous().t()
    _assert_close(linear_int8(t.to(gpu), w8), t, w)
    stack = torch.stack([x[:, :K], x[:, K:2 * K]])
    y = linear_int8(stack.to(gpu), w8)
    assert y.shape == (2, M, N)
    _assert_close(y, stack, w)
    assert linear_int8(xd[0, :K], w8).shape == (N,)
    for dtype, pad, at in ((BF16, 13, 5), (F32, 4, 4), (BF16, 8, 8)):
        big = torch.full((M, N + pad), -7.0, dtype=dtype, device=gpu)
        out = big[:, at:at + N] if at + N <= N + pad else big[:, pad:]
        assert linear_int8(xd[:, :K], w8, out=out) is out
        _assert_close(out, x[:, :K], w)
        rest = big.clone()
        rest.as_strided(out.shape, out.stride(), out.storage_offset()).fill_(-7.0)
        assert (rest == -7).all()
    # a weight whose rows lie apart, and one stored by columns
    wide = torch.zeros(N, K + 3)
    wide[:, :K] = w.float()
    for form in (wide.to(gpu)[:, :K], w.float().t().contiguous().to(gpu).t()):
        _assert_close(linear_int8(xd[:, :K], pack_linear_int8(form)), x[:, :K], w.float())


@pytest.mark.parametrize("M", [16, 200])
def test_rows_with_special_values(gpu, M):
    """Zero rows, subnormal rows, rows with an infinity or a NaN, one value alone, halves."""
    K, N = 130, 40
    x, w = _data(M, N, K, 5, F32, F32)
    x[0] = 0.0
    x[1] = 0.0
    x[1, 129] = 3.0
    x[2, 7] = float("inf")
    x[3, 128] = float("nan")
    x[4] *= 1e-40
    x[5] = 0.0
    x[5, 3] = 1e-45
    x[6, 0] = float("-inf")
    x[7] = (torch.arange(K) % 127).float() + 0.5  # halves in steps of one, whose scale is 1
    x[7, 0] = 127.0
    x[8] *= 2e36
    x[9] *= 1e-33
    x[10, 0] = 3e38
    w[3] = 0.0
    w[5, 1] = float("nan")
    w[6] = 0.0
    w[6, 129] = -1e-30
    got = linear_int8(x.to(gpu), pack_linear_int8(w.to(gpu)))
    nan = got.isnan().cpu()
    rows, cols = torch.zeros(M, dtype=torch.bool), torch.zeros(N, dtype=torch.bool)
    rows[[2, 3, 6]], cols[5] = True, True
    assert torch.equal(nan, rows[:, None] | cols)
    # products below the normal range: a step there is 2^-149, for the scales' product and the result
    want, off = ref.linear(x, w)
    assert want[8].nan_to_num(0.0).abs().max() < 1e38
    diff = (got.cpu().double() - want).abs()
    sums = (want / (ref.rows_to_8_bits(x)[1][:, None] * ref.rows_to_8_bits(w)[1])).abs().nan_to_num(0.0, 0.0, 0.0)
    tol = off + want.abs() * 2.0**-24 + 2.0**-149 * (1 + sums)
    ok = (diff <= tol) | nan
    assert ok.all(), (~ok).nonzero()[:5]


def test_halves_are_decided_by_the_quotient(gpu):
    """Every quotient within a few steps of a half, for scales that are no powers of two:
    the integers are those of the fp32 quotient."""
    scales = torch.tensor([0.013, 0.7, 1.0, 3.3, 1e-3, 977.0, 0.3333333, 1e-30])
    halves = torch.arange(-126, 126).float() + 0.5
    x = torch.zeros(len(scales) * 9, 256)
    for i, s in enumerate(scales):
        for k in range(9):
            near = (halves.double() * s.double()).float()
            for _ in range(abs(k - 4)):
                near = torch.nextafter(near, torch.full_like(near, torch.inf if k > 4 else -torch.inf))
            x[9 * i + k, :252] = near
            x[9 * i + k, 255] = s * 127
    for M in (len(x), 8):
        w = torch.eye(256)
        y = linear_int8(x[:M].to(gpu), pack_linear_int8(w.to(gpu)))
        q, s = ref.rows_to_8_bits(x[:M])
        got = (y.cpu().double() / s[:, None]).round()
        assert torch.equal(got, q)


def test_largest_sums(gpu):
    """127 * 127 * 131,072 is within 32 bits, of either sign."""
    x = torch.ones((3, 131072), dtype=BF16)
    x[1] = -1.0
    w = torch.ones((5, 131072), dtype=BF16)
    y = linear_int8(x.to(gpu), pack_linear_int8(w.to(gpu)), dtype=F32)
    _assert_close(y, x, w)


def test_offsets_past_32_bits(gpu):
    """Inputs, words and outputs of more than 4 GiB."""
    for M, N, K in ((330_000, 16, 8000), (300_000, 4096, 64)):
        x = torch.zeros((M, K), dtype=BF16, device=gpu)
        w = torch.randn((N, K), generator=torch.Generator().manual_seed(0)).bfloat16()
        some = torch.tensor([0, 1, 15, 16, 12345, M // 2, M - 17, M - 2, M - 1])
        g = torch.Generator().manual_seed(1)
        rows = torch.randn((len(some), K), generator=g).bfloat16()
        x[some.to(gpu)] = rows.to(gpu)
        y = linear_int8(x, pack_linear_int8(w.to(gpu)), dtype=F32)
        assert y.numel() * 4 > 2**32 or x.numel() * 2 > 2**32
        _assert_close(y[some.to(gpu)], rows, w)
        assert int((y != 0).any(1).sum()) == len(some)
        del x, y


def test_rows_do_not_depend_on_the_batch(gpu):
    x, w = _data(700, 300, 200, 9)
    w8 = pack_linear_int8(w.to(gpu))
    x = x.to(gpu)
    whole = linear_int8(x, w8)
    for a, e in ((0, 1), (5, 9), (0, 16), (100, 163), (3, 68), (0, 257), (200, 700)):
        assert torch.equal(linear_int8(x[a:e], w8), whole[a:e]), (a, e)


@pytest.mark.parametrize("M", [4, 100, 600])
def test_captured_call_takes_other_inputs(gpu, M):
    K, N = 320, 272
    x, w = _data(M, N, K, 1)
    xs = [x] + [_data(M, N, K, s)[0] for s in (2, 3)]
    w8, bias = pack_linear_int8(w.to(gpu)), torch.randn(N).to(gpu)
    static, out = x.to(gpu), torch.empty((M, N), dtype=BF16, device=gpu)
    ws = torch.empty(linear_int8_workspace_bytes(M, N, K), dtype=torch.uint8, device=gpu)
    linear_int8(static, w8, bias, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        linear_int8(static, w8, bias, out=out, workspace=ws)
    for other in xs + xs:
        static.copy_(other)
        graph.replay()
        eager = linear_int8(other.to(gpu), w8, bias)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_on_a_stream_of_its_own(gpu):
    x, w = _data(200, 300, 200, 4)
    w8, xd = pack_linear_int8(w.to(gpu)), x.to(gpu)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:  # two calls at once, a workspace each
        with torch.cuda.stream(s):
            outs.append(linear_int8(xd, w8))
    torch.cuda.synchronize()
    for y in outs:
        _assert_close(y, x, w)
