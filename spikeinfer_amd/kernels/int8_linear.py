"""Linear layers in 8-bit integers, with a scale for every token and every output channel.

    w8 = pack_linear_int8(w)            # once per weight: [N, K] of any float type
    y = linear_int8(x, w8, bias)        # x [..., K], y [..., N]

A row of x (or of w) becomes ``q = rint(x / s)`` with ``s = max |x| / 127``, both quotients
in single precision; the integer product is exact, and its scales and the bias are applied
in fp32.  From one row (one token) to prompts of thousands the call is the same.  The
reference's weights are bf16 throughout; this has no counterpart there.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from .. import _lib

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


@dataclass(frozen=True)
class Int8Weight:
    """A weight ``[out_features, in_features]`` as :func:`linear_int8` reads it: the integers in
    the matrix instruction's order, and the output channels' scales (padded to 64)."""

    words: torch.Tensor
    scales: torch.Tensor
    out_features: int
    in_features: int

    @property
    def nbytes(self) -> int:
        return self.words.numel() + 4 * self.out_features


def pack_linear_int8(w: torch.Tensor) -> Int8Weight:
    """Quantises the rows of ``w [N, K]`` (fp32, fp16 or bf16, channels contiguous) and lays
    them out for :func:`linear_int8`; done once per weight."""
    dev = _lib.require_gpu(w)
    if w.ndim != 2 or w.dtype not in _FLOATS or 0 in w.shape:
        raise ValueError(f"w must be a float [N, K] tensor, got {w.dtype} {tuple(w.shape)}")
    if w.stride(1) != 1:
        w = w.contiguous()
    N, K = w.shape
    words = torch.empty(int(_lib.load().spk_linear_int8_packed_bytes(N, K)), dtype=torch.uint8, device=dev)
    scales = torch.empty(-(-N // 64) * 64, dtype=torch.float32, device=dev)
    _lib.check(_lib.launch("spk_linear_int8_pack", dev, w.data_ptr(), _lib.dtype_code(w.dtype), w.stride(0), N, K,
                           words.data_ptr(), scales.data_ptr()), "pack_linear_int8")
    return Int8Weight(words, scales, N, K)


@functools.lru_cache(maxsize=1024)
def linear_int8_workspace_bytes(rows: int, out_features: int, in_features: int) -> int:
    """Scratch bytes :func:`linear_int8` needs for this shape."""
    return int(_lib.load().spk_linear_int8_workspace_bytes(rows, out_features, in_features))


def linear_int8(x: torch.Tensor, w: Int8Weight, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
                dtype: torch.dtype | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W^T (+ bias)`` with x's rows and the weight in 8-bit integers.

    Args:
        x: ``[..., K]`` fp32, fp16 or bf16.
        w: the weight, from :func:`pack_linear_int8`.
        bias: optional ``[N]`` of any of these types.
        out: optional ``[..., N]`` of any of these types, columns contiguous and rows one
            distance apart; must not overlap x, nor bias (but for one row in place). By default
            a new tensor of ``dtype`` (x's).
        workspace: optional ``uint8`` scratch of :func:`linear_int8_workspace_bytes`; calls that
            may run at once need one each.

    A row of x with an infinity or a NaN gives a row of NaN (a row of the weight such a
    column).  Rows do not depend on the rows around them.
    """
    native = _lib.native()
    if native is not None:  # the usual form of the arguments, checked and launched in C++
        done = native.linear_int8(x, w.words, w.scales, w.out_features, w.in_features, bias, out, dtype, workspace)
        if done is not None:
            return done
    dev = _lib.require_gpu(x, w.words, w.scales, bias, out, workspace)
    N, K = w.out_features, w.in_features
    if x.dtype not in _FLOATS or x.ndim < 1 or x.shape[-1] != K:
        raise ValueError(f"x must be a float [..., {K}] tensor, got {x.dtype} {tuple(x.shape)}")
    if bias is not None:
        if tuple(bias.shape) != (N,) or bias.dtype not in _FLOATS:
            raise ValueError(f"bias must be a float [{N}] tensor, got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    x2 = x.reshape(-1, K)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    M = x2.shape[0]
    shape = (*x.shape[:-1], N)
    if out is None:
        out = torch.empty(shape, dtype=dtype or x.dtype, device=dev)
    elif tuple(out.shape) != shape or dtype not in (None, out.dtype):
        raise ValueError(f"out must be {shape}{f' of {dtype}' if dtype else ''}, got {out.dtype} {tuple(out.shape)}")
    if out.dtype not in _FLOATS:
        raise ValueError(f"out must be of a float type, got {out.dtype}")
    try:
        y = out.view(-1, N)
    except RuntimeError:
        raise ValueError(f"out's rows must lie one distance apart, got strides {tuple(out.stride())}") from None
    if N > 1 and y.stride(1) != 1:
        raise ValueError(f"out's columns must be contiguous, got strides {tuple(out.stride())}")
    if M == 0:
        return out
    need = linear_int8_workspace_bytes(M, N, K)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
        raise ValueError(f"workspace must hold {need} contiguous bytes")
    _lib.check(
        _lib.launch(
            "spk_linear_int8", dev, x2.data_ptr(), _lib.dtype_code(x2.dtype), x2.stride(0), w.words.data_ptr(),
            w.scales.data_ptr(), _lib.ptr(bias), _lib.dtype_code(bias.dtype) if bias is not None else 0, y.data_ptr(),
            _lib.dtype_code(y.dtype), y.stride(0), M, N, K, workspace.data_ptr(),
            workspace.numel() * workspace.element_size()),
        "linear_int8",
    )
    return out
