"""Outputs that lie on what other workgroups still read are refused on the host; no pointer is
read and nothing is launched."""
from __future__ import annotations

import pytest

from spikeinfer_amd import _lib

P = 1 << 20
M, N, K = 5, 48, 64


def _linear(bias, y, bias_dtype=2, y_dtype=2, y_stride=N, rows=M, ws_bytes=0):
    """With a workspace that is too small: refused behind the checks of the tensors, if not by them."""
    lib = _lib.load()
    rc = lib.spk_linear_int8(1 << 40, 2, K, P, P, bias, bias_dtype, y, y_dtype, y_stride, rows, N, K, P, ws_bytes, None)
    return rc, lib.spk_last_error()


@pytest.mark.parametrize("case", [
    dict(bias=P, y=P),                                        # the first row of several
    dict(bias=P + 2 * 2 * N, y=P),                            # another row
    dict(bias=P + 2 * (M * N - 1), y=P),                      # the last element
    dict(bias=P - 2 * (N - 1), y=P),                          # from before the first
    dict(bias=P, y=P, rows=1, y_dtype=0),                     # one row, but of another type
    dict(bias=P + 2, y=P, rows=1),                            # one row, beside itself
    dict(bias=P + 2 * 60, y=P, y_stride=100),                 # over the end of a row's distance
])
def test_the_result_on_its_bias(case):
    rc, why = _linear(**case)
    assert rc == _lib.SPK_EINVAL and b"y lies on bias" in why


@pytest.mark.parametrize("case", [
    dict(bias=None, y=P),
    dict(bias=P, y=P, rows=1),                                # in place: a lane reads what it writes
    dict(bias=P + 2 * M * N, y=P),
    dict(bias=P - 2 * N, y=P),
    dict(bias=P + 2 * N, y=P, y_stride=2 * N),                # between two rows
])
def test_a_bias_beside_the_result(case):
    rc, why = _linear(**case)
    assert rc == _lib.SPK_EINVAL and b"workspace" in why


@pytest.mark.parametrize("shift", [1, 9, -1, -9])
def test_targets_on_other_rows_tokens(shift):
    lib = _lib.load()
    rows = 10

    def verify(out):
        rc = lib.spk_verify_tree(P, 1 << 30, 1 << 31, 100, 1 << 32, 100, 1 << 33, 1 << 34, rows, 2, 8, 100, 0, out, P, 0, None)
        return rc, lib.spk_last_error()

    rc, why = verify(P + 8 * shift)
    assert rc == _lib.SPK_EINVAL and b"targets lie on" in why
    for beside in (P, P + 8 * rows, P - 8 * rows):
        rc, why = verify(beside)
        assert rc == _lib.SPK_EINVAL and b"workspace" in why
