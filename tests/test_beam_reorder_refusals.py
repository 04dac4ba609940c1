"""Reordering refuses states that hold the parents it goes by (no GPU needed)."""
import ctypes

import pytest

import pesti_beam as pb
import pesti_sampler as ps

P, Q = 1 << 20, 1 << 24  # addresses that are never used: every call below is refused first, or has no device


def _call(rows, parent, G=2, W=4):
    lib = ps.load_library()
    arr = (pb._RowsC * len(rows))(*rows)
    rc = lib.pesti_beam_reorder(ctypes.addressof(arr), len(rows), parent, G, W, None)
    return rc, lib.pesti_last_error().decode()


def _rows(src, dst, stride=64, nbytes=64):
    return pb._RowsC(src, dst, stride, stride, 0, 0, 1, nbytes)


# eight rows of 64 bytes: [dst, dst + 512), parents of 32 bytes
@pytest.mark.parametrize("rows,parent", [
    ([_rows(P, P, 4, 4)], P),                # the parents themselves, in place
    ([_rows(Q, P, 4, 4)], P),
    ([_rows(P, P)], P + 508), ([_rows(P, P)], P - 28), ([_rows(P, P)], P + 64),
    ([_rows(Q, Q), _rows(4 * Q, P)], P + 128),
])
def test_parents_in_a_state(rows, parent):
    rc, msg = _call(rows, parent)
    assert rc == ps.PESTI_E_INVALID_ARG and "parents overlap" in msg


@pytest.mark.parametrize("rows,G,W", [([_rows(P, P)], 1 << 61, 1), ([_rows(P, P)], 1 << 56, 64)])
def test_too_many_parents(rows, G, W):
    rc, msg = _call(rows, Q, G, W)
    assert rc == ps.PESTI_E_INVALID_ARG and "too large" in msg
