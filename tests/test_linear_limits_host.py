"""Which sizes the matrix operators take (no GPU: the C entry points' workspace sizes, which refuse what the calls refuse)."""
import ctypes as C

import pytest


LONG = (1 << 30) - 64  # the longest side of a product of tiles


def fwd(rows, k, n, dt=0):
    from cgan3d_amd import _lib as L
    a = L.LinearArgs(rows=rows, k=k, n=n, dtype=dt, x=64, ldx=k, w=64, ldw=k, y=64, ldy=n)
    return L.load().cgan3d_linear_fwd_ws_bytes(C.byref(a))


def bwd(rows, k, n, dt=0, dx=64, dw=64, dbias=64):
    from cgan3d_amd import _lib as L
    a = L.LinearArgs(rows=rows, k=k, n=n, dtype=dt, x=64, ldx=k, w=64, ldw=k, dy=64, lddy=n, dx=dx, lddx=k, dw=dw,
                     dbias=dbias)
    return L.load().cgan3d_linear_bwd_ws_bytes(C.byref(a))


@pytest.mark.parametrize("dt", [0, 1, 2])
@pytest.mark.parametrize("rows,k,n", [(1, 4_000_000, 8), (8, 8, 4_000_000), (40, 4_096_000, 8), (40, 8, 4_096_000), (1, LONG, 4),
                                      (2, 4, LONG), (3, 1, LONG), (1 << 28, 1, 65), (1 << 40, 64, 64), (1 << 24, 100, 100)])
def test_long_sides_are_taken(rows, k, n, dt):
    """One long side makes no large product: a flattened 160^3 volume as inputs or outputs, a billion rows."""
    assert fwd(rows, k, n, dt) >= 0
    assert bwd(rows, k, n, dt) >= 0


@pytest.mark.parametrize("dt", [0, 1, 2])
def test_what_no_grid_holds_is_refused(dt):
    from cgan3d_amd import _lib as L
    for rows, k, n in (((1 << 30) + 1, 8, 65), (1 << 30, 8, 1 << 13), (1 << 20, 8, 1 << 26), (1 << 41, 8, 8)):
        assert fwd(rows, k, n, dt) == -1, (rows, k, n)
        assert b"too" in L.load().cgan3d_get_last_error()
    assert fwd(1, 1 << 30, 4, dt) >= 0 and fwd(1, 4, 1 << 30, dt) >= 0
    assert bwd(8, LONG, 1 << 10, dt) == -1  # dw of 2^40 values
    assert bwd(8, LONG, 1 << 10, dt, dw=None) >= 0
    assert bwd((1 << 30) + 1, 8, 65, dt) == -1
    assert bwd((1 << 30) + 1, 8, 65, dt, dx=None, dw=None) >= 0  # column sums alone


def test_coefficients_beside_very_long_matrices():
    """Coefficients that take the f32 products: a matrix that their grid does not hold is refused, not left to HIP."""
    from cgan3d_amd import _lib as L
    lib, big = L.load(), 1 << 30
    wild = (C.c_float * 3)(70.0, 0.0, -61.0)
    m = (L.OrthoMat * 1)(L.OrthoMat(64, 64, big, big, 1, big))
    assert lib.cgan3d_orthogonalize(m, 1, L.DT_F32, 5, wild, 1e-7, 256, 1 << 62, None) == 22
    assert b"too large" in lib.cgan3d_get_last_error()
    s = (L.MuonSeg * 1)(L.MuonSeg(0, big, 1, 1.0))
    assert lib.cgan3d_muon_step(64, 64, 64, 64, s, 1, 64, 5, wild, 1e-7, 256, 1 << 62, None) == 22
    assert b"too large" in lib.cgan3d_get_last_error()
