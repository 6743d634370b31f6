"""Gates above 1 on the CPU emulator: products of gates that pass the range of fp32 while the states themselves are finite."""
import ctypes

import numpy as np
import pytest

import block_reference as ref
from test_emu_block import DTYPES, Matrix, emu, floats, operand, run_scan, shape_of, workspace_for  # noqa: F401


def scan_both(emu, dtype, gate, x, g, h0, offsets, hs=None, dh=None, dl=None):
    """Forward and gradient (if dh is given) against the definitions."""
    rows, channels = x.shape
    packed = len(offsets) > 2
    mx, mg, mh = Matrix(x, dtype), Matrix(g, dtype), Matrix(np.full(x.shape, 5.0), dtype)
    s, keep = shape_of(dtype, gate, rows, channels, offsets if packed else None, 32, None if packed else 1)
    f0, last = floats(h0), floats(np.full(h0.shape, 9.0))
    if dh is None:
        assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0
        h, want, e, el = ref.scan(gate, x, g, offsets, h0)
        ref.check(mh.get(), h, e, dtype, "h")
        ref.check(last.reshape(h0.shape), want, el, "f32", "h_last")
        return
    mhs, mdh, mdx, mdg = Matrix(hs, dtype), Matrix(dh, dtype), Matrix(x, dtype), Matrix(x, dtype)
    fl, d0 = floats(dl), floats(np.full(h0.shape, 9.0))
    call = lambda ws, need: emu.emu_gated_scan_backward(ctypes.byref(s), *operand(mdh), *operand(mx), *operand(mg), *operand(mhs), f0.ctypes.data, fl.ctypes.data, *operand(mdx), *operand(mdg), d0.ctypes.data, ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0
    (dx, dg, dh0), (ex, eg, e0) = ref.scan_backward(gate, x, g, hs, dh, offsets, h0, dl)
    ref.check(mdx.get(), dx, ex, dtype, "dx")
    ref.check(mdg.get(), dg, eg, dtype, "dg")
    ref.check(d0.reshape(h0.shape), dh0, e0, "f32", "dh0")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [200, 1000, 2600])
def test_a_state_of_zero_stays_zero_under_growing_gates(emu, dtype, rows):
    """x = 0 up to the last row, h0 = 0, a = e^0.5: h is 0 up to the last row and 1 there, whatever the product of the gates."""
    x, g, h0 = np.zeros((rows, 9)), np.full((rows, 9), 0.5), np.zeros((1, 9))
    x[-1] = 1.0
    scan_both(emu, dtype, "log", x, g, h0, [0, rows])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [200, 1000, 2600, 9000])
def test_the_gradient_of_zeros_under_growing_gates(emu, dtype, rows):
    """dh = 0 but in row 0, which comes last: dx is 0 everywhere else."""
    x, g, h0 = np.zeros((rows, 9)), np.ones((rows, 9)), np.zeros((1, 9))
    dh, hs = np.zeros(x.shape), np.ones(x.shape)
    dh[0] = 2.0
    scan_both(emu, dtype, "log", x, g, h0, [0, rows], hs, dh, np.zeros(h0.shape))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("start,grow", [(0, 700), (150, 900), (300, 2300)])
def test_ordinary_rows_around_growth_from_zero(emu, packed, start, grow):
    """Ordinary rows, a gate of 0 that leaves the state 0, growing gates over it, ordinary rows again: what the zero gate cut off does
    not come back, and what follows is as ever.  Some channels have ordinary gates all along."""
    rng = np.random.default_rng(grow)
    rows, channels = grow + 900, 12
    f = lambda v: ref.to_f64(ref.to_bits(v, "f32"), "f32")
    x, g = f(rng.standard_normal((rows, channels))), f(ref.sigmoid(rng.standard_normal((rows, channels)) * 1.5 + 2))
    h0 = f(rng.standard_normal((1, channels)))
    for c in range(0, channels, 2):
        x[start:grow, c], g[start:grow, c] = 0.0, 1.5
        if start:
            g[start, c] = 0.0
        else:
            h0[0, c] = 0.0
    offsets = [0, rows]
    if packed:
        offsets = [0, grow + 100, rows]
        h0 = np.concatenate([h0, f(rng.standard_normal((1, channels)))])
    scan_both(emu, "f32", "decay", x, g, h0, offsets)
    # the same in place order for the gradient: u[t] = a[t] (dh[t] + u[t+1])
    hs, dh, dl = x[::-1].copy(), x[::-1].copy(), np.zeros(h0.shape)
    scan_both(emu, "f32", "decay", x, g[::-1].copy(), h0, [0, rows] if not packed else [0, rows - grow - 100, rows], hs, dh, dl)


def test_growth_that_passes_the_range_shows(emu):
    """A state that does grow beyond fp32 is an infinity from there on in the definition, and no finite number in the result."""
    rows = 3000
    x, g, h0 = np.zeros((rows, 8)), np.full((rows, 8), 2.0), np.ones((1, 8))
    mx, mg, mh = Matrix(x, "f32"), Matrix(g, "f32"), Matrix(x, "f32")
    s, keep = shape_of("f32", "decay", rows, 8, None, 32, 1)
    f0, last = floats(h0), floats(h0)
    assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0
    got = mh.get()
    assert (got[:127] == 2.0 ** np.arange(1, 128)[:, None]).all() and not np.isfinite(got[127:]).any() and not np.isfinite(last[:8]).any()
