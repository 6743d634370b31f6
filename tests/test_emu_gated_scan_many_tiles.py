"""The gated scan's blocks of 256 threads on the CPU emulator: the library takes them from 1024 tiles on."""
import ctypes

import numpy as np
import pytest

import block_reference as ref
from test_emu_block import Matrix, Shape, ci, emu, floats, operand, run_scan, scan_case, shape_of, workspace_for  # noqa: F401


def takes_256(emu, s, back):
    emu.emu_scan_threads.argtypes = [ctypes.POINTER(Shape), ci]
    return emu.emu_scan_threads(ctypes.byref(s), back) == 256


@pytest.mark.parametrize("back", [False, True])
def test_blocks_of_256_threads(emu, back):
    """Two strips of channels, the second of 5 (rows beginning anywhere); sequences that begin and end inside tiles, at their ends, and over
    more than 64 tiles; rows in front of, between and behind sequences."""
    rows, channels = (34000, 69) if back else (66500, 69)
    offsets = [3, 3, 128, 256, 257, rows // 2, rows - 200, rows - 7]
    rng = np.random.default_rng(5)
    x, g, h0 = scan_case(rng, "f32", "sigmoid", offsets, rows, channels)
    s, keep = shape_of("f32", "sigmoid", rows, channels, offsets, 32)
    assert takes_256(emu, s, back)
    mx, mg, f0 = Matrix(x, "f32"), Matrix(g, "f32", channels + 3), floats(h0)
    if not back:
        mh, last = Matrix(np.full(x.shape, 5.0), "f32"), floats(np.full(h0.shape, 9.0))
        assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0, emu.emu_last_error()
        h, want, e, el = ref.scan("sigmoid", x, g, offsets, h0)
        ref.check(mh.get(), np.where(np.isnan(h), 5.0, h), e, "f32", "h")
        ref.check(last.reshape(h0.shape), want, el, "f32", "h_last")
        return
    hs, dh, dl = x[::-1].copy(), x * 0.5, h0[::-1].copy()
    m = {k: Matrix(v, "f32") for k, v in dict(h=hs, dh=dh, dx=np.full(x.shape, 5.0), dg=np.full(x.shape, 5.0)).items()}
    fl, d0 = floats(dl), floats(np.full(h0.shape, 9.0))
    call = lambda ws, need: emu.emu_gated_scan_backward(ctypes.byref(s), *operand(m["dh"]), *operand(mx), *operand(mg), *operand(m["h"]), f0.ctypes.data, fl.ctypes.data, *operand(m["dx"]), *operand(m["dg"]), d0.ctypes.data,
                                                        ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0, emu.emu_last_error()
    (dx, dg, dh0), (ex, eg, e0) = ref.scan_backward("sigmoid", x, g, hs, dh, offsets, h0, dl)
    ref.check(m["dx"].get(), np.where(np.isnan(dx), 5.0, dx), ex, "f32", "dx")
    ref.check(m["dg"].get(), np.where(np.isnan(dg), 5.0, dg), eg, "f32", "dg")
    ref.check(d0.reshape(h0.shape), dh0, e0, "f32", "dh0")
