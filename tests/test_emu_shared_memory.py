"""Outputs that share memory with other operands: in the place of an input where that is allowed, side by side in one matrix, and refused
everywhere else, on the CPU emulator."""
import ctypes

import numpy as np
import pytest

import block_reference as ref
from test_emu_block import NULL, GemmShape, Matrix, NormShape, aligned, emu, floats, gemm_emu, norm_emu, operand, run_scan, scan_case, shape_of, sz, vector, workspace_for  # noqa: F401

BIG = sz(1 << 40)


@pytest.fixture(scope="module")
def memory():
    buf = aligned(1 << 16, np.uint8, 0)
    return buf, buf.ctypes.data, buf.ctypes.data // 256 * 256 + 32768


def scan_shape(rows=4, channels=8):
    return shape_of("f16", "sigmoid", rows, channels, None, 32, 1)[0]


def test_gated_scan(emu, memory):
    keep, p, ws = memory
    err = lambda: emu.emu_last_error().decode()
    s = scan_shape()
    fwd = lambda x=(p, 8), g=(p + 256, 8), h=(p + 512, 8), h0=None, last=None: emu.emu_gated_scan(ctypes.byref(s), *x, *g, *h, h0, last, ws, ctypes.byref(BIG))
    assert fwd() == 0 and fwd(h=(p, 8)) == 0 and fwd(h=(p + 256, 8)) == 0
    assert fwd(h=(p, 16)) == 1 and "d_h shares memory with d_x" in err()  # another stride
    assert fwd(h=(p + 16, 8)) == 1 and fwd(h=(p - 16 + 64, 8)) == 1 and fwd(h=(p + 240, 8)) == 1
    assert fwd(x=(p, 24), g=(p + 16, 24), h=(p + 32, 24)) == 0  # thirds of one matrix
    assert fwd(x=(p + 32, 24), g=(p, 24), h=(p + 16, 24)) == 0
    assert fwd(x=(p, 20), g=(p + 16, 20), h=(p + 32, 20)) == 1  # the last one runs into the next row
    assert fwd(h0=p + 1024, last=p + 1024) == 0
    assert fwd(h0=p + 1024, last=p + 1040) == 1 and "d_h_last shares memory with d_h0" in err()
    assert fwd(last=p + 528) == 1 and fwd(h0=p + 512) == 1 and fwd(last=p) == 1
    back = lambda dh=(p, 8), x=(p + 256, 8), g=(p + 512, 8), h=(p + 768, 8), h0=None, dl=None, dx=(p + 1024, 8), dg=(p + 1280, 8), d0=None: emu.emu_gated_scan_backward(
        ctypes.byref(s), *dh, *x, *g, *h, h0, dl, *dx, *dg, d0, ws, ctypes.byref(BIG))
    assert back() == 0 and back(dx=(p, 8), dg=(p + 512, 8)) == 0 and back(dx=(p + 256, 8), dg=(p, 8)) == 0
    assert back(dx=(p + 768 + 16, 8)) == 1 and "d_h" in err()
    assert back(dx=(p, 16)) == 1 and back(dg=(p + 1024 + 32, 8)) == 1 and "d_dg" in err()
    assert back(h0=p + 2048, d0=p + 2048) == 0 and back(dl=p + 2048, d0=p + 2048) == 0
    assert back(h0=p + 2048, d0=p + 2064) == 1 and back(d0=p + 768) == 1
    step = lambda x=(p, 8), g=(p + 256, 8), h=(p + 512, 8), state=p + 1024, new=p + 1024, slots=p + 2048: emu.emu_gated_scan_step(0, 2, 8, 4, *x, *g, *h, state, new, 4, slots, 0)
    assert step() == 0 and step(h=(p, 8)) == 0 and step(new=p + 3328) == 0
    assert step(new=p + 1040) == 1 and step(h=(p + 1024, 8)) == 1 and step(h=(p + 2048, 8)) == 1 and step(h=(p, 9)) == 1 and step(new=p) == 1


def test_fused_norm(emu, memory):
    emu = norm_emu(emu)
    keep, p, ws = memory
    err = lambda: emu.emu_last_error().decode()
    shape = NormShape(0, 0, 0, 0, 4, 8, 1e-6, 1.0)
    fwd = lambda x=(p, 8), r=(p + 256, 8), gate=NULL, w=None, out=(p + 512, 8), z=(p + 768, 8): emu.emu_fused_norm(ctypes.byref(shape), *x, *r, *gate, w, None, None, *out, *z)
    assert fwd() == 0 and fwd(out=(p, 8), z=(p + 256, 8)) == 0 and fwd(out=(p + 256, 8), z=(p, 8)) == 0
    assert fwd(x=(p, 16), out=(p + 16, 16)) == 0
    assert fwd(out=(p, 16)) == 1 and "d_out shares memory with d_x" in err()
    assert fwd(out=(p + 32, 8)) == 1 and fwd(z=(p + 512 + 32, 8)) == 1 and fwd(w=p + 512) == 1 and fwd(w=p + 768) == 1
    back = lambda dout=(p, 8), z=(p + 256, 8), gate=NULL, x=NULL, ds=NULL, w=None, dx=(p + 512, 8), dr=NULL, dw=None, db=None: emu.emu_fused_norm_backward(
        ctypes.byref(shape), *dout, *z, *gate, w, None, None, *x, *ds, *dx, *NULL, *dr, dw, db, None, ws, ctypes.byref(BIG))
    assert back() == 0 and back(dx=(p, 8)) == 0 and back(dx=(p, 8), dr=(p + 256, 8)) == 0
    assert back(dx=(p + 32, 8)) == 1 and back(dr=(p + 528, 8)) == 1 and "d_dx shares memory with d_dresidual" in err()
    assert back(dw=p + 1024, db=p + 1024) == 1 and "d_dweight shares memory with d_dbias" in err()
    assert back(dw=p + 1024, db=p + 1056) == 0 and back(dw=p) == 1 and back(w=p + 512) == 1


def test_fused_product(emu, memory):
    emu = gemm_emu(emu)
    keep, p, ws = memory
    err = lambda: emu.emu_last_error().decode()
    fwd = lambda A=(p, 8), B=(p + 256, 8), bias=None, C=(p + 512, 8), D=(p + 768, 8), Z=NULL, beta=1.0: emu.emu_fused_gemm(ctypes.byref(GemmShape(0, 0, 4, 8, 8, beta)), *A, *B, bias, *C, *D, *Z, ws, ctypes.byref(BIG))
    assert fwd() == 0 and fwd(D=(p + 512, 8)) == 0 and fwd(D=(p + 520, 8), beta=0.0) == 0
    assert fwd(A=(p + 4096, 16), D=(p + 4112, 16)) == 0
    assert fwd(D=(p + 512, 16)) == 1 and "d_D shares memory with d_C" in err()
    assert fwd(D=(p + 32, 8)) == 1 and fwd(D=(p + 256 + 64, 8)) == 1 and fwd(Z=(p + 768 + 16, 8)) == 1 and fwd(bias=p + 768) == 1 and fwd(Z=(p + 528, 8)) == 1
    back = lambda dD=(p, 8), A=(p + 256, 8), B=(p + 512, 8), dA=(p + 768, 8), dB=(p + 1024, 8), db=None: emu.emu_fused_gemm_backward(ctypes.byref(GemmShape(0, 0, 4, 8, 8, 0.0)), *dD, *A, *B, *NULL, *dA, *dB, db, ws,
                                                                                                                                   ctypes.byref(BIG))
    assert back() == 0 and back(db=p + 2048) == 0
    assert back(dA=(p + 16, 8)) == 1 and back(dB=(p + 512 + 16, 8)) == 1 and back(dB=(p + 784, 8)) == 1 and back(db=p + 768) == 1 and "d_dA shares memory with d_dbias" in err()


@pytest.mark.parametrize("gate", ["sigmoid", "log"])
def test_scan_gradients_in_the_place_of_inputs(emu, gate):
    rng = np.random.default_rng(2)
    rows, channels, offsets = 900, 20, [0, 300, 300, 900]
    x, g, h0 = scan_case(rng, "f32", gate, offsets, rows, channels)
    hs, dh, dl = x[::-1].copy(), x * 0.5, h0 * 2
    s, keep = shape_of("f32", gate, rows, channels, offsets)
    (dx, dg, dh0), (ex, eg, e0) = ref.scan_backward(gate, x, g, hs, dh, offsets, h0, dl)
    for places in (("dh", "g"), ("x", "dh"), ("g", "x")):
        m = {k: Matrix(v, "f32", channels + 4) for k, v in dict(x=x, g=g, h=hs, dh=dh).items()}
        f0, fl = floats(h0), floats(dl)
        od, og = (m[k] for k in places)
        state = f0 if places[0] == "dh" else fl
        call = lambda ws, need: emu.emu_gated_scan_backward(ctypes.byref(s), *operand(m["dh"]), *operand(m["x"]), *operand(m["g"]), *operand(m["h"]), f0.ctypes.data, fl.ctypes.data, *operand(od), *operand(og),
                                                            state.ctypes.data, ws, need)
        kept, ws, have = workspace_for(call)
        assert call(ws, ctypes.byref(have)) == 0, emu.emu_last_error()
        ref.check(od.get(), dx, ex, "f32", "dx")
        ref.check(og.get(), dg, eg, "f32", "dg")
        ref.check(state.reshape(h0.shape), dh0, e0, "f32", "dh0")
    m = {k: Matrix(v, "f32") for k, v in dict(x=x, g=g).items()}
    f0 = floats(h0)
    assert run_scan(emu, s, m["x"], m["g"], m["g"], f0.ctypes.data, f0.ctypes.data) == 0  # h over g, h_last over h0
    h, last, e, el = ref.scan(gate, x, g, offsets, h0)
    ref.check(m["g"].get(), h, e, "f32", "h")
    ref.check(f0.reshape(h0.shape), last, el, "f32", "h_last")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [24, 1030, 8200])
@pytest.mark.parametrize("order", ["add_norm", "norm_add"])
def test_norm_gradients_in_the_place_of_inputs(emu, dtype, dim, order):
    emu = norm_emu(emu)
    rng = np.random.default_rng(dim)
    rows, add = 3, order == "add_norm"
    f = lambda v: ref.to_f64(ref.to_bits(v, dtype), dtype)
    mat = lambda: f(rng.standard_normal((rows, dim)))
    v = dict(dout=mat(), z=mat(), gate=mat(), x=mat(), stream=mat())
    w, cs = f(rng.standard_normal(dim)), f(rng.standard_normal(dim))
    vw, vc = vector(w, dtype), vector(cs, dtype)
    want, err = ref.norm_backward("layer", order, "silu", v["dout"], v["z"], v["gate"], w, np.zeros(dim), cs, 1e-5, v["x"], v["stream"] if add else None)
    shape = NormShape({"bf16": 1, "f32": 2}[dtype], 1, 0 if add else 1, 3, rows, dim, float(np.float32(1e-5)), 1.0)
    for places in (("dout", "gate", "z"), ("z", "dout", "x"), ("gate", "z", "stream")):
        m = {k: Matrix(a, dtype) for k, a in v.items()}
        dw, dc = floats(np.zeros(dim)), floats(np.zeros(dim))
        odx, odg, odr = (m[k] for k in places)
        call = lambda ws, need: emu.emu_fused_norm_backward(ctypes.byref(shape), *operand(m["dout"]), *operand(m["z"]), *operand(m["gate"]), vw.ctypes.data, None, vc.ctypes.data, *(operand(m["x"]) if add else NULL),
                                                            *(operand(m["stream"]) if add else NULL), *operand(odx), *operand(odg), *(operand(odr) if add else NULL), dw.ctypes.data, None, dc.ctypes.data, ws, need)
        kept, ws, have = workspace_for(call)
        assert call(ws, ctypes.byref(have)) == 0, emu.emu_last_error()
        ref.check(odx.get(), want["dx"], err["dx"], dtype, "dx")
        ref.check(odg.get(), want["dgate"], err["dgate"], dtype, "dgate")
        if add:
            ref.check(odr.get(), want["dresidual"], err["dresidual"], dtype, "dresidual")
        ref.check(dw, want["dweight"], err["dweight"], "f32", "dweight")
        ref.check(dc, want["dscale"], err["dscale"], "f32", "dscale")
