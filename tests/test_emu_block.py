"""The recurrent-block operators' kernel sources (gated scan, fused norm, fused product) run lane by lane on the CPU, as
tests/test_emu_kernels.py does for the others: every array ends at an inaccessible page, so an access out of bounds ends the
run.  References and bounds: tests/block_reference.py."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

import block_reference as ref
from test_emu_kernels import CLANG, EMU, HERE, aligned

DTYPES = {"f16": 0, "bf16": 1, "f32": 2}
GATES = {"decay": 0, "log": 1, "sigmoid": 2}
vp, sz, ci, cf = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_float


class Shape(ctypes.Structure):
    _fields_ = [("dtype", ci), ("gate", ci), ("channels", sz), ("num_rows", sz), ("num_sequences", sz), ("sequence_length", sz), ("d_offsets", vp), ("offset_bits", ci), ("zero_outside", ci)]


@pytest.fixture(scope="module")
def emu():
    if not os.path.exists(CLANG):
        pytest.skip("host clang++ (ROCm LLVM) not available")
    lib = os.path.join(EMU, "libtcu_emu_block.so")
    csrc = os.path.join(HERE, "..", "tcu_scope_amd", "csrc")
    srcs = [os.path.join(EMU, f) for f in ("emu_block_driver.cpp", "block_ops_emu.hpp", "wave_ops_emu.hpp")] + [os.path.join(csrc, f) for f in os.listdir(csrc) if f.endswith(".hpp")]
    srcs.append(os.path.join(HERE, "..", "include", "tcu_scope.h"))
    if not os.path.exists(lib) or any(os.path.getmtime(s) > os.path.getmtime(lib) for s in srcs):
        subprocess.check_call([CLANG, "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wno-psabi", "-I" + EMU, "-o", lib, os.path.join(EMU, "emu_block_driver.cpp")])
    L = ctypes.CDLL(lib)
    shape, psz = ctypes.POINTER(Shape), ctypes.POINTER(sz)
    L.emu_gated_scan.argtypes = [shape, vp, sz, vp, sz, vp, sz, vp, vp, vp, psz]
    L.emu_gated_scan_backward.argtypes = [shape, vp, sz, vp, sz, vp, sz, vp, sz, vp, vp, vp, sz, vp, sz, vp, vp, psz]
    L.emu_gated_scan_step.argtypes = [ci, ci, sz, sz, vp, sz, vp, sz, vp, sz, vp, vp, sz, vp, ci]
    L.emu_waits.argtypes = [ctypes.c_uint, ctypes.c_uint]
    L.emu_last_error.restype = ctypes.c_char_p
    return L


def storage(dtype):
    return np.float32 if dtype == "f32" else np.uint16


class Matrix:
    """rows x width elements of a guarded array, `stride` apart, `shift` elements behind its start; what lies between holds a marker."""

    def __init__(self, values, dtype, stride=None, shift=0):
        self.dtype, (self.rows, self.width), self.shift = dtype, values.shape, shift
        self.stride = stride or self.width
        n = shift + max(self.rows - 1, 0) * self.stride + self.width if self.rows else shift
        self.flat = aligned(max(n, 1), storage(dtype))
        self.flat[:] = ref.to_bits(np.full(self.flat.size, -77.0), dtype)
        self.put(values)

    def view(self):
        return np.lib.stride_tricks.as_strided(self.flat[self.shift:], (self.rows, self.width), (self.stride * self.flat.itemsize, self.flat.itemsize))

    def put(self, values):
        if self.rows:
            self.view()[...] = ref.to_bits(values, self.dtype)

    @property
    def ptr(self):
        return self.flat.ctypes.data + self.shift * self.flat.itemsize

    def get(self):
        return ref.to_f64(np.ascontiguousarray(self.view()), self.dtype) if self.rows else np.zeros((0, self.width))

    def untouched_between(self):
        mark = ref.to_bits(np.full(1, -77.0), self.dtype)[0]
        mask = np.ones(self.flat.size, bool)
        for r in range(self.rows):
            mask[self.shift + r * self.stride:self.shift + r * self.stride + self.width] = False
        return (self.flat[mask] == mark).all()


def floats(values):
    a = aligned(max(values.size, 1), np.float32)
    a[:values.size] = np.asarray(values, dtype=np.float32).reshape(-1)
    return a


def gates(rng, gate, shape):
    z = rng.standard_normal(shape)
    return {"sigmoid": z * 1.5 + 2, "log": -np.exp(z * 1.2 - 3), "decay": ref.sigmoid(z * 1.5 + 2) * np.where(rng.random(shape) < 0.2, -1, 1)}[gate]


def scan_case(rng, dtype, gate, offsets, rows, channels, stride=None, shift=0):
    f = lambda v: ref.to_f64(ref.to_bits(v, dtype), dtype)
    x, g = f(rng.standard_normal((rows, channels))), f(gates(rng, gate, (rows, channels)))
    h0 = rng.standard_normal((len(offsets) - 1, channels)).astype(np.float32).astype(np.float64)
    return x, g, h0


def shape_of(dtype, gate, rows, channels, offsets=None, bits=32, sequences=None, zero_outside=0):
    s = Shape(dtype=DTYPES[dtype], gate=GATES[gate], channels=channels, num_rows=rows, zero_outside=zero_outside)
    keep = None
    if offsets is not None:
        keep = aligned(len(offsets), np.int32 if bits == 32 else np.int64)
        keep[:] = offsets
        s.num_sequences, s.d_offsets, s.offset_bits = len(offsets) - 1, keep.ctypes.data, bits
    else:
        s.num_sequences, s.sequence_length = sequences, rows // sequences if sequences else 0
    return s, keep


def workspace_for(call):
    need = sz(0)
    assert call(None, ctypes.byref(need)) == 0
    # the emulator hands out 16-byte alignment at least; a workspace is 256-byte aligned
    ws = aligned(need.value + 256, np.uint8, 0xA5)
    off = -ws.ctypes.data % 256
    return ws, ws.ctypes.data + off, sz(need.value)


def run_scan(emu, s, x, g, h, h0, last):
    call = lambda ws, need: emu.emu_gated_scan(ctypes.byref(s), x.ptr, x.stride, g.ptr, g.stride, h.ptr, h.stride, h0, last, ws, need)
    keep, ws, have = workspace_for(call)
    return call(ws, ctypes.byref(have))


LAYOUTS = [
    # rows, channels, offsets or number of equal sequences, stride - channels, shift
    (1, 8, 1, 0, 0),
    (5, 1, 1, 0, 0),
    (6, 13, 3, 0, 0),
    (131, 24, 1, 8, 8),
    (300, 136, 2, 0, 0),
    (290, 20, 290, 0, 0),
    (1300, 16, 1, 0, 0),
    (400, 40, [0, 0, 1, 130, 130, 257, 399, 399], 0, 0),
    (257, 9, [3, 3, 100, 129, 240], 5, 3),
    (64, 8, [64, 64], 0, 0),
    (1200, 8, [0, 5, 1190], 0, 0),
]


@pytest.mark.parametrize("dtype,gate", [("f16", "sigmoid"), ("bf16", "log"), ("f32", "decay"), ("f32", "sigmoid"), ("f32", "log")])
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda v: f"{v[0]}x{v[1]}" + ("p" if isinstance(v[2], list) else f"s{v[2]}"))
def test_gated_scan_and_gradient(emu, dtype, gate, layout):
    rows, channels, seqs, gap, shift = layout
    rng = np.random.default_rng(rows * 31 + channels)
    packed = isinstance(seqs, list)
    offsets = seqs if packed else [j * (rows // seqs) for j in range(seqs + 1)]
    x, g, h0 = scan_case(rng, dtype, gate, offsets, rows, channels)
    mx, mg = Matrix(x, dtype, channels + gap, shift), Matrix(g, dtype, channels + 2 * gap, shift)
    mh = Matrix(np.full((rows, channels), 5.0), dtype, channels + gap, 0)
    s, keep = shape_of(dtype, gate, rows, channels, seqs if packed else None, 64 if channels % 2 else 32, None if packed else seqs)
    f0, last = floats(h0), floats(np.full(h0.shape, 9.0))
    assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0, emu.emu_last_error()
    h, want_last, e, elast = ref.scan(gate, x, g, offsets, h0)
    outside = np.isnan(h[:, 0])
    ref.check(mh.get()[~outside], h[~outside], e[~outside], dtype, "h")
    assert (mh.get()[outside] == 5.0).all() and mh.untouched_between() and mx.untouched_between()
    ref.check(last.reshape(h0.shape), want_last, elast, "f32", "h_last")
    # without states, outputs in the place of an input, zeros outside
    s.zero_outside = 1
    inplace = Matrix(x, dtype, channels + gap, 0)
    assert run_scan(emu, s, inplace, mg, inplace, None, None) == 0
    h, _, e, _ = ref.scan(gate, x, g, offsets, np.zeros(h0.shape))
    ref.check(inplace.get(), np.where(np.isnan(h), 0, h), e, dtype, "h in place")
    # the gradient, from states of any origin
    hs = ref.to_f64(ref.to_bits(rng.standard_normal((rows, channels)), dtype), dtype)
    dh = ref.to_f64(ref.to_bits(rng.standard_normal((rows, channels)), dtype), dtype)
    dlast = rng.standard_normal(h0.shape).astype(np.float32).astype(np.float64)
    mhs, mdh = Matrix(hs, dtype, channels + gap, shift), Matrix(dh, dtype)
    mdx, mdg = Matrix(np.full((rows, channels), 5.0), dtype), Matrix(np.full((rows, channels), 5.0), dtype, channels + gap)
    for with_states in (True, False):
        s.zero_outside = 0 if with_states else 1
        fl, d0 = floats(dlast), floats(np.full(h0.shape, 9.0))
        call = lambda ws, need: emu.emu_gated_scan_backward(ctypes.byref(s), mdh.ptr, mdh.stride, mx.ptr if gate == "sigmoid" else None, mx.stride, mg.ptr, mg.stride, mhs.ptr, mhs.stride, f0.ctypes.data if with_states else None,
                                                            fl.ctypes.data if with_states else None, mdx.ptr, mdx.stride, mdg.ptr, mdg.stride, d0.ctypes.data if with_states else None, ws, need)
        kept, ws, have = workspace_for(call)
        assert call(ws, ctypes.byref(have)) == 0, emu.emu_last_error()
        zero = np.zeros(h0.shape)
        (dx, dg, dh0), (ex, eg, e0) = ref.scan_backward(gate, x, g, hs, dh, offsets, h0 if with_states else zero, dlast if with_states else zero)
        fillv = 5.0 if with_states else 0.0
        ref.check(mdx.get(), np.where(np.isnan(dx), fillv, dx), ex, dtype, "dx")
        ref.check(mdg.get(), np.where(np.isnan(dg), fillv, dg), eg, dtype, "dg")
        if with_states:
            ref.check(d0.reshape(h0.shape), dh0, e0, "f32", "dh0")
    assert mdg.untouched_between()


def test_gradient_against_differences(emu):
    """dx, dg and dh0 against central differences of the 64-bit forward recurrence (step 1e-5: off by about 1e-9)."""
    rng = np.random.default_rng(3)
    offsets, rows, channels = [0, 3, 3, 7], 7, 4
    for gate in GATES:
        x, g, h0 = scan_case(rng, "f32", gate, offsets, rows, channels)
        dh = rng.standard_normal((rows, channels))
        dl = rng.standard_normal(h0.shape)
        loss = lambda x, g, h0: (lambda r: float((r[0] * dh).sum() + (r[1] * dl).sum()))(ref.scan(gate, x, g, offsets, h0))
        h = ref.scan(gate, x, g, offsets, h0)[0]
        (dx, dg, dh0), _ = ref.scan_backward(gate, x, g, h, dh, offsets, h0, dl)
        for k, (v, d) in enumerate(((x, dx), (g, dg), (h0, dh0))):
            for at in itertools.product(*(range(n) for n in v.shape)):
                lo, hi = v.copy(), v.copy()
                lo[at] -= 1e-5
                hi[at] += 1e-5
                args = lambda w: tuple(w if i == k else u for i, u in enumerate((x, g, h0)))
                assert abs((loss(*args(hi)) - loss(*args(lo))) / 2e-5 - d[at]) < 1e-7


def test_no_rows_and_empty_sequences(emu):
    h0 = np.arange(12, dtype=np.float64).reshape(3, 4)
    empty = Matrix(np.zeros((0, 4)), "f32")
    for seqs in (3, [0, 0, 0, 0]):
        s, keep = shape_of("f32", "log", 0, 4, seqs if isinstance(seqs, list) else None, 32, seqs)
        f0, last = floats(h0), floats(np.full(h0.shape, 9.0))
        assert run_scan(emu, s, empty, empty, empty, f0.ctypes.data, last.ctypes.data) == 0
        assert (last.reshape(3, 4) == h0).all()
        assert run_scan(emu, s, empty, empty, empty, None, last.ctypes.data) == 0
        assert (last == 0).all()
    s, keep = shape_of("f32", "log", 0, 4, [0], 32)
    assert run_scan(emu, s, empty, empty, empty, None, None) == 0


@pytest.mark.parametrize("zero_outside", [0, 1])
def test_rows_without_any_sequence(emu, zero_outside):
    ones = Matrix(np.ones((5, 12)), "f32")
    s, keep = shape_of("f32", "sigmoid", 5, 12, [0], 32, zero_outside=zero_outside)
    h, dx, dg = (Matrix(np.full((5, 12), 5.0), "f32") for _ in range(3))
    assert run_scan(emu, s, ones, ones, h, None, None) == 0
    call = lambda ws, need: emu.emu_gated_scan_backward(ctypes.byref(s), *(v for m in (ones, ones, ones, ones) for v in (m.ptr, m.stride)), None, None, dx.ptr, dx.stride, dg.ptr, dg.stride, None, ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0
    for m in (h, dx, dg):
        assert (m.get() == (0.0 if zero_outside else 5.0)).all()


def test_offsets_that_pass_the_rows(emu):
    """Only rows that exist count: a sequence that ends behind the last one stops there, one that begins there (or ends in front of the first) has none."""
    rng = np.random.default_rng(12)
    rows, channels, offsets = 20, 12, [-7, -3, 9, 26, 40]
    x, g, _ = scan_case(rng, "f32", "sigmoid", [0, rows], rows, channels)
    h0 = rng.standard_normal((4, channels)).astype(np.float32).astype(np.float64)
    s, keep = shape_of("f32", "sigmoid", rows, channels, offsets, 64)
    mx, mg, mh = Matrix(x, "f32"), Matrix(g, "f32"), Matrix(x, "f32")
    f0, last = floats(h0), floats(np.full(h0.shape, 9.0))
    assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0
    h, want, e, elast = ref.scan("sigmoid", x, g, [0, 0, 9, rows, rows], h0)
    ref.check(mh.get(), h, e, "f32", "h")
    ref.check(last.reshape(h0.shape), want, elast, "f32", "h_last")


def test_states_do_not_pass_between_sequences(emu):
    """An infinite or NaN state stays in its sequence: a sequence's beginning replaces what came before, it does not multiply it by 0."""
    rows, channels = 400, 8
    offsets = [0, 150, 400]
    rng = np.random.default_rng(5)
    for bad in (np.inf, np.nan):
        x, g, h0 = scan_case(rng, "f32", "decay", offsets, rows, channels)
        g = np.abs(g) + 0.01
        x[10] = bad
        mx, mg, mh = Matrix(x, "f32"), Matrix(g, "f32"), Matrix(np.zeros((rows, channels)), "f32")
        s, keep = shape_of("f32", "decay", rows, channels, offsets)
        f0, last = floats(h0), floats(h0)
        assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0
        got = mh.get()
        assert np.isfinite(got[:10]).all() and np.isfinite(got[150:]).all() and not np.isfinite(got[10:150]).any()


def test_gate_extremes(emu):
    """Gates at the ends of their range, and a NaN gate, which has to show."""
    g = np.array([[-np.inf, -200.0, -87.5, 0.0, 87.5, 200.0, np.inf, np.nan]])
    x, h0 = np.full(g.shape, 3.0), np.full(g.shape, 2.0)
    for dtype in DTYPES:
        mx, mg, mh = Matrix(x, dtype), Matrix(g, dtype), Matrix(x, dtype)
        s, keep = shape_of(dtype, "sigmoid", 1, 8, None, 32, 1)
        f0, last = floats(h0), floats(h0)
        assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0
        got = mh.get()[0]
        assert np.allclose(got[:7], [3, 3, 3, 2.5, 2, 2, 2], rtol=2.0 ** -8, atol=0) and np.isnan(got[7])
        gl = np.array([[-np.inf, -200.0, -1.0, 0.0, 1.0, 2.0, np.inf, np.nan]])
        mg = Matrix(gl, dtype)
        s, keep = shape_of(dtype, "log", 1, 8, None, 32, 1)
        assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0
        got = mh.get()[0]
        assert np.allclose(got[:6], [3, 3, 3 + 2 * np.exp(-1), 5, 3 + 2 * np.exp(1), 3 + 2 * np.exp(2)], rtol=2.0 ** -8) and got[6] == np.inf and np.isnan(got[7])


def test_waits_that_expire_leave_nan(emu):
    """A tile that publishes nothing (test switch) and a poll limit of 3: everything that depended on it is NaN up to the end of the sequence, nothing else is."""
    rows, channels = 2600, 8
    offsets = [0, 2000, 2600]
    rng = np.random.default_rng(9)
    x, g, h0 = scan_case(rng, "f16", "sigmoid", offsets, rows, channels)
    want, want_last, e, _ = ref.scan("sigmoid", x, g, offsets, h0)
    mx, mg, mh = Matrix(x, "f16"), Matrix(g, "f16"), Matrix(np.zeros((rows, channels)), "f16")
    s, keep = shape_of("f16", "sigmoid", rows, channels, offsets)
    f0, last = floats(h0), floats(h0)
    emu.emu_waits(3, 1 + 4)  # tile 4 is mute
    try:
        assert run_scan(emu, s, mx, mg, mh, f0.ctypes.data, last.ctypes.data) == 0
    finally:
        emu.emu_waits(1 << 20, 0)
    got, tile = mh.get(), 256  # places of a tile
    ok = np.r_[0:5 * tile, 2000:rows]
    ref.check(got[ok], want[ok], e[ok], "f16", "what did not wait")
    assert np.isnan(got[5 * tile:2000]).all() and np.isnan(last.reshape(2, channels)[0]).all() and np.isfinite(last.reshape(2, channels)[1]).all()


def test_states_handed_on_over_many_tiles(emu):
    """More than 64 tiles along one sequence (entries of one tile, of eight, and states), forwards and backwards; then a mute tile
    in the middle of a group, one that closes eight and one that closes 64: NaN behind it, and nothing else."""
    rows, channels = 9000, 8  # tiles of 128 places backwards
    offsets = [0, rows]
    rng = np.random.default_rng(11)
    x, g, h0 = scan_case(rng, "f32", "decay", offsets, rows, channels)
    g = np.clip(np.abs(g), 0.99, 0.9999).astype(np.float32).astype(np.float64)  # a state that lasts
    hs, dh = x[::-1].copy(), x * 0.5
    m = {k: Matrix(v, "f32") for k, v in dict(g=g, h=hs, dh=dh, dx=x, dg=x).items()}
    s, keep = shape_of("f32", "decay", rows, channels, None, 32, 1)
    f0, d0 = floats(h0), floats(h0)
    call = lambda ws, need: emu.emu_gated_scan_backward(ctypes.byref(s), *operand(m["dh"]), None, 0, *operand(m["g"]), *operand(m["h"]), f0.ctypes.data, None, *operand(m["dx"]), *operand(m["dg"]), d0.ctypes.data, ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0
    (dx, dg, dh0), (ex, eg, e0) = ref.scan_backward("decay", x, g, hs, dh, offsets, h0, np.zeros(h0.shape))
    ref.check(m["dx"].get(), dx, ex, "f32", "dx")
    ref.check(m["dg"].get(), dg, eg, "f32", "dg")
    ref.check(d0.reshape(h0.shape), dh0, e0, "f32", "dh0")
    for mute in (3, 15, 63):
        emu.emu_waits(2, mute + 1)
        try:
            assert call(ws, ctypes.byref(have)) == 0
        finally:
            emu.emu_waits(1 << 20, 0)
        first_bad = rows - (mute + 1) * 128  # places run backwards; the mute tile itself knows its carry
        got = m["dx"].get()
        ref.check(got[first_bad:], dx[first_bad:], ex[first_bad:], "f32", "what did not wait")
        assert np.isnan(got[:first_bad]).all() and np.isnan(d0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("gate", list(GATES))
@pytest.mark.parametrize("rows,channels,slots,gap", [(1, 8, None, 0), (3, 520, None, 8), (5, 13, [4, 0, 6, 1, 2], 3), (7, 16, [3, -1, 3, 9, 3, 1, -5], 0), (70, 8, "many", 0)])
def test_gated_scan_step(emu, dtype, gate, rows, channels, slots, gap):
    rng = np.random.default_rng(rows)
    x, g, _ = scan_case(rng, dtype, gate, [0], rows, channels)
    num_slots = 7 if slots != "many" else 5
    at = list(range(rows)) if slots is None else [int(v) for v in rng.integers(-1, 5, rows)] if slots == "many" else slots
    state = rng.standard_normal((num_slots, channels)).astype(np.float32).astype(np.float64)
    mx, mg, mh = Matrix(x, dtype, channels + gap), Matrix(g, dtype, channels + gap), Matrix(np.full((rows, channels), 5.0), dtype)
    ps = None
    if slots is not None:
        ps = aligned(rows, np.int32)
        ps[:] = at
    a, keep, c = ref.gate_terms(gate, g)
    c = np.broadcast_to(c, g.shape)
    want_state, err = state.copy(), np.zeros(state.shape)
    want_h, eh = np.full((rows, channels), 5.0), np.zeros((rows, channels))
    for i, j in enumerate(at):
        if 0 <= j < num_slots:
            m = np.abs(a[i] * want_state[j]) + np.abs(keep[i] * x[i])
            want_state[j] = a[i] * want_state[j] + keep[i] * x[i]
            err[j] = np.abs(a[i]) * err[j] + (c[i] + 4.0) * ref.EPS32 * m
            want_h[i], eh[i] = want_state[j], err[j]
    for inplace in (False, True):
        st = floats(state)
        new = st if inplace else floats(np.full(state.shape, 9.0))
        assert emu.emu_gated_scan_step(DTYPES[dtype], GATES[gate], channels, rows, mx.ptr, mx.stride, mg.ptr, mg.stride, mh.ptr, mh.stride, st.ctypes.data, new.ctypes.data, num_slots, ps.ctypes.data if ps is not None else None, 0) == 0
        ref.check(mh.get(), want_h, eh, dtype, "h")
        named = sorted({j for j in at if 0 <= j < num_slots})
        ref.check(new.reshape(state.shape)[named], want_state[named], err[named], "f32", "state")
        rest = [j for j in range(num_slots) if j not in named]
        assert (new.reshape(state.shape)[rest] == (state[rest].astype(np.float32) if inplace else 9.0)).all()


def test_gated_scan_refusals(emu):
    buf = aligned(4096, np.uint8, 0)
    p = buf.ctypes.data
    err = lambda: emu.emu_last_error().decode()
    need = sz(0)
    big = sz(1 << 40)

    def scan(s, x=p, xs=8, g=p, gs=8, h=p, hs=8, h0=None, last=None, ws=p // 256 * 256 + 256, have=big):
        return emu.emu_gated_scan(ctypes.byref(s) if s else None, x, xs, g, gs, h, hs, h0, last, ws, ctypes.byref(have) if have else None)

    ok = lambda **k: Shape(**{**dict(dtype=0, gate=2, channels=8, num_rows=0, num_sequences=1, sequence_length=0), **k})
    assert scan(None) == 1 and "null shape" in err()
    assert scan(ok(dtype=3)) == 1 and "dtype" in err()
    assert scan(ok(gate=3)) == 1 and "gate" in err()
    assert scan(ok(channels=0)) == 1 and "channels" in err()
    assert scan(ok(num_rows=5)) == 1 and "num_rows" in err()
    assert scan(ok(num_sequences=1 << 20, sequence_length=1 << 20, num_rows=1 << 40)) == 2 and "rows" in err()
    assert scan(ok(d_offsets=p, offset_bits=16)) == 1 and "offset_bits" in err()
    assert scan(ok(d_offsets=p + 2, offset_bits=32)) == 1 and "aligned" in err()
    assert scan(ok(), have=None) == 1 and "workspace_bytes" in err()
    two = ok(num_rows=2, sequence_length=2)
    assert emu.emu_gated_scan(ctypes.byref(two), None, 8, None, 8, None, 8, None, None, None, ctypes.byref(need)) == 0 and need.value == 256
    assert scan(two, have=sz(255)) == 4 and "workspace" in err()
    assert scan(two, ws=p // 256 * 256 + 264) == 1 and "256-byte" in err()
    assert scan(two, x=None) == 1 and "d_x is null" in err()
    assert scan(two, gs=7) == 1 and "d_g overlap" in err()
    assert scan(two, h=p + 1) == 1 and "d_h is not aligned" in err()
    assert scan(two, xs=1 << 63) == 1 and "overflows" in err()
    assert scan(two, h0=p + 2) == 1 and "d_h0" in err()
    back = lambda s, dx, dg, h=p: emu.emu_gated_scan_backward(ctypes.byref(s), p, 8, p, 8, p, 8, h, 8, None, None, dx, 8, dg, 8, None, p // 256 * 256 + 256, ctypes.byref(big))
    assert back(two, p, p + 64) == 1 and "d_h" in err()
    assert back(two, p + 64, p + 64) == 1 and "same buffer" in err()
    assert back(two, None, p + 64) == 1 and "d_dx is null" in err()
    step = lambda rows=2, num_slots=2, slots=None, state=p, channels=8, dtype=0: emu.emu_gated_scan_step(dtype, 2, channels, rows, p, 8, p, 8, p, 8, state, state, num_slots, slots, 0)
    assert step(num_slots=1) == 1 and "slots" in err()
    assert step(num_slots=0, slots=p) == 1 and "num_slots" in err()
    assert step(slots=p + 2) == 1 and "d_slots" in err()
    assert step(state=None) == 1 and "d_state" in err()
    assert step(dtype=7) == 1 and "dtype" in err()
    assert step(rows=0) == 0


# ---- fused norm -------------------------------------------------------------------------------------------------


class NormShape(ctypes.Structure):
    _fields_ = [("dtype", ci), ("norm", ci), ("order", ci), ("activation", ci), ("rows", sz), ("dim", sz), ("eps", cf), ("scale", cf)]


ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
NULL = (None, 0)
EPS = float(np.float32(1e-5))


def norm_emu(emu):
    shape, psz, m = ctypes.POINTER(NormShape), ctypes.POINTER(sz), [vp, sz]
    emu.emu_fused_norm.argtypes = [shape, *m * 3, vp, vp, vp, *m * 2]
    emu.emu_fused_norm_backward.argtypes = [shape, *m * 3, vp, vp, vp, *m * 5, vp, vp, vp, vp, psz]
    return emu


def vector(values, dtype):
    a = aligned(values.size, storage(dtype))
    a[:] = ref.to_bits(values, dtype)
    return a


def operand(m):
    return (m.ptr, m.stride) if m is not None else NULL


# rows, dim, stride - dim, shift, norm, order, activation of the gate (None: no gate), residual, weight, bias, channel scale, scale
NORMS = [
    (1, 1, 0, 0, "rms", "add_norm", None, False, True, False, False, 1.0),
    (3, 8, 0, 0, "layer", "add_norm", "silu", True, True, True, True, 0.5),
    (5, 100, 3, 1, "rms", "norm_add", "silu", True, True, False, True, 1.5),
    (2, 520, 8, 0, "layer", "norm_add", "sigmoid", False, True, True, False, 1.0),
    (4, 1032, 0, 8, "rms", "add_norm", "gelu", True, False, False, False, 1.0),
    (2, 2056, 0, 0, "layer", "add_norm", None, True, True, True, True, 1.0),
    (3, 2049, 0, 0, "rms", "norm_add", "relu", True, True, True, True, 1.0),
    (2, 4104, 0, 0, "rms", "norm_add", None, True, True, False, False, 0.25),
    (1, 8200, 0, 0, "layer", "norm_add", "silu", True, True, True, True, 1.0),
    (1, 16384, 0, 0, "rms", "add_norm", "silu", True, True, False, True, 1.0),
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", NORMS, ids=lambda c: f"{c[0]}x{c[1]}-{c[4]}-{c[5]}-{c[6]}")
def test_fused_norm_and_gradient(emu, dtype, case):
    rows, dim, gap, shift, kind, order, actn, with_res, with_w, with_b, with_cs, scale = case
    emu = norm_emu(emu)
    rng = np.random.default_rng(dim)
    f = lambda v: ref.to_f64(ref.to_bits(v, dtype), dtype)
    mat = lambda mean=0.0, s=1.0: f(rng.standard_normal((rows, dim)) * s + mean)
    x, res, gate = mat(0.3), mat(0.1, 2.0) if with_res else None, mat() if actn else None
    w, b, cs = (f(rng.standard_normal(dim) * 0.3 + 1) if have else None for have in (with_w, with_b, with_cs))
    s = scale * (cs if with_cs else np.ones(dim))
    one, zero = np.ones(dim), np.zeros(dim)
    out, z, eo, ez = ref.norm(kind, order, actn, x, res, gate, w if with_w else one, b if with_b else zero, s, EPS)
    keep = order == "add_norm" and with_res
    mx, mr, mg = Matrix(x, dtype, dim + gap, shift), Matrix(res, dtype) if with_res else None, Matrix(gate, dtype, dim + gap, shift) if actn else None
    vw, vb, vc = (vector(v, dtype) if v is not None else None for v in (w, b, cs))
    at = lambda v: v.ctypes.data if v is not None else None
    mo, mz = Matrix(x, dtype, dim + gap), Matrix(x, dtype) if keep else None
    shape = NormShape(DTYPES[dtype], {"rms": 0, "layer": 1}[kind], {"add_norm": 0, "norm_add": 1}[order], ACTS[actn or "none"], rows, dim, EPS, scale)
    assert emu.emu_fused_norm(ctypes.byref(shape), *operand(mx), *operand(mr), *operand(mg), at(vw), at(vb), at(vc), *operand(mo), *operand(mz)) == 0, emu.emu_last_error()
    ref.check(mo.get(), out, eo, dtype, "out")
    assert mo.untouched_between() and mx.untouched_between()
    if keep:
        ref.check(mz.get(), z, ez, dtype, "residual_out")
        # outputs in the place of inputs
        assert emu.emu_fused_norm(ctypes.byref(shape), *operand(mx), *operand(mr), *operand(mg), at(vw), at(vb), at(vc), *operand(mx), *operand(mr)) == 0
        assert (mx.get() == mo.get()).all() and (mr.get() == mz.get()).all()
        mx.put(x)
    # the gradient
    dout, dstream = mat(), mat() if keep else None
    zs = f(z)
    md, mzs, mds = Matrix(dout, dtype, dim + gap, shift), Matrix(zs, dtype), Matrix(dstream, dtype) if keep else None
    mdx, mdg, mdr = Matrix(x, dtype, dim + gap), Matrix(x, dtype) if actn else None, Matrix(x, dtype) if keep else None
    dw, db, dc = (floats(np.full(dim, 9.0)) if have else None for have in (with_w, with_b, with_cs))
    call = lambda ws, need: emu.emu_fused_norm_backward(ctypes.byref(shape), *operand(md), *operand(mzs), *operand(mg), at(vw), at(vb), at(vc), *(operand(mx) if with_cs and order == "add_norm" else NULL), *operand(mds),
                                                        *operand(mdx), *operand(mdg), *operand(mdr), at(dw), at(db), at(dc), ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0, emu.emu_last_error()
    got, err = ref.norm_backward(kind, order, actn, dout, zs, gate, w if with_w else one, b if with_b else zero, s, EPS, x, dstream)
    ref.check(mdx.get(), got["dx"], err["dx"], dtype, "dx")
    if actn:
        ref.check(mdg.get(), got["dgate"], err["dgate"], dtype, "dgate")
    if keep:
        ref.check(mdr.get(), got["dresidual"], err["dresidual"], dtype, "dresidual")
    for name, v, factor in (("dweight", dw, 1.0), ("dbias", db, 1.0), ("dscale", dc, scale)):
        if v is not None:
            ref.check(v, got[name] * factor, err[name] * abs(factor) * 1.01, "f32", name)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("actn", ["relu", "gelu", "silu", "sigmoid"])
def test_activations_at_the_ends_of_their_range(emu, dtype, actn):
    """Gates as large as the type holds: the activation is 0, 1 or the gate itself there, its slope 0 or 1, and nothing overflows on the way."""
    emu = norm_emu(emu)
    big = 1e30
    gate = ref.to_f64(ref.to_bits(np.array([[-big, -1e19, -1000.0, -200.0, -90.0, -40.0, 40.0, 90.0, 200.0, 1000.0, 1e19, big]]), dtype), dtype)
    dim = gate.shape[1]
    x, dout = np.ones((1, dim)), np.full((1, dim), 2.0 ** -100)  # y = 1 everywhere up to eps
    low = gate < 0
    want = {"relu": np.where(low, 0, gate), "gelu": np.where(low, 0, gate), "silu": np.where(low, 0, gate), "sigmoid": np.where(low, 0, 1.0)}[actn]
    slope = {"sigmoid": np.zeros_like(gate)}.get(actn, np.where(low, 0.0, 1.0))
    mx, mg, mo, md, mdx, mdg = (Matrix(v, dtype) for v in (x, gate, x, dout, x, x))
    shape = NormShape(DTYPES[dtype], 0, 0, ACTS[actn], 1, dim, 1e-30, 1.0)
    assert emu.emu_fused_norm(ctypes.byref(shape), *operand(mx), *NULL, *operand(mg), None, None, None, *operand(mo), *NULL) == 0
    small = 40 * np.exp(-40.0) * 1.01  # silu and sigmoid at +-40 are this far from their limits
    assert (np.abs(mo.get() - want) <= 2.0 ** -7 * np.abs(want) + small).all()
    call = lambda ws, need: emu.emu_fused_norm_backward(ctypes.byref(shape), *operand(md), *operand(mx), *operand(mg), None, None, None, *NULL, *NULL, *operand(mdx), *operand(mdg), *NULL, None, None, None, ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0
    assert (np.abs(mdg.get() / 2.0 ** -100 - slope) <= 2.0 ** -7 * slope + small).all() and np.isfinite(mdx.get()).all()


def test_fused_norm_many_rows(emu):
    """More rows than blocks in the gradient's kernel, one wave per row with several rows per block, and rows without any content."""
    emu = norm_emu(emu)
    rng = np.random.default_rng(2)
    rows, dim = 2100, 24
    x, dout = rng.standard_normal((rows, dim)), rng.standard_normal((rows, dim))
    x[7] = 0.0
    mx, md, mo, mdx = (Matrix(v, "f32") for v in (x, dout, x, x))
    x, dout = mx.get(), md.get()
    w = rng.standard_normal(dim).astype(np.float32).astype(np.float64)
    vw, dw = vector(w, "f32"), floats(np.full(dim, 9.0))
    shape = NormShape(2, 0, 0, 0, rows, dim, EPS, 1.0)
    assert emu.emu_fused_norm(ctypes.byref(shape), *operand(mx), *NULL, *NULL, vw.ctypes.data, None, None, *operand(mo), *NULL) == 0
    out, _, eo, _ = ref.norm("rms", "add_norm", None, x, None, None, w, 0.0, 1.0, EPS)
    ref.check(mo.get(), out, eo, "f32", "out")
    call = lambda ws, need: emu.emu_fused_norm_backward(ctypes.byref(shape), *operand(md), *operand(mx), *NULL, vw.ctypes.data, None, None, *NULL, *NULL, *operand(mdx), *NULL, *NULL, dw.ctypes.data, None, None, ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0
    got, err = ref.norm_backward("rms", "add_norm", None, dout, x, None, w, 0.0, 1.0, EPS, None, None)
    ref.check(mdx.get(), got["dx"], err["dx"], "f32", "dx")
    ref.check(dw, got["dweight"], err["dweight"], "f32", "dweight")
    shape.rows = 0  # no rows: the vectors' gradients are 0
    assert emu.emu_fused_norm_backward(ctypes.byref(shape), *NULL, *NULL, *NULL, vw.ctypes.data, None, None, *NULL, *NULL, *NULL, *NULL, *NULL, dw.ctypes.data, None, None, ws, ctypes.byref(have)) == 0
    assert (dw == 0).all()


def test_norm_gradient_against_differences(emu):
    rng = np.random.default_rng(3)
    for kind, order, actn in itertools.product(("rms", "layer"), ("add_norm", "norm_add"), ("silu", "gelu", "sigmoid")):
        x, res, gate, dout, dz = (rng.standard_normal((3, 5)) for _ in range(5))
        w, b, s = (rng.standard_normal(5) for _ in range(3))
        add = order == "add_norm"

        def loss(x, res, gate, w, b, s):
            out, z, _, _ = ref.norm(kind, order, actn, x, res, gate, w, b, s, 1e-3)
            return float((out * dout).sum() + ((z * dz).sum() if add else 0.0))

        z = res + s * x if add else x
        got, _ = ref.norm_backward(kind, order, actn, dout, z, gate, w, b, s, 1e-3, x, dz if add else None)
        args = [x, res, gate, w, b, s]
        for k, name in enumerate(("dx", "dresidual", "dgate", "dweight", "dbias", "dscale")):
            if name not in got:
                continue
            for at in itertools.product(*(range(n) for n in args[k].shape)):
                lo, hi = [v.copy() for v in args], [v.copy() for v in args]
                lo[k][at] -= 1e-5
                hi[k][at] += 1e-5
                assert abs((loss(*hi) - loss(*lo)) / 2e-5 - got[name][at]) < 1e-6, (kind, order, actn, name)


def test_fused_norm_refusals(emu):
    emu = norm_emu(emu)
    buf = aligned(8192, np.uint8, 0)
    p = buf.ctypes.data
    err = lambda: emu.emu_last_error().decode()
    big = sz(1 << 40)
    ok = dict(dtype=0, norm=0, order=0, activation=0, rows=2, dim=8, eps=1e-6, scale=1.0)
    m = lambda k: (p + 64 * k, 8)

    def fwd(x=m(0), res=NULL, gate=NULL, cs=None, out=m(1), z=NULL, **k):
        return emu.emu_fused_norm(ctypes.byref(NormShape(**{**ok, **k})), *x, *res, *gate, None, None, cs, *out, *z)

    assert emu.emu_fused_norm(None, *NULL, *NULL, *NULL, None, None, None, *NULL, *NULL) == 1 and "null shape" in err()
    assert fwd(dtype=5) == 1 and "dtype" in err()
    assert fwd(norm=2) == 1 and "norm" in err()
    assert fwd(order=2) == 1 and "order" in err()
    assert fwd(activation=5) == 1 and "activation" in err()
    assert fwd(activation=3) == 1 and "without a gate" in err()
    assert fwd(dim=0) == 1 and fwd(dim=16385) == 2 and fwd(rows=1 << 31) == 2
    assert fwd(scale=2.0) == 1 and "without a residual" in err()
    assert fwd(cs=p) == 1 and "without a residual" in err()
    assert fwd(z=m(2)) == 1 and "residual_out" in err()
    assert fwd(res=m(2), z=m(1)) == 1 and "same buffer" in err()
    assert fwd(x=(None, 8)) == 1 and "d_x is null" in err()
    assert fwd(out=(p + 1, 8)) == 1 and "aligned" in err()
    assert fwd(x=(p, 7)) == 1 and "overlap" in err()
    assert fwd(rows=0, x=NULL, out=NULL) == 0

    def back(dout=m(0), z=m(1), gate=NULL, x=NULL, dro=NULL, dx=m(2), dg=NULL, dr=NULL, dw=None, dc=None, ws=p // 256 * 256 + 1024, have=big, **k):
        return emu.emu_fused_norm_backward(ctypes.byref(NormShape(**{**ok, **k})), *dout, *z, *gate, None, None, None, *x, *dro, *dx, *dg, *dr, dw, None, dc, ws, ctypes.byref(have))

    assert back(have=sz(8)) == 4 and back(ws=p // 256 * 256 + 1032) == 1
    assert back(dg=m(3)) == 1 and "without a gate" in err()
    assert back(order=1, dr=m(3)) == 1 and "d_dout itself" in err()
    assert back(dc=p) == 1 and "needs d_x" in err()
    assert back(dr=m(2)) == 1 and "same buffer" in err()
    assert back(dw=p + 2) == 1 and "d_dweight" in err()
    need = sz(0)
    assert back(ws=None, have=need, dw=p) == 0 and need.value == 512  # 256 says that nothing is kept there
    assert back(ws=None, have=need) == 0 and need.value == 256


# ---- fused product ----------------------------------------------------------------------------------------------


class GemmShape(ctypes.Structure):
    _fields_ = [("dtype", ci), ("activation", ci), ("M", sz), ("N", sz), ("K", sz), ("beta", cf)]


def gemm_emu(emu):
    shape, psz, m = ctypes.POINTER(GemmShape), ctypes.POINTER(sz), [vp, sz]
    emu.emu_fused_gemm.argtypes = [shape, *m * 2, vp, *m * 3, vp, psz]
    emu.emu_fused_gemm_backward.argtypes = [shape, *m * 6, vp, vp, psz]
    emu.emu_fused_gemm_tiles.argtypes = [ci, ctypes.c_uint, ci, ci, sz, sz, sz, cf, *m * 2, vp, *m * 3, vp]
    emu.emu_fused_gemm_down.argtypes = [ci, ci, ctypes.c_uint, ci, sz, sz, sz, *m * 3, vp]
    return emu


def gemm_operands(rng, dtype, M, N, K, with_bias, with_c):
    f = lambda v: ref.to_f64(ref.to_bits(v, dtype), dtype)
    A, B = f(rng.standard_normal((M, K))), f(rng.standard_normal((N, K)) / max(K, 1) ** 0.5)
    return A, B, f(rng.standard_normal(N)) if with_bias else None, f(rng.standard_normal((M, N))) if with_c else None


# M, N, K, gap of the operands' rows, activation, bias, C, Z
GEMMS = [
    (1, 1, 1, 0, "none", False, False, False),
    (1, 40, 0, 0, "silu", True, True, True),
    (3, 17, 100, 0, "gelu", True, True, False),
    (5, 64, 1032, 8, "none", True, True, False),
    (16, 33, 2100, 0, "relu", False, False, True),
    (20, 24, 72, 1, "sigmoid", True, False, True),
    (64, 16, 4160, 0, "silu", True, True, True),
    (65, 136, 64, 0, "silu", True, True, True),
    (70, 130, 200, 8, "gelu", True, False, True),
    (129, 40, 37, 0, "none", False, True, False),
    (66, 9, 1100, 3, "sigmoid", True, True, False),
    (70, 20, 0, 0, "silu", True, True, True),
    (80, 30, 1, 0, "none", True, False, False),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", GEMMS, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{c[4]}")
def test_fused_gemm(emu, dtype, case):
    M, N, K, gap, name, with_bias, with_c, with_z = case
    emu = gemm_emu(emu)
    rng = np.random.default_rng(M * 7 + N)
    A, B, bias, C = gemm_operands(rng, dtype, M, N, K, with_bias, with_c)
    mA, mB = Matrix(A, dtype, K + gap) if K else None, Matrix(B, dtype, K + 2 * gap) if K else None
    mD, mZ = Matrix(np.zeros((M, N)), dtype, N + gap), Matrix(np.zeros((M, N)), dtype) if with_z else None
    mC = Matrix(C, dtype, N + gap) if with_c else None
    vb = vector(bias, dtype) if with_bias else None
    beta = 0.5 if with_c else 0.0
    s = GemmShape(DTYPES[dtype], ACTS[name], M, N, K, beta)
    run = lambda out: (lambda call: (lambda kept, ws, have: call(ws, ctypes.byref(have)))(*workspace_for(call)))(
        lambda ws, need: emu.emu_fused_gemm(ctypes.byref(s), *operand(mA), *operand(mB), vb.ctypes.data if with_bias else None, *operand(mC), *operand(out), *operand(mZ), ws, need))
    assert run(mD) == 0, emu.emu_last_error()
    d, z, ed, ez = ref.product(A, B, bias if with_bias else np.zeros(N), name, C, beta)
    ref.check(mD.get(), d, ed, dtype, "D")
    assert mD.untouched_between()
    if with_z:
        ref.check(mZ.get(), z, ez, dtype, "Z")
    if with_c:
        assert run(mC) == 0
        assert (mC.get() == mD.get()).all() and mC.untouched_between()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("w8,splits,M,N,K", [(4, 1, 130, 250, 136), (4, 3, 140, 100, 328), (8, 1, 300, 257, 208), (8, 2, 256, 40, 192), (8, 1, 33, 300, 448), (4, 2, 100, 30, 128), (6, 1, 200, 193, 152), (6, 2, 192, 384, 256)])
def test_fused_gemm_tiles(emu, dtype, w8, splits, M, N, K):
    emu = gemm_emu(emu)
    rng = np.random.default_rng(M)
    A, B, bias, C = gemm_operands(rng, dtype, M, N, K, True, True)
    ld = (K + 7) // 8 * 8
    mA, mB, mC, mD, mZ = Matrix(A, dtype, ld), Matrix(B, dtype, ld + 8), Matrix(C, dtype), Matrix(C, dtype, N + 3), Matrix(C, dtype)
    vb = vector(bias, dtype)
    shares = floats(np.full(splits * M * ((N + 7) // 8 * 8), np.nan))
    emu.emu_fused_gemm_tiles(w8, splits, DTYPES[dtype], ACTS["silu"], M, N, K, 0.5, *operand(mA), *operand(mB), vb.ctypes.data, *operand(mC), *operand(mD), *operand(mZ), shares.ctypes.data)
    d, z, ed, ez = ref.product(A, B, bias, "silu", C, 0.5)
    ref.check(mD.get(), d, ed, dtype, "D")
    ref.check(mZ.get(), z, ez, dtype, "Z")
    assert mD.untouched_between()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", [1, 2])
@pytest.mark.parametrize("w8,splits,M,N,K", [(4, 1, 130, 248, 131), (4, 3, 33, 104, 328), (8, 1, 301, 264, 207), (8, 2, 40, 256, 192), (6, 1, 200, 200, 151), (6, 2, 192, 384, 256)])
def test_fused_gemm_tiles_down_the_rows(emu, dtype, layout, w8, splits, M, N, K):
    """Operands whose K runs down their rows: parts of a step, of a chunk of columns, and rows further apart than they are long.  What the padding
    of a row holds beyond the operand must not be used."""
    emu = gemm_emu(emu)
    rng = np.random.default_rng(M + layout)
    A, B, _, _ = gemm_operands(rng, dtype, M, N, K, False, False)
    up = lambda n: (n + 7) // 8 * 8
    wide = lambda m: np.concatenate([m, np.zeros((m.shape[0], up(m.shape[1]) - m.shape[1]))], 1)
    mA = Matrix(wide(A.T if layout == 2 else A), dtype)
    mB, mD = Matrix(B.T, dtype, N + 16), Matrix(np.zeros((M, N)), dtype, N + 8)
    shares = floats(np.full(splits * M * N, np.nan))
    emu.emu_fused_gemm_down(w8, layout, splits, DTYPES[dtype], M, N, K, *operand(mA), *operand(mB), *operand(mD), shares.ctypes.data)
    d, _, ed, _ = ref.product(A, B, np.zeros(N), "none", None, 0.0)
    ref.check(mD.get(), d, ed, dtype, "D")
    assert mD.untouched_between()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,gap,name", [(1, 1, 1, 0, "silu"), (70, 100, 72, 0, "silu"), (130, 8, 65, 1, "gelu"), (9, 67, 130, 0, "none"), (100, 16, 24, 3, "none"), (40, 80, 16, 8, "sigmoid"), (0, 5, 9, 0, "relu"), (66, 70, 68, 0, "relu"), (150, 67, 136, 8, "silu"), (65, 144, 72, 0, "none"), (20, 200, 64, 0, "none"), (130, 24, 80, 8, "none"), (70, 0, 72, 0, "none"), (3, 0, 8, 0, "none")])
def test_fused_gemm_gradient(emu, dtype, M, N, K, gap, name):
    emu = gemm_emu(emu)
    rng = np.random.default_rng(M + N)
    f = lambda v: ref.to_f64(ref.to_bits(v, dtype), dtype)
    A, B, _, _ = gemm_operands(rng, dtype, M, N, K, False, False)
    dD, Z = f(rng.standard_normal((M, N))), f(rng.standard_normal((M, N))) if name != "none" else None
    mA, mB, mD, mZ = Matrix(A, dtype, K + gap), Matrix(B, dtype, K + gap), Matrix(dD, dtype, N + gap), Matrix(Z, dtype) if name != "none" else None
    dA, dB, db = Matrix(np.full((M, K), 5.0), dtype), Matrix(np.full((N, K), 5.0), dtype), floats(np.full(N, 9.0))
    s = GemmShape(DTYPES[dtype], ACTS[name], M, N, K, 0.0)
    got, err = ref.product_backward(dD, A, B, Z, name, dtype)
    for wanted in ("AB+", "A", "B", "+"):
        call = lambda ws, need: emu.emu_fused_gemm_backward(ctypes.byref(s), *operand(mD), *operand(mA), *operand(mB), *operand(mZ), *(operand(dA) if "A" in wanted else NULL), *(operand(dB) if "B" in wanted else NULL),
                                                            db.ctypes.data if "+" in wanted else None, ws, need)
        dA.put(np.full((M, K), 5.0))
        dB.put(np.full((N, K), 5.0))
        kept, ws, have = workspace_for(call)
        assert call(ws, ctypes.byref(have)) == 0, emu.emu_last_error()
        if "A" in wanted:
            ref.check(dA.get(), got["dA"], err["dA"], dtype, "dA")
        if "B" in wanted:
            ref.check(dB.get(), got["dB"], err["dB"], dtype, "dB")
        if "+" in wanted:
            ref.check(db[:N], got["dbias"], err["dbias"], "f32", "dbias")


def test_product_gradient_against_differences():
    rng = np.random.default_rng(4)
    for name in ACTS:
        A, B, bias, dD = rng.standard_normal((3, 4)), rng.standard_normal((5, 4)), rng.standard_normal(5), rng.standard_normal((3, 5))
        loss = lambda A, B, bias: float((ref.product(A, B, bias, name, None, 0.0)[0] * dD).sum())
        got, _ = ref.product_backward(dD, A, B, A @ B.T + bias, name, "f32")
        args = [A, B, bias]
        for k, key in enumerate(("dA", "dB", "dbias")):
            for at in itertools.product(*(range(n) for n in args[k].shape)):
                lo, hi = [v.copy() for v in args], [v.copy() for v in args]
                lo[k][at] -= 1e-5
                hi[k][at] += 1e-5
                assert abs((loss(*hi) - loss(*lo)) / 2e-5 - got[key][at]) < 1e-7, (name, key)


def test_fused_gemm_refusals(emu):
    emu = gemm_emu(emu)
    buf = aligned(1 << 16, np.uint8, 0)
    p = buf.ctypes.data
    ws0 = p // 256 * 256 + 32768
    err = lambda: emu.emu_last_error().decode()
    big = sz(1 << 40)
    m = lambda k: (p + 1024 * k, 8)
    ok = dict(dtype=0, activation=0, M=2, N=8, K=8, beta=0.0)

    def fwd(A=m(0), B=m(1), bias=None, C=NULL, D=m(2), Z=NULL, ws=ws0, have=big, **k):
        return emu.emu_fused_gemm(ctypes.byref(GemmShape(**{**ok, **k})), *A, *B, bias, *C, *D, *Z, ws, ctypes.byref(have) if have else None)

    assert emu.emu_fused_gemm(None, *NULL, *NULL, None, *NULL, *NULL, *NULL, None, None) == 1 and "null shape" in err()
    assert fwd(dtype=2) == 1 and "dtype" in err()
    assert fwd(activation=9) == 1 and "activation" in err()
    assert fwd(K=(1 << 22) + 1) == 2 and fwd(M=1 << 31) == 2 and fwd(M=1 << 30, N=1 << 30) == 2
    assert fwd(N=(1 << 28) + 1) == 2 and fwd(D=(p, (1 << 28) + 8)) == 2 and "leading dimension" in err()
    assert fwd(have=None) == 1 and fwd(have=sz(16)) == 4 and fwd(ws=ws0 + 8) == 1
    assert fwd(beta=1.0) == 1 and "beta without d_C" in err()
    assert fwd(A=(None, 8)) == 1 and "d_A" in err()
    assert fwd(B=(p, 7)) == 1 and "overlap" in err()
    assert fwd(D=(p + 1, 8)) == 1 and "aligned" in err()
    assert fwd(D=m(0)) == 1 and fwd(D=m(1)) == 1 and fwd(Z=m(2)) == 1 and fwd(Z=m(1)) == 1 and "in the place" in err()
    assert fwd(C=m(3), Z=m(3), beta=1.0) == 1
    assert fwd(bias=p + 1) == 1 and "d_bias" in err()
    assert fwd(M=0, A=NULL, D=NULL) == 0
    back = lambda dA=m(4), dB=m(5), Z=NULL, db=None, **k: emu.emu_fused_gemm_backward(ctypes.byref(GemmShape(**{**ok, **k})), *m(0), *m(1), *m(2), *Z, *dA, *dB, db, ws0, ctypes.byref(big))
    assert back(activation=3) == 1 and "needs d_Z" in err()
    assert back(M=(1 << 22) + 1) == 2
    assert back(dA=m(0)) == 1 and back(dA=m(5)) == 1 and back(dB=m(1)) == 1 and "in the place" in err()
    assert back(db=p + 2) == 1 and "d_dbias" in err()
