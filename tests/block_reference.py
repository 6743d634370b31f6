"""The recurrent-block operators in 64 bits, step by step from their definitions, with bounds on what fp32 arithmetic and
one rounding of each result may add.

Rounding of a value v to a type: at most U[type] |v|, and half the smallest subnormal step for fp16.  Arithmetic in fp32:
every operation is off by at most 2^-24 of its result (2^-23 for the hardware's exp2, reciprocal and square root), so a
result built by c of them from terms of magnitudes m is off by at most c 2^-24 m.  The bounds are written next to the
formulas; for recurrences they follow the same recurrence."""
import numpy as np

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}
EPS32 = 2.0 ** -24


def to_bits(v, dtype):
    """float64 array -> storage (uint16 or float32), rounded to nearest even."""
    v32 = np.asarray(v, dtype=np.float32)
    if dtype == "f32":
        return v32.copy()
    if dtype == "f16":
        return v32.astype(np.float16).view(np.uint16)
    u = v32.view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def to_f64(bits, dtype):
    if dtype == "f32":
        return bits.astype(np.float64)
    if dtype == "f16":
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def sigmoid(x):
    return np.where(x >= 0, 1.0 / (1.0 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1.0 + np.exp(-np.abs(x))))


def gate_terms(gate, g):
    """a, the weight of x, and how many roundings of 2^-24 they carry: for exp(g), |g| of them from the product with log2(e)
    (16-bit types), 2 from the instruction; for sigmoid besides those the sum, the reciprocal and one product: |g| + 6."""
    if gate == "decay":
        return g, np.ones_like(g), 0.0
    with np.errstate(over="ignore"):
        if gate == "log":
            return np.exp(g), np.ones_like(g), np.minimum(np.abs(g), 128) + 2.0
        return sigmoid(g), sigmoid(-g), np.minimum(np.abs(g), 128) + 6.0


def scan(gate, x, g, offsets, h0):
    """(h, h_last, bound of fp32 arithmetic on h, on h_last); rows outside all sequences are NaN in h."""
    a, keep, c = gate_terms(gate, g)
    c = np.broadcast_to(c, g.shape)
    b = keep * x
    h, e = np.full(x.shape, np.nan), np.zeros(x.shape)
    last, elast = np.array(h0, dtype=np.float64), np.zeros(h0.shape)
    for j in range(len(offsets) - 1):
        m, err, v = np.abs(last[j]), np.zeros(x.shape[1]), last[j]
        for t in range(offsets[j], offsets[j + 1]):
            v = a[t] * v + b[t]
            # whatever the order in which the steps are combined, a step multiplies what it carries by a (c + 1 roundings) or
            # by a product with a in it, and adds: 3 more roundings on the sum of the magnitudes
            m = np.abs(a[t]) * m + np.abs(b[t])
            err = np.abs(a[t]) * err + (c[t] + 5.0) * EPS32 * m
            h[t], e[t] = v, err
        last[j], elast[j] = v, err
    return h, last, e, elast


def scan_backward(gate, x, g, h, dh, offsets, h0, dh_last):
    """(dx, dg, dh0) and the bounds on each."""
    a, keep, c = gate_terms(gate, g)
    c = np.broadcast_to(c, g.shape)
    dx, dg = np.full(g.shape, np.nan), np.full(g.shape, np.nan)
    ex, eg = np.zeros(g.shape), np.zeros(g.shape)
    dh0, e0 = np.array(dh_last, dtype=np.float64), np.zeros(dh_last.shape)
    for j in range(len(offsets) - 1):
        u, m, err = dh0[j], np.abs(dh0[j]), np.zeros(g.shape[1])
        for t in reversed(range(offsets[j], offsets[j + 1])):
            delta = dh[t] + u
            m = np.abs(dh[t]) + m
            err = err + 2.0 * EPS32 * m
            before = h0[j] if t == offsets[j] else h[t - 1]
            if gate == "sigmoid":
                slope, mag = (before - x[t]) * a[t] * keep[t], (np.abs(before) + np.abs(x[t])) * a[t] * keep[t]
                dx[t] = keep[t] * delta
            else:
                f = a[t] if gate == "log" else 1.0
                slope, mag = before * f, np.abs(before) * np.abs(f)
                dx[t] = delta
            dg[t] = delta * slope
            ex[t] = keep[t] * (err + (c[t] + 2.0) * EPS32 * np.abs(delta))
            eg[t] = np.abs(slope) * err + (2.0 * c[t] + 5.0) * EPS32 * np.abs(delta) * mag
            u = a[t] * delta
            err = np.abs(a[t]) * err + (c[t] + 4.0) * EPS32 * np.abs(a[t]) * m
            m = np.abs(a[t]) * m
        dh0[j], e0[j] = u, err
    return (dx, dg, dh0), (ex, eg, e0)


def check(got, want, err, dtype, what):
    """|got - want| <= err + U |want| + U err (+ the subnormal step); NaN and infinities in the same places."""
    got, want, err = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64), np.asarray(err, dtype=np.float64)
    assert got.shape == want.shape, f"{what}: shape {got.shape} for {want.shape}"
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places ({np.isnan(got).sum()} for {np.isnan(want).sum()})"
    same = ~fine & ~np.isnan(want)
    assert np.array_equal(got[same], want[same]), f"{what}: infinities differ"
    off = np.abs(got[fine] - want[fine])
    may = err[fine] + U[dtype] * (np.abs(want[fine]) + err[fine]) + TINY[dtype]
    bad = ~(off <= may)
    if bad.any():
        k = int(np.argmax(np.where(bad, off / np.maximum(may, 1e-300), 0)))
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside the bound, worst {got[fine][k]} for {want[fine][k]}, {off[k]:.3g} off where {may[k]:.3g} is allowed")
