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


# ---- activations and norms --------------------------------------------------------------------------------------

GELU_A, GELU_B = np.sqrt(2.0 / np.pi), 0.044715


def act(name, z):
    """act(z), act'(z), and how many roundings relative to |act(z)| (+ |z| |act'| for the slope) their fp32 forms carry: the
    sigmoid's |argument| + 6 (gate_terms), the argument of gelu 4 more that the exponential turns into 4 |argument|, and the products."""
    one = np.ones_like(z)
    with np.errstate(over="ignore", invalid="ignore"):
        if name == "none":
            return z, one, 0.0 * one
        if name == "relu":
            return np.where(z < 0, 0.0, z), (z > 0).astype(np.float64), 0.0 * one
        v = 2 * GELU_A * (z + GELU_B * z ** 3) if name == "gelu" else z
        s, r = sigmoid(v), sigmoid(-v)
        c = np.minimum(np.abs(v), 128) * (5.0 if name == "gelu" else 1.0) + 10.0
        if name == "sigmoid":
            return s, s * r, c
        dv = 2 * GELU_A * (1 + 3 * GELU_B * z ** 2) if name == "gelu" else one
        return z * s, s + z * s * r * dv, c


def _stats(kind, z, ez, eps):
    """centred rows, 1 / sigma, and their bounds.  A sum over a row adds along chains of at most 64 + 24 values."""
    chain = 100.0 * EPS32
    mean = z.mean(-1, keepdims=True) if kind == "layer" else 0.0
    c = z - mean
    ec = ez + (chain * np.abs(z).mean(-1, keepdims=True) + ez.mean(-1, keepdims=True) + EPS32 * np.abs(c) if kind == "layer" else 0.0)
    var = (c * c).mean(-1, keepdims=True)
    rho = 1.0 / np.sqrt(var + eps)
    rel = 0.5 * ((chain * var + 2 * (np.abs(c) * ec).mean(-1, keepdims=True)) / (var + eps) + 2 * EPS32) + 4 * EPS32
    return c, ec, rho, rel


def norm(kind, order, name, x, residual, gate, weight, bias, scale, eps):
    """(out, z, bound on out, on z); scale: the vector s."""
    add = order == "add_norm" and residual is not None
    z = residual + scale * x if add else x
    ez = 3 * EPS32 * (np.abs(residual) + np.abs(scale * x)) if add else np.zeros_like(x)
    c, ec, rho, rel = _stats(kind, z, ez, eps)
    y = c * rho * weight + bias
    ey = np.abs(weight) * rho * (ec + np.abs(c) * (rel + 2 * EPS32)) + 2 * EPS32 * (np.abs(c * rho * weight) + np.abs(bias))
    f, _, cf = act(name, gate) if gate is not None else (np.ones_like(x), None, np.zeros_like(x))
    u, eu = y * f, ey * np.abs(f) + (cf + 1) * EPS32 * np.abs(y * f)
    if order == "norm_add":
        base = residual if residual is not None else np.zeros_like(x)
        return base + scale * u, z, np.abs(scale) * eu + 3 * EPS32 * (np.abs(scale * u) + np.abs(base)), ez
    return u, z, eu, ez


def norm_backward(kind, order, name, dout, z, gate, weight, bias, scale, eps, x, dstream):
    """dict of gradients (dscale with respect to the vector s) and dict of bounds."""
    c, ec, rho, rel = _stats(kind, z, np.zeros_like(z), eps)
    n, en = c * rho, rho * ec + np.abs(c * rho) * (rel + EPS32)
    y, ey = n * weight + bias, np.abs(weight) * en + 2 * EPS32 * (np.abs(n * weight) + np.abs(bias))
    f, slope, cf = act(name, gate) if gate is not None else (np.ones_like(z), np.zeros_like(z), np.zeros_like(z))
    mag = np.abs(f) + np.abs(gate) if gate is not None else np.abs(f)  # terms of the slope: s and z s (1 - s) v', each below this
    up = scale * dout if order == "norm_add" else dout
    dy, edy = up * f, (cf + 3) * EPS32 * np.abs(up * f)
    dn, edn = dy * weight, (cf + 4) * EPS32 * np.abs(dy * weight)
    mean = lambda v: v.mean(-1, keepdims=True)
    m1, em1 = mean(dn * n), 104 * EPS32 * mean(np.abs(dn * n)) + mean(np.abs(dn) * en + edn * np.abs(n)) + rel * np.abs(mean(dn * n))
    m2, em2 = (mean(dn), 104 * EPS32 * mean(np.abs(dn)) + mean(edn)) if kind == "layer" else (0.0, 0.0)
    inner = dn - n * m1 - m2
    einner = edn + en * np.abs(m1) + np.abs(n) * em1 + em2 + 4 * EPS32 * (np.abs(dn) + np.abs(n * m1) + np.abs(m2))
    dz, edz = rho * inner, rho * einner + (rel + EPS32) * rho * (np.abs(dn) + np.abs(n * m1) + np.abs(m2))
    got, err = {}, {}
    # a column's sum: the rows of one block in a chain, then the blocks' partial sums
    rows = z.shape[0]
    column = lambda t, e: (t.sum(0), (rows / 512 + 100) * EPS32 * np.abs(t).sum(0) + e.sum(0))
    got["dgate"], err["dgate"] = up * y * slope, np.abs(up) * (ey * np.abs(slope) + (3 * cf + 8) * EPS32 * np.abs(y) * mag)
    got["dweight"], err["dweight"] = column(dy * n, edy * np.abs(n) + np.abs(dy) * en + EPS32 * np.abs(dy * n))
    got["dbias"], err["dbias"] = column(dy, edy)
    if order == "norm_add":
        got["dscale"], err["dscale"] = column(dout * f * y, np.abs(dout) * (np.abs(f) * ey + (cf + 3) * EPS32 * np.abs(f * y)))
    else:
        extra = dstream if dstream is not None else 0.0
        dz, edz = dz + extra, edz + 2 * EPS32 * (np.abs(dz) + np.abs(extra))
        got["dresidual"], err["dresidual"] = dz, edz
        if x is not None:
            got["dscale"], err["dscale"] = column(dz * x, np.abs(x) * edz + EPS32 * np.abs(dz * x))
        dz, edz = scale * dz, np.abs(scale) * (edz + 2 * EPS32 * np.abs(dz))
    got["dx"], err["dx"] = dz, edz
    return got, err


# ---- product ----------------------------------------------------------------------------------------------------


def product(A, B, bias, name, C, beta):
    """(D, Z, bound on D, on Z) of D = act(A B^T + bias) + beta C; B as N rows of K.  A sum of K products in any order is off by at
    most 2 K 2^-24 times the sum of their magnitudes (two roundings an addition: the matrix unit's own and the accumulator's)."""
    k = A.shape[1]
    z = A @ B.T + bias
    ez = (2 * k + 8) * EPS32 * (np.abs(A) @ np.abs(B).T) + 2 * EPS32 * (np.abs(z) + np.abs(bias))
    f, _, c = act(name, z)
    d = f + (beta * C if C is not None else 0.0)
    steepest = 1.2  # no activation's slope is above it
    ed = steepest * ez + (c + 2) * EPS32 * np.abs(f) + 2 * EPS32 * (np.abs(d) + (np.abs(beta * C) if C is not None else 0.0))
    return d, z, ed, ez


def product_backward(dD, A, B, Z, name, dtype):
    """dict of gradients and of bounds; dZ is rounded to `dtype` in front of the products."""
    _, slope, c = act(name, Z) if Z is not None else (None, np.ones_like(dD), np.zeros_like(dD))
    mag = 1.0 + np.abs(Z) if Z is not None and name != "relu" else np.abs(slope)
    dz = dD * slope
    e = (3 * c + 8) * EPS32 * np.abs(dD) * mag if Z is not None else np.zeros_like(dD)
    er = e + U[dtype] * (np.abs(dz) + e) + TINY[dtype] if Z is not None else e
    m, n = dD.shape
    got = {"dA": dz @ B, "dB": dz.T @ A, "dbias": dz.sum(0)}
    err = {"dA": er @ np.abs(B) + (2 * n + 8) * EPS32 * ((np.abs(dz) + er) @ np.abs(B)), "dB": er.T @ np.abs(A) + (2 * m + 8) * EPS32 * ((np.abs(dz) + er).T @ np.abs(A)),
           "dbias": e.sum(0) + (m + 8) * EPS32 * np.abs(dz).sum(0)}
    return got, err
