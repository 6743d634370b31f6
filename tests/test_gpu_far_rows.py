"""Rows that lie far apart (slices of very wide matrices, some 64-bit offsets), on the GPU: operands and results side by side in one buffer."""
import numpy as np
import pytest

import block_reference as ref
from test_gpu_gated_scan import NAMES, gates, host, rounded, tcu  # noqa: F401

pytestmark = pytest.mark.gpu


class Wide:
    """One buffer whose rows are `stride` elements apart; place() gives the next columns of it."""

    def __init__(self, rows, stride, dtype, used):
        import torch

        self.rows, self.stride, self.at = rows, stride, 0
        self.flat = torch.empty((rows - 1) * stride + used, dtype=getattr(torch, NAMES[dtype]), device="cuda")

    def place(self, values, rows=None):
        import torch

        t = self.flat.as_strided((rows or self.rows, values.shape[-1]), (self.stride, 1), self.at)
        self.at += values.shape[-1]
        t.copy_(torch.from_numpy(np.ascontiguousarray(values)))
        return t


# 2^23 elements is where the scan's kernel stops to address a wave's rows by 32-bit offsets
@pytest.mark.parametrize("dtype,gate", [("bf16", "sigmoid"), ("f32", "log")])
@pytest.mark.parametrize("stride", [(1 << 23) - 8, 1 << 23, (1 << 23) + 7])
@pytest.mark.parametrize("offsets", [None, [0, 100, 100, 599]])
def test_scan(tcu, dtype, gate, stride, offsets):
    import torch

    rng = np.random.default_rng(stride)
    rows, channels = 600, 24
    offs = offsets or [0, rows]
    x, g = rounded(rng.standard_normal((rows, channels)), dtype), rounded(gates(rng, gate, (rows, channels)), dtype)
    hs, dh = rounded(rng.standard_normal((rows, channels)), dtype), rounded(rng.standard_normal((rows, channels)), dtype)
    wide = Wide(rows, stride, dtype, 7 * channels)
    tx, tg, ths, tdh, out, dx, dg = (wide.place(v) for v in (x, g, hs, dh, x * 0 + 5, x * 0 + 5, x * 0 + 5))
    to = torch.tensor(offsets, dtype=torch.int32, device="cuda") if offsets else None
    zero = np.zeros((len(offs) - 1, channels))
    _, last = tcu.gated_scan(tx, tg, gate, offsets=to, out=out)
    wh, wl, e, el = ref.scan(gate, x, g, offs, zero)
    ref.check(host(out), np.where(np.isnan(wh), 5, wh), e, dtype, "h")
    ref.check(host(last), wl, el, "f32", "h_last")
    _, _, d0 = tcu.gated_scan_backward(tdh, tx, tg, ths, gate, offsets=to, dx=dx, dg=dg)
    (wx, wg, w0), (ex, eg, e0) = ref.scan_backward(gate, x, g, hs, dh, offs, zero, zero)
    ref.check(host(dx), np.where(np.isnan(wx), 5, wx), ex, dtype, "dx")
    ref.check(host(dg), np.where(np.isnan(wg), 5, wg), eg, dtype, "dg")
    ref.check(host(d0), w0, e0, "f32", "dh0")
    assert (host(tx) == x).all() and (host(tg) == g).all()  # the neighbours are what they were


def test_norm(tcu):
    rng = np.random.default_rng(3)
    rows, dim, eps = 600, 136, float(np.float32(1e-6))
    x, r, gate, dout = (rounded(rng.standard_normal((rows, dim)), "bf16") for _ in range(4))
    wide = Wide(rows, (1 << 23) + 8, "bf16", 8 * dim)
    tx, tr, tg, td, out, z = (wide.place(v) for v in (x, r, gate, dout, x, x))
    tcu.fused_norm(tx, residual=tr, gate=tg, out=out, residual_out=z, eps=eps)
    want, wz, e, ez = ref.norm("rms", "add_norm", "silu", x, r, gate, 1.0, 0.0, 1.0, eps)
    ref.check(host(out), want, e, "bf16", "out")
    ref.check(host(z), wz, ez, "bf16", "z")
    got = tcu.fused_norm_backward(td, z, gate=tg, eps=eps)
    want, err = ref.norm_backward("rms", "add_norm", "silu", dout, host(z), gate, np.ones(dim), np.zeros(dim), np.ones(dim), eps, None, None)
    for name, t in got.items():
        ref.check(host(t), want[name], err[name], "bf16", name)


@pytest.mark.parametrize("M,stride", [(20, (1 << 22) + 8), (600, 1 << 22), (600, (1 << 22) + 8), (600, (1 << 22) + 3)])
def test_product(tcu, M, stride):
    """Up to rows 2^22 apart the operands are taken as they are, beyond that (and off 16 bytes) they are copied first."""
    rng = np.random.default_rng(M)
    N, K = 200, 136
    A, B, C, dD = (rounded(rng.standard_normal(s), "f16") for s in ((M, K), (N, K), (M, N), (M, N)))
    wide = Wide(max(M, N), stride, "f16", 2 * K + 4 * N)
    tA, tB, tC, tD, out, z = wide.place(A, M), wide.place(B, N), wide.place(C, M), wide.place(dD, M), wide.place(C, M), wide.place(C, M)
    tcu.fused_gemm(tA, tB, None, "silu", C=tC, beta=0.5, out=out, preactivation=z)
    d, wz, ed, ez = ref.product(A, B, np.zeros(N), "silu", C, 0.5)
    ref.check(host(out), d, ed, "f16", "D")
    ref.check(host(z), wz, ez, "f16", "Z")
    Z = host(z)
    got = tcu.fused_gemm_backward(tD, tA, tB, z, "silu")
    want, err = ref.product_backward(dD, A, B, Z, "silu", "f16")
    for k, t in got.items():
        ref.check(host(t), want[k], err[k], "f32" if k == "dbias" else "f16", k)
