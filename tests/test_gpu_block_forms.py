"""Every form of the gated scan's and the fused product's kernels on the GPU, at sizes of tests/block_shapes.py.  The products' references are
64-bit products on the GPU with the bounds of tests/block_reference.py."""
import numpy as np
import pytest

import block_reference as ref
from block_shapes import GRADIENTS, PRODUCTS, SCANS
from test_gpu_gated_scan import NAMES, dev, gates, host, rounded, tcu  # noqa: F401

pytestmark = pytest.mark.gpu


def check(got, want, err, dtype, what):
    """block_reference.check on the GPU, for finite values."""
    assert got.shape == want.shape and bool(got.isfinite().all()), what
    may = err + ref.U[dtype] * (want.abs() + err) + ref.TINY[dtype]
    off = (got.double() - want).abs()
    bad = off > may
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, worst {float(off[bad].max())}"


def normal(seed, dtype):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *shape, scale=1.0: torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(getattr(torch, NAMES[dtype]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,w8,shared", PRODUCTS)
def test_products(tcu, dtype, M, N, K, w8, shared):
    import torch

    mk = normal(M + N, dtype)
    A, B, bias, C = mk(M, K), mk(N, K, scale=K ** -0.5), mk(N), mk(M, N)
    D, Z = tcu.fused_gemm(A, B, bias, "none", C=C, beta=0.5, return_preactivation=True)
    a, b, c = A.double(), B.double(), 0.5 * C.double()
    z = a @ b.t().contiguous() + bias.double()
    ez = (2 * K + 8) * ref.EPS32 * (a.abs() @ b.abs().t().contiguous()) + 2 * ref.EPS32 * (z.abs() + bias.double().abs())
    check(Z, z, ez, dtype, "Z")
    check(D, z + c, ez + 2 * ref.EPS32 * ((z + c).abs() + c.abs()), dtype, "D")
    for _ in range(3):
        assert torch.equal(tcu.fused_gemm(A, B, bias, "none", C=C, beta=0.5), D)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,for_a,for_b", GRADIENTS, ids=lambda v: str(v) if isinstance(v, int) else "")
def test_gradients(tcu, dtype, M, N, K, for_a, for_b):
    import torch

    mk = normal(M + N, dtype)
    A, B, dD, Z = mk(M, K), mk(N, K, scale=K ** -0.5), mk(M, N), mk(M, N)
    got = tcu.fused_gemm_backward(dD, A, B, Z, "relu")  # its slope is exact, so dZ is dD or 0 without another rounding
    dz, a, b = dD.double() * (Z > 0), A.double(), B.double()
    check(got["dA"], dz @ b, (2 * N + 8) * ref.EPS32 * (dz.abs() @ b.abs()), dtype, "dA")
    t = dz.t().contiguous()
    check(got["dB"], t @ a, (2 * M + 8) * ref.EPS32 * (t.abs() @ a.abs()), dtype, "dB")
    check(got["dbias"], dz.sum(0), (M + 8) * ref.EPS32 * dz.abs().sum(0), "f32", "dbias")
    for _ in range(3):
        again = tcu.fused_gemm_backward(dD, A, B, Z, "relu")
        assert all(torch.equal(again[k], got[k]) for k in got)


@pytest.mark.parametrize("rows,channels,dtype,seqs", SCANS, ids=lambda v: "packed" if isinstance(v, list) else str(v))
def test_scans(tcu, rows, channels, dtype, seqs):
    import torch

    gate = {"bf16": "sigmoid", "f16": "log", "f32": "decay"}[dtype]
    rng = np.random.default_rng(channels)
    packed = isinstance(seqs, list)
    offs = seqs if packed else [j * (rows // seqs) for j in range(seqs + 1)]
    x, g = rounded(rng.standard_normal((rows, channels)), dtype), rounded(gates(rng, gate, (rows, channels)), dtype)
    hs, dh = rounded(rng.standard_normal((rows, channels)), dtype), rounded(rng.standard_normal((rows, channels)), dtype)
    h0, dl = (rng.standard_normal((len(offs) - 1, channels)).astype(np.float32).astype(np.float64) for _ in range(2))
    to = torch.tensor(offs, dtype=torch.int64, device="cuda") if packed else None
    shaped = (lambda v: v) if packed else (lambda v: v.reshape(seqs, rows // seqs, channels))
    tx, tg, ths, tdh = (shaped(dev(v, dtype)) for v in (x, g, hs, dh))
    t0, tl = dev(h0, "f32"), dev(dl, "f32")
    flat = lambda t: host(t).reshape(rows, channels)
    h, last = tcu.gated_scan(tx, tg, gate, h0=t0, offsets=to)
    wh, wl, e, el = ref.scan(gate, x, g, offs, h0)
    ref.check(flat(h), np.where(np.isnan(wh), 0, wh), e, dtype, "h")
    ref.check(host(last), wl, el, "f32", "h_last")
    dx, dg, d0 = tcu.gated_scan_backward(tdh, tx, tg, ths, gate, h0=t0, dh_last=tl, offsets=to)
    (wx, wg, w0), (ex, eg, e0) = ref.scan_backward(gate, x, g, hs, dh, offs, h0, dl)
    ref.check(flat(dx), np.where(np.isnan(wx), 0, wx), ex, dtype, "dx")
    ref.check(flat(dg), np.where(np.isnan(wg), 0, wg), eg, dtype, "dg")
    ref.check(host(d0), w0, e0, "f32", "dh0")
    for _ in range(3):
        assert torch.equal(tcu.gated_scan(tx, tg, gate, h0=t0, offsets=to)[0], h)
