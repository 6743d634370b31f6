"""The fused norm and its gradient on the GPU, against the 64-bit formulas and bounds of tests/block_reference.py."""
import numpy as np
import pytest

import block_reference as ref
from test_gpu_gated_scan import dev, host, rounded

pytestmark = pytest.mark.gpu
EPS = float(np.float32(1e-6))


@pytest.fixture(scope="module")
def tcu():
    import tcu_scope_amd as t

    t.init(0)
    return t


CASES = [
    # rows, dim, stride, norm, order, activation of the gate, residual, weight, bias, channel scale, scale
    (1, 1, None, "rms", "add_norm", None, False, True, False, False, 1.0),
    (12, 2048, None, "rms", "norm_add", "silu", True, True, False, True, 1.0),
    (3000, 256, 272, "layer", "add_norm", "silu", True, True, True, True, 0.5),
    (2500, 1000, None, "rms", "norm_add", "sigmoid", True, True, False, True, 1.0),
    (700, 4096, None, "rms", "add_norm", None, True, True, False, False, 1.0),
    (2100, 2048, None, "layer", "norm_add", "gelu", False, True, True, False, 2.0),
    (2050, 4001, None, "rms", "add_norm", "silu", True, False, False, False, 1.0),
    (40, 8200, None, "layer", "norm_add", "relu", True, True, True, True, 1.0),
    (9, 16384, None, "rms", "add_norm", "silu", True, True, True, True, 1.0),
    (5, 16001, None, "layer", "add_norm", "silu", True, True, True, True, 1.0),
]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}-{c[3]}-{c[4]}-{c[5]}")
def test_norm_and_gradient(tcu, dtype, case):
    import torch

    rows, dim, stride, kind, order, actn, with_res, with_w, with_b, with_cs, scale = case
    rng = np.random.default_rng(dim)
    mat = lambda mean=0.0, s=1.0: rounded(rng.standard_normal((rows, dim)) * s + mean, dtype)
    x, res, gate = mat(0.3), mat(0.1, 2.0) if with_res else None, mat() if actn else None
    w, b, cs = (rounded(rng.standard_normal(dim) * 0.3 + 1, dtype) if have else None for have in (with_w, with_b, with_cs))
    s = scale * (cs if with_cs else np.ones(dim))
    one, zero = np.ones(dim), np.zeros(dim)
    out, z, eo, ez = ref.norm(kind, order, actn, x, res, gate, w if with_w else one, b if with_b else zero, s, EPS)
    keep = order == "add_norm" and with_res
    d = lambda v, st=None: None if v is None else dev(v, dtype, st)
    tx, tr, tg, tw, tb, tc = d(x, stride), d(res), d(gate, stride), d(w), d(b), d(cs)
    kw = dict(gate=tg, scale=scale, channel_scale=tc, norm=kind, order=order, activation=actn or "none", eps=EPS)
    got = tcu.fused_norm(tx, tw, tb, residual=tr, **kw)
    to, tz = got if keep else (got, None)
    ref.check(host(to), out, eo, dtype, "out")
    if keep:
        ref.check(host(tz), z, ez, dtype, "residual_out")
    dout, dstream = mat(), mat() if keep else None
    zs = rounded(z, dtype)
    args = (d(dout), d(zs), tw, tb)
    kw.update(x=tx, dresidual_out=d(dstream))
    got = tcu.fused_norm_backward(*args, **kw)
    want, err = ref.norm_backward(kind, order, actn, dout, zs, gate, w if with_w else one, b if with_b else zero, s, EPS, x, dstream)
    assert set(got) == {"dx"} | ({"dgate"} if actn else set()) | ({"dweight"} if with_w else set()) | ({"dbias"} if with_b else set()) | ({"dscale"} if with_cs else set()) | ({"dresidual"} if keep else set())
    for name, t in got.items():
        f = scale if name == "dscale" else 1.0
        ref.check(host(t), want[name] * f, err[name] * abs(f) * 1.01, "f32" if t.dtype == torch.float32 else dtype, name)
    again = tcu.fused_norm_backward(*args, **kw)
    assert all(torch.equal(t, again[name]) for name, t in got.items())


def test_rows_of_no_content_and_of_no_number(tcu):
    """A row of zeros is 0 (eps keeps it finite); a NaN or an infinity stays in its row."""
    import torch

    x = torch.randn(5, 512, device="cuda").half()
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    for kind in ("rms", "layer"):
        y = tcu.fused_norm(x, norm=kind)
        assert (y[1] == 0).all() and y[2].isnan().all() and not y[3].isfinite().all() and y[0].isfinite().all() and y[4].isfinite().all()
        d = tcu.fused_norm_backward(torch.ones_like(x), x, norm=kind)["dx"]
        assert d[2].isnan().all() and d[0].isfinite().all() and d[4].isfinite().all()


def test_in_place_empty_and_graph(tcu):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    x, r, w = mk(2, 150, 1024), mk(2, 150, 1024), mk(1024)
    out, z = tcu.fused_norm(x, w, residual=r)
    x2, r2 = x.clone(), r.clone()
    tcu.fused_norm(x2, w, residual=r2, out=x2, residual_out=r2)
    assert torch.equal(x2, out) and torch.equal(r2, z)
    e = mk(0, 64)
    assert tcu.fused_norm(e).shape == (0, 64)
    got = tcu.fused_norm_backward(e, e, weight=mk(64))
    assert (got["dweight"] == 0).all() and got["dx"].shape == (0, 64)
    want = tcu.fused_norm_backward(x, z, w, dresidual_out=r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go, gz = tcu.fused_norm(x, w, residual=r)
        gd = tcu.fused_norm_backward(x, z, w, dresidual_out=r)
    for _ in range(3):
        go.zero_(), gd["dweight"].zero_()
        graph.replay()
        assert torch.equal(tcu.fused_norm(x, w, residual=r)[0], out)
        torch.cuda.synchronize()
        assert torch.equal(go, out) and torch.equal(gz, z) and all(torch.equal(gd[k], want[k]) for k in want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    so, _ = tcu.fused_norm(x, w, residual=r, stream=s)
    s.synchronize()
    assert torch.equal(so, out)


def test_refusals(tcu):
    import torch

    x = torch.zeros(4, 64, device="cuda", dtype=torch.float16)
    v = x[0]
    for call, kind, words in [
        (lambda: tcu.fused_norm(x, weight=v.float()), ValueError, "weight"),
        (lambda: tcu.fused_norm(x, weight=v[:32]), ValueError, "weight"),
        (lambda: tcu.fused_norm(x, residual=x[:2]), ValueError, "residual must have"),
        (lambda: tcu.fused_norm(v), ValueError, "two dimensions"),
        (lambda: tcu.fused_norm(x.int()), TypeError, "float16"),
        (lambda: tcu.fused_norm(x, activation="silu"), tcu.TcuError, "without a gate"),
        (lambda: tcu.fused_norm(x, scale=2.0), tcu.TcuError, "without a residual"),
        (lambda: tcu.fused_norm(x, residual_out=x), ValueError, "residual_out"),
        (lambda: tcu.fused_norm(x, norm="group"), ValueError, "rms"),
        (lambda: tcu.fused_norm(torch.zeros(1, 16385, device="cuda")), tcu.TcuError, "16384"),
        (lambda: tcu.fused_norm_backward(x, x, channel_scale=v), ValueError, "needs x"),
        (lambda: tcu.fused_norm_backward(x, x, order="norm_add", dresidual_out=x), tcu.TcuError, "d_dout itself"),
    ]:
        with pytest.raises(kind, match=words):
            call()
