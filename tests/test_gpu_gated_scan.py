"""The gated scan, its gradient and its one-token form on the GPU, against the 64-bit recurrences and bounds of
tests/block_reference.py."""
import numpy as np
import pytest

import block_reference as ref

pytestmark = pytest.mark.gpu

NAMES = {"f16": "float16", "bf16": "bfloat16", "f32": "float32"}


@pytest.fixture(scope="module")
def tcu():
    import tcu_scope_amd as t

    t.init(0)
    return t


def dev(values, dtype, stride=None):
    """values on the GPU in `dtype`; with `stride`, as the first columns of a wider matrix."""
    import torch

    t = torch.from_numpy(np.ascontiguousarray(values)).cuda().to(getattr(torch, NAMES[dtype]))
    if stride is None:
        return t
    wide = torch.full((*values.shape[:-1], stride), -77.0, dtype=t.dtype, device="cuda")
    wide[..., :values.shape[-1]] = t
    return wide[..., :values.shape[-1]]


def host(t):
    return t.detach().cpu().double().numpy()


def rounded(values, dtype):
    return ref.to_f64(ref.to_bits(values, dtype), dtype)


def gates(rng, gate, shape):
    z = rng.standard_normal(shape)
    return {"sigmoid": z * 1.5 + 2, "log": -np.exp(z * 1.2 - 3), "decay": ref.sigmoid(z * 1.5 + 2) * np.where(rng.random(shape) < 0.2, -1, 1)}[gate]


@pytest.mark.parametrize("dtype,gate", [("f16", "sigmoid"), ("bf16", "log"), ("f32", "decay"), ("bf16", "sigmoid"), ("f32", "sigmoid")])
@pytest.mark.parametrize("rows,channels,offsets,stride", [(1, 8, None, None), (7, 1, None, None), (129, 24, None, 40), (4000, 136, None, None), (3001, 77, None, None), (2600, 256, [0, 0, 1, 130, 1900, 1900, 2590], 264),
                                                          (20000, 16, None, None), (1200, 130, [5, 700, 1199], None)])
def test_scan_and_gradient(tcu, dtype, gate, rows, channels, offsets, stride):
    import torch

    rng = np.random.default_rng(rows + channels)
    offs = offsets or [0, rows]
    x, g = rounded(rng.standard_normal((rows, channels)), dtype), rounded(gates(rng, gate, (rows, channels)), dtype)
    h0 = rng.standard_normal((len(offs) - 1, channels)).astype(np.float32).astype(np.float64)
    dl = rng.standard_normal(h0.shape).astype(np.float32).astype(np.float64)
    hs, dh = rounded(rng.standard_normal((rows, channels)), dtype), rounded(rng.standard_normal((rows, channels)), dtype)
    tx, tg, t0 = dev(x, dtype, stride), dev(g, dtype, stride), dev(h0, "f32")
    to = torch.tensor(offsets, dtype=torch.int64 if channels % 2 else torch.int32, device="cuda") if offsets else None
    h, last = tcu.gated_scan(tx, tg, gate, h0=t0, offsets=to)
    wh, wl, e, el = ref.scan(gate, x, g, offs, h0)
    ref.check(host(h), np.where(np.isnan(wh), 0, wh), e, dtype, "h")
    ref.check(host(last), wl, el, "f32", "h_last")
    again, _ = tcu.gated_scan(tx, tg, gate, h0=t0, offsets=to)
    assert torch.equal(h, again)
    dx, dg, d0 = tcu.gated_scan_backward(dev(dh, dtype), tx, tg, dev(hs, dtype, stride), gate, h0=t0, dh_last=dev(dl, "f32"), offsets=to)
    (wx, wg, w0), (ex, eg, e0) = ref.scan_backward(gate, x, g, hs, dh, offs, h0, dl)
    ref.check(host(dx), np.where(np.isnan(wx), 0, wx), ex, dtype, "dx")
    ref.check(host(dg), np.where(np.isnan(wg), 0, wg), eg, dtype, "dg")
    ref.check(host(d0), w0, e0, "f32", "dh0")
    out = torch.full_like(h, 5.0)
    tcu.gated_scan(tx, tg, gate, h0=t0, offsets=to, out=out)
    assert torch.equal(out, torch.where(torch.from_numpy(np.isnan(wh)).cuda(), 5.0, h.float()).to(out.dtype))


def test_batches_and_slices(tcu):
    """(sequences, tokens, channels), gate and input as halves of one wider product, an output in the place of the input."""
    import torch

    rng = np.random.default_rng(1)
    both = rounded(rng.standard_normal((3, 300, 256)), "bf16")
    t = dev(both, "bf16")
    x, g = both[..., :128].reshape(900, 128), both[..., 128:].reshape(900, 128)
    wh, wl, e, el = ref.scan("sigmoid", x, g, [0, 300, 600, 900], np.zeros((3, 128)))
    h, last = tcu.gated_scan(t[..., :128], t[..., 128:])
    assert h.shape == (3, 300, 128)
    ref.check(host(h).reshape(900, 128), wh, e, "bf16", "h")
    ref.check(host(last), wl, el, "f32", "h_last")
    tcu.gated_scan(t[..., :128], t[..., 128:], out=t[..., :128])
    assert torch.equal(t[..., :128], h)
    with pytest.raises(ValueError, match="evenly"):
        tcu.gated_scan(dev(both, "bf16").transpose(0, 1)[..., :128], dev(both, "bf16").transpose(0, 1)[..., 128:])


def test_empty(tcu):
    import torch

    x = torch.zeros(0, 8, device="cuda", dtype=torch.float16)
    h0 = torch.arange(16.0, device="cuda").reshape(2, 8)
    h, last = tcu.gated_scan(x, x, h0=h0, offsets=torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert h.shape == (0, 8) and torch.equal(last, h0)
    h, last = tcu.gated_scan(x.reshape(2, 0, 8), x.reshape(2, 0, 8), h0=h0)
    assert torch.equal(last, h0)
    _, _, d0 = tcu.gated_scan_backward(x, x, x, x, dh_last=h0, offsets=torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert torch.equal(d0, h0)
    # rows, and no sequence that has them
    x, none = torch.ones(5, 8, device="cuda", dtype=torch.float16), torch.zeros(1, dtype=torch.int32, device="cuda")
    h, last = tcu.gated_scan(x, x, offsets=none)
    dx, dg, d0 = tcu.gated_scan_backward(x, x, x, x, offsets=none)
    assert last.shape == d0.shape == (0, 8) and all((t == 0).all() for t in (h, dx, dg))


def test_side_stream_and_graph(tcu):
    """The same bits on a side stream and from a captured graph replayed between eager calls; two graphs with a workspace each."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(1)
    mk = lambda: torch.randn(2, 1500, 192, generator=gen, device="cuda").bfloat16()
    x, g, h0 = mk(), mk(), torch.randn(2, 192, generator=gen, device="cuda")
    want, wlast = tcu.gated_scan(x, g, h0=h0)
    dwant = tcu.gated_scan_backward(x, x, g, want, h0=h0, dh_last=h0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got, last = tcu.gated_scan(x, g, h0=h0, stream=s)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(last, wlast)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h, last = tcu.gated_scan(x, g, h0=h0)
            d = tcu.gated_scan_backward(x, x, g, h, h0=h0, dh_last=h0)
        graphs.append((graph, h, last, d))
    for r in range(4):
        for graph, h, last, d in graphs:
            h.zero_()
            graph.replay()
        eager, _ = tcu.gated_scan(x, g, h0=h0)
        torch.cuda.synchronize()
        assert torch.equal(eager, want)
        for _, h, last, d in graphs:
            assert torch.equal(h, want) and torch.equal(last, wlast) and all(torch.equal(a, b) for a, b in zip(d, dwant))


@pytest.mark.parametrize("dtype,gate", [("f16", "sigmoid"), ("bf16", "log"), ("f32", "decay")])
@pytest.mark.parametrize("rows,channels", [(1, 8), (48, 2048), (200, 333)])
def test_step(tcu, dtype, gate, rows, channels):
    import torch

    rng = np.random.default_rng(rows)
    x, g = rounded(rng.standard_normal((rows, channels)), dtype), rounded(gates(rng, gate, (rows, channels)), dtype)
    state = rng.standard_normal((60, channels)).astype(np.float32).astype(np.float64)
    at = rng.integers(-1, 60, rows)  # repeated slots and padding among them
    t = dev(state, "f32")
    h = tcu.gated_scan_step(dev(x, dtype), dev(g, dtype), t, gate, slots=torch.from_numpy(at.astype(np.int32)).cuda())
    a, keep, c = ref.gate_terms(gate, g)
    c = np.broadcast_to(c, g.shape)
    want, err, wh, eh = state.copy(), np.zeros(state.shape), np.zeros(x.shape), np.zeros(x.shape)
    for i, j in enumerate(at):
        if j >= 0:
            m = np.abs(a[i] * want[j]) + np.abs(keep[i] * x[i])
            want[j] = a[i] * want[j] + keep[i] * x[i]
            err[j] = np.abs(a[i]) * err[j] + (c[i] + 4.0) * ref.EPS32 * m
            wh[i], eh[i] = want[j], err[j]
    ref.check(host(h), wh, eh, dtype, "h")
    ref.check(host(t), want, err, "f32", "state")
    # a sequence advanced token by token ends where the scan ends
    one = torch.zeros(1, channels, device="cuda")
    xs, gs = dev(x, dtype), dev(g, dtype)
    steps = torch.cat([tcu.gated_scan_step(xs[i:i + 1], gs[i:i + 1], one, gate) for i in range(min(rows, 20))])
    hh, last = tcu.gated_scan(xs[:20], gs[:20], gate)
    _, _, e, el = ref.scan(gate, x[:20], g[:20], [0, min(rows, 20)], np.zeros((1, channels)))
    ref.check(host(steps), host(hh), 2 * e + ref.U[dtype] * np.abs(host(hh)), dtype, "steps")
    ref.check(host(one), host(last), 2 * el, "f32", "state behind the steps")


def test_refusals(tcu):
    import torch

    x = torch.zeros(4, 8, device="cuda", dtype=torch.float16)
    for call, kind, words in [
        (lambda: tcu.gated_scan(x, x[:3]), ValueError, "g must have the shape"),
        (lambda: tcu.gated_scan(x, x.float()), ValueError, "g must have"),
        (lambda: tcu.gated_scan(x.double(), x.double()), TypeError, "float16, bfloat16 or float32"),
        (lambda: tcu.gated_scan(x.cpu(), x.cpu()), ValueError, "CUDA"),
        (lambda: tcu.gated_scan(x.t().contiguous().t(), x), ValueError, "contiguous along its last"),
        (lambda: tcu.gated_scan(x, x, gate="relu"), ValueError, "decay"),
        (lambda: tcu.gated_scan(x, x, h0=torch.zeros(2, 8, device="cuda")), ValueError, "h0"),
        (lambda: tcu.gated_scan(x, x, offsets=torch.zeros(3, device="cuda")), ValueError, "offsets"),
        (lambda: tcu.gated_scan(x[None], x[None], offsets=torch.zeros(3, device="cuda", dtype=torch.int32)), ValueError, "matrix of all rows"),
        (lambda: tcu.gated_scan(x, x, workspace=torch.empty(16, dtype=torch.uint8, device="cuda")), tcu.TcuError, "workspace"),
        (lambda: tcu.gated_scan(x[:1].expand(4, 8), x), tcu.TcuError, "overlap"),
        (lambda: tcu.gated_scan_backward(x, None, x, x), ValueError, "needs x"),
        (lambda: tcu.gated_scan_backward(x, x, x, x, dx=x), ValueError, "both or neither"),
        (lambda: tcu.gated_scan_step(x, x, torch.zeros(3, 8, device="cuda")), tcu.TcuError, "fewer slots"),
        (lambda: tcu.gated_scan_step(x, x, torch.zeros(3, 8, device="cuda"), slots=torch.zeros(4, dtype=torch.int64, device="cuda")), ValueError, "slots"),
    ]:
        with pytest.raises(kind, match=words):
            call()
