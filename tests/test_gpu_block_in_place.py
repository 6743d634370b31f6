"""Gradients in the place of the operands they may replace, on the GPU: the same bits as in buffers of their own."""
import pytest

from test_gpu_block_forms import normal
from test_gpu_gated_scan import tcu  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,gate", [("bf16", "sigmoid"), ("f32", "log")])
@pytest.mark.parametrize("rows,channels,packed", [(20000, 1032, False), (20000, 1001, True), (700, 40, True)])
def test_scan(tcu, dtype, gate, rows, channels, packed):
    import torch

    mk = normal(rows, dtype)
    base = dict(dh=mk(rows, channels), x=mk(rows, channels), g=mk(rows, channels) - 3.0)
    h, offsets = mk(rows, channels), torch.tensor([0, 100, 100, 650, rows], device="cuda") if packed else None
    states = (4 if packed else 1, channels)
    h0, dl = torch.randn(states, device="cuda"), torch.randn(states, device="cuda")
    run = lambda m, **out: tcu.gated_scan_backward(m["dh"], m["x"], m["g"], h, gate, h0=h0, dh_last=dl, offsets=offsets, **out)
    want = run(base)
    for to_x, to_g in (("dh", "g"), ("x", "dh"), ("g", "x")):
        m = {k: t.clone() for k, t in base.items()}
        got = run(m, dx=m[to_x], dg=m[to_g])
        assert got[0] is m[to_x] and got[1] is m[to_g] and all(torch.equal(a, b) for a, b in zip(got, want))
    out, last = tcu.gated_scan(base["x"], base["g"], gate, h0=h0, offsets=offsets)
    m, state = base["g"].clone(), h0.clone()
    tcu.gated_scan(base["x"], m, gate, h0=state, offsets=offsets, out=m, h_last=state)
    assert torch.equal(m, out) and torch.equal(state, last)


def test_step(tcu):
    import torch

    mk = normal(5, "bf16")
    x, g, state = mk(200, 333), mk(200, 333), torch.randn(50, 333, device="cuda")
    slots = torch.randint(-1, 50, (200,), device="cuda", dtype=torch.int32)
    new = state.clone()
    h = tcu.gated_scan_step(x, g, state, slots=slots, new_state=new)
    for place in (x.clone(), g.clone()):
        own, keep = state.clone(), place.clone()
        ops = (place, g) if torch.equal(place, x) else (x, place)
        tcu.gated_scan_step(*ops, own, slots=slots, out=place)
        padding = (slots < 0)[:, None]
        assert torch.equal(place, torch.where(padding, keep, h)) and torch.equal(own, new)
