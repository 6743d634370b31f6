"""A gated recurrent block of the operators together, as a model has them: norm with the residual stream, projection, gated scan
on slices of the projection, gated norm, projection back onto the stream; its gradient against autograd in 64 bits; and token
by token with the states of the sequences in slots.

Bounds: along any path at most twelve tensors are rounded to the type, each by at most U of its values; the norms of the errors add
up to at most 12 U of the results' norms where the block's operations do not amplify (norms and gates keep values near 1; the
projections' weights are scaled to keep variances; 2 for what the norms' gradients amplify)."""
import pytest

import block_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tcu():
    import tcu_scope_amd as t

    t.init(0)
    return t


def make(dtype, B, T, D, E):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(D)
    mk = lambda *s, scale=1.0, mean=0.0: (torch.randn(*s, generator=gen, device="cuda") * scale + mean).to(dtype)
    return dict(u=mk(B, T, D), stream=mk(B, T, D), w1=mk(D, scale=0.1, mean=1.0), w_in=mk(3 * E, D, scale=D ** -0.5), b_in=mk(3 * E, scale=0.5), w2=mk(E, scale=0.1, mean=1.0), w_out=mk(D, E, scale=E ** -0.5))


def forward(tcu, p, E, scan):
    n1, s1 = tcu.fused_norm(p["u"], p["w1"], residual=p["stream"])
    proj = tcu.fused_gemm(n1, p["w_in"], p["b_in"])
    v, g, og = proj[..., :E], proj[..., E:2 * E], proj[..., 2 * E:]
    h = scan(v, g)
    y = tcu.fused_norm(h, p["w2"], gate=og, norm="layer")
    return tcu.fused_gemm(y, p["w_out"], C=s1), (n1, s1, proj, h, y)


def exact(p, E, B, T):
    import torch

    x = {k: t.double().requires_grad_(True) for k, t in p.items()}
    s1 = x["stream"] + x["u"]
    n1 = s1 / (s1.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * x["w1"]
    proj = torch.nn.functional.linear(n1, x["w_in"], x["b_in"])
    v, g, og = proj.split(E, -1)
    a = torch.sigmoid(g)
    h, hs = torch.zeros(B, E, dtype=torch.float64, device="cuda"), []
    for t in range(T):
        h = a[:, t] * h + (1 - a[:, t]) * v[:, t]
        hs.append(h)
    h = torch.stack(hs, 1)
    y = (h - h.mean(-1, keepdim=True)) / (h.var(-1, unbiased=False, keepdim=True) + 1e-6).sqrt() * x["w2"] * torch.nn.functional.silu(og)
    return torch.nn.functional.linear(y, x["w_out"]) + s1, x


def near(got, want, dtype, what, amplified=1.0):
    u = ref.U[{"torch.float16": "f16", "torch.bfloat16": "bf16"}[str(dtype)]]
    off = ((got.double() - want).norm() / want.norm()).item()
    assert off <= 12 * u * amplified, f"{what}: {off:.3g} off, {12 * u * amplified:.3g} allowed"


@pytest.mark.parametrize("name,B,T,D,E", [("bfloat16", 2, 300, 256, 192), ("float16", 3, 65, 136, 72), ("bfloat16", 1, 130, 100, 50)])
def test_block(tcu, name, B, T, D, E):
    import torch

    dtype = getattr(torch, name)
    p = make(dtype, B, T, D, E)
    out, (n1, s1, proj, h, y) = forward(tcu, p, E, lambda v, g: tcu.gated_scan(v, g)[0])
    want, x = exact(p, E, B, T)
    near(out, want.detach(), dtype, "out")
    dout = torch.randn(B, T, D, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dtype)
    grads = dict(zip(x, torch.autograd.grad(want, list(x.values()), dout.double())))
    g_out = tcu.fused_gemm_backward(dout, y, p["w_out"], bias_gradient=False)
    v, g, og = proj[..., :E], proj[..., E:2 * E], proj[..., 2 * E:]
    g_n2 = tcu.fused_norm_backward(g_out["dA"], h, p["w2"], gate=og, norm="layer")
    dproj = torch.empty_like(proj)
    tcu.gated_scan_backward(g_n2["dx"], v, g, h, dx=dproj[..., :E], dg=dproj[..., E:2 * E])
    dproj[..., 2 * E:] = g_n2["dgate"]
    g_in = tcu.fused_gemm_backward(dproj, n1, p["w_in"])
    g_n1 = tcu.fused_norm_backward(g_in["dA"], s1, p["w1"], dresidual_out=dout)
    got = {"u": g_n1["dx"], "stream": g_n1["dresidual"], "w1": g_n1["dweight"], "w_in": g_in["dB"], "b_in": g_in["dbias"], "w2": g_n2["dweight"], "w_out": g_out["dB"]}
    for k, t in got.items():
        near(t, grads[k], dtype, "gradient of " + k, 2.0)


def test_block_token_by_token(tcu):
    """The block advanced one token at a time, requests in slots of a pool and one row of padding, ends where the whole sequences do."""
    import torch

    B, T, D, E = 3, 20, 128, 64
    p = make(torch.bfloat16, B, T, D, E)
    whole, _ = forward(tcu, p, E, lambda v, g: tcu.gated_scan(v, g)[0])
    state = torch.zeros(9, E, device="cuda")
    slots = torch.tensor([7, 2, -1, 4], dtype=torch.int32, device="cuda")
    rows = [0, 1, 0, 2]  # the third row is padding
    outs = []
    for t in range(T):
        q = dict(p, u=p["u"][rows, t].contiguous(), stream=p["stream"][rows, t].contiguous())
        outs.append(forward(tcu, q, E, lambda v, g: tcu.gated_scan_step(v, g, state, slots=slots))[0][[0, 1, 3]])
    near(torch.stack(outs, 1), whole.double(), torch.bfloat16, "token by token", 2.0)
    assert (state[[0, 1, 3, 5, 6, 8]] == 0).all()


def test_block_in_a_graph(tcu):
    """The whole block, forward and gradient, captured and replayed with new inputs between eager runs."""
    import torch

    B, T, D, E = 2, 700, 128, 64
    p = make(torch.bfloat16, B, T, D, E)

    def step():
        out, (n1, s1, proj, h, y) = forward(tcu, p, E, lambda v, g: tcu.gated_scan(v, g)[0])
        g_out = tcu.fused_gemm_backward(p["u"], y, p["w_out"])
        g_n2 = tcu.fused_norm_backward(g_out["dA"], h, p["w2"], gate=proj[..., 2 * E:], norm="layer")
        dv, dg, _ = tcu.gated_scan_backward(g_n2["dx"], proj[..., :E], proj[..., E:2 * E], h)
        return [out, dv, dg, *g_out.values(), *g_n2.values()]

    eager = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for r in range(3):
        p["u"].copy_(torch.randn(B, T, D, generator=torch.Generator(device="cuda").manual_seed(r), device="cuda"))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


def test_two_streams_at_once(tcu):
    """Blocks on two streams that run side by side get what each gets alone, to the bit: no call keeps anything where another finds it."""
    import torch

    sets = [(make(torch.bfloat16, B, T, D, E), E) for B, T, D, E in ((2, 1500, 256, 320), (3, 900, 256, 264))]

    def step(p, E):
        out, (n1, s1, proj, h, y) = forward(tcu, p, E, lambda v, g: tcu.gated_scan(v, g)[0])
        g_out = tcu.fused_gemm_backward(out, y, p["w_out"])
        g_n2 = tcu.fused_norm_backward(g_out["dA"], h, p["w2"], gate=proj[..., 2 * E:], norm="layer")
        return [out, *g_out.values(), *g_n2.values(), *tcu.gated_scan_backward(g_n2["dx"], proj[..., :E], proj[..., E:2 * E], h)]

    alone = [step(*a) for a in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (a, s) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(s):
                got[i].append(step(*a))
    torch.cuda.synchronize()
    for want, runs in zip(alone, got):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(r, want))
