"""What is measured of the recurrent-block operators: the gated scan, the fused norm and the fused matrix product.

Each case below is one pass through one operator.  Where `own` is false the operator is computed from elementary torch
operations in 32 bits, rounded once at the end; where it is true the framework's entry points are called on the same
inputs.  `exact` computes the same outputs from the definitions in 64 bits, step by step along the sequence where the
plain form doubles its stride.

Formulas (rows are tokens, channels are independent of each other):

  gated scan       h[t] = a[t] h[t-1] + b[t] inside a sequence, h[-1] = h0 of the sequence; from a gate g and an input x
                     decay    a = g            b = x
                     log      a = exp(g)       b = x
                     sigmoid  a = sigmoid(g)   b = (1 - a) x
  fused norm       order add_norm:  z = residual + s x,  out = act(gate) (norm(z) weight + bias),  z is returned as well
                   order norm_add:  out = residual + s act(gate) (norm(x) weight + bias)
                   norm: rms (z / sqrt(mean z^2 + eps)) or layer ((z - mean) / sqrt(var + eps)); s one number per channel
  fused product    D = act(A B + bias) + beta C, with the argument of act returned where a backward pass will want it
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6
GELU_A, GELU_B = math.sqrt(2.0 / math.pi), 0.044715


def listed():
    return [
        # a whole long document at once: one sequence, its state coming from an earlier part; work is split along time
        {"name": "scan_long_document", "op": "scan", "type": "f16", "gate": "sigmoid", "sequences": 1, "tokens": 65536, "channels": 2048, "packed": False},
        # a training batch, sequences of equal length
        {"name": "scan_training", "op": "scan", "type": "bf16", "gate": "sigmoid", "sequences": 8, "tokens": 8 * 4096, "channels": 2048, "packed": False},
        # prompts of unequal length packed behind each other, an odd number of tokens and of channels
        {"name": "scan_packed_prompts", "op": "scan", "type": "bf16", "gate": "log", "sequences": 37, "tokens": 8191, "channels": 1000, "packed": True},
        # the gradient of the training batch
        {"name": "scan_training_backward", "op": "scan_backward", "type": "bf16", "gate": "sigmoid", "sequences": 8, "tokens": 8 * 4096, "channels": 2048, "packed": False},
        # the gradient over packed sequences in 32 bits, decays given as they are
        {"name": "scan_packed_backward", "op": "scan_backward", "type": "f32", "gate": "decay", "sequences": 19, "tokens": 4099, "channels": 769, "packed": True},
        # one new token for each running request, states in a pool of slots
        {"name": "scan_one_token", "op": "scan_step", "type": "bf16", "gate": "sigmoid", "requests": 48, "slots": 256, "channels": 2048},
        # the norm in front of a block in training: the residual stream takes the last block's output, then the norm
        {"name": "norm_training", "op": "norm", "type": "bf16", "norm": "rms", "order": "add_norm", "act": "none", "rows": 16384, "dim": 4096, "residual": True, "bias": False, "scale": False},
        # the gated norm behind a block for a few new tokens: latency
        {"name": "norm_few_tokens", "op": "norm", "type": "f16", "norm": "rms", "order": "norm_add", "act": "silu", "rows": 12, "dim": 2048, "residual": True, "bias": False, "scale": True},
        # the gradient of a gated norm with a learned scale of the residual branch
        {"name": "norm_gated_backward", "op": "norm_backward", "type": "bf16", "norm": "layer", "order": "norm_add", "act": "silu", "rows": 8192, "dim": 4096, "residual": True, "bias": True, "scale": True},
        # the projection into gates of a training batch: bias and activation, the activation's argument kept
        {"name": "product_training", "op": "product", "type": "bf16", "act": "silu", "rows": 8192, "out": 8192, "in": 4096, "bias": True, "residual": False, "keep": True},
        # the projection back onto the residual stream for a few new tokens: bound by the weights
        {"name": "product_few_tokens", "op": "product", "type": "f16", "act": "none", "rows": 5, "out": 4096, "in": 8192, "bias": True, "residual": True, "keep": False},
        # the gradient of a projection, odd sizes
        {"name": "product_backward", "op": "product_backward", "type": "bf16", "act": "silu", "rows": 4001, "out": 4096, "in": 2056, "bias": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width as models have them (a multiple of 64, or of 8) or, one time in four, any number."""
    n = _spread(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    return max(lo, n // step * step)


def draw(rng):
    op = rng.choice(("scan", "scan", "scan_backward", "scan_backward", "scan_step", "norm", "norm", "norm_backward", "product", "product", "product_backward"))
    kind = rng.choice(("f16", "bf16"))
    if op in ("scan", "scan_backward"):
        channels = _width(rng, 64, 4096)
        tokens = _spread(rng, 64, min(65536, (1 << 26) // channels))
        packed = rng.random() < 0.5
        sequences = _spread(rng, 1, max(1, min(64, tokens // 16)))
        if not packed:
            tokens = tokens // sequences * sequences
        return {"op": op, "type": rng.choice((kind, kind, kind, "f32")), "gate": rng.choice(("sigmoid", "sigmoid", "log", "decay")), "sequences": sequences, "tokens": tokens, "channels": channels, "packed": packed}
    if op == "scan_step":
        requests = _spread(rng, 1, 512)
        return {"op": op, "type": kind, "gate": rng.choice(("sigmoid", "log")), "requests": requests, "slots": requests + rng.randint(0, 300), "channels": _width(rng, 256, 8192)}
    if op in ("norm", "norm_backward"):
        dim = _width(rng, 128, 8192)
        rows = _spread(rng, 1 if op == "norm" else 16, (1 << 26) // dim if op == "norm" else (1 << 25) // dim)
        order = rng.choice(("add_norm", "norm_add"))
        residual = order == "norm_add" or rng.random() < 0.7
        return {"op": op, "type": rng.choice((kind, kind, kind, "f32")), "norm": rng.choice(("rms", "rms", "layer")), "order": order, "act": rng.choice(("none", "silu", "sigmoid")), "rows": rows, "dim": dim,
                "residual": residual, "bias": rng.random() < 0.3, "scale": residual and rng.random() < 0.5}
    rows, out, inner = _spread(rng, 1 if op == "product" else 64, 8192), _width(rng, 256, 8192), _width(rng, 256, 8192)
    while rows * out * inner > 8192 * 4096 * 4096 // (2 if op == "product_backward" else 1):
        rows = max(1, rows // 2)
    act = rng.choice(("none", "relu", "gelu", "silu", "sigmoid"))
    if op == "product_backward":
        return {"op": op, "type": kind, "act": act, "rows": rows, "out": out, "in": inner, "bias": rng.random() < 0.7}
    return {"op": op, "type": kind, "act": act, "rows": rows, "out": out, "in": inner, "bias": rng.random() < 0.7, "residual": rng.random() < 0.5, "keep": act != "none" and rng.random() < 0.4}


# ---- inputs -----------------------------------------------------------------------------------------------------


def _gates(gate, shape, gen):
    """Gates as a trained recurrence has them: most of the state is kept from token to token."""
    g = torch.randn(shape, generator=gen, device="cuda")
    if gate == "sigmoid":
        return g.mul_(1.5).add_(2.0)
    if gate == "log":
        return g.mul_(1.2).sub_(3.0).exp_().neg_()
    return g.mul_(1.5).add_(2.0).sigmoid_()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = TYPES[case["type"]]

    def normal(*shape, scale=1.0, mean=0.0, to=None):
        return torch.randn(shape, generator=gen, device="cuda").mul_(scale).add_(mean).to(to or dtype)

    st = {"case": case}
    op = case["op"]
    if op in ("scan", "scan_backward"):
        n, d, seqs = case["tokens"], case["channels"], case["sequences"]
        if case["packed"]:  # cut points anywhere: sequences of one token and empty ones among them
            cuts = torch.randint(0, n + 1, (seqs - 1,), generator=gen, device="cuda").sort().values
            offsets = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), n)]).to(torch.int32)
            st["offsets"], st["longest"] = offsets, int((offsets[1:] - offsets[:-1]).max())
            shape = (n, d)
        else:
            st["offsets"], st["longest"] = None, n // seqs
            shape = (seqs, n // seqs, d)
        st["x"] = normal(*shape)
        st["g"] = _gates(case["gate"], shape, gen).to(dtype)
        st["h0"] = normal(seqs, d, to=torch.float32)
        if op == "scan_backward":
            st["h"] = normal(*shape, scale=0.7)
            st["dh"] = normal(*shape)
            st["dh_last"] = normal(seqs, d, to=torch.float32)
    elif op == "scan_step":
        n, d = case["requests"], case["channels"]
        st["x"], st["g"] = normal(n, d), _gates(case["gate"], (n, d), gen).to(dtype)
        st["state"] = normal(case["slots"], d, to=torch.float32)
        st["new_state"] = st["state"].clone()
        st["slots"] = torch.randperm(case["slots"], generator=gen, device="cuda")[:n].to(torch.int32)
    elif op in ("norm", "norm_backward"):
        n, d = case["rows"], case["dim"]
        st["x"] = normal(n, d, mean=0.1)
        st["weight"] = normal(d, scale=0.2, mean=1.0)
        st["bias"] = normal(d, scale=0.2) if case["bias"] else None
        st["gate"] = normal(n, d) if case["act"] != "none" else None
        st["scale"] = normal(d, scale=0.3, mean=0.8) if case["scale"] else None
        st["residual"] = normal(n, d, scale=2.0) if case["residual"] else None
        if op == "norm_backward":
            st["dout"] = normal(n, d)
            adds = case["order"] == "add_norm" and case["residual"]
            st["z"] = normal(n, d, scale=2.0, mean=0.1) if adds else st["x"]
            st["dstream"] = normal(n, d) if adds else None
    else:
        m, n, k = case["rows"], case["out"], case["in"]
        st["A"] = normal(m, k)
        st["B"] = normal(n, k, scale=1.0 / math.sqrt(k))
        st["bias"] = normal(n, scale=0.3) if case["bias"] else None
        if op == "product":
            st["C"] = normal(m, n) if case["residual"] else None
        else:
            st["dD"] = normal(m, n)
            st["Z"] = normal(m, n) if case["act"] != "none" else None
    return st


# ---- the plain forms, in 32 bits --------------------------------------------------------------------------------


def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "gelu":  # the tanh form
        return 0.5 * z * (1.0 + torch.tanh(GELU_A * (z + GELU_B * z * z * z)))
    s = 1.0 / (1.0 + torch.exp(-z))
    return s if name == "sigmoid" else z * s


def _act_slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        t = torch.tanh(GELU_A * (z + GELU_B * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_A * (1.0 + 3.0 * GELU_B * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 - s) if name == "sigmoid" else s * (1.0 + z * (1.0 - s))


def _decays(gate, g):
    """a and 1 - a, the second without the cancellation of a subtraction."""
    if gate == "decay":
        return g, None
    if gate == "log":
        return torch.exp(g), None
    return 1.0 / (1.0 + torch.exp(-g)), 1.0 / (1.0 + torch.exp(g))


def _rows(st):
    """(index of the first row of each non-empty sequence, of its last row, the numbers of these sequences, of the empty ones)."""
    n, seqs = st["case"]["tokens"], st["case"]["sequences"]
    if st["offsets"] is None:
        first = torch.arange(seqs, device="cuda") * (n // seqs)
        which = torch.arange(seqs, device="cuda")
        return first, first + (n // seqs - 1), which
    lo, hi = st["offsets"][:-1].long(), st["offsets"][1:].long()
    which = torch.nonzero(hi > lo).reshape(-1)
    return lo[which], hi[which] - 1, which


def _doubling(A, B, longest):
    """y[t] = A[t] y[t-1] + B[t] down the rows, by steps of doubled stride (A is 0 where a sequence begins)."""
    step = 1
    while step < longest:
        upper = B[step:] + A[step:] * B[:-step]
        B = torch.cat([B[:step], upper])
        A = torch.cat([A[:step], A[step:] * A[:-step]])
        step *= 2
    return B


def _scan_plain(st):
    case, shape, dtype = st["case"], st["x"].shape, st["x"].dtype
    x, g = st["x"].reshape(-1, shape[-1]).float(), st["g"].reshape(-1, shape[-1]).float()
    a, keep = _decays(case["gate"], g)
    b = x if keep is None else keep * x
    first, last, which = _rows(st)
    b = b.index_add(0, first, a[first] * st["h0"][which])
    a = a.index_fill(0, first, 0.0)
    h = _doubling(a, b, st["longest"])
    h_last = st["h0"].clone()
    h_last[which] = h[last]
    return h.to(dtype).reshape(shape), h_last


def _scan_backward_plain(st):
    case, shape, dtype = st["case"], st["x"].shape, st["x"].dtype
    x, g, h, dh = (st[k].reshape(-1, shape[-1]).float() for k in ("x", "g", "h", "dh"))
    a, keep = _decays(case["gate"], g)
    first, last, which = _rows(st)
    after = torch.cat([a[1:], a[:1]]).index_fill(0, last, 0.0)
    delta = _doubling(after.flip(0), dh.index_add(0, last, st["dh_last"][which]).flip(0), st["longest"]).flip(0)
    before = torch.cat([h[:1], h[:-1]])
    before[first] = st["h0"][which]
    dh0 = st["dh_last"].clone()
    dh0[which] = a[first] * delta[first]
    if case["gate"] == "sigmoid":
        dx, dg = keep * delta, delta * (before - x) * a * keep
    else:
        dx, dg = delta, delta * before * (a if case["gate"] == "log" else 1.0)
    return dx.to(dtype).reshape(shape), dg.to(dtype).reshape(shape), dh0


def _step_plain(st):
    a, keep = _decays(st["case"]["gate"], st["g"].float())
    x = st["x"].float()
    at = st["slots"].long()
    h = a * st["state"][at] + (x if keep is None else keep * x)
    st["new_state"][at] = h
    return h.to(st["x"].dtype), st["new_state"]


def _normed(case, z):
    if case["norm"] == "layer":
        z = z - z.mean(-1, keepdim=True)
    return z, 1.0 / torch.sqrt((z * z).mean(-1, keepdim=True) + EPS)


def _norm_plain(st):
    case, dtype = st["case"], st["x"].dtype
    x = st["x"].float()
    s = st["scale"].float() if st["scale"] is not None else 1.0
    z = st["residual"].float() + s * x if case["order"] == "add_norm" and st["residual"] is not None else x
    c, rho = _normed(case, z)
    y = c * rho * st["weight"].float()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    if st["gate"] is not None:
        y = y * _act(case["act"], st["gate"].float())
    if case["order"] == "norm_add":
        return (st["residual"].float() + s * y).to(dtype)
    return (y.to(dtype), z.to(dtype)) if st["residual"] is not None else y.to(dtype)


def _norm_backward_plain(st):
    case, dtype = st["case"], st["x"].dtype
    w = st["weight"].float()
    dout = st["dout"].float()
    c, rho = _normed(case, st["z"].float())
    n = c * rho
    y = n * w if st["bias"] is None else n * w + st["bias"].float()
    got = {}
    s = st["scale"].float() if st["scale"] is not None else 1.0
    gate = st["gate"].float() if st["gate"] is not None else None
    f = 1.0 if gate is None else _act(case["act"], gate)
    if case["order"] == "norm_add":
        if st["scale"] is not None:
            got["dscale"] = (dout * y * f).sum(0)
        dout = dout * s
    if gate is not None:
        got["dgate"] = (dout * y * _act_slope(case["act"], gate)).to(dtype)
    dy = dout * f
    got["dweight"] = (dy * n).sum(0)
    if st["bias"] is not None:
        got["dbias"] = dy.sum(0)
    dn = dy * w
    inner = dn - n * (dn * n).mean(-1, keepdim=True)
    if case["norm"] == "layer":
        inner = inner - dn.mean(-1, keepdim=True)
    dz = rho * inner
    if st["dstream"] is not None:
        dz = dz + st["dstream"].float()
        got["dresidual"] = dz.to(dtype)
        if st["scale"] is not None:
            got["dscale"] = (dz * st["x"].float()).sum(0)
        dz = dz * s
    got["dx"] = dz.to(dtype)
    return got


def _product_plain(st):
    case, dtype = st["case"], st["A"].dtype
    z = st["A"].float() @ st["B"].float().t()
    if st["bias"] is not None:
        z = z + st["bias"].float()
    d = _act(case["act"], z)
    if st["C"] is not None:
        d = d + st["C"].float()
    return (d.to(dtype), z.to(dtype)) if case["keep"] else d.to(dtype)


def _product_backward_plain(st):
    case, dtype = st["case"], st["A"].dtype
    dz = st["dD"].float()
    if st["Z"] is not None:
        dz = dz * _act_slope(case["act"], st["Z"].float())
    got = {"dA": (dz @ st["B"].float()).to(dtype), "dB": (dz.t() @ st["A"].float()).to(dtype)}
    if case["bias"]:
        got["dbias"] = dz.sum(0)
    return got


# ---- one pass ---------------------------------------------------------------------------------------------------


def run(state):
    st, case = state, state["case"]
    op = case["op"]
    if own:
        import tcu_scope_amd as tcu

        if op == "scan":
            return tcu.gated_scan(st["x"], st["g"], gate=case["gate"], h0=st["h0"], offsets=st["offsets"])
        if op == "scan_backward":
            return tcu.gated_scan_backward(st["dh"], st["x"], st["g"], st["h"], gate=case["gate"], h0=st["h0"], dh_last=st["dh_last"], offsets=st["offsets"])
        if op == "scan_step":
            return tcu.gated_scan_step(st["x"], st["g"], st["state"], gate=case["gate"], slots=st["slots"], new_state=st["new_state"]), st["new_state"]
        if op == "norm":
            return tcu.fused_norm(st["x"], st["weight"], bias=st["bias"], residual=st["residual"], gate=st["gate"], channel_scale=st["scale"], norm=case["norm"], order=case["order"], activation=case["act"], eps=EPS)
        if op == "norm_backward":
            return tcu.fused_norm_backward(st["dout"], st["z"], st["weight"], bias=st["bias"], gate=st["gate"], channel_scale=st["scale"], x=st["x"], dresidual_out=st["dstream"], norm=case["norm"], order=case["order"],
                                           activation=case["act"], eps=EPS)
        if op == "product":
            return tcu.fused_gemm(st["A"], st["B"], bias=st["bias"], activation=case["act"], C=st["C"], return_preactivation=case["keep"])
        return tcu.fused_gemm_backward(st["dD"], st["A"], st["B"], Z=st["Z"], activation=case["act"], bias_gradient=case["bias"])
    plain = {"scan": _scan_plain, "scan_backward": _scan_backward_plain, "scan_step": _step_plain, "norm": _norm_plain, "norm_backward": _norm_backward_plain, "product": _product_plain,
             "product_backward": _product_backward_plain}
    return plain[op](st)


def work(case):
    """Each input read once, each output written once; a flop is an addition or a multiplication, an exponential counts as one."""
    e, op = BYTES[case["type"]], case["op"]
    if op in ("scan", "scan_backward"):
        n, d, s = case["tokens"], case["channels"], case["sequences"]
        sig = case["gate"] == "sigmoid"
        streams = 3 if op == "scan" else (6 if sig else 5)  # x g -> h; dh g h (x) -> dx dg
        return {"bytes": streams * n * d * e + 2 * s * d * 4 + (s * d * 4 if op != "scan" else 0), "flops": (6 if op == "scan" else 10) * n * d}
    if op == "scan_step":
        n, d = case["requests"], case["channels"]
        return {"bytes": 3 * n * d * e + 2 * n * d * 4 + 4 * n, "flops": 6 * n * d}
    if op in ("norm", "norm_backward"):
        n, d = case["rows"], case["dim"]
        gate, res = case["act"] != "none", case["residual"]
        adds = case["order"] == "add_norm" and res
        if op == "norm":
            streams = 2 + gate + res + adds
        else:  # dout z -> dx; gate -> dgate; the stream's gradient in and out, x for the scale's
            streams = 3 + 2 * gate + 2 * adds + (adds and case["scale"])
        vectors = 1 + case["bias"] + case["scale"]
        return {"bytes": streams * n * d * e + vectors * d * (e + (4 if op == "norm_backward" else 0)), "flops": (8 if op == "norm" else 20) * n * d}
    m, n, k = case["rows"], case["out"], case["in"]
    if op == "product":
        return {"bytes": e * (m * k + n * k + m * n * (1 + case["residual"] + case["keep"]) + n * case["bias"]), "flops": 2 * m * n * k}
    return {"bytes": e * (2 * m * k + 2 * n * k + m * n * (2 if case["act"] != "none" else 1)) + 4 * n * case["bias"], "flops": 4 * m * n * k}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------


def _exact_gate(gate, g):
    if gate == "decay":
        return g, torch.ones_like(g)
    if gate == "log":
        return g.exp(), torch.ones_like(g)
    return torch.sigmoid(g), torch.sigmoid(-g)


def _exact_segments(st):
    n, seqs = st["case"]["tokens"], st["case"]["sequences"]
    if st["offsets"] is None:
        return [(j * (n // seqs), (j + 1) * (n // seqs)) for j in range(seqs)]
    o = st["offsets"].tolist()
    return list(zip(o[:-1], o[1:]))


def _exact_act(name, z):
    """The activation and its slope, the slope by way of other identities than the plain form's."""
    z = z.detach().requires_grad_(True)
    f = {"none": lambda v: v * 1.0, "relu": torch.relu, "gelu": lambda v: torch.nn.functional.gelu(v, approximate="tanh"), "silu": lambda v: v * torch.sigmoid(v), "sigmoid": torch.sigmoid}[name](z)
    (slope,) = torch.autograd.grad(f.sum(), z)
    return f.detach(), slope


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "scan":
        shape = st["x"].shape
        x, g = st["x"].double().reshape(-1, shape[-1]), st["g"].double().reshape(-1, shape[-1])
        a, keep = _exact_gate(case["gate"], g)
        b = keep * x
        out, last = torch.empty_like(x), st["h0"].double()
        if st["offsets"] is None:  # all sequences side by side
            av, bv, ov = (t.view(shape) for t in (a, b, out))
            for t in range(shape[1]):
                last = torch.addcmul(bv[:, t], av[:, t], last)
                ov[:, t] = last
        else:
            for j, (lo, hi) in enumerate(_exact_segments(st)):
                h = last[j]
                for t in range(lo, hi):
                    h = torch.addcmul(b[t], a[t], h, out=out[t])
                last[j] = h
        return out.view(shape), last
    if op == "scan_backward":
        shape = st["x"].shape
        x, g, h, dh = (st[k].double().reshape(-1, shape[-1]) for k in ("x", "g", "h", "dh"))
        a, keep = _exact_gate(case["gate"], g)
        delta, before = torch.empty_like(x), torch.empty_like(x)
        carry = st["dh_last"].double()
        h0 = st["h0"].double()
        if st["offsets"] is None:
            av, dv, sv, bv, hv = (t.view(shape) for t in (a, dh, delta, before, h))
            for t in reversed(range(shape[1])):
                sv[:, t] = dv[:, t] + carry
                carry = av[:, t] * sv[:, t]
            bv[:, 1:] = hv[:, :-1]
            bv[:, 0] = h0
        else:
            for j, (lo, hi) in enumerate(_exact_segments(st)):
                u = carry[j].clone()
                for t in reversed(range(lo, hi)):
                    torch.add(dh[t], u, out=delta[t])
                    u = a[t] * delta[t]
                carry[j] = u
                if hi > lo:
                    before[lo] = h0[j]
                    before[lo + 1:hi] = h[lo:hi - 1]
        slope = {"decay": lambda: before, "log": lambda: before * a, "sigmoid": lambda: (before - x) * a * keep}[case["gate"]]()
        return (delta * keep).view(shape), (delta * slope).view(shape), carry
    if op == "scan_step":
        a, keep = _exact_gate(case["gate"], st["g"].double())
        new = st["state"].double()
        at = st["slots"].long()
        new[at] = a * new[at] + keep * st["x"].double()
        return new[at], new
    if op in ("norm", "norm_backward"):
        names = ("x", "weight", "bias", "gate", "scale", "residual")
        v = {k: (st[k].double().requires_grad_(True) if st[k] is not None else None) for k in names}
        s = v["scale"] if v["scale"] is not None else 1.0
        adds = case["order"] == "add_norm" and case["residual"]
        back = op == "norm_backward"
        z = st["z"].double().requires_grad_(True) if back and adds else (v["residual"] + s * v["x"] if adds else v["x"])
        if case["norm"] == "layer":
            y = (z - z.mean(-1, keepdim=True)) / (z.var(-1, unbiased=False, keepdim=True) + EPS).sqrt()
        else:
            y = z / (z.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        y = y * v["weight"]
        if v["bias"] is not None:
            y = y + v["bias"]
        if v["gate"] is not None:
            y = y * (torch.sigmoid(v["gate"]) * (v["gate"] if case["act"] == "silu" else 1.0))
        out = v["residual"] + s * y if case["order"] == "norm_add" else y
        if not back:
            return (out.detach(), z.detach()) if adds else out.detach()
        wrt = {"dweight": v["weight"], "dbias": v["bias"], "dgate": v["gate"]}
        wrt["dz"] = z if adds else v["x"]
        if case["order"] == "norm_add":
            wrt["dscale"] = v["scale"]
        wrt = {k: t for k, t in wrt.items() if t is not None}
        got = dict(zip(wrt, torch.autograd.grad(out, list(wrt.values()), st["dout"].double())))
        dz = got.pop("dz")
        if adds:
            dz = dz + st["dstream"].double()
            got["dresidual"] = dz
            if v["scale"] is not None:
                got["dscale"] = (dz * st["x"].double()).sum(0)
                dz = dz * st["scale"].double()
        got["dx"] = dz
        return got
    if op == "product":
        z = torch.mm(st["A"].double(), st["B"].double().t().contiguous())
        if st["bias"] is not None:
            z += st["bias"].double()
        d = _exact_act(case["act"], z)[0]
        if st["C"] is not None:
            d = d + st["C"].double()
        return (d, z) if case["keep"] else d
    dz = st["dD"].double()
    if st["Z"] is not None:
        dz = dz * _exact_act(case["act"], st["Z"].double())[1]
    got = {"dA": torch.mm(dz, st["B"].double()), "dB": torch.mm(dz.t().contiguous(), st["A"].double())}
    if case["bias"]:
        got["dbias"] = dz.sum(0)
    return got
