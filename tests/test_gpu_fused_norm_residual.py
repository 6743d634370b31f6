"""The residual's gradient of a norm whose written stream nothing else uses (the last norm of a model), on the GPU."""
import numpy as np
import pytest

import block_reference as ref
from test_gpu_fused_norm import EPS, tcu  # noqa: F401
from test_gpu_gated_scan import dev, host, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,dim,actn,with_scale", [(70, 256, None, True), (33, 1001, "silu", True), (12, 6000, None, False)])
def test_residual_gradient_without_a_stream_gradient(tcu, dtype, rows, dim, actn, with_scale):
    rng = np.random.default_rng(dim)
    mat = lambda: rounded(rng.standard_normal((rows, dim)), dtype)
    x, z, dout, gate = mat(), mat(), mat(), mat() if actn else None
    w = rounded(rng.standard_normal(dim) * 0.3 + 1, dtype)
    cs = rounded(rng.standard_normal(dim) * 0.3, dtype) if with_scale else None
    if with_scale:
        cs[::3] = 0.0  # there the residual's gradient does not follow from dx
    d = lambda v: None if v is None else dev(v, dtype)
    args, kw = (d(dout), d(z), d(w)), dict(gate=d(gate), scale=0.5, channel_scale=d(cs), x=d(x), norm="rms", order="add_norm", activation=actn or "none", eps=EPS)
    got = tcu.fused_norm_backward(*args, residual_gradient=True, **kw)
    s = 0.5 * (cs if with_scale else np.ones(dim))
    want, err = ref.norm_backward("rms", "add_norm", actn, dout, z, gate, w, np.zeros(dim), s, EPS, x, None)
    for name in ("dx", "dresidual", "dweight"):
        ref.check(host(got[name]), want[name], err[name], "f32" if name == "dweight" else dtype, name)
    assert "dresidual" not in tcu.fused_norm_backward(*args, **kw)
    assert "dresidual" not in tcu.fused_norm_backward(*args, dresidual_out=d(x), residual_gradient=False, **kw)
    with pytest.raises(tcu.TcuError, match="d_dout itself"):
        tcu.fused_norm_backward(*args, residual_gradient=True, **{**kw, "order": "norm_add", "x": None})
