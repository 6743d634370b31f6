"""Gates above 1 on the GPU: products of gates that pass the range of fp32 over states of zero."""
import numpy as np
import pytest

import block_reference as ref
from test_gpu_gated_scan import dev, host, rounded, tcu  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,channels", [(300, 24), (5000, 136), (70000, 40)])
def test_zeros_under_growing_gates(tcu, dtype, rows, channels):
    """Even channels: x = 0 up to the last rows under a = e^0.5, odd ones ordinary; then the gradient with dh = 0 but in the first rows."""
    rng = np.random.default_rng(rows)
    x, g = rounded(rng.standard_normal((rows, channels)), dtype), rounded(-np.exp(rng.standard_normal((rows, channels)) * 1.2 - 3), dtype)
    x[:-20, ::2], g[:-20, ::2] = 0.0, 0.5
    h0 = np.zeros((1, channels))
    h, last = tcu.gated_scan(dev(x, dtype), dev(g, dtype), "log")
    wh, wl, e, el = ref.scan("log", x, g, [0, rows], h0)
    ref.check(host(h), wh, e, dtype, "h")
    ref.check(host(last), wl, el, "f32", "h_last")
    x, g = np.ascontiguousarray(x[::-1]), np.ascontiguousarray(g[::-1])
    dx, dg, d0 = tcu.gated_scan_backward(dev(x, dtype), None, dev(g, dtype), dev(x, dtype), "log")
    (wx, wg, w0), (ex, eg, e0) = ref.scan_backward("log", x, g, x, x, [0, rows], h0, h0)
    ref.check(host(dx), wx, ex, dtype, "dx")
    ref.check(host(dg), wg, eg, dtype, "dg")
    ref.check(host(d0), w0, e0, "f32", "dh0")
