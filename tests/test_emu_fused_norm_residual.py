"""The residual's gradient without a gradient of the written stream, on the CPU emulator."""
import ctypes

import numpy as np
import pytest

import block_reference as ref
from test_emu_block import ACTS, DTYPES, EPS, NULL, Matrix, NormShape, emu, norm_emu, operand, vector, workspace_for  # noqa: F401


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,dim,gap,actn,with_scale", [(3, 64, 0, None, True), (4, 100, 3, "silu", True), (2, 2056, 0, None, False)])
def test_residual_gradient_without_a_stream_gradient(emu, dtype, rows, dim, gap, actn, with_scale):
    emu = norm_emu(emu)
    rng = np.random.default_rng(dim)
    f = lambda v: ref.to_f64(ref.to_bits(v, dtype), dtype)
    mat = lambda: f(rng.standard_normal((rows, dim)))
    z, dout, gate = mat(), mat(), mat() if actn else None
    w, cs = f(rng.standard_normal(dim)), f(rng.standard_normal(dim)) if with_scale else None
    mz, md, mg = Matrix(z, dtype, dim + gap), Matrix(dout, dtype), Matrix(gate, dtype) if actn else None
    mdx, mdr = Matrix(z, dtype), Matrix(z, dtype, dim + gap)
    vw, vc = vector(w, dtype), vector(cs, dtype) if with_scale else None
    shape = NormShape(DTYPES[dtype], 0, 0, ACTS[actn or "none"], rows, dim, EPS, 0.5)
    call = lambda ws, need: emu.emu_fused_norm_backward(ctypes.byref(shape), *operand(md), *operand(mz), *operand(mg), vw.ctypes.data, None, vc.ctypes.data if with_scale else None, *NULL, *NULL, *operand(mdx), *NULL,
                                                        *operand(mdr), None, None, None, ws, need)
    kept, ws, have = workspace_for(call)
    assert call(ws, ctypes.byref(have)) == 0, emu.emu_last_error()
    s = 0.5 * (cs if with_scale else np.ones(dim))
    got, err = ref.norm_backward("rms", "add_norm", actn, dout, z, gate, w, np.zeros(dim), s, EPS, None, None)
    ref.check(mdx.get(), got["dx"], err["dx"], dtype, "dx")
    ref.check(mdr.get(), got["dresidual"], err["dresidual"], dtype, "dresidual")
    assert mdr.untouched_between()
