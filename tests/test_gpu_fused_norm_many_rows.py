"""More rows than one launch of the fused norm takes, on the GPU."""
import pytest

from test_gpu_fused_norm import tcu  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim,stride", [((1 << 22) + 5, 16, 24), ((1 << 21) + 1, 600, 600), ((1 << 26) + 3, 8, 8)])
def test_every_row_as_in_a_call_of_its_own(tcu, rows, dim, stride):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(1)
    mk = lambda width: torch.randn(rows, width, generator=gen, device="cuda", dtype=torch.bfloat16)[:, :dim]
    x, r = mk(stride), mk(dim)
    w = mk(dim)[0].clone()
    gate = mk(dim) if rows < 1 << 23 else None
    out, z = tcu.fused_norm(x, w, residual=r, gate=gate)
    step = (1 << 21) // 3  # slices whose ends are no ends of a launch
    for lo in range(0, rows, step):
        part = slice(lo, min(lo + step, rows))
        o, zz = tcu.fused_norm(x[part], w, residual=r[part], gate=None if gate is None else gate[part])
        assert torch.equal(out[part], o) and torch.equal(z[part], zz)
    if gate is None:
        got = tcu.fused_norm(x, w, order="norm_add", residual=r, out=x)  # in the place of the input
        assert got is x
