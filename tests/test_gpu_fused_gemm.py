"""The fused product and its gradient on the GPU, against the 64-bit formulas and bounds of tests/block_reference.py."""
import numpy as np
import pytest

import block_reference as ref
from test_gpu_gated_scan import dev, host, rounded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tcu():
    import tcu_scope_amd as t

    t.init(0)
    return t


def operands(rng, dtype, M, N, K):
    return rounded(rng.standard_normal((M, K)), dtype), rounded(rng.standard_normal((N, K)) / max(K, 1) ** 0.5, dtype), rounded(rng.standard_normal(N), dtype), rounded(rng.standard_normal((M, N)), dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,stride,name", [(1, 1, 1, None, "silu"), (1, 4096, 1024, None, "none"), (5, 250, 8200, None, "gelu"), (16, 1000, 777, None, "relu"), (33, 64, 4096, 4104, "sigmoid"), (64, 513, 320, None, "silu"),
                                               (65, 128, 64, None, "silu"), (100, 2000, 2051, None, "gelu"), (700, 520, 136, 144, "relu"), (129, 130, 8192, None, "none"), (2000, 4100, 200, None, "silu"), (2049, 4096, 64, None, "sigmoid"),
                                               (4000, 2050, 130, None, "gelu")])
def test_product(tcu, dtype, M, N, K, stride, name):
    import torch

    rng = np.random.default_rng(M + N + K)
    A, B, bias, C = operands(rng, dtype, M, N, K)
    tA, tB, tb, tC = dev(A, dtype, stride), dev(B, dtype), dev(bias, dtype), dev(C, dtype)
    d, z, ed, ez = ref.product(A, B, bias, name, C, 0.5)
    D, Z = tcu.fused_gemm(tA, tB, tb, name, C=tC, beta=0.5, return_preactivation=True)
    ref.check(host(D), d, ed, dtype, "D")
    ref.check(host(Z), z, ez, dtype, "Z")
    again = tcu.fused_gemm(tA, tB, tb, name, C=tC, beta=0.5)
    assert torch.equal(again, D)
    plain = tcu.fused_gemm(tA, tB, activation=name)
    d, _, ed, _ = ref.product(A, B, np.zeros(N), name, None, 0.0)
    ref.check(host(plain), d, ed, dtype, "D without bias and C")
    tcu.fused_gemm(tA, tB, tb, name, C=tC, beta=0.5, out=tC)
    assert torch.equal(tC, D)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,stride,name", [(1, 1, 1, None, "silu"), (200, 520, 264, None, "silu"), (333, 77, 129, None, "gelu"), (64, 2048, 512, None, "none"), (1000, 96, 40, 48, "none"), (2100, 600, 4097, None, "relu"), (4111, 512, 64, None, "sigmoid"), (31, 700, 1032, None, "gelu"), (130, 2120, 1064, 1072, "none"),
                                               (1100, 4096, 4096, 4104, "silu")])
def test_gradient(tcu, dtype, M, N, K, stride, name):
    import torch

    rng = np.random.default_rng(M + N)
    A, B, _, dD = operands(rng, dtype, M, N, K)
    Z = rounded(rng.standard_normal((M, N)), dtype) if name != "none" else None
    tA, tB, tD, tZ = dev(A, dtype, stride), dev(B, dtype), dev(dD, dtype), dev(Z, dtype) if Z is not None else None
    want, err = ref.product_backward(dD, A, B, Z, name, dtype)
    got = tcu.fused_gemm_backward(tD, tA, tB, tZ, name)
    for k, t in got.items():
        ref.check(host(t), want[k], err[k], "f32" if k == "dbias" else dtype, k)
    for k in got:
        one = tcu.fused_gemm_backward(tD, tA, tB, tZ, name, bias_gradient=k == "dbias", input_gradient=k == "dA", weight_gradient=k == "dB")
        assert list(one) == [k] and torch.equal(one[k], got[k])


def test_infinities_stay_in_their_rows(tcu):
    """What lies behind a ragged K or beside a ragged tile does not reach a result: only the row and column with an infinity show one."""
    import torch

    for M, N, K in ((5, 48, 100), (130, 140, 100), (300, 200, 1000)):
        A, B = torch.randn(M, K + 28, device="cuda").half(), torch.randn(N, K + 28, device="cuda").half()
        A[:, K:] = float("nan")
        B[:, K:] = float("inf")
        A[M - 1, 0] = float("inf")
        D = tcu.fused_gemm(A[:, :K], B[:, :K])
        assert D[:M - 1].isfinite().all() and not D[M - 1].isfinite().any()


def test_stream_graph_and_empty(tcu):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()
    for M in (3, 300):
        A, B, b, dD = mk(M, 1001), mk(700, 1001), mk(700), mk(M, 700)
        want, z = tcu.fused_gemm(A, B, b, "silu", return_preactivation=True)
        dwant = tcu.fused_gemm_backward(dD, A, B, z, "silu")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = tcu.fused_gemm(A, B, b, "silu", stream=s)
        s.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gD, gz = tcu.fused_gemm(A, B, b, "silu", return_preactivation=True)
            gd = tcu.fused_gemm_backward(dD, A, B, gz, "silu")
        for _ in range(3):
            gD.zero_()
            graph.replay()
            assert torch.equal(tcu.fused_gemm(A, B, b, "silu"), want)
            torch.cuda.synchronize()
            assert torch.equal(gD, want) and all(torch.equal(gd[k], dwant[k]) for k in dwant)
    assert tcu.fused_gemm(mk(0, 8), mk(16, 8)).shape == (0, 16)
    got = tcu.fused_gemm_backward(mk(0, 16), mk(0, 8), mk(16, 8))
    assert (got["dB"] == 0).all() and (got["dbias"] == 0).all()


def test_refusals(tcu):
    import torch

    a, b = torch.zeros(4, 64, device="cuda", dtype=torch.float16), torch.zeros(32, 64, device="cuda", dtype=torch.float16)
    for call, kind, words in [
        (lambda: tcu.fused_gemm(a, b[:, :32]), ValueError, "Bt must be"),
        (lambda: tcu.fused_gemm(a, b.bfloat16()), ValueError, "type and device"),
        (lambda: tcu.fused_gemm(a.float(), b.float()), tcu.TcuError, "TCU_F16 or TCU_BF16"),
        (lambda: tcu.fused_gemm(a, b, bias=b[0]), ValueError, "bias"),
        (lambda: tcu.fused_gemm(a, b, C=a), ValueError, "C must be 4 x 32"),
        (lambda: tcu.fused_gemm(a, b, activation="tanh"), ValueError, "relu"),
        (lambda: tcu.fused_gemm(a, b, workspace=torch.empty(8, device="cuda")), tcu.TcuError, "workspace"),
        (lambda: tcu.fused_gemm_backward(torch.zeros(4, 32, device="cuda", dtype=torch.float16), a, b, activation="silu"), tcu.TcuError, "needs d_Z"),
    ]:
        with pytest.raises(kind, match=words):
            call()
