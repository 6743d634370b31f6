"""Sizes whose launches would have 2^32 threads or more are refused before anything is launched (asked for the workspace, which
goes by the same rules)."""
import ctypes

from test_emu_block import GemmShape, Shape, emu, gemm_emu, sz  # noqa: F401

MOST = (1 << 31) - 4096


def test_gated_scan(emu):
    need = sz(0)
    fwd = lambda **k: emu.emu_gated_scan(ctypes.byref(Shape(dtype=0, gate=0, num_sequences=1, sequence_length=k["num_rows"], **k)), None, 1, None, 1, None, 1, None, None, None, ctypes.byref(need))
    back = lambda **k: emu.emu_gated_scan_backward(ctypes.byref(Shape(dtype=0, gate=0, num_sequences=1, sequence_length=k["num_rows"], **k)), None, 1, None, 1, None, 1, None, 1, None, None, None, 1, None, 1, None, None, ctypes.byref(need))
    assert fwd(channels=1, num_rows=MOST) == 0 and fwd(channels=129, num_rows=MOST) == 2  # 128 rows x 128 channels to 256 threads
    assert b"tiles" in emu.emu_last_error()
    assert back(channels=1, num_rows=(1 << 30) - 64) == 0 and back(channels=1, num_rows=1 << 30) == 2 and back(channels=256, num_rows=1 << 29) == 2
    buf = (ctypes.c_char * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    step = lambda rows, channels: emu.emu_gated_scan_step(0, 0, channels, rows, p, channels, p, channels, p, channels, p, p, 1, p, 0)
    assert step(1 << 26, 8) == 2 and step(1 << 25, 1024) == 2 and b"blocks" in emu.emu_last_error()


def test_fused_product(emu):
    emu = gemm_emu(emu)
    need = sz(0)
    fwd = lambda M, N, K: emu.emu_fused_gemm(ctypes.byref(GemmShape(0, 0, M, N, K, 0.0)), None, K, None, K, None, None, 0, None, N, None, 0, None, ctypes.byref(need))
    assert fwd(4, 1 << 26, 8) == 0 and fwd(4, 1 << 27, 8) == 2 and b"tiles" in emu.emu_last_error()  # 16 columns to 512 threads
    assert fwd(1 << 17, 1 << 18, 64) == 2 and b"2^35" in emu.emu_last_error()
    assert fwd((1 << 31) - 1, 1, 8) == 2 and fwd(1 << 30, 1, 8) == 0
    assert fwd(1 << 22, 40, 1 << 14) == 0 and fwd(1 << 22, 40, (1 << 14) + 1) == 2  # A would be copied to rows of whole chunks
    back = lambda M, N, K: emu.emu_fused_gemm_backward(ctypes.byref(GemmShape(0, 0, M, N, K, 0.0)), *[None, 0] * 4, 16, K, 32, K, None, None, ctypes.byref(need))
    assert back(1 << 17, (1 << 18) - 64, 1 << 16) == 0 and back(1 << 17, (1 << 18) - 64, 1 << 17) == 2  # three matrices in one launch
