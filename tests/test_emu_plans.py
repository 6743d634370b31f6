"""The sizes of tests/block_shapes.py take the forms that they are listed for."""
import ctypes

import pytest

from block_shapes import GRADIENTS, PRODUCTS, SCANS
from test_emu_block import DTYPES, Shape, ci, emu, sz  # noqa: F401


@pytest.fixture(scope="module")
def tile(emu):
    emu.emu_gemm_tile.argtypes = [sz, sz, sz, ci, ctypes.POINTER(sz)]

    def of(M, N, K, layout):
        splits = sz(0)
        w8 = emu.emu_gemm_tile(M, N, K, layout, ctypes.byref(splits))
        return w8, splits.value > 1

    return of


def test_products(tile):
    seen = set()
    for M, N, K, w8, shared in PRODUCTS:
        assert tile(M, N, K, 0) == (w8, shared), (M, N, K)
        seen.add((w8, shared, K % 64 != 0))
    assert len(seen) == 12  # three tiles, alone or sharing, with and without a tail


def test_gradients(tile):
    seen = set()
    for M, N, K, a, b in GRADIENTS:
        assert K % 8 == 0 and M >= 64 and N >= 64  # the operands are taken as they lie
        if a:
            assert tile(M, K, N, 1) == a, (M, N, K)
            seen.add((1, *a))
        if b:
            assert tile(N, K, M, 2) == b, (M, N, K)
            seen.add((2, *b))
    assert len(seen) == 12


def test_scans(emu):
    emu.emu_scan_threads.argtypes = [ctypes.POINTER(Shape), ci]
    for rows, channels, dtype, seqs in SCANS:
        packed = isinstance(seqs, list)
        s = Shape(dtype=DTYPES[dtype], channels=channels, num_rows=rows, num_sequences=len(seqs) - 1 if packed else seqs, sequence_length=0 if packed else rows // seqs)
        if packed:
            s.d_offsets, s.offset_bits = 64, 32
        assert emu.emu_scan_threads(ctypes.byref(s), 0) == 256 and emu.emu_scan_threads(ctypes.byref(s), 1) == 256, (rows, channels)
    small = Shape(dtype=1, channels=64, num_rows=1000, num_sequences=1, sequence_length=1000)
    assert emu.emu_scan_threads(ctypes.byref(small), 0) == 512
