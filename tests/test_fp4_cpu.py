"""Microscaled 4-bit matrices and clipping, what needs no GPU: sizes, refusals of the C entries and of the PyTorch door, and the reference that the GPU
tests compare with."""
import ctypes as C
import importlib

import numpy as np
import pytest

import fp4_reference as ref

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


@pytest.mark.parametrize("fmt", [ref.MXFP4, ref.NVFP4])
@pytest.mark.parametrize("rows,cols", [(0, 1), (1, 1), (1, 16), (1, 33), (127, 64), (129, 65), (4096, 14336), (70000, 5), (5, 70000)])
def test_packed_bytes(lib, ops, fmt, rows, cols):
    assert lib.bsq_fp4_packed_bytes(fmt, rows, cols) == ref.packed_bytes(rows, cols, fmt) == ops._packed_bytes(fmt, rows, cols)


def test_sizes_that_do_not_exist(lib):
    assert lib.bsq_fp4_packed_bytes(7, 4, 4) == 0 and lib.bsq_fp4_packed_bytes(8, 4, 0) == 0
    assert lib.bsq_fp4_packed_bytes(9, 1 << 31, 4) == 0 and lib.bsq_fp4_packed_bytes(9, 4, 1 << 31) == 0


def test_reference_rounds_to_even_and_saturates():
    x = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.0001, 6.0, 7.9, -0.25, -0.75, -5.5, 0.0, 4.0, 0.2501] + [0] * 16])
    codes, byte, g = ref.quantize(x, ref.MXFP4)
    assert byte[0, 0] == 127 and list(codes[0, :16]) == [0, 2, 2, 4, 4, 6, 6, 7, 7, 7, 8, 10, 15, 0, 6, 1]


def test_reference_round_trip_of_its_own_values():
    rng = np.random.default_rng(3)
    for fmt in (ref.MXFP4, ref.NVFP4):
        x = rng.standard_normal((5, 70))
        v = ref.values(*ref.quantize(x, fmt), fmt, 70)
        assert np.max(np.abs(v - x) / np.abs(x).max()) < 0.26       # (half the widest step, 4 to 6, of a block's largest, and what saturates)


P = C.c_void_p


def refused(f, *args):
    return f(*args) == 1


def test_c_entries_refuse(lib):
    """Every call below is turned down on the host; no pointer is looked at."""
    a, odd, f = 4096, 4097, lib
    q = f.bsq_fp4_quantize
    ok = [9, a, 2, 1024, 64, 64, None, a, a, None]

    def but(base, i, v):
        args = list(base)
        args[i] = v
        return args
    for i, v in ((0, 7), (0, 10), (1, None), (1, odd), (2, 3), (2, -1), (3, 1 << 31), (4, 0), (4, 1 << 31), (5, 63), (7, None), (7, a + 8), (8, None), (8, odd)):
        assert refused(q, *but(ok, i, v)), (i, v)
    ok = [9, a, 4, 64, a, 2, 64, None]
    for i, v in ((0, 7), (1, None), (1, a + 8), (2, 1 << 31), (3, 0), (4, None), (4, odd), (5, 5), (6, 63)):
        assert refused(f.bsq_fp4_dequantize, *but(ok, i, v)), (i, v)
    ok = [9, a, 4, a, 8, 64, a, 2, 8, None, None]
    for i, v in ((0, 0), (1, None), (1, a + 4), (2, 1 << 31), (3, None), (4, 1 << 31), (5, 0), (6, None), (6, odd), (7, 9), (8, 7)):
        assert refused(f.bsq_fp4_matmul, *but(ok, i, v)), (i, v)
    ok = [9, a, 4, 8, a, 8, 64, a, 2, 64, a, None, None]
    for i, v in ((0, 0), (1, None), (1, odd), (2, 1 << 31), (3, 7), (4, None), (4, a + 4), (5, 1 << 31), (6, 0), (7, None), (8, 4), (9, 63)):
        assert refused(f.bsq_fp4_grad_input, *but(ok, i, v)), (i, v)
    assert refused(f.bsq_fp4_grad_input, 9, a + 2, 4, 8, a, 8, 64, a, 2, 64, None, None, None)          # rows off 16 bytes need scratch
    assert refused(f.bsq_fp4_grad_input, 9, a, 4, 9, a, 9, 64, a, 2, 64, a + 8, None, None)
    ok = [9, a, 4, 8, 8, a, 64, a, 2, 64, a, None, None]
    for i, v in ((0, 0), (1, None), (4, 7), (5, None), (6, 0), (7, None), (8, 4), (9, 63), (3, 1 << 31)):
        assert refused(f.bsq_fp4_grad_weight, *but(ok, i, v)), (i, v)


def test_scratch_of_quantisation(lib):
    f = lib.bsq_fp4_scratch_bytes
    assert f(8, 0, 4096, 4096) == 0 and f(9, 2, 1, 4096) == 0 and f(9, 2, 8, 4096) == 0 and f(9, 2, 9, 4096) == 4096 and f(9, 0, 8, 4096) == 4096 and f(7, 0, 4096, 64) == 0


def test_scratch_of_gradients(lib):
    f = lib.bsq_fp4_grad_scratch_bytes
    assert f(4096, 10, 64, 64) == 0 and f(4096, 1, 7, 7) == 0
    assert f(4096, 10, 63, 63) == 10 * 64 * 2 and f(4098, 10, 64, 64) == 10 * 64 * 2 and f(4098, 1, 7, 7) == 16


def call_norm(lib, ptrs, counts, types, outs, max_norm=1.0, kind=2, norm=8192, scratch=16384):
    n = len(ptrs)
    arr = (P * n)(*ptrs) if n else None
    return lib.bsq_grad_norm_clip(arr, (C.c_uint64 * n)(*counts) if n else None, (C.c_int * n)(*types) if n else None, n,
                                  None if outs is None else (P * n)(*outs), max_norm, kind, norm, scratch, None)


def test_norm_entry_refuses(lib):
    a = 1 << 20
    assert call_norm(lib, [a], [4], [3], None) == 1                                  # type
    assert call_norm(lib, [None], [4], [0], None) == 1 and call_norm(lib, [a + 2], [4], [0], None) == 1
    assert call_norm(lib, [a], [4], [0], [None]) == 1 and call_norm(lib, [a], [4], [0], [a + 1]) == 1
    assert call_norm(lib, [a], [4], [0], [a], max_norm=-1.0) == 1 and call_norm(lib, [a], [4], [0], [a], max_norm=float("nan")) == 1
    assert call_norm(lib, [a], [4], [0], None, kind=1) == 1
    assert call_norm(lib, [a], [4], [0], None, norm=None) == 1 and call_norm(lib, [a], [4], [0], None, scratch=None) == 1
    assert call_norm(lib, [a], [4], [0], None, scratch=4) == 1 and call_norm(lib, [a], [1 << 50], [0], None) == 1
    assert lib.bsq_grad_norm_clip(None, None, None, -1, None, 1.0, 2, 8192, 16384, None) == 1
    assert lib.bsq_grad_norm_clip(None, None, None, 1, None, 1.0, 2, 8192, 16384, None) == 1
    # the same memory twice, overlapping results, a result over another input
    assert call_norm(lib, [a, a], [8, 8], [0, 0], [a, a]) == 1
    assert call_norm(lib, [a, a + 4096], [8, 8], [0, 0], [a + 8192, a + 8192 + 16]) == 1
    assert call_norm(lib, [a, a + 4096], [8, 8], [0, 0], [a + 4096, a + 8192]) == 1
    assert call_norm(lib, [a, a + 4096], [8, 8], [0, 0], [a + 16, a + 4096]) == 1


def test_door_refuses_host_tensors(ops):
    x = torch.zeros(4, 64)
    for call in (lambda: ops.fp4_quantize(x), lambda: ops.fp4_quantize(x, 11), lambda: ops.Fp4Matrix(torch.zeros(9999, dtype=torch.uint8), 4, 64),
                 lambda: ops.Fp4Matrix(x, 4, 0), lambda: ops.fp4_matmul(x, x), lambda: ops.fp4_dequantize(x), lambda: ops.fp4_grad_input(x, x),
                 lambda: ops.fp4_linear(x, x), lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.clip_grad_norm([], 1.0), lambda: ops.clip_grad_norm([x], -1.0),
                 lambda: ops.clip_grad_norm([x], 1.0, norm_type=1)):
        with pytest.raises(ValueError):
            call()
