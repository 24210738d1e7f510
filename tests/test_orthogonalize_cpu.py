"""What orthogonalised updates refuse before anything is launched, and the scratch that they ask for."""
import ctypes as C
import importlib

import pytest

torch = pytest.importorskip("torch")

A = 1 << 20                                                    # addresses that are never looked at: every call here is refused
QUINTIC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def call(lib, ins=(A,), rows=(64,), cols=(32,), lds=(32,), types=(0,), outs=(A + 65536,), ld_outs=(32,), out_type=2, steps=5, k=QUINTIC * 5, eps=1e-7, scale=1.0, scratch=A, n=None):
    u64, ptr = C.c_uint64 * len(rows), C.c_void_p * len(rows)
    return lib.bsq_orthogonalize(ptr(*ins), u64(*rows), u64(*cols), u64(*lds), (C.c_int * len(rows))(*types), len(rows) if n is None else n, ptr(*outs), u64(*ld_outs), out_type, steps,
                                 (C.c_float * len(k))(*k), eps, scale, scratch, None, None)


BAD = [dict(ins=(None,)), dict(ins=(A + 2,)), dict(rows=(65537,)), dict(cols=(65537,), lds=(65537,)), dict(lds=(31,)), dict(types=(3,)), dict(types=(-1,)), dict(outs=(None,)), dict(outs=(A + 65537,)),
       dict(ld_outs=(31,)), dict(out_type=3), dict(steps=0), dict(steps=65, k=QUINTIC * 65), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(scale=float("inf")),
       dict(scale=float("nan")), dict(scratch=None), dict(scratch=A + 64), dict(n=-1), dict(k=(float("nan"),) * 15), dict(k=(float("inf"),) * 15), dict(k=(10.0, 10.0, 10.0) * 5),
       dict(outs=(A,)), dict(outs=(A + 64 * 32 * 4 - 2,)), dict(outs=(A - 64 * 32 * 2 + 2,)),
       dict(ins=(A, A + (1 << 20)), rows=(64, 64), cols=(32, 32), lds=(32, 32), types=(0, 0), outs=(A + 65536, A + 65536 + 64 * 32 * 2 - 2), ld_outs=(32, 32))]


@pytest.mark.parametrize("bad", range(len(BAD)))
def test_refuses(lib, bad):
    assert call(lib, **BAD[bad]) == 1


def test_null_arrays(lib):
    assert lib.bsq_orthogonalize(None, None, None, None, None, 1, None, None, 2, 5, None, 1e-7, 1.0, A, None, None) == 1


def test_nothing_to_do(lib):
    assert call(lib, n=0) == 0 and call(lib, rows=(0,), scratch=None) == 0 and call(lib, cols=(0,), lds=(0,), ld_outs=(0,), scratch=None) == 0


def test_scratch(lib):
    def f(shapes, type=0, out=2):
        n = len(shapes)
        return lib.bsq_orthogonalize_scratch_bytes((C.c_uint64 * n)(*[s[0] for s in shapes]), (C.c_uint64 * n)(*[s[1] for s in shapes]), (C.c_int * n)(*[type] * n), n, out)
    assert f([(64, 64)], type=5) == 0 and f([(64, 64)], out=5) == 0 and f([(65537, 1)]) == 0 and lib.bsq_orthogonalize_scratch_bytes(None, None, None, 1, 2) == 0 and f([(0, 9)]) == 0
    one = f([(1024, 4096)])
    assert 4 * 2 * 1024 * 4096 + 2 * 2 * 1024 * 1024 <= one < 4 * 2 * 1024 * 4096 + 2 * 2 * 1024 * 1024 + 65536
    assert f([(1024, 4096)], out=0) > one
    assert one < f([(1024, 4096)] * 3) <= 3 * one and f([(1024, 4096)] * 500) < 1 << 30
    assert f([(1024, 4096), (64, 64), (4096, 1024)]) == one        # shapes go one behind the other
    assert f([(14336, 14336)]) > 1 << 30                           # one matrix is always taken


def test_python_refuses(ops):
    g = torch.zeros(8, 8)
    for f in (lambda: ops.orthogonalize(g), lambda: ops.orthogonalize([g]), lambda: ops.orthogonalize(g, steps=0), lambda: ops.orthogonalize(g, coefficients=[1.0, 2.0]),
              lambda: ops.orthogonalize(g, dtype=torch.float64), lambda: ops.orthogonalize(g, eps=-1.0)):
        with pytest.raises(ValueError):
            f()
    assert ops.orthogonalize([]) == []


def why(lib, ins=(A,), rows=(64,), cols=(32,), lds=(32,), types=(0,), outs=(A + 65536,), ld_outs=(32,), out_type=2, steps=5, k=QUINTIC * 5, eps=1e-7, scale=1.0, n=None):
    u64, ptr = C.c_uint64 * len(rows), C.c_void_p * len(rows)
    return lib.bsq_orthogonalize_check(ptr(*ins), u64(*rows), u64(*cols), u64(*lds), (C.c_int * len(rows))(*types), len(rows) if n is None else n, ptr(*outs), u64(*ld_outs), out_type, steps,
                                       (C.c_float * len(k))(*k), eps, scale)


def test_why(lib):
    assert why(lib) == 0 and why(lib, rows=(0,)) == 0 and why(lib, n=0) == 0
    for bad in BAD:
        if "scratch" not in bad:
            assert why(lib, **bad) == (2 if "k" in bad and bad.get("steps", 5) == 5 else 3 if "outs" in bad and bad["outs"][0] not in (None, A + 65537) else 1), bad
    assert why(lib, k=(10.0, 10.0, 10.0) * 5, outs=(A,)) == 2


B, E = A + (1 << 24), 2                                        # results in BF16: E bytes an element


@pytest.mark.parametrize("n", [2, 3, 70])
def test_results_side_by_side(lib, n):
    """Columns of one tensor, in whatever order they are listed, are no overlap; one more column is."""
    def many(width, ld=32 * n, order=1):
        at = [B + 32 * E * i for i in range(n)][::order]
        return why(lib, ins=[A + 65536 * i for i in range(n)], rows=[64] * n, cols=[width] * n, lds=[width] * n, types=[2] * n, outs=at, ld_outs=[ld] * n)
    assert many(32) == 0 and many(32, order=-1) == 0 and many(31) == 0
    assert many(33) == 3 and many(33, order=-1) == 3
    assert many(32, ld=32 * n - 1) == 3 and many(32, ld=32 * n + 1) == 0       # (the last one wraps into the next row of the first)


def test_side_by_side_with_others(lib):
    two = dict(rows=(64, 64), cols=(32, 32), types=(2, 2), ld_outs=(64, 64))
    # an update and its own result, or another's, as halves of one buffer; the update in FP32: the same distance in bytes
    assert why(lib, ins=(B + 32 * E,), lds=(64,), types=(2,), outs=(B,), ld_outs=(64,)) == 0
    assert why(lib, ins=(B + 31 * E,), lds=(64,), types=(2,), outs=(B,), ld_outs=(64,)) == 3
    assert why(lib, ins=(B + 64,), lds=(48,), types=(0,), outs=(B,), ld_outs=(96,)) == 0
    assert why(lib, ins=(B + 64,), lds=(47,), types=(0,), outs=(B,), ld_outs=(96,)) == 3            # rows that pass one another
    assert why(lib, ins=(A, A), lds=(32, 32), outs=(B, B + 32 * E), **two) == 0                      # one update twice
    assert why(lib, ins=(A, A), lds=(32, 32), outs=(B, B + 64 * 64 * E - 32 * E), **two) == 0        # the second one begins beside the last row of the first
    assert why(lib, ins=(A, A), lds=(32, 32), outs=(B, B + 63 * 64 * E), **two) == 3                 # ... at the last row
    assert why(lib, ins=(A, A), lds=(32, 32), outs=(B, B + 63 * 64 * E + 32 * E), **two) == 0
    # a single row beside the columns of a matrix, and through them
    row = dict(rows=(64, 1), types=(2, 2), ld_outs=(64, 7), lds=(32, 1))
    assert why(lib, ins=(A, A), cols=(32, 32), outs=(B, B + 5 * 64 * E + 32 * E), **row) == 0
    assert why(lib, ins=(A, A), cols=(32, 33), outs=(B, B + 5 * 64 * E + 32 * E), **row) == 3
    assert why(lib, ins=(A, A), cols=(32, 200), outs=(B, B + 5 * 64 * E + 32 * E), **row) == 3
    assert why(lib, rows=(1, 1), ins=(A, A), cols=(32, 32), lds=(1, 1), types=(2, 2), ld_outs=(1, 1), outs=(B, B + 31 * E)) == 3
