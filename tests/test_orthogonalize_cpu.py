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
