"""What lies beside a result is left as it was: rows of a wider tensor that start on 16 bytes and end anywhere, a single row in the middle of a buffer."""
import importlib

import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def ints(gen, rows, cols):
    return torch.randint(-2, 3, (rows, cols), generator=gen, device="cuda").to(torch.bfloat16)


def check(call, want, dtype):
    """`call` writes the tensor it is given: at several places of a wider one, with guards all around."""
    rows, cols = want.shape
    step = 128 // torch.finfo(dtype).bits                          # elements of 16 bytes
    for first in (0, step, 1):
        for width in (-(-(first + cols) // step) * step, first + cols + 1):
            big = torch.full((rows + 2, width), -7.0, dtype=dtype, device="cuda")
            out = big[1: rows + 1, first: first + cols]
            call(out)
            assert torch.equal(out, want)
            out.fill_(-7.0)
            assert (big == -7.0).all(), (first, width, (big != -7.0).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,N,K", [(1, 77, 300), (3, 131, 200), (129, 93, 100), (300, 21, 4500), (300, 517, 2100), (807, 129, 40), (2309, 2301, 70), (2309, 2301, 4200)])
def test_product(ops, dtype, M, N, K):
    gen, t = torch.Generator(device="cuda").manual_seed(M), DTYPES[dtype]
    a, b = ops.fp4_quantize(ints(gen, M, K), ref.MXFP4), ops.fp4_quantize(ints(gen, N, K), ref.MXFP4)
    want = (ops.fp4_dequantize(a).double() @ ops.fp4_dequantize(b).double().t()).float().to(t)
    check(lambda out: ops.fp4_matmul(a, b, t, out=out), want, t)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("M,N,K", [(9, 10, 77), (77, 1, 93), (4, 1, 2654), (180, 13, 1209), (1, 40, 301), (300, 700, 131), (2309, 33, 2301), (1100, 1300, 1501), (2309, 1100, 2301)])
def test_gradients(ops, dtype, M, N, K):
    gen, t = torch.Generator(device="cuda").manual_seed(N), DTYPES[dtype]
    dy = ints(gen, M, N)
    w, x = ops.fp4_quantize(ints(gen, N, K), ref.MXFP4), ops.fp4_quantize(ints(gen, M, K), ref.MXFP4)
    dx = (dy.double() @ ops.fp4_dequantize(w).double()).float().to(t)
    dw = (dy.double().t() @ ops.fp4_dequantize(x).double()).float().to(t)
    check(lambda out: ops.fp4_grad_input(dy, w, t, out=out), dx, t)
    check(lambda out: ops.fp4_grad_weight(dy, x, t, out=out), dw, t)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("fmt", [ref.MXFP4, ref.NVFP4])
@pytest.mark.parametrize("M,K", [(1, 77), (5, 301), (140, 1031), (700, 93)])
def test_values(ops, dtype, fmt, M, K):
    t = DTYPES[dtype]
    m = ops.fp4_quantize(torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(K), device="cuda"), fmt)
    check(lambda out: ops.fp4_dequantize(m, t, out=out), ops.fp4_dequantize(m, t), t)


@pytest.mark.parametrize("fmt", [ref.MXFP4, ref.NVFP4])
@pytest.mark.parametrize("M,K", [(1, 77), (5, 301), (140, 1031), (700, 93), (128, 64)])
def test_packed(ops, fmt, M, K):
    """A packed matrix in the middle of a buffer; scale bytes of rows behind the last one are within it and may be anything."""
    x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(K), device="cuda")
    alone = ops.fp4_quantize(x, fmt)
    buffer = torch.full((alone.nbytes + 128,), 0xA5, dtype=torch.uint8, device="cuda")
    m = ops.Fp4Matrix(buffer[48: 48 + alone.nbytes], M, K, fmt)
    ops.fp4_quantize(x, fmt, out=m)
    assert torch.equal(m.codes, alone.codes) and torch.equal(m.block_scales(), alone.block_scales())
    assert (buffer[:48] == 0xA5).all() and (buffer[48 + alone.nbytes:] == 0xA5).all()
