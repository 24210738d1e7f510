"""Matrix scales at the ends of their range: results that FP32 can hold are right although a factor on the way to them could not be."""
import importlib

import numpy as np
import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FORMATS = [ref.MXFP4, ref.NVFP4]


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def packed(ops, rng, rows, cols, fmt, scale):
    """Multiples of 0.5 up to 24, times `scale`."""
    codes, byte, _ = ref.random_parts(rng, rows, cols, fmt)
    data = torch.from_numpy(ref.pack(codes, byte, scale, fmt, cols, fill=0xFF)).cuda()
    return ops.Fp4Matrix(data, rows, cols, fmt), ref.values(codes, byte, scale, fmt, cols)


def two(e):
    return float(2.0 ** e)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(5, 200, 300), (40, 512, 4096), (300, 260, 64), (300, 300, 2048), (2100, 2300, 100)])
def test_product(ops, fmt, M, N, K):
    """One CTA a tile, clusters, pairs.  Sums are multiples of 0.25 below 2^22, and the scales powers of two: results are exact, infinite from 2^128 on."""
    rng = np.random.default_rng(M)
    for sa, sb in ((117, -110), (-110, 117), (-149, 100), (100, -149), (-60, -60), (60, 60), (-110, -20), (-20, -110), (126, 1), (64, 64)):
        a, va = packed(ops, rng, M, K, fmt, -two(sa))
        b, vb = packed(ops, rng, N, K, fmt, two(sb))
        with np.errstate(over="ignore"):
            want = (va @ vb.T).astype(np.float32)
        assert np.array_equal(ops.fp4_matmul(a, b, torch.float32).cpu().numpy(), want), (sa, sb)


def test_product_of_quantised_matrices(ops):
    for M in (5, 300):
        for big, small in ((1e36, 1e-30), (1e-30, 1e36)):
            a, b = ops.fp4_quantize(torch.full((M, 4096), big, device="cuda")), ops.fp4_quantize(torch.full((300, 4096), small, device="cuda"))
            want = ops.fp4_dequantize(a).double() @ ops.fp4_dequantize(b).double().t()
            assert torch.equal(ops.fp4_matmul(a, b, torch.float32).double(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(7, 300, 200), (140, 1200, 300), (300, 100, 260), (2300, 64, 2200), (2100, 1300, 1500)])
def test_gradients(ops, fmt, M, N, K):
    """Few rows, clusters, one CTA a tile, pairs.  dy holds integers up to 8 times a power of two."""
    rng = np.random.default_rng(N)
    for scale, factor in ((117, -30), (126, -20), (-110, -27), (-126, -10), (-149, 40)):
        w, vw = packed(ops, rng, N, K, fmt, two(scale))
        x, vx = packed(ops, rng, M, K, fmt, -two(scale))
        dy = rng.integers(-8, 9, (M, N)) * two(factor)
        d = torch.from_numpy(dy).to(torch.bfloat16).cuda()
        assert np.array_equal(ops.fp4_grad_input(d, w, torch.float32).cpu().numpy(), (dy @ vw).astype(np.float32)), scale
        assert np.array_equal(ops.fp4_grad_weight(d, x, torch.float32).cpu().numpy(), (dy.T @ vx).astype(np.float32)), scale
