"""Gradients summed over many terms, against 64 bits.

The tensor core cuts an addition off instead of rounding it, so what a chain of additions in one accumulator loses grows with its length, all to one side.  FP32 results are
summed in chains of 1024 terms, 64 additions, whose sums are added rounded.  With terms of random sign a chain is off by 1.5e-7 of itself and so is the sum of all chains
(their errors are to the side of their signs, as their sum is); n rounded additions come to 2^-25 sqrt(n / 2) in the mean, 3.4e-7 for the 256 chains of 262144 terms.
5e-7 holds with room; chains of 8192 terms are 2.6e-6 off."""
import importlib

import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FORMATS = [ref.MXFP4, ref.NVFP4]
SLACK = 5e-7


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def product(a, b):
    """a b in 64 bits, a piece of the sum at a time."""
    out = torch.zeros(a.shape[0], b.shape[1], dtype=torch.float64, device="cuda")
    for i in range(0, a.shape[1], 8192):
        out += a[:, i: i + 8192].double() @ b[i: i + 8192].double()
    return out


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


# outputs, columns, tokens: clusters with slices of up to and beyond four chains, odd lengths; one CTA a tile; pairs; both with rows off 16 bytes
WEIGHT = [(1024, 1024, 16384), (1024, 1024, 65536), (64, 4096, 32768), (64, 300, 262144), (257, 260, 100003), (100, 100, 33000), (1036, 1040, 6001), (2304, 2304, 9000),
          (1036, 1037, 6001), (2100, 2201, 4100)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,K,M", WEIGHT)
def test_fp32_weight_gradient(ops, fmt, N, K, M):
    gen = torch.Generator(device="cuda").manual_seed(M)
    x = ops.fp4_quantize(torch.randn(M, K, generator=gen, device="cuda"), fmt)
    dy = torch.randn(M, N, generator=gen, device="cuda").to(torch.bfloat16)
    want = product(dy.t(), ops.fp4_dequantize(x))
    got = ops.fp4_grad_weight(dy, x, torch.float32)
    assert off(got, want) < SLACK
    assert torch.equal(ops.fp4_grad_weight(dy, x, torch.float32), got)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(200, 65536, 1024), (40, 131072, 520), (128, 20000, 4096), (300, 9001, 8191)])
def test_fp32_input_gradient(ops, fmt, M, N, K):
    gen = torch.Generator(device="cuda").manual_seed(N)
    w = ops.fp4_quantize(torch.randn(N, K, generator=gen, device="cuda"), fmt)
    dy = torch.randn(M, N, generator=gen, device="cuda").to(torch.bfloat16)
    want = product(dy, ops.fp4_dequantize(w))
    got = ops.fp4_grad_input(dy, w, torch.float32)
    assert off(got, want) < SLACK
    assert torch.equal(ops.fp4_grad_input(dy, w, torch.float32), got)


@pytest.mark.parametrize("M", [5000, 100000])
def test_longer_slices_exact(ops, M):
    """Sums that FP32 holds exactly, over slices that end inside a chain, inside a stage, and of every CTA of a cluster its own."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    for N, K in ((33, 70), (300, 300), (700, 130)):
        for extra in (0, 1, 63, 1000):
            x = ops.fp4_quantize(torch.randint(-1, 2, (M + extra, K), generator=gen, device="cuda").float(), ref.MXFP4)
            dy = torch.randint(-2, 3, (M + extra, N), generator=gen, device="cuda").to(torch.bfloat16)
            want = product(dy.t(), ops.fp4_dequantize(x))
            assert torch.equal(ops.fp4_grad_weight(dy, x, torch.float32).double(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 131072, 520), (16, 131072, 1024), (16, 65536, 4100), (7, 30001, 14336), (16, 32769, 14336), (3, 1100, 100000),
                                   (16, 70000, 14336), (1, 131072, 14336), (5, 9000, 70000)])
def test_fp32_input_gradient_of_few_rows(ops, fmt, M, N, K):
    gen = torch.Generator(device="cuda").manual_seed(N + M)
    w = ops.fp4_quantize(torch.randn(N, K, generator=gen, device="cuda"), fmt)
    dy = torch.randn(M, N, generator=gen, device="cuda").to(torch.bfloat16)
    want = product(dy, ops.fp4_dequantize(w))
    got = ops.fp4_grad_input(dy, w, torch.float32)
    assert off(got, want) < SLACK
    assert torch.equal(ops.fp4_grad_input(dy, w, torch.float32), got)


def test_few_rows_of_long_sums_exact(ops):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for N, K in ((131072, 64), (70001, 300), (32800, 14336)):
        w = ops.fp4_quantize(torch.randint(-1, 2, (N, K), generator=gen, device="cuda").float(), ref.MXFP4)
        dy = torch.randint(-2, 3, (16, N), generator=gen, device="cuda").to(torch.bfloat16)
        want = product(dy, ops.fp4_dequantize(w))
        for M in (1, 9, 16):
            assert torch.equal(ops.fp4_grad_input(dy[:M], w, torch.float32).double(), want[:M])


# one CTA a tile, a second chain of one term, pairs, clusters
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,K,M", [(1036, 1040, 200000), (1036, 1037, 65537), (2304, 2304, 140001), (300, 300, 600000)])
def test_fp16_weight_gradient(ops, fmt, N, K, M):
    """Chains of FP16 results are 65536 terms long: 4096 additions, 0.33e-4 of a result, towards 0 (64 additions lose 1.5e-7; the loss grows faster than their number,
    as larger partial sums are cut more coarsely).  FP16's own rounding goes to either side: over 90000 results 2^-12 / 300 = 8e-7.  6e-5 holds with room; 140001
    terms in one chain lose 0.8e-4, 262144 1.9e-4."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    x = ops.fp4_quantize(torch.randn(M, K, generator=gen, device="cuda").to(torch.bfloat16), fmt)
    dy = torch.randn(M, N, generator=gen, device="cuda").to(torch.bfloat16)
    want = torch.zeros(N, K, dtype=torch.float64, device="cuda")
    v = ops.fp4_dequantize(x, torch.bfloat16)                      # (exact: 6 bits times a power of two)
    for i in range(0, M, 8192):
        want += dy[i: i + 8192].double().t() @ v[i: i + 8192].double()
    got = ops.fp4_grad_weight(dy, x, torch.float16).double()
    assert abs(float(((got - want) * want.sign()).sum() / want.abs().sum())) < 6e-5
    bound = 2.0 ** -11 * want.abs() + 2.0 ** -25 + 1e-3 * want.abs().mean()     # a rounding, and 1e-3 of a typical result: what a chain loses, many times over
    assert ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("N,K,M", [(300, 300, 600000), (1036, 1040, 70000), (2304, 2304, 70001), (1500, 1036, 530000), (2100, 2304, 530001)])
def test_fp16_and_bf16_exact(ops, N, K, M):
    """As many chains as there are ways, sums that every one of them holds exactly."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = ops.fp4_quantize(torch.randint(-1, 2, (M, K), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16), ref.MXFP4)
    dy = torch.randint(-2, 3, (M, N), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    v = ops.fp4_dequantize(x, torch.bfloat16)
    want = torch.zeros(N, K, dtype=torch.float64, device="cuda")
    for i in range(0, M, 8192):
        want += dy[i: i + 8192].double().t() @ v[i: i + 8192].double()
    for t in (torch.float16, torch.bfloat16):
        assert torch.equal(ops.fp4_grad_weight(dy, x, t), want.float().to(t))


# pairs that add in memory; tiles of 128 columns where results are off 16 bytes; clusters with tokens as columns and as rows; one CTA a tile
LONG_PRODUCT = [(2048, 4096, 131072), (2049, 4097, 66000), (16, 4096, 131072), (777, 1031, 131072), (300, 300, 70001), (100, 20000, 20001), (1, 4096, 262144)]


@pytest.mark.parametrize("M,N,K", LONG_PRODUCT)
def test_fp32_product(ops, M, N, K):
    """Of NVFP4 matrices with some columns 20 to 100 times the others', in chains of 4096 terms, 64 additions each.  A column that is large in both matrices can make up most of
    a result: the additions behind it in its chain, 32 in the mean, are cut off at full size, 1.5e-8 (2^-26) each, 4.8e-7 at most where it makes up all of it; it does in
    half of the results (the others are sums of many), 3.4e-7 in the mean square.  The 32 chains of 131072 terms are added up by roundings of 2^-23.5 / sqrt(12), 1.4e-7 in
    all (64 of 262144 terms: 2.0e-7).  Together 4.0e-7.  Chains of 256 additions are 3.9e-6 off, FP32 sums that are rounded at each term 3e-7."""
    gen = torch.Generator(device="cuda").manual_seed(K)

    def matrix(rows):
        x = torch.randn(rows, K, generator=gen, device="cuda")
        at = torch.randperm(K, generator=gen, device="cuda")[: K // 1000]
        x[:, at] *= 20 + 80 * torch.rand(K // 1000, generator=gen, device="cuda")
        return ops.fp4_quantize(x)
    a, b = matrix(M), matrix(N)
    want = product(ops.fp4_dequantize(a), ops.fp4_dequantize(b).t())
    got = ops.fp4_matmul(a, b, torch.float32)
    assert off(got, want) < SLACK
    assert torch.equal(ops.fp4_matmul(a, b, torch.float32), got)


@pytest.mark.parametrize("M,N,K", LONG_PRODUCT + [(700, 900, 600000), (2100, 2300, 270000), (50, 130, 600000), (130, 20000, 263000)])
def test_product_of_long_rows_exact(ops, M, N, K):
    gen = torch.Generator(device="cuda").manual_seed(K)
    a, b = (ops.fp4_quantize(torch.randint(-1, 2, (n, K), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16), ref.MXFP4) for n in (M, N))
    va, vb = ops.fp4_dequantize(a, torch.bfloat16), ops.fp4_dequantize(b, torch.bfloat16)
    want = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    for i in range(0, K, 8192):
        want += va[:, i: i + 8192].double() @ vb[:, i: i + 8192].double().t()
    for t in (torch.float32, torch.float16, torch.bfloat16):
        assert torch.equal(ops.fp4_matmul(a, b, t), want.float().to(t))


def test_16_bit_results_of_few_rows_and_millions_of_terms_exact(ops):
    """A weight of 4300001 x 100: more than 65536 rows for each of the 64 warps that share its columns."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    N, K = 4300001, 100
    w = ops.fp4_quantize(torch.randint(-1, 2, (N, K), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16), ref.MXFP4)
    v = ops.fp4_dequantize(w, torch.bfloat16)
    dy = torch.randint(-2, 3, (16, N), generator=gen, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    want = torch.zeros(16, K, dtype=torch.float64, device="cuda")
    for i in range(0, N, 1 << 16):
        want += dy[:, i: i + (1 << 16)].double() @ v[i: i + (1 << 16)].double()
    for t in (torch.float32, torch.float16, torch.bfloat16):
        assert torch.equal(ops.fp4_grad_input(dy, w, t), want.float().to(t))
