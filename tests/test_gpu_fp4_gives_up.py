"""Waits that run out in the products of 4-bit matrices: NaN in the whole result, the status bit, and a device that works on.  Inputs are valid; the waits that give up
are those for finished tiles, at once, while copies, decoding and MMAs of the same tile are still under way."""
import importlib

import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


@pytest.fixture
def no_tries(lib):
    lib.bsq_test_limit_waits(0)
    yield
    torch.cuda.synchronize()
    lib.bsq_test_limit_waits(1 << 16)


@pytest.fixture
def status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def ptr(t):
    return t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


# clusters that share a tile (tokens as columns, as rows), one CTA a tile, pairs
MATMUL = [(40, 512, 4096), (1, 1024, 8192), (300, 515, 4096), (300, 260, 64), (100, 300, 200), (2049, 2300, 300)]
# clusters, one CTA a tile, pairs of CTAs (16-bit results: tiles of 512 rows); more rows of dY than the kernel of few rows takes
GRAD = [(40, 4096, 300), (200, 2048, 512), (300, 140, 260), (2500, 200, 2600)]


@pytest.mark.parametrize("fmt", [ref.MXFP4, ref.NVFP4])
@pytest.mark.parametrize("M,N,K", MATMUL)
def test_product(ops, lib, status, request, fmt, M, N, K):
    torch.manual_seed(M)
    a, b = ops.fp4_quantize(torch.randn(M, K, device="cuda"), fmt), ops.fp4_quantize(torch.randn(N, K, device="cuda"), fmt)
    want = ops.fp4_matmul(a, b, torch.float32)
    request.getfixturevalue("no_tries")
    for _ in range(5):
        out = torch.zeros(M, N, device="cuda")
        status.zero_()
        assert lib.bsq_fp4_matmul(fmt, ptr(a.data), M, ptr(b.data), N, K, ptr(out), 0, N, ptr(status), stream()) == 0
        assert torch.isnan(out).all() and status.item() == 1
    assert torch.isnan(ops.fp4_matmul(a, b)).all()
    lib.bsq_test_limit_waits(1 << 16)
    status.zero_()
    assert lib.bsq_fp4_matmul(fmt, ptr(a.data), M, ptr(b.data), N, K, ptr(out), 0, N, ptr(status), stream()) == 0
    assert torch.equal(out, want) and status.item() == 0


@pytest.mark.parametrize("fmt", [ref.MXFP4, ref.NVFP4])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", GRAD)
def test_gradients(ops, lib, status, request, fmt, dtype, M, N, K):
    torch.manual_seed(M)
    t, code = (torch.float32, 0) if dtype == "f32" else (torch.bfloat16, 2)
    w, x = ops.fp4_quantize(torch.randn(N, K, device="cuda"), fmt), ops.fp4_quantize(torch.randn(M, K, device="cuda"), fmt)
    dy = torch.randn(M, N + (-N) % 8, device="cuda").to(torch.bfloat16)[:, :N]
    ld = dy.stride(0)
    dx, dw = ops.fp4_grad_input(dy, w, t), ops.fp4_grad_weight(dy, x, t)
    gx, gw = torch.zeros_like(dx), torch.zeros_like(dw)

    def both():
        status.zero_()
        assert lib.bsq_fp4_grad_input(fmt, ptr(dy), M, ld, ptr(w.data), N, K, ptr(gx), code, K, None, ptr(status), stream()) == 0
        first = status.item()
        status.zero_()
        assert lib.bsq_fp4_grad_weight(fmt, ptr(dy), M, N, ld, ptr(x.data), K, ptr(gw), code, K, None, ptr(status), stream()) == 0
        return first, status.item()
    request.getfixturevalue("no_tries")
    for _ in range(5):
        gx.zero_()
        gw.zero_()
        assert both() == (1, 1) and torch.isnan(gx).all() and torch.isnan(gw).all()
    lib.bsq_test_limit_waits(1 << 16)
    assert both() == (0, 0) and torch.equal(gx, dx) and torch.equal(gw, dw)


def test_more_tiles_than_accumulators(ops, lib, no_tries):
    """Whoever has given up hands no accumulators back, so the next tile waits in vain: that wait is bounded too, and everything is NaN."""
    a, b = ops.fp4_quantize(torch.randn(5200, 128, device="cuda")), ops.fp4_quantize(torch.randn(5200, 128, device="cuda"))
    dy = torch.randn(5200, 64, device="cuda").to(torch.bfloat16)
    w = ops.fp4_quantize(torch.randn(64, 5200, device="cuda"))
    results = [ops.fp4_matmul(a, b), ops.fp4_grad_input(dy, w), ops.fp4_grad_input(dy, w, torch.float32)]
    assert all(torch.isnan(r).all() for r in results)
    lib.bsq_test_limit_waits(1 << 16)
    assert not any(torch.isnan(r).any() for r in (ops.fp4_matmul(a, b), ops.fp4_grad_input(dy, w), ops.fp4_grad_input(dy, w, torch.float32)))


def test_sums_of_several_chains(ops, lib, no_tries):
    """Accumulators that are handed back between the chains of a tile: none is, and every result is NaN."""
    torch.manual_seed(1)
    a, b, c = (ops.fp4_quantize(torch.randn(n, 40000, device="cuda")) for n in (300, 20, 2400))
    dy = torch.randn(300, 40000, device="cuda").to(torch.bfloat16)
    w = ops.fp4_quantize(torch.randn(40000, 130, device="cuda"))
    x = ops.fp4_quantize(torch.randn(70000, 1040, device="cuda"))
    dz = torch.randn(70000, 1040, device="cuda").to(torch.bfloat16)
    calls = [lambda: ops.fp4_matmul(a, a, torch.float32), lambda: ops.fp4_matmul(b, a, torch.float32), lambda: ops.fp4_matmul(c, c, torch.float32),
             lambda: ops.fp4_grad_input(dy, w, torch.float32), lambda: ops.fp4_grad_weight(dz, x, torch.float16), lambda: ops.fp4_grad_weight(dz[:, :200], x, torch.float32)]
    for call in calls:
        assert torch.isnan(call()).all()
    lib.bsq_test_limit_waits(1 << 16)
    for call in calls:
        assert not torch.isnan(call()).any()
