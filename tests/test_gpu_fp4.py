"""Microscaled 4-bit matrices on the GPU against the definition in 64 bits (fp4_reference.py): packed bytes are equal, products of values whose sums are
exact in FP32 are equal, others are within a bound on FP32 sums."""
import importlib

import numpy as np
import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FORMATS = [ref.MXFP4, ref.NVFP4]
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def live(packed, rows, cols, fmt):
    """A packed form without the scale bytes of rows behind the last one, which may hold anything."""
    ld, at, groups, quads = ref.sizes(rows, cols, fmt)
    packed = packed[: at + groups * quads * 512].copy()
    packed[128 + rows * ld: at] = 0
    r = (np.arange(512) // 16) + (np.arange(512) % 16) // 4 * 32
    for grp in range(groups):
        dead = grp * 128 + r >= rows
        tiles = packed[at + grp * quads * 512: at + (grp + 1) * quads * 512].reshape(quads, 512)
        tiles[:, dead] = 0
    return packed


def check_quantised(ops, x, fmt, amax=None, **kw):
    rows, cols = x.shape
    got = ops.fp4_quantize(x, fmt, **kw)
    codes, byte, g = ref.quantize(x.double().cpu().numpy(), fmt, amax)
    want = ref.pack(codes, byte, g, fmt, cols)
    have = live(got.data.cpu().numpy(), rows, cols, fmt)
    assert np.array_equal(have[:128], want[:128]), (have[:4].view(np.float32), g)
    ld, at, _, _ = ref.sizes(rows, cols, fmt)
    assert np.array_equal(have[at:], want[at:])
    assert np.array_equal(have[128:at], want[128:at])
    assert np.array_equal(got.block_scales().cpu().numpy(), byte) and got.shape == (rows, cols) and got.nbytes == want.size
    v = ref.values(codes, byte, g, fmt, cols)
    for dtype in DTYPES.values():
        back = ops.fp4_dequantize(got, dtype)
        expect = torch.from_numpy(v).to(torch.float32).to(dtype)
        assert torch.equal(torch.nan_to_num(back.cpu(), nan=12345.0), torch.nan_to_num(expect, nan=12345.0))
    return got


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (1, 4096), (3, 31), (2, 33), (127, 64), (129, 65), (33, 257), (200, 1000), (257, 518), (5, 20000)])
def test_quantise(ops, fmt, dtype, rows, cols):
    rng = np.random.default_rng(rows * 7 + cols)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-6, 7, (rows, 1)))
    check_quantised(ops, torch.from_numpy(x).to(DTYPES[dtype]).cuda(), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_quantise_rows_apart_and_off_alignment(ops, fmt, dtype):
    base = torch.randn(70, 300, generator=torch.Generator().manual_seed(1)).to(DTYPES[dtype]).cuda()
    for first, cols in ((0, 256), (1, 255), (2, 200), (4, 64), (3, 1)):
        check_quantised(ops, base[:, first: first + cols], fmt)
    x = base.view(7, 10, 300)
    assert torch.equal(ops.fp4_quantize(x, fmt).codes, ops.fp4_quantize(base, fmt).codes)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_quantise_every_tie(ops, fmt, dtype):
    """Halfway points times every block scale that the type can hold, and the values beside them."""
    t = DTYPES[dtype]
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    scales = ref.E4M3[1:] if fmt == ref.NVFP4 else 2.0 ** np.arange(-12, 12)
    for s in scales:
        x = torch.from_numpy(np.concatenate([mids * s, [6.0 * s]])).to(t)
        up = torch.nextafter(x, torch.full_like(x, float("inf")))
        down = torch.nextafter(x, torch.full_like(x, 0.0))
        row = torch.zeros(32, dtype=t)
        row[:8], row[16:24] = x, -x
        row[8:15], row[24:31] = up[:7], -down[:7]
        rows.append(row)
    x = torch.stack(rows)
    if fmt == ref.NVFP4:                                          # (the largest magnitude is 2688, so that the matrix scale is 1)
        x = torch.cat([x, torch.full((1, 32), 2688.0, dtype=t)])
    check_quantised(ops, x.cuda(), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantise_every_block_scale_boundary(ops, fmt):
    """Largest magnitudes beside the points where the block scale changes."""
    if fmt == ref.MXFP4:
        tops = 2.0 ** np.arange(-20.0, 20.0)
    else:
        tops = 6.0 * (ref.E4M3[1:] + ref.E4M3[:-1]) / 2
    t = torch.from_numpy(tops).to(torch.float32)
    x = torch.stack([t, torch.nextafter(t, torch.full_like(t, 1e9)), torch.nextafter(t, torch.zeros_like(t))], dim=1).reshape(-1, 1)
    x = torch.cat([x, x / 3, -x / 5, torch.zeros(x.shape[0], 13)], dim=1)
    if fmt == ref.NVFP4:
        x = torch.cat([x, torch.full((1, 16), 2688.0)])
    check_quantised(ops, x.cuda(), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_quantise_special_values(ops, fmt, dtype):
    t = DTYPES[dtype]
    top, tiny = torch.finfo(t).max, torch.finfo(t).smallest_normal
    x = torch.randn(12, 96, generator=torch.Generator().manual_seed(2)).to(t)
    x[0, 5], x[1, 40], x[2, 95], x[3, 0] = float("inf"), float("-inf"), float("nan"), float("nan")
    x[4] = 0
    x[5] = -0.0
    x[6] *= tiny
    x[7, :32] = 0
    x[8, 33] = float("nan")
    check_quantised(ops, x.cuda(), fmt)
    y = torch.zeros(3, 64, dtype=t)
    check_quantised(ops, y.cuda(), fmt)
    y[0, :] = top
    y[1, 3] = -top
    y[2, 10] = tiny
    check_quantised(ops, y.cuda(), fmt)
    check_quantised(ops, (torch.arange(1, 65, dtype=torch.float32) * float(torch.finfo(t).tiny) / 64).to(t).view(1, 64).cuda(), fmt)      # subnormals


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("amax", [1e-30, 0.5, 3.0, 2688.0, 2688.0001, 1e9, 0.0, float("inf"), float("nan")])
def test_quantise_with_a_given_largest_magnitude(ops, dtype, amax):
    x = (torch.randn(9, 100, generator=torch.Generator().manual_seed(4)) * 2).to(DTYPES[dtype])
    x[3, 7] = 60000.0
    given = torch.tensor([amax], dtype=torch.float32)
    got = ops.fp4_quantize(x.cuda(), ref.NVFP4, amax=given.cuda())
    codes, byte, g = ref.quantize(x.double().numpy(), ref.NVFP4, given.item())
    assert np.array_equal(live(got.data.cpu().numpy(), 9, 100, ref.NVFP4), ref.pack(codes, byte, g, ref.NVFP4, 100))


@pytest.mark.parametrize("fmt", FORMATS)
def test_matrices_large_enough_for_every_pass(ops, fmt):
    """More tiles than resident CTAs; the largest magnitude found by a pass of its own; the last row group partly filled."""
    x = torch.randn(1300, 4100, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    x[1299, 4099] = 900.0
    got = ops.fp4_quantize(x.cuda(), fmt)
    codes, byte, g = ref.quantize(x.double().numpy(), fmt)
    assert np.array_equal(got.block_scales().cpu().numpy(), byte) and float(got.tensor_scale) == g
    c = got.codes.cpu().numpy()
    assert np.array_equal(np.stack([c & 15, c >> 4], axis=2).reshape(1300, -1)[:, :4100], codes[:, :4100])


def packed(ops, rng, rows, cols, fmt, exact=True, fill=0xFF):
    parts = ref.random_parts(rng, rows, cols, fmt, exact)
    data = torch.from_numpy(ref.pack(*parts, fmt, cols, fill=fill)).cuda()
    return ops.Fp4Matrix(data, rows, cols, fmt), ref.values(*parts, fmt, cols)


MATMUL = [(1, 16, 32), (1, 128, 64), (1, 1031, 300), (3, 257, 1000), (16, 300, 128), (17, 130, 96), (63, 640, 257), (64, 1000, 512), (65, 100, 31), (100, 129, 700),
          (128, 256, 256), (129, 257, 258), (200, 1500, 640), (777, 515, 1030), (1, 4096, 2048), (40, 40, 4096), (300, 3000, 100), (2500, 2600, 64), (2049, 2600, 700), (1800, 2304, 1031)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", MATMUL)
def test_matmul_exact_sums(ops, fmt, M, N, K):
    """Values are multiples of 0.5 up to 24, products multiples of 0.25 up to 576: sums of up to 4096 of them fit 24 bits (576 * 4096 / 0.25 = 2^23.2)."""
    rng = np.random.default_rng(M + N + K)
    a, va = packed(ops, rng, M, K, fmt)
    b, vb = packed(ops, rng, N, K, fmt)
    want = torch.from_numpy(va @ vb.T)
    assert torch.equal(ops.fp4_matmul(a, b, torch.float32).cpu().double(), want)
    assert torch.equal(ops.fp4_matmul(a, b).cpu(), want.float().to(torch.bfloat16))
    assert torch.equal(ops.fp4_matmul(a, b, torch.float16).cpu(), want.float().to(torch.float16))


def sum_bound(a, b, terms):
    """FP32 sums of `terms` products: every addition is off by at most 2^-23 of the sum of magnitudes (cut off, not rounded), the products are exact."""
    return (terms + 4) * 2.0 ** -23 * (np.abs(a) @ np.abs(b))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 300, 1000), (130, 270, 512), (300, 700, 2000)])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_matmul_random_scales(ops, fmt, M, N, K, dtype):
    rng = np.random.default_rng(M * 3 + N)
    a, va = packed(ops, rng, M, K, fmt, exact=False)
    b, vb = packed(ops, rng, N, K, fmt, exact=False)
    got = ops.fp4_matmul(a, b, DTYPES[dtype]).double().cpu().numpy()
    want = va @ vb.T
    # the two matrix scales are two more roundings of 2^-24; then the result's own, half a step
    tol = sum_bound(va, vb.T, K) + np.abs(want) * (2.0 ** -22 + torch.finfo(DTYPES[dtype]).eps / 2) + torch.finfo(DTYPES[dtype]).smallest_normal
    over = np.abs(want) > torch.finfo(DTYPES[dtype]).max
    assert np.all((np.abs(got - want) <= tol) | over)


@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_results_in_place_and_strided(ops, fmt):
    rng = np.random.default_rng(9)
    for M, N in ((5, 70), (130, 300)):
        a, va = packed(ops, rng, M, 96, fmt)
        b, vb = packed(ops, rng, N, 96, fmt)
        for dtype in DTYPES.values():
            big = torch.full((M + 2, N + 9), -7.0, dtype=dtype, device="cuda")
            out = big[1: M + 1, 5: N + 5]
            assert ops.fp4_matmul(a, b, dtype, out=out) is out
            want = torch.full((M + 2, N + 9), -7.0, dtype=dtype)
            want[1: M + 1, 5: N + 5] = torch.from_numpy(va @ vb.T).to(dtype)
            assert torch.equal(big.cpu(), want)                   # nothing beside the result was written


@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_scales_stay_in_their_rows_and_columns(ops, fmt):
    a = torch.ones(130, 128).cuda()
    b = torch.ones(260, 128).cuda()
    a[5, 100], b[200, 3] = float("nan"), float("inf")
    y = ops.fp4_matmul(ops.fp4_quantize(a, fmt), ops.fp4_quantize(b, fmt), torch.float32).cpu()
    bad = torch.zeros(130, 260, dtype=torch.bool)
    bad[5], bad[:, 200] = True, True
    # 1 in NVFP4: the matrix scale is 2^-11, the block scale E4M3(2^11 / 6 = 341.3) = 352, the largest element 6 * 352 / 2048
    one = 1.0 if fmt == ref.MXFP4 else 1.03125
    assert torch.equal(torch.isnan(y), bad) and (y[~bad] == 128 * one * one).all()
    x = ops.fp4_quantize(a, fmt)
    dy = torch.ones(130, 70, dtype=torch.bfloat16, device="cuda")
    dw = ops.fp4_grad_weight(dy, x, torch.float32).cpu()
    block = ref.BLOCK[fmt]
    col = torch.zeros(128, dtype=torch.bool)
    col[100 // block * block: 100 // block * block + block] = True
    assert torch.isnan(dw[:, col]).all() and (dw[:, ~col] == 130 * one).all()


def test_scale_extremes(ops):
    """Block scales at the ends of their ranges, subnormal ones among them."""
    for fmt, lo, hi in ((ref.MXFP4, 1, 160), (ref.NVFP4, 1, 126)):
        for M in (1, 70):
            codes = np.full((M, 64), 3, np.uint8)                # 1.5
            ones = np.full((40, 64), 2, np.uint8)                # 1
            blocks = 64 // ref.BLOCK[fmt]
            one = 127 if fmt == ref.MXFP4 else 56
            for s in (lo, hi):
                x = (codes, np.full((M, blocks), s, np.uint8), 1.0)
                w = (ones, np.full((40, blocks), one, np.uint8), 1.0)
                a = ops.Fp4Matrix(torch.from_numpy(ref.pack(*x, fmt, 64)).cuda(), M, 64, fmt)
                b = ops.Fp4Matrix(torch.from_numpy(ref.pack(*w, fmt, 64)).cuda(), 40, 64, fmt)
                want = ref.values(*x, fmt, 64) @ ref.values(*w, fmt, 64).T
                assert np.array_equal(ops.fp4_matmul(a, b, torch.float32).double().cpu().numpy(), want)
                dy = torch.full((M, 40), 2.0, dtype=torch.bfloat16, device="cuda")
                got = ops.fp4_grad_weight(dy, a, torch.float32).double().cpu().numpy()
                assert np.array_equal(got, np.full((40, M), 2.0) @ ref.values(*x, fmt, 64))


GRAD = [(2, 33, 129), (9, 2000, 390), (15, 4090, 1000), (1, 16, 32), (1, 1031, 300), (3, 257, 1000), (16, 300, 128), (63, 640, 257), (65, 100, 31), (128, 256, 256), (129, 257, 258), (200, 1500, 640),
        (777, 515, 1030), (1, 4096, 512), (40, 40, 4096), (2500, 72, 64), (130, 64, 9000), (2600, 2500, 520), (4100, 200, 4100), (200, 4100, 4100)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", GRAD)
def test_gradients_exact_sums(ops, fmt, M, N, K):
    """dy holds integers up to 8 in magnitude: products are multiples of 0.5 up to 192, sums of up to 4096 of them fit 24 bits."""
    rng = np.random.default_rng(M + 2 * N + 3 * K)
    w, vw = packed(ops, rng, N, K, fmt)
    x, vx = packed(ops, rng, M, K, fmt)
    dy = rng.integers(-8, 9, (M, N)).astype(np.float64)
    d = torch.from_numpy(dy).to(torch.bfloat16).cuda()
    dx, dw = torch.from_numpy(dy @ vw), torch.from_numpy(dy.T @ vx)
    for dtype in DTYPES.values():
        assert torch.equal(ops.fp4_grad_input(d, w, dtype).cpu(), dx.float().to(dtype))
        assert torch.equal(ops.fp4_grad_weight(d, x, dtype).cpu(), dw.float().to(dtype))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(5, 700, 300), (300, 270, 512), (1100, 600, 1000)])
def test_gradients_random(ops, fmt, M, N, K):
    rng = np.random.default_rng(M + N + K)
    w, vw = packed(ops, rng, N, K, fmt, exact=False)
    x, vx = packed(ops, rng, M, K, fmt, exact=False)
    d = torch.from_numpy(rng.standard_normal((M, N))).to(torch.bfloat16)
    dy = d.double().numpy()
    for got, a, b, terms in ((ops.fp4_grad_input(d.cuda(), w, torch.float32), dy, vw, N), (ops.fp4_grad_weight(d.cuda(), x, torch.float32), dy.T, vx, M)):
        want = a @ b
        assert np.all(np.abs(got.double().cpu().numpy() - want) <= sum_bound(a, b, terms) + np.abs(want) * 2.0 ** -22)


@pytest.mark.parametrize("fmt", FORMATS)
def test_gradients_against_differences(ops, fmt):
    """<dy, f(x + h e) - f(x - h e)> / 2h with f the product of the values in 64 bits, which is linear in either operand."""
    rng = np.random.default_rng(12)
    M, N, K, h = 33, 40, 70, 0.5
    w, vw = packed(ops, rng, N, K, fmt)
    x, vx = packed(ops, rng, M, K, fmt)
    dy = rng.integers(-4, 5, (M, N)).astype(np.float64)
    d = torch.from_numpy(dy).to(torch.bfloat16).cuda()
    dx, dw = ops.fp4_grad_input(d, w, torch.float32).cpu().numpy(), ops.fp4_grad_weight(d, x, torch.float32).cpu().numpy()
    for _ in range(20):
        i, j, k = rng.integers(M), rng.integers(N), rng.integers(K)
        e = np.zeros((M, K))
        e[i, k] = h
        assert np.sum(dy * ((vx + e) @ vw.T - (vx - e) @ vw.T)) / (2 * h) == dx[i, k]
        e = np.zeros((N, K))
        e[j, k] = h
        assert np.sum(dy * (vx @ (vw + e).T - vx @ (vw - e).T)) / (2 * h) == dw[j, k]


@pytest.mark.parametrize("fmt", FORMATS)
def test_gradients_of_strided_and_offset_dy(ops, fmt):
    rng = np.random.default_rng(13)
    M, N, K = 70, 96, 300
    w, vw = packed(ops, rng, N, K, fmt)
    x, vx = packed(ops, rng, M, K, fmt)
    base = torch.from_numpy(rng.integers(-8, 9, (M, N + 40)).astype(np.float64)).to(torch.bfloat16).cuda()
    for first in (0, 1, 8, 13):
        d = base[:, first: first + N]
        dy = d.double().cpu().numpy()
        big = torch.full((M, K + 3), -7.0, device="cuda")
        ops.fp4_grad_input(d, w, torch.float32, out=big[:, 1: K + 1])
        assert np.array_equal(big[:, 1: K + 1].double().cpu().numpy(), dy @ vw) and (big[:, 0] == -7).all() and (big[:, K + 1:] == -7).all()
        assert np.array_equal(ops.fp4_grad_weight(d, x, torch.float32).double().cpu().numpy(), dy.T @ vx)
    d3 = base[:, :N].contiguous().view(7, 10, N)
    assert torch.equal(ops.fp4_grad_input(d3, w).view(M, K), ops.fp4_grad_input(base[:, :N], w))
    assert torch.equal(ops.fp4_grad_weight(d3, x), ops.fp4_grad_weight(base[:, :N], x))


@pytest.mark.parametrize("fmt", FORMATS)
def test_no_tokens(ops, fmt):
    w = ops.fp4_quantize(torch.randn(64, 96, device="cuda"), fmt)
    x = ops.fp4_quantize(torch.empty(0, 96, device="cuda"), fmt)
    assert ops.fp4_dequantize(x).shape == (0, 96) and ops.fp4_matmul(x, w).shape == (0, 64) and ops.fp4_matmul(w, x).shape == (64, 0)
    dy = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    assert ops.fp4_grad_input(dy, w).shape == (0, 96)
    for dtype in DTYPES.values():
        assert torch.equal(ops.fp4_grad_weight(dy, x, dtype), torch.zeros(64, 96, dtype=dtype, device="cuda"))


def test_one_product_does_not_depend_on_what_else_runs(ops):
    """Two products on two streams at once, again and again, against their results alone."""
    rng = np.random.default_rng(21)
    a, va = packed(ops, rng, 700, 1024, ref.NVFP4)
    b, vb = packed(ops, rng, 900, 1024, ref.NVFP4)
    dy = torch.from_numpy(rng.integers(-8, 9, (700, 900)).astype(np.float64)).to(torch.bfloat16).cuda()
    y, dx, dw = ops.fp4_matmul(a, b), ops.fp4_grad_input(dy, b), ops.fp4_grad_weight(dy, a)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((ops.fp4_matmul(a, b), ops.fp4_grad_input(dy, b), ops.fp4_grad_weight(dy, a)))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], y) and torch.equal(g[1], dx) and torch.equal(g[2], dw)


def test_captured_and_replayed(ops):
    """Two graphs of the same calls with inputs of their own, replayed in turn with new contents."""
    graphs = []
    w = ops.fp4_quantize(torch.randn(300, 200, device="cuda"), ref.NVFP4)
    for _ in range(2):
        x = torch.randn(50, 200, device="cuda").to(torch.bfloat16)
        dy = torch.randn(50, 300, device="cuda").to(torch.bfloat16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.fp4_matmul(ops.fp4_quantize(x), w)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x4 = ops.fp4_quantize(x)
            outs = [ops.fp4_matmul(x4, w), ops.fp4_grad_input(dy, w), ops.fp4_grad_weight(dy, x4, torch.float32), ops.fp4_dequantize(x4)]
        graphs.append((g, x, dy, outs))
    for _ in range(3):
        for g, x, dy, _ in graphs:
            x.copy_(torch.randn(50, 200, device="cuda"))
            dy.copy_(torch.randn(50, 300, device="cuda"))
        for g, *_ in graphs:
            g.replay()
        for g, x, dy, outs in graphs:
            x4 = ops.fp4_quantize(x)
            want = [ops.fp4_matmul(x4, w), ops.fp4_grad_input(dy, w), ops.fp4_grad_weight(dy, x4, torch.float32), ops.fp4_dequantize(x4)]
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_linear_under_autograd(ops):
    """The pieces that fp4_linear is made of, and a frozen packed weight."""
    torch.manual_seed(5)
    x = torch.randn(3, 20, 96, device="cuda").to(torch.bfloat16).requires_grad_()
    w = (torch.randn(130, 96, device="cuda") * 0.1).requires_grad_()
    y = ops.fp4_linear(x, w)
    dy = torch.randn_like(y)
    y.backward(dy)
    x4, w4 = ops.fp4_quantize(x.detach()), ops.fp4_quantize(w.detach())
    assert torch.equal(y.detach().view(60, 130), ops.fp4_matmul(x4, w4)) and y.shape == (3, 20, 130)
    assert torch.equal(x.grad, ops.fp4_grad_input(dy, w4)) and torch.equal(w.grad, ops.fp4_grad_weight(dy, x4, torch.float32))
    x.grad = None
    ops.fp4_linear(x, w4).sum().backward()                        # (the gradient of a sum is a broadcast one)
    assert torch.equal(x.grad, ops.fp4_grad_input(torch.ones_like(y), w4))
    with torch.no_grad():
        assert not ops.fp4_linear(x, w4).requires_grad
    with pytest.raises(ValueError):
        ops.fp4_linear(x, ops.fp4_quantize(w.detach(), ref.MXFP4))
    with pytest.raises(ValueError):
        ops.fp4_linear(x.float(), w)


def test_training_step(ops):
    """Two layers with parked activations, gradients clipped together, against the same step in 64 bits on the values that the operators hold."""
    torch.manual_seed(6)
    x = torch.randn(200, 128, device="cuda").to(torch.bfloat16)
    w1 = (torch.randn(256, 128, device="cuda") * 0.1).requires_grad_()
    w2 = (torch.randn(64, 256, device="cuda") * 0.1).requires_grad_()
    h = ops.fp4_linear(x, w1)
    y = ops.fp4_linear(torch.relu(h), w2)
    dy = torch.randn_like(y)
    y.backward(dy)
    q = lambda t: ops.fp4_dequantize(ops.fp4_quantize(t.detach())).double()  # noqa: E731
    hv = torch.relu(h.detach())
    dw2 = dy.double().t() @ q(hv)
    dh = ((dy.double() @ q(w2)).to(torch.bfloat16).double() * (h.detach() > 0)).to(torch.bfloat16).double()
    dw1 = dh.t() @ q(x)
    # sums of 200 products in FP32; dh rounds to BF16 in both, which may fall differently where the FP32 sum is beside a tie: 2^-8 of it
    bound2 = 204 * 2.0 ** -23 * (dy.double().abs().t() @ q(hv).abs())
    bound1 = (204 * 2.0 ** -23 + 2.0 ** -8) * (dh.abs().t() @ q(x).abs())
    assert ((w2.grad.double() - dw2).abs() <= bound2 + dw2.abs() * 2.0 ** -23).all()
    assert ((w1.grad.double() - dw1).abs() <= bound1 + dw1.abs() * 2.0 ** -23).all()
    before = [w1.grad.clone(), w2.grad.clone()]
    want = torch.sqrt(sum((g.double() ** 2).sum() for g in before))
    norm = ops.clip_grad_norm([w1.grad, w2.grad], 1.0)
    assert abs(norm.double() - want) <= want * 2.0 ** -23
    for g, b in zip((w1.grad, w2.grad), before):
        assert ((g.double() - b.double() / (want + 1e-6)).abs() <= b.double().abs() / want * 2.0 ** -22).all()


def test_door_refusals(ops):
    x = torch.randn(8, 64, device="cuda")
    q, q8 = ops.fp4_quantize(x), ops.fp4_quantize(x, ref.MXFP4)
    d = torch.randn(8, 8, device="cuda").to(torch.bfloat16)
    out = torch.empty(8, 8, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: ops.fp4_quantize(x.double()), lambda: ops.fp4_quantize(x.t()), lambda: ops.fp4_quantize(x[:, ::2]), lambda: ops.fp4_quantize(x[:, :0]),
                 lambda: ops.fp4_quantize(x[:1].expand(4, 64)), lambda: ops.fp4_quantize(x, ref.MXFP4, amax=x[0, :1]), lambda: ops.fp4_quantize(x, amax=x[0, :2]),
                 lambda: ops.fp4_quantize(x, out=q8), lambda: ops.fp4_quantize(x[:4], out=q), lambda: ops.fp4_quantize(x.view(2, 4, 64)[:, :3]),
                 lambda: ops.Fp4Matrix(q.data[:-1], 8, 64), lambda: ops.Fp4Matrix(q.data[8:], 1, 64), lambda: ops.Fp4Matrix(q.data, 8, 64, 3),
                 lambda: ops.fp4_matmul(q, q8), lambda: ops.fp4_matmul(q, ops.fp4_quantize(x[:, :32])), lambda: ops.fp4_matmul(q, q, torch.float64),
                 lambda: ops.fp4_matmul(q, q, out=out.t()), lambda: ops.fp4_matmul(q, q, out=out[:4]), lambda: ops.fp4_matmul(q, q, out=out.float()),
                 lambda: ops.fp4_matmul(q, q, out=q.data[: 128].view(torch.bfloat16).view(8, 8)),
                 lambda: ops.fp4_grad_input(d.float(), q), lambda: ops.fp4_grad_input(d[:, :4], q), lambda: ops.fp4_grad_input(d.half(), q),
                 lambda: ops.fp4_grad_weight(d[:4], q), lambda: ops.fp4_grad_input(d, x), lambda: ops.fp4_grad_weight(d.t(), q),
                 lambda: ops.fp4_grad_input(d, ops.fp4_quantize(x[:, :8]), out=d),
                 lambda: ops.fp4_dequantize(q, out=x.requires_grad_())):
        with pytest.raises(ValueError):
            call()


def test_quantise_into_a_given_matrix(ops):
    x = torch.randn(20, 100, device="cuda")
    q = ops.fp4_quantize(torch.zeros(20, 100, device="cuda"))
    assert ops.fp4_quantize(x, out=q) is q and torch.equal(q.codes, ops.fp4_quantize(x).codes)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_large_rows_apart(ops, fmt, dtype):
    """Rows that are not neighbours in a matrix large enough for a pass of its own over the magnitudes, and values written to such rows."""
    base = torch.randn(700, 310, generator=torch.Generator().manual_seed(7)).to(DTYPES[dtype])
    base[:, 300:] = 1000.0                                        # (not part of the matrix: must not count)
    base[699, 299] = -77.0
    base = base.cuda()
    for first, cols in ((0, 300), (1, 299), (5, 256)):
        x = base[:, first: first + cols]
        q = check_quantised(ops, x, fmt)
        wide = torch.full((702, cols + 11), -7.0, dtype=DTYPES[dtype], device="cuda")
        out = wide[1:701, 3: 3 + cols]
        assert ops.fp4_dequantize(q, DTYPES[dtype], out=out) is out
        assert torch.equal(out, ops.fp4_dequantize(q, DTYPES[dtype]))
        assert (wide[0] == -7).all() and (wide[701] == -7).all() and (wide[:, :3] == -7).all() and (wide[:, 3 + cols:] == -7).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_packed_matrices_on_any_16_bytes(ops, fmt):
    x = torch.randn(150, 200, device="cuda").to(torch.bfloat16)
    w = torch.randn(90, 200, device="cuda").to(torch.bfloat16)
    dy = torch.randn(150, 90, device="cuda").to(torch.bfloat16)
    x4, w4 = ops.fp4_quantize(x, fmt), ops.fp4_quantize(w, fmt)

    def moved(m, by):
        buffer = torch.full((m.nbytes + by + 64,), 0xFF, dtype=torch.uint8, device="cuda")
        buffer[by: by + m.nbytes] = m.data[: m.nbytes]
        return ops.Fp4Matrix(buffer[by: by + m.nbytes], m.rows, m.cols, m.format)
    xm, wm = moved(x4, 16), moved(w4, 48)
    assert torch.equal(ops.fp4_matmul(xm, wm), ops.fp4_matmul(x4, w4)) and torch.equal(ops.fp4_dequantize(xm), ops.fp4_dequantize(x4))
    assert torch.equal(ops.fp4_grad_input(dy, wm), ops.fp4_grad_input(dy, w4)) and torch.equal(ops.fp4_grad_weight(dy, xm), ops.fp4_grad_weight(dy, x4))
    assert torch.equal(ops.fp4_grad_input(dy[:9], wm), ops.fp4_grad_input(dy[:9], w4))
    ops.fp4_quantize(w, fmt, out=xm if xm.shape == w.shape else wm)
    assert torch.equal(wm.codes, w4.codes)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [7, 140])
def test_non_finite_gradients_stay_where_they_belong(ops, fmt, M):
    w, x = ops.fp4_quantize(torch.ones(90, 200, device="cuda"), fmt), ops.fp4_quantize(torch.ones(M, 200, device="cuda"), fmt)
    dy = torch.ones(M, 90, dtype=torch.bfloat16, device="cuda")
    dx0, dw0 = ops.fp4_grad_input(dy, w, torch.float32), ops.fp4_grad_weight(dy, x, torch.float32)
    dy[3, 60], dy[5, 89] = float("nan"), float("inf")
    dx, dw = ops.fp4_grad_input(dy, w, torch.float32), ops.fp4_grad_weight(dy, x, torch.float32)
    rows, cols = [i for i in range(M) if i not in (3, 5)], [i for i in range(90) if i not in (60, 89)]
    assert torch.isnan(dx[3]).all() and torch.isinf(dx[5]).all() and torch.equal(dx[rows], dx0[rows])
    assert torch.isnan(dw[60]).all() and torch.isinf(dw[89]).all() and torch.equal(dw[cols], dw0[cols])


def test_the_same_bits_every_time(ops):
    """Shapes that take every way through the products, ten times over."""
    torch.manual_seed(3)
    for M, N, K in ((1, 600, 3000), (40, 4096, 2048), (300, 1000, 4096), (2100, 2200, 2050), (4100, 300, 4100)):
        x, w = ops.fp4_quantize(torch.randn(M, K, device="cuda")), ops.fp4_quantize(torch.randn(N, K, device="cuda"))
        dy = torch.randn(M, N, device="cuda").to(torch.bfloat16)
        calls = [lambda: ops.fp4_matmul(x, w, torch.float32), lambda: ops.fp4_grad_input(dy, w), lambda: ops.fp4_grad_input(dy, w, torch.float32),
                 lambda: ops.fp4_grad_weight(dy, x), lambda: ops.fp4_grad_weight(dy, x, torch.float32), lambda: ops.fp4_grad_input(dy[: min(M, 9)], w)]
        for call in calls:
            first = call()
            assert not torch.isnan(first).any()
            for _ in range(10):
                assert torch.equal(call(), first)


@pytest.mark.parametrize("fmt", FORMATS)
def test_few_rows_are_the_rows_of_many(ops, fmt):
    """The kernel for up to 16 rows against the one for more: sums of values that are exact in FP32."""
    rng = np.random.default_rng(31)
    for N, K in ((16, 33), (1000, 700), (4096, 300), (100, 5000)):
        w, vw = packed(ops, rng, N, K, fmt)
        dy = torch.from_numpy(rng.integers(-8, 9, (33, N)).astype(np.float64)).to(torch.bfloat16).cuda()
        many = ops.fp4_grad_input(dy, w, torch.float32)
        for a, b in ((0, 1), (1, 17), (5, 13), (16, 33)):
            assert torch.equal(ops.fp4_grad_input(dy[a:b], w, torch.float32), many[a:b])


def test_few_rows_with_small_scales(ops):
    """MXFP4 scales up to 2 take a shorter way; 0.25 to 1 keeps sums exact, the ends of the range (2^-127, 2) are in a matrix of their own."""
    rng = np.random.default_rng(32)
    for N, K, bytes_ in ((500, 300, (125, 126, 127)), (4096, 128, (126, 127, 128)), (64, 96, (0, 0, 0)), (64, 96, (128, 128, 128)), (64, 96, (129, 129, 128))):
        codes = rng.integers(0, 16, (N, -(-K // 32) * 32)).astype(np.uint8)
        codes[:, K:] = 0
        byte = rng.choice(np.array(bytes_, np.uint8), (N, -(-K // 32)))
        w = ops.Fp4Matrix(torch.from_numpy(ref.pack(codes, byte, 1.0, ref.MXFP4, K, fill=0xFF)).cuda(), N, K, ref.MXFP4)
        dy = rng.integers(-8, 9, (16, N)).astype(np.float64)
        want = dy @ ref.values(codes, byte, 1.0, ref.MXFP4, K)
        got = ops.fp4_grad_input(torch.from_numpy(dy).to(torch.bfloat16).cuda(), w, torch.float32).double().cpu().numpy()
        assert np.array_equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_status_word_of_the_c_entries(ops, lib, fmt):
    x, w = ops.fp4_quantize(torch.randn(40, 64, device="cuda"), fmt), ops.fp4_quantize(torch.randn(50, 64, device="cuda"), fmt)
    dy = torch.randn(40, 50, device="cuda").to(torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty(50, 64, device="cuda")
    scratch = torch.empty(lib.bsq_fp4_grad_scratch_bytes(dy.data_ptr(), 40, 50, 50), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.bsq_fp4_matmul(fmt, x.data.data_ptr(), 40, w.data.data_ptr(), 50, 64, out.data_ptr(), 0, 50, status.data_ptr(), stream) == 0
    assert torch.equal(out.view(-1)[: 2000].view(40, 50), ops.fp4_matmul(x, w, torch.float32))
    assert lib.bsq_fp4_grad_weight(fmt, dy.data_ptr(), 40, 50, 50, x.data.data_ptr(), 64, out.data_ptr(), 0, 64, scratch.data_ptr(), status.data_ptr(), stream) == 0
    assert torch.equal(out, ops.fp4_grad_weight(dy, x, torch.float32)) and status.item() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(700, 4100, 2100), (2650, 2660, 1984), (4100, 700, 2070), (300, 2100, 140)])
def test_partly_filled_tiles_again_and_again(ops, dtype, M, N, K):
    """Tiles whose last columns are not there, on their way out through two boxes in turn: what is left out must not let a box be overwritten while it is read.
    Sums are exact, so every call gives the same bits; one call in some hundred went wrong when it did."""
    rng = np.random.default_rng(M)
    w, vw = packed(ops, rng, N, K, ref.MXFP4)
    dy = rng.integers(-2, 3, (M, N)).astype(np.float64)
    d = torch.from_numpy(dy).to(torch.bfloat16).cuda()
    want = torch.from_numpy(dy @ vw).float().to(DTYPES[dtype]).cuda()
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        wrong += (ops.fp4_grad_input(d, w, DTYPES[dtype]) != want).any()
    assert wrong.item() == 0


def test_copies_that_land_in_any_order(ops):
    """Products of operands that were made just before, a library product in between: copies then land late and out of order.  A wait that took one round of a
    ring for another let one call in a hundred decode what had not arrived."""
    import random
    rnd, gen = random.Random(5), torch.Generator(device="cuda").manual_seed(5)
    wrong = []
    for i in range(2500):
        fmt, dtype = rnd.choice(FORMATS), rnd.choice(list(DTYPES.values()))
        M, N, K = rnd.randint(2300, 3000), rnd.randint(2300, 3000), rnd.randint(1, 32)
        q = ops.fp4_quantize(torch.randint(-3, 4, (N, K), generator=gen, device="cuda").float(), fmt)
        v = ops.fp4_dequantize(q).double()
        off, pad = rnd.choice([(0, 0), (0, 8), (1, 3), (8, 8)])
        dy = torch.randint(-8, 9, (M, off + N + pad), generator=gen, device="cuda").to(torch.bfloat16)[:, off: off + N]
        d = dy.double()
        want = d @ v
        got = ops.fp4_grad_input(dy, q, dtype).double()
        bound = (N + 4) * 2.0 ** -23 * (d.abs() @ v.abs()) + want.abs() * (2.0 ** -22 + torch.finfo(dtype).eps / 2)   # as sum_bound, and the result's rounding
        if bool(((got - want).abs() > bound).any()):
            wrong.append((i, fmt, M, N, K))
    assert not wrong


def test_linear_of_tensors_that_do_not_lie_as_rows(ops):
    """A transposed attention output, a broadcast one, columns of a wider matrix, a transposed weight: as contiguous copies of them."""
    torch.manual_seed(11)
    heads = torch.randn(2, 4, 10, 16, device="cuda").to(torch.bfloat16)
    wide = torch.randn(2, 10, 200, device="cuda").to(torch.bfloat16)
    w = torch.randn(48, 64, device="cuda") * 0.1
    for make in (lambda: heads.transpose(1, 2).flatten(2), lambda: heads.permute(0, 2, 3, 1).reshape(2, 64, 10).transpose(1, 2), lambda: heads[:1, :1, :, :1].expand(2, 4, 10, 64),
                 lambda: wide[:, :5, ::2][..., :64], lambda: wide[..., 8:72]):
        results = []
        for x, weight in ((make(), w), (make().contiguous(), w), (make(), w.t().contiguous().t())):
            x, weight = x.detach(), weight.detach()
            x.requires_grad_()
            weight.requires_grad_()
            y = ops.fp4_linear(x, weight)
            y.backward(torch.arange(y.numel(), device="cuda").view(y.shape).to(torch.bfloat16) / 64)
            results.append((y.detach(), x.grad, weight.grad))
        for r in results[1:]:
            assert all(torch.equal(a, b) for a, b in zip(results[0], r))
    frozen = ops.fp4_quantize(w)
    x = heads.permute(0, 2, 3, 1).reshape(2, 64, 10).transpose(1, 2)
    assert torch.equal(ops.fp4_linear(x, frozen), ops.fp4_linear(x.contiguous(), frozen))
