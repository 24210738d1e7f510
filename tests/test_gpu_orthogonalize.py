"""Orthogonalised updates (bsq_orthogonalize, orthogonalize) against the steps in 64 bits, and a training step that uses everything from the linear layer to the update."""
import importlib
import math
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
QUINTIC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def make(m, n, kind="noise", seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 7 * m + n)
    g = torch.randn(m, n, generator=gen, device="cuda")
    if kind == "shared":                                           # a few directions far above the noise
        g += 6 * torch.randn(m, 4, generator=gen, device="cuda") @ torch.randn(4, n, generator=gen, device="cuda")
    elif kind == "decay":                                          # singular values from 1 to 1 / 300
        k = min(m, n)
        u = torch.linalg.qr(torch.randn(m, k, generator=gen, device="cuda"))[0]
        v = torch.linalg.qr(torch.randn(n, k, generator=gen, device="cuda"))[0]
        g = (u * torch.logspace(0, -2.5, k, device="cuda")) @ v.t()
    return g * scale


def exact(g, steps=5, table=None, eps=1e-7):
    x = g.double()
    x = x / (x.square().sum().sqrt() + eps)
    for a, b, c in table or [QUINTIC] * steps:
        if x.size(0) <= x.size(1):
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
        else:
            s = x.t() @ x
            x = a * x + x @ (b * s + c * (s @ s))
    return x


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def tolerance(g, want, dtype, table=None):
    """In the 2-norm.  Products of one half: what the three roundings of a step to 2^-12 leave is below 2^-9 in a model of them for these spectra (0.1e-3 to 1.4e-3), and a rounding to
    BF16 is at most 2^-8 / sqrt(3) of the norm: 2^-8 holds both.  Products of both halves: X is rounded to 2^-22 and FP32 sums of (long + 2 short) / 16 additions are cut off at
    2^-23 each; what is left on the small singular values grows with them, by the product of the a's, against a result whose norm is that of `want`; then the result's own rounding."""
    m, n = g.shape
    if dtype == torch.bfloat16 and min(m, n) > 128:
        return 2.0 ** -8
    grown = math.prod(abs(t[0]) for t in table or [QUINTIC] * 5) / want.norm().item()
    return (grown + 8) * (2.0 ** -21 + (max(m, n) + 2 * min(m, n)) / 16 * 2.0 ** -23) + torch.finfo(dtype).eps / 2


def check(ops, g, dtype=torch.bfloat16, **more):
    got = ops.orthogonalize(g, dtype=dtype, **more)
    assert got.dtype == dtype and got.shape == g.shape
    want = exact(g)
    assert off(got, want) <= tolerance(g, want, dtype), (off(got, want), tolerance(g, want, dtype))
    return got


SIDES = [(1, 1), (1, 9), (9, 1), (2, 3), (16, 16), (33, 7), (64, 1024), (65, 130), (128, 128), (129, 129), (130, 300), (300, 130), (257, 256), (777, 2051), (2051, 777), (513, 1100), (1030, 200), (200, 5000)]


@pytest.mark.parametrize("m,n", SIDES)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_sides(ops, dtype, m, n):
    check(ops, make(m, n).to(DTYPES[dtype]))


@pytest.mark.parametrize("m,n", SIDES)
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_both_halves(ops, out, m, n):
    check(ops, make(m, n), DTYPES[out])


@pytest.mark.parametrize("m,n", [(40, 300), (200, 200), (1500, 300), (300, 1500), (2304, 2304), (4000, 2500)])
@pytest.mark.parametrize("kind", ["shared", "decay"])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_spectra(ops, dtype, kind, m, n):
    for out in (torch.bfloat16, torch.float32):
        check(ops, make(m, n, kind).to(DTYPES[dtype]), out)


@pytest.mark.parametrize("scale", [1e-4, 1e-2, 1e4, 1e18, 1e30])
def test_magnitudes(ops, scale):
    check(ops, make(150, 300, scale=scale))
    check(ops, make(150, 300, scale=scale), torch.float32)
    if scale < 1e4:
        check(ops, make(300, 150, scale=scale).half())


@pytest.mark.parametrize("m,n", [(33000, 65536), (65536, 33000)])
def test_beyond_32_bits(ops, m, n):
    """2.2 10^9 elements of rank one, u v^T: the one singular value goes the way of a number, the rest stays what it is, nothing."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    u, v = torch.randint(1, 9, (m, 1), generator=gen, device="cuda").bfloat16(), torch.randint(1, 9, (1, n), generator=gen, device="cuda").bfloat16()
    g = u * v                                                      # (whole numbers up to 64: exact)
    got = ops.orthogonalize(g)
    s, (a, b, c) = 1.0, QUINTIC
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    scale = s / (u.double().norm() * v.double().norm()).item()
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        want = u[rows].double() @ v.double() * scale
        assert off(got[rows], want) <= 2.0 ** -8


@pytest.mark.parametrize("m,n", [(16384, 32768), (32768, 16384)])
def test_long_sums_of_one_sign(ops, m, n):
    """Rank one in FP32.  What the sums of P X lose need not be of X's rank: each later step pulls it up by a = 3.4445.  A chain has 92 additions of 16 products at most (23 stages of 64); each cuts
    off up to 2^-23 of what it has by then, so the sum loses up to (92 + 1) / 2 * 2^-23 = 5.5e-6 of |P| s.  With s = 1, 0.701, 1.114, 0.721, 1.090 and |P| = 2.74, 1.86, 2.80, 1.93, 2.81, and 3.4445^4
    ... 1 for the steps that follow: 2.8e-3 of s = 0.696 at the end, 4.1e-3 of it; roundings to 22 bits are in that, and A and P, whose errors share u or v with X and grow by 1.6 a step at most, add 2.5e-4."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    u, v = torch.randint(1, 9, (m, 1), generator=gen, device="cuda").bfloat16(), torch.randint(1, 9, (1, n), generator=gen, device="cuda").bfloat16()
    got = ops.orthogonalize(u * v, dtype=torch.float32)
    s, (a, b, c) = 1.0, QUINTIC
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    scale = s / (u.double().norm() * v.double().norm()).item()
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        assert off(got[rows], u[rows].double() @ v.double() * scale) <= 4.5e-3


def test_eps(ops):
    g = make(150, 300, scale=1e-9)                                 # |G| about 2e-7
    for eps in (0.0, 1e-7, 1e-6):
        want = exact(g, eps=eps)
        assert off(ops.orthogonalize(g, eps=eps), want) <= 2.0 ** -8


@pytest.mark.parametrize("m,n", [(1, 1), (5, 70), (140, 300), (600, 131)])
@pytest.mark.parametrize("out", sorted(DTYPES))
def test_zeros(ops, out, m, n):
    assert (ops.orthogonalize(torch.zeros(m, n, device="cuda"), dtype=DTYPES[out]) == 0).all()
    assert (ops.orthogonalize(torch.zeros(m, n, device="cuda"), dtype=DTYPES[out], eps=0.0) == 0).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("m,n", [(5, 70), (140, 300), (600, 131)])
def test_not_finite(ops, value, m, n):
    """In one matrix of three: that one is NaN, the others are what they were."""
    g = torch.stack([make(m, n, seed=i) for i in range(3)])
    want = ops.orthogonalize(g)
    g[1, m // 2, n // 3] = value
    got = ops.orthogonalize(g)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_a_matrix_of_lower_rank(ops):
    g = torch.zeros(200, 400, device="cuda")
    g[7] = 3.0
    check(ops, g)
    g[:, 5] = 1.0
    check(ops, g, torch.float32)


@pytest.mark.parametrize("steps", [1, 2, 3, 8])
@pytest.mark.parametrize("m,n", [(64, 100), (150, 300), (300, 150)])
def test_steps_and_scale(ops, m, n, steps):
    g = make(m, n)
    want = exact(g, steps) * 0.2
    assert off(ops.orthogonalize(g, steps=steps, scale=0.2), want) <= 2.0 ** -8


@pytest.mark.parametrize("m,n", [(64, 100), (150, 300), (300, 150)])
def test_coefficients(ops, m, n):
    """The classic cubic steps, ones of each step's own, and none at all."""
    for table in ([(1.5, -0.5, 0.0)] * 10, [(4.0, -7.0, 4.0), (3.0, -4.0, 2.0), (1.875, -1.25, 0.375)], [(1.0, 0.0, 0.0)], [(0.0, 0.0, 0.0)]):
        g = make(m, n)
        got, want = ops.orthogonalize(g, steps=len(table), coefficients=table), exact(g, table=table)
        assert (got == 0).all() if not want.any() else off(got, want) <= 2.0 ** -8
    same = ops.orthogonalize(g, coefficients=[QUINTIC] * 5)
    assert torch.equal(same, ops.orthogonalize(g))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_lists_and_stacks(ops, dtype):
    t = DTYPES[dtype]
    one = [make(m, n, seed=i).to(t) for i, (m, n) in enumerate([(64, 100), (300, 140), (64, 100), (5, 5), (64, 100), (140, 300), (300, 140)])]
    want = [ops.orthogonalize(g) for g in one]
    assert all(torch.equal(a, b) for a, b in zip(ops.orthogonalize(one), want))
    mixed = one[:3] + [make(64, 100, seed=9).to(torch.float16), torch.empty(0, 5, device="cuda"), torch.empty(3, 7, 0, device="cuda")] + one[3:]
    got = ops.orthogonalize(mixed)
    assert [g.shape for g in got] == [g.shape for g in mixed]
    assert all(torch.equal(a, b) for a, b in zip(got[:3] + got[6:], want)) and torch.equal(got[3], ops.orthogonalize(mixed[3]))
    stack = torch.stack([make(150, 200, seed=i).to(t) for i in range(6)]).view(2, 3, 150, 200)
    got = ops.orthogonalize(stack)
    assert got.shape == stack.shape and all(torch.equal(got[i, j], ops.orthogonalize(stack[i, j])) for i in range(2) for j in range(3))


@pytest.mark.parametrize("count", [63, 64, 65, 150])
def test_many(ops, count):
    g = [make(17, 40, seed=i) for i in range(count)]
    got = ops.orthogonalize(g)
    assert torch.equal(got[-1], ops.orthogonalize(g[-1])) and torch.equal(got[0], ops.orthogonalize(g[0]))
    for a, b in zip(got, g):
        assert off(a, exact(b)) <= 2.0 ** -8


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_strides(ops, dtype):
    t = DTYPES[dtype]
    g = make(150, 201).to(t)
    want = ops.orthogonalize(g)
    wide = torch.full((150, 333), 9.0, dtype=t, device="cuda")
    wide[:, 77:278] = g
    assert torch.equal(ops.orthogonalize(wide[:, 77:278]), want)
    assert torch.equal(ops.orthogonalize(g.t().contiguous().t()), want)
    stack = torch.stack([g, g * 2, g * 4], dim=1)                  # the matrices of a stack row by row
    assert torch.equal(ops.orthogonalize(stack.transpose(0, 1)), torch.stack([want] * 3))    # (powers of two change nothing but the scale)
    assert torch.equal(ops.orthogonalize(g.expand(4, 150, 201)), want.expand(4, 150, 201))


def test_transposed_is_the_transpose(ops):
    g = make(300, 700)
    assert off(ops.orthogonalize(g.t()).t(), exact(g)) <= 2.0 ** -8


@pytest.mark.parametrize("out", sorted(DTYPES))
@pytest.mark.parametrize("m,n", [(3, 77), (129, 93), (300, 513), (513, 300)])
def test_into_other_tensors(ops, out, m, n):
    t = DTYPES[out]
    g = make(m, n)
    want = ops.orthogonalize(g, dtype=t)
    for first in (0, 8, 1):
        big = torch.full((m + 2, n + 11), -7.0, dtype=t, device="cuda")
        to = big[1:-1, first: first + n]
        assert ops.orthogonalize(g, dtype=t, out=to) is to and torch.equal(to, want)
        to.fill_(-7.0)
        assert (big == -7.0).all()


def test_out_is_refused(ops):
    g = make(64, 64)
    stack = torch.empty(3, 64, 64, dtype=torch.bfloat16, device="cuda")
    for o in (g, g.bfloat16()[:32], stack[0].float(), [stack[0]], torch.empty(64, 64, dtype=torch.bfloat16), torch.empty(64, 64, dtype=torch.bfloat16, device="cuda").t(),
              torch.empty(64, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)):
        with pytest.raises(ValueError):
            ops.orthogonalize(g, out=o)
    half = g.bfloat16()
    for call in (lambda: ops.orthogonalize(half, out=half), lambda: ops.orthogonalize([half, half], out=[stack[0], stack[0]]), lambda: ops.orthogonalize([half], out=[stack[0], stack[1]]),
                 lambda: ops.orthogonalize(torch.stack([half, half]), out=stack[:1].expand(2, 64, 64)), lambda: ops.orthogonalize(g, coefficients=(10.0, 10.0, 10.0)),
                 lambda: ops.orthogonalize(g, steps=2.5), lambda: ops.orthogonalize(g, scale=math.inf), lambda: ops.orthogonalize(g[0]), lambda: ops.orthogonalize(g.double()),
                 lambda: ops.orthogonalize(g, coefficients=[QUINTIC] * 4), lambda: ops.orthogonalize([g, g.cpu()])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("m,n", [(64, 1024), (777, 2051), (2051, 777), (2304, 2304)])
def test_same_bits_every_time(ops, m, n):
    g = make(m, n)
    want = ops.orthogonalize(g)
    for _ in range(5):
        assert torch.equal(ops.orthogonalize(g), want)


def test_captured(ops):
    g = [torch.empty(150, 300, device="cuda"), torch.empty(64, 100, device="cuda"), torch.empty(150, 300, device="cuda")]
    for t, i in zip(g, range(3)):
        t.copy_(make(*t.shape, seed=i))
    ops.orthogonalize(g)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                             # two graphs, each with memory of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.orthogonalize(g)
        graphs.append((graph, got))
    for seed in (5, 6):
        for t, i in zip(g, range(3)):
            t.copy_(make(*t.shape, seed=seed + i))
        for graph, got in graphs:
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, ops.orthogonalize(g)))


def test_side_by_side(ops):
    cases = [[make(100 + 80 * i, 90 + 70 * j, seed=i) for j in range(3)] for i in range(4)]
    want = [ops.orthogonalize(c) for c in cases]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = ops.orthogonalize(cases[i])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))


@pytest.mark.parametrize("m,n", [(64, 100), (300, 200), (2304, 2304)])
def test_waits_that_run_out(ops, lib, m, n):
    g = make(m, n)
    want = ops.orthogonalize(g)
    try:
        lib.bsq_test_limit_waits(0)
        assert torch.isnan(ops.orthogonalize(g)).all()
        torch.cuda.synchronize()
    finally:
        lib.bsq_test_limit_waits(1 << 16)
    assert torch.equal(ops.orthogonalize(g), want)


def test_a_training_step(ops):
    """A layer in 4 bits, the loss over a vocabulary, its backward pass, the norm of all gradients, and the update: each against the formulas from what the step before it gave."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(300, 256, generator=gen, device="cuda").bfloat16()
    layer = (torch.randn(512, 256, generator=gen, device="cuda") / 16).bfloat16().requires_grad_()
    head = (torch.randn(3001, 512, generator=gen, device="cuda") / 20).bfloat16().requires_grad_()
    target = torch.randint(0, 3001, (300,), generator=gen, device="cuda")
    target[::7] = -100
    hidden = ops.fp4_linear(x, layer)
    loss = ops.linear_cross_entropy(hidden, head, target)
    loss.backward()
    logits = hidden.detach().double() @ head.detach().double().t()
    assert abs(loss.item() - torch.nn.functional.cross_entropy(logits, target).item()) <= 1e-4
    a = hidden.detach().double().requires_grad_()
    b = head.detach().double().requires_grad_()
    da, db = torch.autograd.grad(torch.nn.functional.cross_entropy(a @ b.t(), target), (a, b))
    assert off(head.grad, db) <= 2.0 ** -7                         # dl and the result, each rounded to BF16
    want = da.t() @ ops.fp4_dequantize(ops.fp4_quantize(x)).double()
    assert off(layer.grad, want) <= 2.0 ** -7 + 2.0 ** -8          # ... and rounded once more
    grads = [layer.grad, head.grad]
    before = [g.double() for g in grads]
    norm = ops.clip_grad_norm(grads, 0.01)
    assert abs(norm.item() - math.sqrt(sum((g ** 2).sum().item() for g in before))) <= norm.item() * 2.0 ** -19
    updates = ops.orthogonalize(grads, scale=0.2)
    for u, g in zip(updates, grads):
        assert off(u, exact(g) * 0.2) <= 2.0 ** -8
    with torch.no_grad():
        for p, u in zip((layer, head), updates):
            p.sub_(u, alpha=0.02)
    assert all(torch.isfinite(p).all() for p in (layer, head))
