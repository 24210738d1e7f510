"""The norm of many tensors and clipping (bsq_grad_norm_clip, clip_grad_norm) against the formula in 64 bits."""
import importlib
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def make(shapes, dtype, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    dtypes = [dtype] * len(shapes) if not isinstance(dtype, list) else [dtype[i % len(dtype)] for i in range(len(shapes))]
    return [(torch.randn(s, generator=gen) * scale).to(d).cuda() for s, d in zip(shapes, dtypes)]


def exact_norm(grads):
    return math.sqrt(math.fsum((g.double() ** 2).sum().item() for g in grads))


def check(ops, grads, max_norm):
    """Squares in FP32 sums of at most 32 terms (32 * 2^-24 relative, all of one sign), FP64 from there; the norm halves that and is rounded once: 2^-19 holds
    with room.  A result: the factor is off by the norm's 2^-19 and its own rounding, the product by half a step of its type."""
    before = [g.clone() for g in grads]
    norm = ops.clip_grad_norm(grads, max_norm)
    want = exact_norm(before)
    assert norm.shape == () and norm.dtype == torch.float32 and abs(norm.item() - want) <= want * 2.0 ** -19
    f = min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        if f == 1.0:
            assert torch.equal(g, b)
            continue
        w = b.double() * f
        step = torch.finfo(g.dtype).eps / 2
        assert ((g.double() - w).abs() <= w.abs() * (2.0 ** -18 + step) + torch.finfo(g.dtype).smallest_normal * step).all()


SHAPES = [[(1,)], [(7,)], [(16384,)], [(16385,), (1,), (16383,)], [(300, 200), (200,), (3, 5, 7), (1,), (64, 1024)], [(1000, 1000)] * 3 + [(17,)] * 40]


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
def test_norm_and_clipping(ops, shapes, dtype, max_norm):
    check(ops, make(shapes, DTYPES[dtype]), max_norm)


def test_mixed_types_and_no_elements(ops):
    grads = make([(30, 20), (0,), (777,), (5, 0, 2), (50,), (2, 3, 4)], [torch.float32, torch.bfloat16, torch.float16])
    check(ops, grads, 1.0)
    empty = [torch.empty(0, device="cuda")]
    assert ops.clip_grad_norm(empty, 1.0).item() == 0.0


@pytest.mark.parametrize("count", [64, 65, 640, 641, 1500])
def test_many_tensors(ops, count):
    """Around the sizes of the table that a launch takes."""
    check(ops, make([(3 + i % 29,) for i in range(count)], [torch.float32, torch.bfloat16], seed=count), 0.75)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_tensors_off_alignment(ops, dtype):
    base = make([(70000,)], DTYPES[dtype])[0]
    for a, n in ((1, 40000), (3, 7), (5, 16384), (2, 1), (7, 33333)):
        check(ops, [base[a: a + n]], 0.5)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_into_other_tensors(ops, dtype):
    grads = make([(123, 45), (9,), (20000,)], DTYPES[dtype])
    for max_norm in (0.5, 1e9):
        pad = [torch.full((g.numel() + 5,), -7.0, dtype=g.dtype, device="cuda") for g in grads]
        outs = [p[3: 3 + g.numel()].view(g.shape) for p, g in zip(pad, grads)]                   # off the inputs' alignment
        before = [g.clone() for g in grads]
        n1 = ops.clip_grad_norm(grads, max_norm, out=outs)
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
        n2 = ops.clip_grad_norm(before, max_norm)
        assert torch.equal(n1, n2) and all(torch.equal(o, b) for o, b in zip(outs, before))
        assert all((p[:3] == -7).all() and (p[-2:] == -7).all() for p in pad)


@pytest.mark.parametrize("scale", [1e-37, 1e-30, 1e-25, 1e-18, 1e15, 1e19, 1e30, 1e34])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_magnitudes_whose_squares_leave_fp32(ops, scale, dtype):
    check(ops, make([(1000,), (17, 300)], DTYPES[dtype], scale=scale), scale)
    mixed = make([(1000,)], DTYPES[dtype]) + make([(1000,)], DTYPES[dtype], seed=1, scale=scale)
    check(ops, mixed, 1.0)


def test_zeros(ops):
    grads = [torch.zeros(5000, device="cuda"), torch.zeros(40000, dtype=torch.bfloat16, device="cuda")]
    check(ops, grads, 0.0)
    grads[0][4999] = 1e-30
    check(ops, grads, 1.0)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_non_finite_gradients(ops, bad, dtype):
    """As torch.nn.utils.clip_grad_norm_: a NaN goes into everything, an Inf makes the factor 0."""
    for where in (0, 4097, 16383):
        grads = make([(20000,), (50,)], DTYPES[dtype])
        grads[0][where] = bad
        norm = ops.clip_grad_norm(grads, 1.0)
        if math.isnan(bad):
            assert math.isnan(norm.item()) and all(torch.isnan(g).all() for g in grads)
        else:
            assert norm.item() == math.inf and torch.isnan(grads[0][where]) and (grads[1] == 0).all()
        grads = make([(20000,), (50,)], DTYPES[dtype])
        grads[0][where] = bad
        n = ops.clip_grad_norm(grads, None, norm_type=math.inf).item()
        assert math.isnan(n) if math.isnan(bad) else n == math.inf


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_largest_magnitude(ops, dtype):
    grads = make([(20000,), (50,), (1,)], DTYPES[dtype])
    grads[1][3] = -37.5
    before = [g.clone() for g in grads]
    assert ops.clip_grad_norm(grads, None, norm_type=math.inf).item() == 37.5 and all(torch.equal(g, b) for g, b in zip(grads, before))
    assert ops.clip_grad_norm(grads, 3.75, norm_type=math.inf).item() == 37.5
    f = 3.75 / (37.5 + 1e-6)
    step = torch.finfo(DTYPES[dtype]).eps / 2
    for g, b in zip(grads, before):
        assert ((g.double() - b.double() * f).abs() <= b.double().abs() * f * (2.0 ** -23 + step) + 1e-30).all() if dtype != "f16" else \
            ((g.double() - b.double() * f).abs() <= b.double().abs() * f * (2.0 ** -23 + step) + 2.0 ** -25).all()


def test_dense_tensors_of_any_order_and_what_is_refused(ops):
    g = make([(40, 60)], torch.float32)[0]
    check(ops, [g.t()], 1.0)
    check(ops, [g.view(4, 10, 60).permute(1, 2, 0)], 0.5)
    for call in (lambda: ops.clip_grad_norm([g[:, ::2]], 1.0), lambda: ops.clip_grad_norm([g, g], 1.0), lambda: ops.clip_grad_norm([g[:20], g[10:30]], 1.0),
                 lambda: ops.clip_grad_norm([g], 1.0, out=[g.t()]), lambda: ops.clip_grad_norm([g.double()], 1.0), lambda: ops.clip_grad_norm([g], float("nan")),
                 lambda: ops.clip_grad_norm([g[:20]], 1.0, out=[g[10:30]]), lambda: ops.clip_grad_norm([g, g + 1], 1.0, out=[g + 2]),
                 lambda: ops.clip_grad_norm([g], None, out=[g]), lambda: ops.clip_grad_norm([g.cpu()], 1.0)):
        with pytest.raises(ValueError):
            call()
    twice = ops.clip_grad_norm([g, g], None)                       # the norm alone may count a tensor twice
    assert abs(twice.item() - math.sqrt(2) * exact_norm([g])) <= 1e-5 * twice.item()


def test_the_same_bits_every_time_and_under_capture(ops):
    grads = make([(300000,), (77,), (1000, 333)], [torch.float32, torch.bfloat16], seed=8)
    outs = [torch.empty_like(g) for g in grads]
    first = ops.clip_grad_norm(grads, 1.0, out=outs)
    kept = [o.clone() for o in outs]
    for _ in range(5):
        assert torch.equal(ops.clip_grad_norm(grads, 1.0, out=outs), first) and all(torch.equal(o, k) for o, k in zip(outs, kept))
    graphs = []
    for i in range(2):
        mine = [g * (i + 1) for g in grads]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = ops.clip_grad_norm(mine, 1.0)
        graphs.append((graph, mine, norm))
    for i in range(3):
        for _, mine, _ in graphs:
            for m, g in zip(mine, grads):
                m.copy_(g * (i + 2))
        for graph, *_ in graphs:
            graph.replay()
        want = [g * (i + 2) for g in grads]
        n = ops.clip_grad_norm(want, 1.0)
        for _, mine, norm in graphs:
            assert torch.equal(norm, n) and all(torch.equal(m, w) for m, w in zip(mine, want))


def test_in_place_is_seen_by_autograd(ops):
    g = torch.randn(100, device="cuda")
    v = g._version
    ops.clip_grad_norm([g], 1.0)
    assert g._version > v


def test_parameters_are_not_scaled_in_place(ops):
    """Called as PyTorch's own function is, with the parameters: their values would be scaled, not their gradients."""
    model = torch.nn.Linear(30, 20, device="cuda")
    before = [p.detach().clone() for p in model.parameters()]
    model(torch.randn(5, 30, device="cuda")).sum().backward()
    params = list(model.parameters())
    for grads in (model.parameters(), [params[0].grad, params[1]], [params[0] * 2.0]):
        with pytest.raises(ValueError):
            ops.clip_grad_norm(grads, 0.5)
    with torch.no_grad(), pytest.raises(ValueError):
        ops.clip_grad_norm(params, 0.5)
    assert all(torch.equal(p, b) for p, b in zip(params, before))
    assert abs(ops.clip_grad_norm(params, None).item() - exact_norm(before)) <= 1e-5 * exact_norm(before)     # the norm alone of whatever there is
    outs = [torch.empty_like(b) for b in before]
    ops.clip_grad_norm(params, 0.5, out=outs)                      # and into other tensors
    assert all(torch.equal(p, b) for p, b in zip(params, before))
    check(ops, [p.grad for p in params], 0.5)
