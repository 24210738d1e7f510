"""Calls of the loss over a vocabulary and of orthogonalised updates that other parts of PyTorch make, and combinations of their arguments."""
import importlib

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def operands(tokens=8, cols=64, vocab=100, dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(tokens + cols + vocab)
    x, w = torch.randn(tokens, cols, generator=gen, device="cuda"), torch.randn(vocab, cols, generator=gen, device="cuda") / cols ** 0.5
    return x.to(dtype), w.to(dtype), torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")


@pytest.mark.parametrize("which", ["x", "weight", "strided x"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(ops, which, grad):
    """A derivative that is asked for is not left out of a sum without a word."""
    x, w, t = operands()
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
        if which == "x":
            x = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        elif which == "weight":
            w = torch.autograd.forward_ad.make_dual(w, torch.ones_like(w))
        else:
            x = torch.autograd.forward_ad.make_dual(x.t().contiguous(), torch.ones_like(x).t().contiguous()).t()
        with pytest.raises(NotImplementedError):
            ops.linear_cross_entropy(x, w, t)
        assert torch.isfinite(ops.linear_cross_entropy(*operands()))            # nothing carries a tangent


def test_results_of_a_list_are_tensors_of_their_own(ops):
    """Changing one in place is no change of another, and is allowed with a tensor that requires a gradient."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    updates = [torch.randn(*s, generator=gen, device="cuda") for s in ((64, 80), (64, 80), (64, 80), (2, 200, 150), (2, 200, 150), (64, 80), (0, 5), (0, 5), (3, 0), (3, 0))]
    out = ops.orthogonalize(updates)
    assert [o.shape for o in out] == [u.shape for u in updates] and all(o.is_contiguous() and not o._is_view() for o in out)
    assert all(torch.equal(a, ops.orthogonalize(b)) for a, b in zip(out, updates) if b.numel())
    p, kept = torch.ones(64, 80, dtype=torch.bfloat16, device="cuda", requires_grad=True), out[0].clone()
    y = (p * out[0]).sum()                                         # saves out[0]
    out[1].mul_(2), out[3].zero_()
    y.backward()
    assert torch.equal(p.grad, kept) and [o._version for o in out[:5]] == [0, 1, 0, 1, 0]
    out[2].mul_(p)
    assert out[2].requires_grad


@pytest.mark.parametrize("m,k,n", [(64, 3, 80), (300, 2, 200), (150, 5, 33), (40, 70, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_side_by_side(ops, dtype, m, k, n):
    """Written by columns of one tensor, as a list and as a stack; input and output as halves of one."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    updates = torch.randn(k, m, n, generator=gen, device="cuda")
    want = ops.orthogonalize(updates, dtype=dtype)
    big = torch.full((m, k, n), -7.0, dtype=dtype, device="cuda")
    assert torch.equal(ops.orthogonalize(updates, dtype=dtype, out=big.transpose(0, 1)), want) and torch.equal(big.transpose(0, 1), want)
    big = torch.full((m, k * n + 1), -7.0, dtype=dtype, device="cuda")
    outs = [big[:, i * n: (i + 1) * n] for i in range(k)][::-1]
    got = ops.orthogonalize(list(updates)[::-1], dtype=dtype, out=outs)
    assert all(a is b for a, b in zip(got, outs)) and torch.equal(torch.stack(outs[::-1]), want) and (big[:, -1] == -7).all()
    both = torch.zeros(m, 2 * n, dtype=dtype, device="cuda")
    both[:, :n] = updates[0]
    one = ops.orthogonalize(both[:, :n].clone(), dtype=dtype)
    ops.orthogonalize(both[:, :n], dtype=dtype, out=both[:, n:])
    assert torch.equal(both[:, n:], one) and torch.equal(both[:, :n], updates[0].to(dtype))


def test_what_is_said_of_a_call_that_fails(ops, monkeypatch):
    """An overlap where there is one; the library's own error otherwise, also with `out`."""
    g = torch.randn(64, 64, device="cuda").bfloat16()
    out = torch.empty(2, 64, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="apart"):
        ops.orthogonalize([g, g], out=[out[0], out[0]])
    with pytest.raises(ValueError, match="apart"):
        ops.orthogonalize([g, g], out=[out.view(64, 128)[:, :64], out.view(64, 128)[:, 60:124]])
    with pytest.raises(ValueError, match="coefficients"):
        ops.orthogonalize(g, out=out[0], coefficients=(10.0, 10.0, 10.0))

    def fails(*args):
        raise RuntimeError("bsq_orthogonalize failed")
    monkeypatch.setattr(ops, "_call", fails)
    with pytest.raises(RuntimeError, match="failed"):
        ops.orthogonalize(g, out=out[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("m,n", [(64, 100), (300, 513), (513, 300), (1100, 1100)])
def test_products_of_both_halves_of_several(ops, dtype, m, n):
    """FP32 and FP16 results of a list and of a stack: what each gives alone, and X's formula."""
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    updates = [torch.randn(m, n, generator=gen, device="cuda") * 10.0 ** i for i in range(5)]
    alone = [ops.orthogonalize(u, dtype=dtype) for u in updates]
    assert all(torch.equal(a, b) for a, b in zip(ops.orthogonalize(updates, dtype=dtype), alone))
    assert torch.equal(ops.orthogonalize(torch.stack(updates), dtype=dtype), torch.stack(alone))
    for u, a in zip(updates, alone):
        x = u.double() / u.double().norm()
        for _ in range(5):
            s = x @ x.t()
            x = 3.4445 * x + (-4.7750 * s + 2.0315 * s @ s) @ x
        # noise keeps its digits: sums of FP32 and operands of 22 bits, 2^-13 at most, and the result's rounding
        assert (a.double() - x).norm() <= (2.0 ** -13 + torch.finfo(dtype).eps / 2) * x.norm()


@pytest.mark.parametrize("m,n,dtype", [(1024, 4096, torch.bfloat16), (4096, 1024, torch.float32), (128, 65536, torch.bfloat16)])
def test_more_than_share_the_scratch(ops, m, n, dtype):
    """More matrices than 1 GB of scratch takes: several runs, one behind the other."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    two = [torch.randn(m, n, generator=gen, device="cuda").bfloat16() for _ in range(2)]
    want = [ops.orthogonalize(u, dtype=dtype) for u in two]
    got = ops.orthogonalize([two[i % 2] for i in range(61)], dtype=dtype)
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("e", [0.1, 1.0])
@pytest.mark.parametrize("tokens,cols,vocab", [(300, 64, 70001), (2, 40, 140000), (1025, 72, 66000)])
def test_smoothing_over_several_pieces(ops, dtype, e, tokens, cols, vocab):
    """dl = p - e / V, less 1 - e at the target, a piece of the vocabulary at a time: against the formula in 64 bits."""
    x, w, t = operands(tokens, cols, vocab, dtype)
    t[0], t[-1] = vocab - 1, -100
    live = t != -100
    l = x.double() @ w.double().t()
    logp = torch.log_softmax(l, 1)
    want = torch.full_like(l, e / vocab)
    want[live.nonzero()[:, 0], t[live]] += 1 - e
    loss = -(want * logp).sum(1) * live
    dl = (torch.exp(logp) - want) * live[:, None]
    dx, dw = dl @ w.double(), dl.t() @ x.double()
    x.requires_grad_(), w.requires_grad_()
    got = ops.linear_cross_entropy(x, w, t, label_smoothing=e, reduction="none")
    a, b = torch.autograd.grad(got.sum(), (x, w))
    assert ((got - loss).abs() <= 1e-4).all()                      # (sums of 1100 products and of 140000 terms in FP32: a few 2^-23 of 12, 300 additions of 2^-24)
    # each row or column of the gradients: dl and the result rounded once each, 2^-8 or 2^-11, and 2^-20 of what e / V takes from p before dl is rounded
    half = torch.finfo(dtype).eps / 2
    near = (dl.abs() @ w.double().abs(), dl.abs().t() @ x.double().abs())
    for got, want, by in ((a, dx, near[0]), (b, dw, near[1])):
        assert ((got.double() - want).norm(dim=1) <= 2.02 * half * by.norm(dim=1) + 2.0 ** -20 * (x.abs().max() + w.abs().max()) * by.size(1) ** 0.5).all()
