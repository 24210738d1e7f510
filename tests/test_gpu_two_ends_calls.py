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
