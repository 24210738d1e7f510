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
