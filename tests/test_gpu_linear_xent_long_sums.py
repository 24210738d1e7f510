"""The loss over a vocabulary and its gradient where sums are long and of one sign, so that what additions lose adds up."""
import importlib

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# What a chain of n additions of 16 products cuts off: the tensor core aligns the 17 terms of an addition with the largest and drops what is below 2^-25 of it, 17 * 2^-25 of the sum so far at most,
# which grows evenly: (n + 1) / 2 * 17 * 2^-25 of the chain's sum.  A chain has 1536 of K at most, 96 additions; chains are added up rounded, 2^-24 each.
CHAIN = 97 / 2 * 17 * 2.0 ** -25
# On average half a step, of which the sum over a hundred additions is near (a tenth more).  The gradient's chains have 6144 of K at most, 384 additions.
USUAL, USUAL_BACK = 1.1 * CHAIN / 2, 1.1 * 385 / 2 * 17 * 2.0 ** -26


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def one_sign(tokens, cols, vocab, dtype, top):
    """Logits of `top`, all products of one sign; the target's row is 0, so that its logit is none of them."""
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.rand(tokens, cols, generator=gen, device="cuda") + 0.5
    w = (torch.rand(vocab, cols, generator=gen, device="cuda") + 0.5) * (top / cols)
    w[0] = 0
    return x.to(dtype), w.to(dtype), torch.zeros(tokens, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("tokens", [5, 40, 300])
@pytest.mark.parametrize("cols", [4096, 16384, 40000, 65536])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_loss(ops, dtype, cols, tokens):
    """lse - 0: chains of logits of 40, exponentials of 2^-21, at most 288 additions of 2^-24 of positive terms, and lse rounded to FP32 twice.  One chain for all loses 8e-4 to 1.3e-2."""
    x, w, t = one_sign(tokens, cols, 300, DTYPES[dtype], 40.0)
    l = x.double() @ w.double().t()
    want = torch.logsumexp(l, 1) - l[:, 0]
    got = ops.linear_cross_entropy(x, w, t, reduction="none")
    off = l.amax() * (CHAIN + (cols // 1024 + 1) * 2.0 ** -24) + 2.0 ** -21 + 288 * 2.0 ** -24 + want.amax() * 2.0 ** -23
    assert (got - want).abs().max() <= off


@pytest.mark.parametrize("tokens", [2, 40, 300])
@pytest.mark.parametrize("cols", [4096, 16384, 40000, 65536])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_gradient_of_long_logits(ops, dtype, cols, tokens):
    """dl = p for all but the target: p is exp of a logit less lse, each off by what its chains lose; then two roundings, of dl and of the result, and the sums' own cut-offs.  With logits of one chain dx
    was 4e-3 (16384 columns) to 1.7e-2 (65536) too small, all of it."""
    x, w, t = one_sign(tokens, cols, 300, DTYPES[dtype], 40.0)
    l = x.double() @ w.double().t()
    dl = torch.softmax(l, 1)
    dl[:, 0] -= 1
    dx, dw = dl @ w.double(), (dl.t() @ x.double())[1:]
    x.requires_grad_(), w.requires_grad_()
    a, b = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
    off = (l.amax() * (USUAL + USUAL_BACK + (cols // 1024 + 1) * 2.0 ** -24)).item() + 2.0 ** -21 + 288 * 2.0 ** -24 + 45 * 2.0 ** -23 + USUAL_BACK
    half = torch.finfo(x.dtype).eps / 2
    for got, want in ((a.double(), dx), (b[1:].double(), dw)):
        rel = (got - want) / want
        assert rel.abs().max() <= off + 2.01 * half
        # (roundings of either sign: of many elements of many values a tenth of one is left at most)
        assert rel.mean().abs() <= off + half / 10


@pytest.mark.parametrize("tokens,dtype", [(65536, "f16"), (65536, "bf16"), (524288, "bf16")])
def test_weight_gradient_of_many_tokens(ops, tokens, dtype):
    """An element of dW is a sum over the tokens, here of positive terms: one chain of 524288 lost 3.2e-3, nearly a rounding, of every element."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x = (torch.rand(tokens, 64, generator=gen, device="cuda") + 0.5).to(DTYPES[dtype])
    w = (torch.randn(300, 64, generator=gen, device="cuda") * 0.02).to(DTYPES[dtype])
    t = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    dl = torch.softmax(x.double() @ w.double().t(), 1)
    want = (dl.t() @ x.double())[1:]
    w.requires_grad_()
    got, = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction="sum"), w)
    rel, half = (got[1:].double() - want) / want, torch.finfo(w.dtype).eps / 2
    # (the sum; logits of up to 1 and lse of some 6; roundings of dl of either sign average out over the tokens)
    off = USUAL_BACK + USUAL_BACK + 6 * USUAL + (tokens // 1024 + 1) * 2.0 ** -24 + 2.0 ** -20
    assert rel.abs().max() <= off + half * 1.2
    assert rel.mean().abs() <= off + half / 10


@pytest.mark.parametrize("tokens,cols,vocab", [(2048, 2304, 40000), (300, 2304, 140000), (130, 200, 70001)])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_input_gradient_of_a_large_vocabulary(ops, dtype, tokens, cols, vocab):
    """An element of dx is a sum over the vocabulary, here of positive terms, in pieces and in slices."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.rand(tokens, cols, generator=gen, device="cuda").to(DTYPES[dtype])
    w = ((torch.rand(vocab, cols, generator=gen, device="cuda") + 0.5) * (4 / cols)).to(DTYPES[dtype])
    w[0] = 0
    t = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    rows = slice(0, 130)
    want = torch.softmax(x[rows].double() @ w.double().t(), 1) @ w.double()
    x.requires_grad_()
    got, = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction="sum"), x)
    rel, half = (got[rows].double() - want) / want, torch.finfo(x.dtype).eps / 2
    off = 4 * USUAL_BACK + 15 * USUAL + (vocab // 1024 + 70) * 2.0 ** -24 + 2.0 ** -20     # (logits of some 3 and the sum; lse of some 15)
    assert rel.abs().max() <= off + half * 1.2
    assert rel.mean().abs() <= off + half / 10


@pytest.mark.parametrize("tokens,cols,vocab", [(40, 9000, 700), (300, 13000, 515), (9000, 64, 300)])
def test_waits_that_run_out_between_chains(ops, lib, tokens, cols, vocab):
    """Sums of several chains, given up: NaN, and the next call is as before."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x, w = torch.randn(tokens, cols, generator=gen, device="cuda").bfloat16().requires_grad_(), (torch.randn(vocab, cols, generator=gen, device="cuda") / cols ** 0.5).bfloat16().requires_grad_()
    t = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    want = torch.autograd.grad(ops.linear_cross_entropy(x, w, t), (x, w))
    try:
        lib.bsq_test_limit_waits(0)
        got = torch.autograd.grad(ops.linear_cross_entropy(x, w, t), (x, w))
        assert all(torch.isnan(g).all() for g in got)
        torch.cuda.synchronize()
    finally:
        lib.bsq_test_limit_waits(1 << 16)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(ops.linear_cross_entropy(x, w, t), (x, w)), want))
