"""The loss over a vocabulary and its gradient (bsq_linear_xent, linear_cross_entropy) against the formulas in 64 bits."""
import importlib
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def make(tokens, cols, vocab, dtype, seed=0, ignored=0.2, lift=6.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(vocab, cols, generator=gen, device="cuda") * (1.5 / cols ** 0.5)
    t = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    x = torch.randn(tokens, cols, generator=gen, device="cuda") + w[t] * (lift / 2.25) * torch.rand(tokens, 1, generator=gen, device="cuda")
    if tokens > 1:
        t[torch.rand(tokens, generator=gen, device="cuda") < ignored] = IGNORE
        t[-1] = vocab - 1
    return x.to(dtype), w.to(dtype), t


def exact(x, w, t, e, g):
    """Losses, and for the gradients `g` of the losses: dx, dw; with each how far off it may be."""
    dtype, vocab, cols, tokens = x.dtype, w.size(0), x.size(1), x.size(0)
    x, w, live = x.double(), w.double(), t != IGNORE
    l = x @ w.t()
    lse = torch.logsumexp(l, dim=1)
    want = torch.full_like(l, e / vocab)
    want[live.nonzero()[:, 0], t[live]] += 1 - e
    loss = torch.where(live, lse - (want * l).sum(dim=1), torch.zeros_like(lse))
    # A logit: a chain of cols / 16 additions that are cut off (a step of 2^-23 each, of at most the sum of magnitudes), the 16 products within one likewise.
    off_l = ((cols / 16 + 2) * 2.0 ** -23) * (x.abs() @ w.abs().t()).amax(dim=1)
    # lse: logits, exponentials good to 2^-21, at most 288 additions of 2^-24 in a tile and behind it, and the logarithm's value rounded to FP32.  The loss takes a logit (or their mean) away.
    off_lse = off_l + 2.0 ** -21 + 288 * 2.0 ** -24 + lse.abs() * 2.0 ** -23
    off_loss = live * (off_lse + off_l + e * 2.0 ** -16 * l.abs().amax(dim=1) + loss.abs() * 2.0 ** -24)
    p = torch.exp(l - lse[:, None])
    dl = (p - want) * (g * live)[:, None]
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    # dl: the logits' and lse's errors and the exponential's in p, the subtraction's, one rounding; FP16: scaled so that the largest g is 2^13 or more, steps of 2^-25 there
    off_dl = (p * (off_l + off_lse + 2.0 ** -21)[:, None] + 2.0 ** -23) * (g * live).abs()[:, None] * (1 + half) + dl.abs() * half
    # (FP32's rounding of p - want is relative to the larger of the two; where p is near want it is at most 2^-23 of 1)
    if dtype == torch.float16:
        off_dl += (g * live).abs().max() * 2.0 ** -38
    a = dl.abs() + off_dl
    dx, dw = dl @ w, dl.t() @ x
    # sums: chains of vocab / 16 and tokens / 16 additions, a few more where pieces and slices are joined; then one rounding
    off_dx = off_dl @ w.abs() + ((vocab / 16 + 80) * 2.0 ** -23) * (a @ w.abs()) + dx.abs() * half * 1.01 + tiny
    off_dw = off_dl.t() @ x.abs() + ((tokens / 16 + 3) * 2.0 ** -23) * (a.t() @ x.abs()) + dw.abs() * half * 1.01 + tiny
    return loss, off_loss, dx, off_dx, dw, off_dw


def near(got, want, off):
    assert got.shape == want.shape
    bad = ((got.double() - want).abs() > off) | torch.isnan(got)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), got[bad][:3].tolist(), want[bad][:3].tolist(), off[bad][:3].tolist())


def check(ops, x, w, t, e=0.0, seed=0):
    """Each token's loss with a gradient of its own; the sum and the mean from the same formulas."""
    g = torch.rand(t.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") + 0.25
    loss, off_loss, dx, off_dx, dw, off_dw = exact(x, w, t, e, g.double())
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    got = ops.linear_cross_entropy(x, w, t, label_smoothing=e, reduction="none")
    assert got.dtype == torch.float32
    near(got.detach(), loss, off_loss)
    a, b = torch.autograd.grad(got, (x, w), g)
    assert a.dtype == x.dtype and b.dtype == w.dtype
    near(a, dx, off_dx)
    near(b, dw, off_dw)
    count = int((t != IGNORE).sum())
    for how, n in (("sum", 1), ("mean", count)):
        total = ops.linear_cross_entropy(x, w, t, label_smoothing=e, reduction=how)
        assert total.shape == ()
        if n:
            near(total.detach(), loss.sum() / n, off_loss.sum() / n + (loss.sum() / n).abs() * 2.0 ** -24)


SIZES = [(1, 1, 1), (1, 8, 2), (2, 7, 3), (1, 64, 300), (3, 65, 129), (31, 200, 127), (33, 16, 128), (64, 128, 1000), (128, 72, 257), (129, 1031, 131), (300, 333, 515), (130, 257, 12801),
         (300, 64, 6400), (300, 96, 6529), (1000, 520, 5001), (5, 1000, 20001), (1, 4096, 5000)]


@pytest.mark.parametrize("tokens,cols,vocab", SIZES)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_sizes(ops, dtype, tokens, cols, vocab):
    check(ops, *make(tokens, cols, vocab, DTYPES[dtype], seed=tokens + cols + vocab))


@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("cols,vocab", [(1, 1), (7, 3), (8, 33), (66, 5000), (1000, 9473), (1031, 20001), (4104, 700), (2, 40000)])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_few_tokens(ops, dtype, cols, vocab, tokens):
    """Around the kernel that takes up to four: its three widths of loads, rows and CTAs that have nothing."""
    check(ops, *make(tokens, cols, vocab, DTYPES[dtype], seed=tokens + vocab, ignored=0.3), e=0.1 * (vocab % 2))


def test_few_tokens_of_many_columns(ops):
    """More than fit into shared memory."""
    check(ops, *make(1, 50000, 300, torch.bfloat16))
    check(ops, *make(4, 12296, 300, torch.bfloat16))
    check(ops, *make(4, 12288, 300, torch.float16))


@pytest.mark.parametrize("tokens", [2, 40, 300])
def test_infinite_weights(ops, tokens):
    """A logit of -Inf has no probability; one of +Inf leaves nothing to compute with."""
    x, w, t = make(tokens, 64, 7000, torch.bfloat16, ignored=0.0)
    x = x.abs()
    t.clamp_(min=300)
    want = ops.linear_cross_entropy(x, torch.cat([w[300:]]), t - 300, reduction="none")
    low = w.clone()
    low[:300, 3] = float("-inf")
    got = ops.linear_cross_entropy(x, low, t, reduction="none")
    assert torch.isfinite(got).all() and (got - want).abs().max() <= 1e-5
    own = torch.full_like(t, 7)                                    # a target without probability
    assert (ops.linear_cross_entropy(x, low, own, reduction="none") == float("inf")).all()
    low[5000, 3] = float("inf")
    assert torch.isnan(ops.linear_cross_entropy(x, low, torch.full_like(t, 5000), reduction="none")).all()
    assert torch.isnan(ops.linear_cross_entropy(x, low, t, reduction="none")).all()


@pytest.mark.parametrize("tokens,cols,vocab", [(1, 8, 2), (7, 65, 129), (300, 96, 6529), (40, 256, 3001)])
@pytest.mark.parametrize("e", [0.1, 0.5, 1.0])
def test_label_smoothing(ops, e, tokens, cols, vocab):
    for dtype in DTYPES.values():
        check(ops, *make(tokens, cols, vocab, dtype, seed=vocab), e=e)


@pytest.mark.parametrize("tokens,cols,vocab", [(300, 64, 70001), (1025, 72, 66000), (2, 40, 140000), (140, 1100, 65537)])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_several_pieces(ops, dtype, tokens, cols, vocab):
    check(ops, *make(tokens, cols, vocab, DTYPES[dtype], seed=vocab))


def test_many_tokens(ops):
    check(ops, *make(9001, 40, 1031, torch.bfloat16))
    check(ops, *make(40000, 16, 513, torch.float16))


@pytest.mark.parametrize("tokens", [2, 9])
def test_weights_beyond_32_bits(ops, tokens):
    """2.2 10^9 elements, rows off 16 bytes; targets and the rows that are looked at on both sides of 2^31."""
    cols, vocab = 4100, 530000
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    w = torch.empty(vocab, cols, dtype=torch.bfloat16, device="cuda").normal_(0, 1.5 / cols ** 0.5, generator=gen)
    x = torch.randn(tokens, cols, generator=gen, device="cuda").bfloat16()
    t = torch.tensor([vocab - 1 - 3000 * i for i in range(tokens)], device="cuda")
    l = torch.cat([x.double() @ w[i: i + 50000].double().t() for i in range(0, vocab, 50000)], dim=1)
    loss = torch.nn.functional.cross_entropy(l, t, reduction="none")
    dl = torch.softmax(l, 1)
    dl[torch.arange(tokens), t] -= 1
    x.requires_grad_(), w.requires_grad_()
    got = ops.linear_cross_entropy(x, w, t, reduction="none")
    assert ((got - loss).abs() <= 1e-4).all()                      # (cols / 16 steps of 2^-23 of sums of magnitudes of some 80, and more)
    dx, dw = torch.autograd.grad(got.sum(), (x, w))
    with torch.no_grad():
        want = sum(dl[:, i: i + 50000] @ w[i: i + 50000].double() for i in range(0, vocab, 50000))
        assert ((dx.double() - want).norm(dim=1) <= 2.0 ** -7 * want.norm(dim=1)).all()
        for first in (0, 500, (1 << 31) // cols - 50, vocab - 100):
            part = dl[:, first: first + 100].t() @ x.double()
            assert ((dw[first: first + 100].double() - part).norm() <= 2.0 ** -7 * part.norm())
        for v in t.tolist():
            part = dl[:, v] @ x.double()
            assert ((dw[v].double() - part).norm() <= 2.0 ** -7 * part.norm())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_strides(ops, dtype):
    x, w, t = make(150, 100, 1000, DTYPES[dtype])
    wide_x, wide_w = torch.full((150, 131), 9.0, dtype=x.dtype, device="cuda"), torch.full((1000, 120), 9.0, dtype=x.dtype, device="cuda")
    wide_x[:, 3:103], wide_w[:, 8:108] = x, w
    for a, b in ((wide_x[:, 3:103], w), (x, wide_w[:, 8:108]), (wide_x[:, 3:103], wide_w[:, 8:108]), (x.t().contiguous().t(), w.t().contiguous().t())):
        assert torch.equal(a, x) and torch.equal(b, w)
        check(ops, a, b, t)
    check(ops, x[:1].expand(150, 100), w, t)


def test_leading_dimensions(ops):
    x, w, t = make(60, 64, 500, torch.bfloat16)
    flat = ops.linear_cross_entropy(x, w, t, reduction="none")
    assert torch.equal(ops.linear_cross_entropy(x.view(3, 4, 5, 64), w, t.view(3, 4, 5), reduction="none"), flat.view(3, 4, 5))
    assert torch.equal(ops.linear_cross_entropy(x[7], w, t[7], reduction="none"), ops.linear_cross_entropy(x[7:8], w, t[7:8], reduction="none")[0])
    other = t.view(6, 10).t()                                      # a target whose elements do not lie in order
    y = x.view(6, 10, 64).transpose(0, 1)
    assert torch.equal(ops.linear_cross_entropy(y, w, other, reduction="none"), flat.view(6, 10).t())


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_nothing_counts(ops, dtype):
    x, w, t = make(50, 64, 300, DTYPES[dtype])
    t.fill_(IGNORE)
    x.requires_grad_(), w.requires_grad_()
    assert torch.equal(ops.linear_cross_entropy(x, w, t, reduction="none"), torch.zeros(50, device="cuda"))
    assert ops.linear_cross_entropy(x, w, t, reduction="sum").item() == 0 and torch.isnan(ops.linear_cross_entropy(x, w, t))
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
    assert (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("cols,vocab", [(64, 300), (30, 7000)])
def test_no_tokens(ops, cols, vocab):
    x, w, t = torch.empty(0, cols, dtype=torch.bfloat16, device="cuda", requires_grad=True), make(2, cols, vocab, torch.bfloat16)[1].requires_grad_(), torch.empty(0, dtype=torch.int64, device="cuda")
    assert ops.linear_cross_entropy(x, w, t, reduction="none").shape == (0,)
    total = ops.linear_cross_entropy(x, w, t, reduction="sum")
    assert total.item() == 0 and torch.isnan(ops.linear_cross_entropy(x, w, t))
    dx, dw = torch.autograd.grad(total, (x, w))
    assert dx.shape == x.shape and (dw == 0).all()


def test_another_ignored_index(ops):
    x, w, t = make(40, 64, 300, torch.bfloat16)
    want = ops.linear_cross_entropy(x, w, t, reduction="none")
    for index in (7, -1, 1 << 40):
        t7 = torch.where(t == IGNORE, torch.full_like(t, index), torch.where(t == 7, torch.full_like(t, 8), t))
        got = ops.linear_cross_entropy(x, w, t7, ignore_index=index, reduction="none")
        same = t != 7
        assert torch.equal(got[same], want[same])


def test_targets_that_are_none(ops):
    """NaN for their tokens, and nothing else."""
    x, w, t = make(40, 64, 300, torch.bfloat16, ignored=0.0)
    want = ops.linear_cross_entropy(x, w, t, reduction="none")
    bad = t.clone()
    at = {3: 300, 5: -1, 9: 1 << 40, 11: -(1 << 40), 39: (1 << 32) + 5}
    for i, v in at.items():
        bad[i] = v
    x.requires_grad_()
    got = ops.linear_cross_entropy(x, w, bad, reduction="none")
    nan = torch.zeros(40, dtype=torch.bool, device="cuda")
    nan[list(at)] = True
    assert torch.isnan(got[nan]).all() and torch.equal(got[~nan], want[~nan])
    assert torch.isnan(ops.linear_cross_entropy(x, w, bad))
    dx, = torch.autograd.grad(got.nan_to_num().sum(), x)
    assert torch.isfinite(dx[~nan]).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), 65504.0])
def test_values_in_ignored_rows(ops, value):
    x, w, t = make(300, 64, 7000, torch.float16)
    want = ops.linear_cross_entropy(x, w, t, reduction="none")
    y = torch.where((t == IGNORE)[:, None], torch.full_like(x, value), x).requires_grad_()
    got = ops.linear_cross_entropy(y, w, t, reduction="none")
    assert torch.equal(got, want)
    dx, = torch.autograd.grad(got.sum(), y)
    assert torch.isfinite(dx).all() and (dx[t == IGNORE] == 0).all()


def test_nan_stays_in_its_row(ops):
    x, w, t = make(300, 64, 7000, torch.bfloat16, ignored=0.0)
    want = ops.linear_cross_entropy(x, w, t, reduction="none")
    for value in (float("nan"), float("inf")):
        y = x.clone()
        y[17, 5] = value
        y.requires_grad_()
        got = ops.linear_cross_entropy(y, w, t, reduction="none")
        keep = torch.arange(300, device="cuda") != 17
        assert torch.isnan(got[17]) and torch.equal(got[keep], want[keep])
        dx, = torch.autograd.grad(got.sum(), y)
        assert torch.isnan(dx[17]).any() and torch.isfinite(dx[keep]).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_far_logits(ops, dtype):
    """Logits of some hundred: exponentials underflow, the loss is a difference of large numbers."""
    x, w, t = make(64, 256, 1000, DTYPES[dtype])
    check(ops, x * 16, w * 4, t)
    check(ops, x * 0, w, t)
    check(ops, x[:3] * 64, w * 64, t[:3])                          # some thousand
    check(ops, x * 64, w * 64, t)


@pytest.mark.parametrize("tokens", [1, 30, 300])
@pytest.mark.parametrize("cols,vocab", [(64, 200), (1600, 3000)])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_sure_tokens(ops, dtype, cols, vocab, tokens):
    """Targets of a probability of 0.99 to 0.99999: the loss and the gradient are what is left of 1, and as good as any other.  The loss is a sum of what is left and its
    logarithm: its logits' errors and some 2^-18 of itself (exponentials of 2^-21, 300 additions); gradients: two roundings of 2^-12 or 2^-9, each row for itself."""
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    w = torch.randn(vocab, cols, generator=gen, device="cuda") * (1.5 / cols ** 0.5)
    t = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
    p = 1 - 10 ** (-2 - 3 * torch.rand(tokens, 1, generator=gen, device="cuda", dtype=torch.float64))
    x = torch.randn(tokens, cols, generator=gen, device="cuda").double()
    for _ in range(30):                                            # (moved along the target's row until it has that probability)
        l = x @ w.double().t()
        left = torch.log(p / (1 - p)) - (l.gather(1, t[:, None]) - torch.logsumexp(l.scatter(1, t[:, None], float("-inf")), 1, keepdim=True))
        x = x + left * w[t].double() / w[t].double().square().sum(1, keepdim=True)
    x, w = x.to(DTYPES[dtype]), w.to(DTYPES[dtype])
    l = x.double() @ w.double().t()
    loss = torch.nn.functional.cross_entropy(l, t, reduction="none")
    dl = torch.softmax(l, 1)
    dl[torch.arange(tokens), t] = torch.expm1(-loss)
    dx = dl @ w.double()
    x.requires_grad_()
    got = ops.linear_cross_entropy(x, w, t, reduction="none")
    # (a logit's own error, of the products and their chains, moves the loss by its part of 1 - p)
    off_l = ((cols / 16 + 2) * 2.0 ** -23) * (x.detach().double().abs() @ w.double().abs().t()).amax(dim=1)
    assert ((got - loss).abs() <= loss * (2 * off_l + 2.0 ** -18)).all()
    a, = torch.autograd.grad(got.sum(), x)
    # (FP16 holds what is below 2^-14 in steps of 2^-24: each element of such a row is off by up to 2^-25, the row by sqrt(cols) of that)
    steps = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2 * cols ** 0.5
    row, norm = (a.double() - dx).norm(dim=1), dx.norm(dim=1)
    assert (row <= norm * (2.5 * torch.finfo(x.dtype).eps / 2 + 2.0 ** -18 + 2 * off_l) + steps).all(), (row / norm).max()


@pytest.mark.parametrize("scale", [2.0 ** -30, 2.0 ** -15, 1.0, 2.0 ** 16, -3.0])
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_small_and_large_gradients(ops, dtype, scale):
    """dl is held so that a loss scale, or a mean over many tokens, costs no bits."""
    x, w, t = make(100, 64, 800, DTYPES[dtype])
    loss, _, dx, off_dx, dw, off_dw = exact(x, w, t, 0.0, torch.full((100,), scale, dtype=torch.float64, device="cuda"))
    x.requires_grad_(), w.requires_grad_()
    a, b = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction="sum"), (x, w), torch.tensor(scale, device="cuda"))
    top = torch.finfo(x.dtype).max
    for got, want, off in ((a, dx, off_dx), (b, dw, off_dw)):
        fits = want.abs() < top * 0.99
        near(torch.where(fits, got, torch.zeros_like(got)), torch.where(fits, want, torch.zeros_like(want)), off)


def test_gradient_against_differences(ops):
    """The loss along a direction: a central difference of the 64-bit loss at the 16-bit points."""
    x, w, t = make(60, 64, 500, torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(x, w, t), (x, w))
    gen = torch.Generator(device="cuda").manual_seed(5)
    for got, which in ((dx, 0), (dw, 1)):
        d = torch.randn(got.shape, generator=gen, device="cuda", dtype=torch.float64)

        def loss(s):
            a, b = x.detach().double() + (s * d if which == 0 else 0), w.detach().double() + (s * d if which == 1 else 0)
            return torch.nn.functional.cross_entropy(a @ b.t(), t)
        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        # every element is off by at most 2^-8 of itself twice over (dl and the result); 2^-6 of the sum of magnitudes leaves room for the difference's own error
        assert abs((got.double() * d).sum() - want) <= 2.0 ** -6 * (got.double() * d).abs().sum()


@pytest.mark.parametrize("need", ["x", "w", "none"])
def test_only_what_is_asked_for(ops, need):
    x, w, t = make(70, 64, 900, torch.bfloat16)
    xa, wa = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(xa, wa, t), (xa, wa))
    if need == "x":
        assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(xa, w, t), xa)[0], dx)
    elif need == "w":
        assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(x, wa, t), wa)[0], dw)
    else:
        assert not ops.linear_cross_entropy(x, w, t).requires_grad


def test_saved_tensors_that_move(ops):
    """Hooks that put what is kept for the backward pass elsewhere and bring back other tensors, with other strides."""
    x, w, t = make(70, 64, 900, torch.bfloat16)
    xa, wa = x.clone().requires_grad_(), w.clone().requires_grad_()
    want = torch.autograd.grad(ops.linear_cross_entropy(xa, wa, t), (xa, wa))
    for unpack in (lambda v: v.cuda(), lambda v: v.cuda().t().contiguous().t() if v.dim() == 2 else v.cuda()):
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), unpack):
            xb, wb = x.clone().requires_grad_(), w.clone().requires_grad_()
            loss = ops.linear_cross_entropy(xb * 1, wb * 1, t)
        filler = [torch.full_like(v, float("nan")) for v in (x, w) for _ in range(4)]            # (over what the products with 1 had)
        got = torch.autograd.grad(loss, (xb, wb))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and len(filler) == 8


def test_what_was_kept_and_changed(ops):
    x, w, t = make(70, 64, 900, torch.bfloat16)
    w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t)
    x.add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, w)


@pytest.mark.parametrize("tokens,cols,vocab", [(5, 64, 20000), (300, 72, 70001), (2000, 512, 9000)])
def test_same_bits_every_time(ops, tokens, cols, vocab):
    x, w, t = make(tokens, cols, vocab, torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()
    first = None
    for _ in range(4):
        loss = ops.linear_cross_entropy(x, w, t)
        a = torch.autograd.grad(loss, (x, w), retain_graph=True)
        b = torch.autograd.grad(loss, (x, w))
        now = (loss.detach(), *a)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        first = first or now
        assert all(torch.equal(p, q) for p, q in zip(first, now))


def test_captured(ops):
    x, w, t = make(200, 64, 9000, torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear_cross_entropy(x, w, t), (x, w))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = ops.linear_cross_entropy(x, w, t)
        dx, dw = torch.autograd.grad(loss, (x, w))
    for seed in (1, 2):
        x2, w2, t2 = make(200, 64, 9000, torch.bfloat16, seed=seed)
        with torch.no_grad():
            x.copy_(x2), w.copy_(w2), t.copy_(t2)
        graph.replay()
        x2.requires_grad_(), w2.requires_grad_()
        want = ops.linear_cross_entropy(x2, w2, t2)
        a, b = torch.autograd.grad(want, (x2, w2))
        assert torch.equal(loss, want) and torch.equal(dx, a) and torch.equal(dw, b)


def test_side_by_side(ops):
    """Calls from several threads on streams of their own."""
    cases = [make(50 + 90 * i, 64 + 8 * i, 3000 + 1111 * i, torch.bfloat16, seed=i) for i in range(4)]
    want = [ops.linear_cross_entropy(*c, reduction="none") for c in cases]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = ops.linear_cross_entropy(*cases[i], reduction="none")
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("tokens,cols,vocab", [(3, 77, 300), (200, 93, 7001), (2, 5, 70000), (700, 1000, 3001)])
def test_beside_the_results(ops, lib, dtype, tokens, cols, vocab):
    """Gradients into rows of wider tensors: what lies beside is left as it was."""
    x, w, t = make(tokens, cols, vocab, DTYPES[dtype])
    xa, wa = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(xa, wa, t, reduction="sum"), (xa, wa))
    type, stream = {"f16": 1, "bf16": 2}[dtype], torch.cuda.current_stream().cuda_stream
    loss, stats, one = torch.empty(1, device="cuda"), torch.empty(2 * tokens + 1, device="cuda"), torch.ones(1, device="cuda")
    base = (type, x.data_ptr(), tokens, cols, cols, w.data_ptr(), vocab, cols)
    room = torch.empty(lib.bsq_linear_xent_scratch_bytes(*base, 0.0), dtype=torch.uint8, device="cuda")
    assert lib.bsq_linear_xent(*base, t.data_ptr(), IGNORE, 0.0, 1, loss.data_ptr(), stats.data_ptr(), room.data_ptr(), None, stream) == 0
    room = torch.empty(lib.bsq_linear_xent_grad_scratch_bytes(*base, 1), dtype=torch.uint8, device="cuda")
    for first in (0, 8, 1):
        ld = (first + cols + 8) // 8 * 8 if first != 1 else first + cols + 1
        big = [torch.full((n + 2, ld), -7.0, dtype=x.dtype, device="cuda") for n in (tokens, vocab)]
        outs = [b[1:-1, first: first + cols] for b in big]
        assert lib.bsq_linear_xent_grad(*base, t.data_ptr(), IGNORE, 0.0, 1, stats.data_ptr(), one.data_ptr(), outs[0].data_ptr(), ld, outs[1].data_ptr(), ld, room.data_ptr(), None, stream) == 0
        assert torch.equal(outs[0], dx) and torch.equal(outs[1], dw)
        for b, o in zip(big, outs):
            o.fill_(-7.0)
            assert (b == -7.0).all()


@pytest.mark.parametrize("tokens,cols,vocab", [(40, 128, 1000), (300, 256, 7000), (200, 64, 30000)])
def test_waits_that_run_out(ops, lib, tokens, cols, vocab):
    x, w, t = make(tokens, cols, vocab, torch.bfloat16, ignored=0.0)
    x.requires_grad_(), w.requires_grad_()
    want = ops.linear_cross_entropy(x, w, t, reduction="none")
    a, b = torch.autograd.grad(want.sum(), (x, w))
    try:
        lib.bsq_test_limit_waits(0)
        assert torch.isnan(ops.linear_cross_entropy(x, w, t, reduction="none")).all()
        loss = ops.linear_cross_entropy(x, w, t, reduction="sum")
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert torch.isnan(loss) and torch.isnan(dx).all() and torch.isnan(dw).all()
        torch.cuda.synchronize()
    finally:
        lib.bsq_test_limit_waits(1 << 16)
    assert torch.equal(ops.linear_cross_entropy(x, w, t, reduction="none"), want)
    c, d = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, reduction="sum"), (x, w))
    assert torch.equal(a, c) and torch.equal(b, d)


def test_refusals(ops):
    x, w, t = make(10, 64, 100, torch.bfloat16)
    for call in (lambda: ops.linear_cross_entropy(x.float(), w.float(), t), lambda: ops.linear_cross_entropy(x, w.half(), t), lambda: ops.linear_cross_entropy(x, w[:, :63], t),
                 lambda: ops.linear_cross_entropy(x, w, t.int()), lambda: ops.linear_cross_entropy(x, w, t[:9]), lambda: ops.linear_cross_entropy(x, w, t.cpu()),
                 lambda: ops.linear_cross_entropy(x, w, t, reduction="max"), lambda: ops.linear_cross_entropy(x, w, t, label_smoothing=1.5),
                 lambda: ops.linear_cross_entropy(x, w, t, label_smoothing=float("nan")), lambda: ops.linear_cross_entropy(x, w, t, ignore_index=1 << 63),
                 lambda: ops.linear_cross_entropy(x, w[:0], t), lambda: ops.linear_cross_entropy(x[:, :0], w[:, :0], t), lambda: ops.linear_cross_entropy(x, w.cpu(), t),
                 lambda: ops.linear_cross_entropy(torch.zeros(65537, 8, dtype=torch.float16, device="cuda"), w.half()[:, :8], torch.zeros(65537, dtype=torch.int64, device="cuda")),
                 lambda: ops.linear_cross_entropy(torch.zeros(1, 65537, dtype=torch.float16, device="cuda"), torch.zeros(2, 65537, dtype=torch.float16, device="cuda"), t[:1])):
        with pytest.raises(ValueError):
            call()
