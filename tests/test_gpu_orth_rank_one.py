"""Updates of exactly rank one with both sides above 128, the gradient of one token: what the documentation says of them."""
import importlib

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

VALUES = {"gaussian": None, "3, 5, 7": [3, 5, 7], "11, 13": [11, 13], "1 to 8": list(range(1, 9)), "1, 2": [1, 2], "0, 1": [0, 1], "1": [1]}


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


@pytest.mark.parametrize("kind", sorted(VALUES))
@pytest.mark.parametrize("m,n", [(130, 300), (300, 300), (300, 2000), (2000, 300), (1024, 4096), (4096, 1024), (2304, 2304)])
def test_rank_one(ops, m, n, kind):
    """The one singular value goes the way of a number: s = 1, 0.701, 1.114, 0.721, 1.090, 0.696.
    BF16 results.  P is held in 11 bits beside its diagonal.  Where a row's elements are all alike so are their roundings, 2^-11 of them: that turns or scales X's vectors by 2^-11 |P| s / s' at each step,
    (3.9 + 1.2 + 4.3 + 1.3 + 4.4) 2^-11 = 7.4e-3, and is not of another rank, so that later steps leave it as it is.  With a short side above 512 X's low part is left out off P's diagonal: as much again.
    A's 11 bits give (1.0 + 0.9 + 0.5 + 0.9 + 0.1) 2^-11 = 1.7e-3.  Half of it on average, and a rounding to BF16, 2^-8: 8.5e-3, or 1.2e-2.  (A factor of ones is of few values too.)
    FP32 results: what the sums of P X lose, 4.1e-3 where each addition cuts off 2^-23 of what it has (see the sums of one sign of longer matrices); on average it is 0.36 of that."""
    gen = torch.Generator(device="cuda").manual_seed(m + n)

    def vector(*shape):
        if kind == "gaussian":
            return torch.randn(*shape, generator=gen, device="cuda")
        values = torch.tensor(VALUES[kind], dtype=torch.float32, device="cuda")
        return values[torch.randint(0, len(values), shape, generator=gen, device="cuda")]
    for other in (True, False):
        u, v = vector(m, 1), vector(1, n) if other else torch.ones(1, n, device="cuda")
        g, s = u * v, 1.0
        for _ in range(5):
            s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
        # (products of Gaussian factors are rounded to FP32, 2^-25 of which is not of rank one and grows by 485)
        want = u.double() * v.double() * (s / (u.double().norm() * v.double().norm()))
        for dtype, off in ((torch.bfloat16, 2.0 ** -8 if kind == "gaussian" and other else 8.5e-3 if min(m, n) <= 512 else 1.2e-2), (torch.float32, 1.5e-3)):
            got = ops.orthogonalize(g, dtype=dtype)
            assert (got.double() - want).norm() <= off * want.norm(), (dtype, other)


@pytest.mark.parametrize("m,n", [(129, 129), (129, 357), (357, 129), (160, 5000), (5000, 160), (256, 256), (512, 600), (513, 600), (1000, 1000)])
def test_gaussian_factors(ops, m, n):
    """Elements of many values: a rounding to BF16, 2^-8 / sqrt(3) of the norm at most; P's and A's 11 bits, 2e-4 of an element, at random: (7.5 + 1.7) 2e-4 sqrt(3 / s) (7.5 and 1.7 the root sums of
    squares of the figures above), 2.8e-4 at 129.  Above 512, where P's diagonal alone goes with X's low part, that is not of X's rank: 2.74 * 2e-4 sqrt(15) / s, 140 times as much four steps later,
    0.43 / s of the result.  (All sides that way: 129 x 357 5.4e-3, 3.7e-3 on average.)"""
    s = 1.0
    for _ in range(5):
        s = 3.4445 * s - 4.7750 * s ** 3 + 2.0315 * s ** 5
    short = min(m, n)
    for seed in range(10):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        u, v = torch.randn(m, 1, generator=gen, device="cuda"), torch.randn(1, n, generator=gen, device="cuda")
        want = u.double() * v.double() * (s / (u.double().norm() * v.double().norm()))
        off = (ops.orthogonalize(u * v).double() - want).norm() / want.norm()
        assert off <= 2.0 ** -8 / 3 ** 0.5 + 3e-4 + (0.45 / short if short > 512 else 0)
