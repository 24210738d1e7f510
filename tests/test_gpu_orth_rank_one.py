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
    """The one singular value goes the way of a number.
    BF16 results: P has 11 bits beside its diagonal and A too.  Where all elements of a row are alike so are their roundings, 2^-12: 6.7e-4, 4.5e-4, 6.8e-4 ... of X at each step from P and 0.2e-4 to 3.4e-4
    from A, which later steps multiply by 0.8 to 1.4: 5.6e-3 of the result, 0.696, along it; across it there is as much again at most where elements take few values; and its rounding to BF16, 2^-8.
    Where both factors take many values they do not round alike: 2^-8 in all.  (A factor of ones is of few: P = p 1 1^T, if it is that side's, has one value.)
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
        for dtype, off in ((torch.bfloat16, 2.0 ** -8 if kind == "gaussian" and other else 1.2e-2), (torch.float32, 1.5e-3)):
            got = ops.orthogonalize(g, dtype=dtype)
            assert (got.double() - want).norm() <= off * want.norm(), (dtype, other)
