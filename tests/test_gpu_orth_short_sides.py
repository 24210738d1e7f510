"""Updates of matrices with a short side of up to 128, results in BF16: alone and in lists, wide and tall, of rank one."""
import importlib
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

QUINTIC = (3.4445, -4.7750, 2.0315)
SIDES = [(16, 65536), (32, 16384), (48, 2000), (64, 1024), (64, 16384), (96, 2000), (100, 16384), (128, 2000), (128, 16384), (128, 65536)]


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def make(kind, s, l, tall, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + s + l)
    m, n = (l, s) if tall else (s, l)
    if kind == "noise":
        return torch.randn(m, n, generator=gen, device="cuda")
    if kind == "rank 8":
        return torch.randn(m, 8, generator=gen, device="cuda") @ torch.randn(8, n, generator=gen, device="cuda")
    if kind == "gaussian":
        return torch.randn(m, 1, generator=gen, device="cuda") * torch.randn(1, n, generator=gen, device="cuda")
    few = torch.tensor({"1 to 8": list(range(1, 9)), "3, 5, 7": [3, 5, 7], "11, 13": [11, 13]}[kind], dtype=torch.float32, device="cuda")
    pick = [few[torch.randint(0, len(few), shape, generator=gen, device="cuda")] for shape in ((m, 1), (1, n))]
    return pick[0] * pick[1]


def exact(g):
    x = g.double()
    x = x / (x.square().sum().sqrt() + 1e-7)
    for a, b, c in [QUINTIC] * 5:
        if x.size(0) <= x.size(1):
            s = x @ x.t()
            x = a * x + (b * s + c * (s @ s)) @ x
        else:
            s = x.t() @ x
            x = a * x + x @ (b * s + c * (s @ s))
    return x


def off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("kind", ["noise", "3, 5, 7"])
@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("s,l", SIDES)
def test_alone_and_in_a_list(ops, s, l, tall, kind):
    """What a matrix becomes does not depend on how many go with it, nor on what they are."""
    g, other = make(kind, s, l, tall), make("noise", s, l, tall, seed=1) * 3
    want = ops.orthogonalize(g)
    for count in (15, 24, 64):
        got = ops.orthogonalize([other] * (count // 2) + [g] * (count - count // 2 - 1) + [other])
        assert torch.equal(got[count // 2], want) and torch.equal(got[count - 2], want) and torch.equal(got[0], got[-1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,n", [(300, 500), (500, 300), (1100, 1100)])
def test_longer_sides_alone_and_in_a_list(ops, m, n, dtype):
    """The paths of longer sides likewise: tiles of another size, norms of another number of shares."""
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    g = [make("noise", m, n, False, seed=i) for i in range(9)]
    assert all(torch.equal(ops.orthogonalize(a, dtype=t), b) for a, b in zip(g, ops.orthogonalize(g, dtype=t)))


@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("s,l", SIDES)
def test_long_sides_in_lists(ops, s, l, tall):
    """Full rank and rank 8 among 64: FP32 sums and products of 22 bits leave 2^-12 at most, a rounding to BF16 2^-8 / sqrt(3) of the norm."""
    for kind in ("noise", "rank 8"):
        g = make(kind, s, l, tall)
        assert off(ops.orthogonalize([g] * 64)[40], exact(g)) <= 2.0 ** -8 / math.sqrt(3) + 2.0 ** -12


def test_slices_of_one_length(ops):
    """A long side's sums in a list of 63 and alone: rank one of few values, 1.3e-1 off where a chain had 16384 terms."""
    for kind, s, l, count in (("3, 5, 7", 32, 65536, 63), ("3, 5, 7", 16, 65536, 64), ("11, 13", 64, 16384, 64), ("1 to 8", 16, 65536, 64)):
        g = make(kind, s, l, False)
        alone, among = ops.orthogonalize(g), ops.orthogonalize([g] * count)[count // 2]
        assert torch.equal(alone, among)


@pytest.mark.parametrize("tall", [False, True])
@pytest.mark.parametrize("s,l", SIDES + [(40, 300), (64, 200), (128, 200), (128, 1024)])
def test_rank_one(ops, s, l, tall):
    """The gradient of one token.  A rounding to BF16 is 2^-8 of an element at most.  Beside it: the result is R u v^T + q u v^T, -484 and 485 of u v^T for 0.7.  Each of the four products that make R adds
    up to h = s / 32 times in either accumulator what is of its size, and each time cuts 16 terms off at 2^-25 of the sum so far, by half a step on average: (h + 1) / 2 * 16 * 2^-26 * 484 / 0.7
    where all elements lose alike, 1.7e-4 up to 32 and 4.1e-4 at 128; what is lost stays in proportion, so four times that.  The FP32 additions of R's rounding and R G, (s + 1) / 2 * 2^-24 * 484 / 0.7:
    6.8e-4 and 2.7e-3.  1.4e-3 and 4.3e-3 in all.  Elements of many values do not lose alike: 1.3e-3 whatever the side."""
    for kind in ("gaussian", "1 to 8", "3, 5, 7", "11, 13"):
        g = make(kind, s, l, tall)
        beside = 1.3e-3 if kind == "gaussian" else 1.4e-3 if s <= 32 else 4.3e-3
        assert off(ops.orthogonalize(g), exact(g)) <= 2.0 ** -8 + beside, kind


@pytest.mark.parametrize("m,n", [(8, 300), (300, 8), (16, 65536), (5, 7), (32, 32), (32, 100), (31, 5000), (33, 40), (128, 200)])
def test_few_rows_of_far_singular_values(ops, m, n):
    """Noise beside a mean thirty times as large, singular values from 1 to 1 / 1000, one far above the others.  A_0 in 22 bits is 2^-23 off; a direction of singular value x then |Q'(x^2)| x 2^-23, at
    most 3.6e4 * 2^-23 = 4.3e-3 (at x = 0.004), of some 0.7 to 1.1, if all of it fell into that direction; it is spread over as many as there are rows.  A rounding to BF16 is 2^-8 / sqrt(3) of the norm."""
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    noise = torch.randn(m, n, generator=gen, device="cuda")
    u, v = (torch.linalg.qr(torch.randn(k, min(m, n), generator=gen, device="cuda"))[0] for k in (m, n))
    one = torch.randn(m, 1, generator=gen, device="cuda") * torch.randn(1, n, generator=gen, device="cuda")
    for g in (noise + 30, noise + 300, u * torch.logspace(0, -3, min(m, n), device="cuda") @ v.t(), one + 1e-2 * noise, one + 1e-3 * noise):
        assert off(ops.orthogonalize(g), exact(g)) <= 2.0 ** -8 / math.sqrt(3) + 4.3e-3 / 0.69 / math.sqrt(min(m, n))
