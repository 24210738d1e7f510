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
