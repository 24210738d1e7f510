"""What the loss over a vocabulary refuses before anything is launched, and the scratch that it asks for."""
import importlib

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


A = 1 << 20                                                    # addresses that are never looked at: every call here is refused
LOSS = [2, A, 4, 64, 64, A, 100, 64, A, -100, 0.0, 2, A, A, A, None, None]
GRAD = [2, A, 4, 64, 64, A, 100, 64, A, -100, 0.0, 2, A, A, A, 64, A, 64, A, None, None]
NAN = float("nan")
SHARED = [(0, 0), (0, 3), (1, None), (1, A + 1), (2, 524289), (3, 0), (3, 65537), (4, 63), (4, 1 << 38), (5, None), (5, A + 1), (6, 0), (6, 1 << 31), (7, 63), (7, 1 << 38), (8, None), (8, A + 4),
          (10, -0.1), (10, 1.1), (10, NAN), (11, -1), (11, 3)]


def but(args, i, v):
    return args[:i] + [v] + args[i + 1:]


@pytest.mark.parametrize("i,v", SHARED + [(12, None), (12, A + 2), (13, None), (13, A + 2), (14, None), (14, A + 64)])
def test_loss_refuses(lib, i, v):
    assert lib.bsq_linear_xent(*but(LOSS, i, v)) == 1


@pytest.mark.parametrize("i,v", SHARED + [(12, None), (12, A + 2), (13, None), (13, A + 2), (14, A + 1), (15, 63), (16, A + 1), (17, 63), (18, None), (18, A + 64)])
def test_gradient_refuses(lib, i, v):
    assert lib.bsq_linear_xent_grad(*but(GRAD, i, v)) == 1


def test_fp16_takes_fewer_tokens(lib):
    assert lib.bsq_linear_xent(*but(but(LOSS, 0, 1), 2, 65537)) == 1 and lib.bsq_linear_xent_grad(*but(but(GRAD, 0, 1), 2, 65537)) == 1


def test_nothing_wanted(lib):
    assert lib.bsq_linear_xent_grad(*but(but(GRAD, 14, None), 16, None)) == 0


def test_scratch(lib):
    f, g = lib.bsq_linear_xent_scratch_bytes, lib.bsq_linear_xent_grad_scratch_bytes
    assert f(0, A, 4, 64, 64, A, 100, 64, 0.0) == 0 and f(2, A, 0, 64, 64, A, 100, 64, 0.0) == 0 and g(2, A, 4, 0, 64, A, 100, 64, 1) == 0
    plain = f(2, A, 40, 64, 64, A, 100, 64, 0.0)
    assert 0 < plain < 8192 and f(2, A, 40, 64, 64, A, 100, 64, 0.1) > plain
    assert f(2, A + 2, 40, 64, 64, A, 100, 64, 0.0) >= plain + 40 * 64 * 2                   # x off 16 bytes is copied
    assert f(2, A, 40, 64, 64, A, 100, 65, 0.0) >= plain + 100 * 64 * 2                      # the weight's rows too
    assert f(2, A, 4, 64, 64, A, 100, 65, 0.0) == f(2, A, 4, 64, 64, A, 100, 64, 0.0)        # a few tokens read them as they are
    # logits are not kept: a piece of their gradient at a time, and the sums of dx
    tokens, cols, vocab = 16384, 4096, 131072
    assert g(2, A, tokens, cols, cols, A, vocab, cols, 1) < (tokens * vocab * 2) // 8
    assert g(2, A, tokens, cols, cols, A, vocab, cols, 0) < (tokens * vocab * 2) // 16


def test_python_refuses(ops):
    x, w, t = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(9, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w, t)
