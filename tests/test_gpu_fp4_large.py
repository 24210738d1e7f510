"""Matrices whose offsets pass 32 bits, and calls made from several threads and streams."""
import importlib
import threading

import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def last_rows(ops, m, n):
    """The last n rows of a packed matrix of a multiple of 128 rows, n a multiple of 128, as a matrix of their own."""
    ld = -(-m.cols // 32) * 16
    at = (128 + m.rows * ld + 127) // 128 * 128
    per = -(-m.cols // (4 * ref.BLOCK[m.format])) * 512
    out = torch.zeros(ops._packed_bytes(m.format, n, m.cols), dtype=torch.uint8, device="cuda")
    out[:128] = m.data[:128]
    out[128: 128 + n * ld] = m.data[128 + (m.rows - n) * ld: 128 + m.rows * ld]
    out[out.numel() - n // 128 * per:] = m.data[at + (m.rows - n) // 128 * per: at + m.rows // 128 * per]
    return ops.Fp4Matrix(out, n, m.cols, m.format)


@pytest.mark.parametrize("fmt", [ref.MXFP4, ref.NVFP4])
def test_more_than_two_to_the_31_elements(ops, fmt):
    """65664 x 33024: 2.17e9 elements, 4.3 GB in BF16, 1.1 GB packed."""
    rows, cols = 65664, 33024
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    block = torch.randint(-3, 4, (128, cols), generator=gen, device="cuda").to(torch.bfloat16)
    x.view(rows // 128, 128, cols)[:] = block
    tail = (torch.randint(-3, 4, (128, cols), generator=gen, device="cuda")).to(torch.bfloat16)
    x[-128:] = tail
    m = ops.fp4_quantize(x, fmt)
    small = last_rows(ops, m, 128)
    want = ops.fp4_quantize(torch.cat([block[:1], tail]), fmt)             # (the same largest magnitude, 3)
    assert torch.equal(small.codes, want.codes[1:]) and torch.equal(small.block_scales(), want.block_scales()[1:])
    back = ops.fp4_dequantize(m, torch.bfloat16, out=x)
    assert torch.equal(back[-128:], ops.fp4_dequantize(small, torch.bfloat16))
    assert torch.equal(back[:128], back[128 * 300: 128 * 301])
    del x, back
    # one token, and a few hundred, against the large weight; gradients from it and with it
    for tokens in (1, 300):
        a = ops.fp4_quantize(torch.randint(-3, 4, (tokens, cols), generator=gen, device="cuda").to(torch.bfloat16), fmt)
        y = ops.fp4_matmul(a, m, torch.float32)
        assert torch.equal(y[:, -128:], ops.fp4_matmul(a, small, torch.float32)) and torch.equal(y[:, :128], y[:, 12800: 12928])
        # dy is 0 but at the last 128 outputs, so that the gradient is theirs
        dy = torch.zeros(tokens, rows, dtype=torch.bfloat16, device="cuda")
        dy[:, -128:] = torch.randint(-3, 4, (tokens, 128), generator=gen, device="cuda").to(torch.bfloat16)
        dx = ops.fp4_grad_input(dy, m, torch.float32)
        assert torch.equal(dx, ops.fp4_grad_input(dy[:, -128:], small, torch.float32))
    # dW of 65664 x 33024 in BF16 (4.3 GB) from 128 rows
    dy = torch.zeros(128, rows, dtype=torch.bfloat16, device="cuda")
    dy[:, -1], dy[:, 0] = 1, 2
    dw = ops.fp4_grad_weight(dy, small)
    s = ops.fp4_dequantize(small).double().sum(dim=0)
    assert torch.equal(dw[-1].double(), s.float().to(torch.bfloat16).double()) and torch.equal(dw[0].double(), (2 * s).float().to(torch.bfloat16).double())
    assert (dw[1:-1:1000] == 0).all()
    del dw
    # a product with more than 2^31 results
    b = ops.fp4_quantize(torch.eye(128, device="cuda")[torch.arange(50048, device="cuda") % 128].to(torch.bfloat16), fmt)
    y = ops.fp4_matmul(b, b)
    one = float(y[0, 0])
    assert one > 0.9 and float(y[50047, 50047]) == one and float(y[50047, 0]) == 0.0 and float(y[50046, 50047]) == 0.0
    assert torch.equal(y[-256:, -256:], y[:256, :256])


def test_calls_from_several_threads(ops):
    """Four host threads, a stream each, all operators: the results of a thread alone."""
    torch.manual_seed(1)
    x = torch.randn(300, 512, device="cuda").to(torch.bfloat16)
    w = ops.fp4_quantize(torch.randn(700, 512, device="cuda") * 0.1)
    dy = torch.randn(300, 700, device="cuda").to(torch.bfloat16)

    def step():
        x4 = ops.fp4_quantize(x)
        y, dx, dw = ops.fp4_matmul(x4, w), ops.fp4_grad_input(dy, w), ops.fp4_grad_weight(dy, x4, torch.float32)
        few = ops.fp4_grad_input(dy[:7], w)
        return [y, dx, dw, few, ops.clip_grad_norm([dw], 0.5), ops.fp4_dequantize(x4)]
    want = step()
    torch.cuda.synchronize()
    wrong, errors = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step()
                    torch.cuda.current_stream().synchronize()
                    wrong.extend(i for i, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))
        except Exception as e:                                    # (an assertion in a thread would not fail the test)
            errors.append(e)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong


def test_beside_the_framework_s_own_products(ops, pkg):
    """The products of the low-rank path and these on two streams at once: tensor memory and shared memory are shared by whoever is there."""
    api = importlib.import_module(pkg.__name__ + ".torch_api")
    comp = api.Compressor(2048, 4096, rank=64)
    m = torch.randn(2048, 4096, device="cuda")
    alone = comp.compress(m).to_bytes()[200:]
    a, b = ops.fp4_quantize(torch.randn(1000, 2048, device="cuda")), ops.fp4_quantize(torch.randn(1500, 2048, device="cuda"))
    dy = torch.randn(1000, 1500, device="cuda").to(torch.bfloat16)
    y, dx = ops.fp4_matmul(a, b), ops.fp4_grad_input(dy, b)
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        pending = comp.compress_async(m)
        for _ in range(10):
            got.append((ops.fp4_matmul(a, b), ops.fp4_grad_input(dy, b)))
        assert (pending.wait().to_bytes()[200:] == alone).all()
    torch.cuda.synchronize()
    assert all(torch.equal(p, y) and torch.equal(q, dx) for p, q in got)
    comp.close()
