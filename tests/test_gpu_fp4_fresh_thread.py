"""Operators as the first thing that a host thread asks of the GPU, as in the thread of a backward pass."""
import importlib
import threading

import pytest

import fp4_reference as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(pkg):
    return importlib.import_module(pkg.__name__ + ".torch_ops")


def in_a_thread(call):
    errors = []

    def work():
        try:
            call()
        except Exception as e:                                    # (an exception in a thread would not fail the test)
            errors.append(e)
    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not errors, errors
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", [ref.MXFP4, ref.NVFP4])
@pytest.mark.parametrize("M", [5, 40, 300])
def test_every_operator(ops, fmt, M):
    torch.manual_seed(M)
    x, dy = torch.randn(M, 512, device="cuda").to(torch.bfloat16), torch.randn(M, 264, device="cuda").to(torch.bfloat16)
    x4, w4 = ops.fp4_quantize(x, fmt), ops.fp4_quantize(torch.randn(264, 512, device="cuda"), fmt)
    y, dx, dw, back = ops.fp4_matmul(x4, w4), ops.fp4_grad_input(dy, w4), ops.fp4_grad_weight(dy, x4, torch.float32), ops.fp4_dequantize(x4)
    out, again = [torch.zeros_like(t) for t in (y, dx, dw, back)], ops.fp4_quantize(torch.zeros_like(x), fmt)
    torch.cuda.synchronize()
    in_a_thread(lambda: ops.fp4_matmul(x4, w4, out=out[0]))
    in_a_thread(lambda: ops.fp4_grad_input(dy, w4, out=out[1]))
    in_a_thread(lambda: ops.fp4_grad_weight(dy, x4, torch.float32, out=out[2]))
    in_a_thread(lambda: ops.fp4_dequantize(x4, out=out[3]))
    in_a_thread(lambda: ops.fp4_quantize(x, fmt, out=again))
    assert all(torch.equal(a, b) for a, b in zip(out, (y, dx, dw, back))) and torch.equal(again.codes, x4.codes)
    want = [dw.clone()]
    norm = ops.clip_grad_norm(want, 1.0)
    got = []
    in_a_thread(lambda: got.append(ops.clip_grad_norm([out[2]], 1.0)))
    assert torch.equal(got[0], norm) and torch.equal(out[2], want[0])


@pytest.mark.parametrize("M", [20, 200])
def test_first_call_of_a_captured_graph_s_thread(ops, M):
    """... and under capture, on a stream of the thread's own."""
    x4, w4 = ops.fp4_quantize(torch.randn(M, 512, device="cuda")), ops.fp4_quantize(torch.randn(264, 512, device="cuda"))
    dy = torch.randn(M, 264, device="cuda").to(torch.bfloat16)
    want = ops.fp4_matmul(x4, w4), ops.fp4_grad_input(dy, w4)
    out = [torch.zeros_like(t) for t in want]
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        def call():
            with torch.cuda.stream(side):
                ops.fp4_matmul(x4, w4, out=out[0])
                ops.fp4_grad_input(dy, w4, out=out[1])
        errors = []

        def work():
            try:
                call()
            except Exception as e:
                errors.append(e)
        t = threading.Thread(target=work)
        t.start()
        t.join()
    assert not errors, errors
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
