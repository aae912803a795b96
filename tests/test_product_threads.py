"""Products as the first thing that a thread does on the GPU, as autograd's threads may."""
import threading

import pytest
import torch

from ramtorch_b200 import microscaling as mx


def in_a_new_thread(call):
    out = []

    def run():
        try:
            out.append(call())
        except Exception as e:      # noqa: BLE001
            out.append(e)
    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(out[0], Exception):
        raise out[0]
    return out[0]


@pytest.mark.gpu
@pytest.mark.parametrize("host_side", ["C++", "ctypes"])
def test_products_are_the_first_call_of_a_thread(host_side, monkeypatch):
    if host_side == "ctypes":
        monkeypatch.setattr(mx, "_fast", False)
    x, g = torch.randn(64, 96, device="cuda").bfloat16(), torch.randn(64, 128, device="cuda").bfloat16()
    q, a, b = mx.quantize_mxint8(x), mx.quantize_mxfp4(x), mx.quantize_mxfp4(torch.randn(200, 96, device="cuda"))
    for call in (lambda: mx.weight_grad(g, q), lambda: mx.weight_grad(g, q, out=torch.zeros(128, 96, device="cuda"), accumulate=True),
                 lambda: mx.mxfp4_matmul(a, b), lambda: mx.mxfp4_matmul(b, a)):
        want = call()               # plans and memory are there already
        torch.cuda.synchronize()
        assert torch.equal(in_a_new_thread(call), want)


@pytest.mark.gpu
def test_products_on_two_streams_and_in_two_threads_at_once():
    """Every way of summing at the same time: nothing is shared between calls."""
    r = lambda *s: torch.randn(*s, device="cuda").bfloat16()      # noqa: E731
    g, q = r(4096, 130), mx.quantize_mxint8(r(4096, 200))           # parts that a second kernel joins
    h, p = r(700, 1000), mx.quantize_mxint8(r(700, 600))
    f = torch.randn(300, 200, device="cuda")
    u = mx.quantize_mxint8(r(300, 100))                             # planes in a workspace
    a, b, c = mx.quantize_mxfp4(r(3, 4096)), mx.quantize_mxfp4(r(900, 4096)), mx.quantize_mxfp4(r(1500, 4096))
    calls = [lambda: mx.weight_grad(g, q), lambda: mx.weight_grad(h, p), lambda: mx.weight_grad(f, u), lambda: mx.mxfp4_matmul(a, b), lambda: mx.mxfp4_matmul(b, c)]
    want = [call() for call in calls]
    torch.cuda.synchronize()

    def run(order):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [(i, calls[i]()) for _ in range(20) for i in order]
        stream.synchronize()
        return all(torch.equal(t, want[i]) for i, t in got)

    done = []
    threads = [threading.Thread(target=lambda o=o: done.append(run(o))) for o in ((0, 1, 2, 3, 4), (4, 3, 2, 1, 0), (2, 4, 1, 3, 0))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert done == [True, True, True]
    mx.check_faults()
