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
