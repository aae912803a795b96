"""Waits that ran out inside a product's kernel are reported.  The count is set here on the host: no kernel is made to fail."""
import ctypes

import pytest
import torch

from ramtorch_b200 import _native as N
from ramtorch_b200 import microscaling as mx


class Library:
    """Stands for the library: a count for each device that was current when it was asked."""

    def __init__(self, monkeypatch):
        self.counts, self.current, self.asked = {}, 0, []
        monkeypatch.setattr(mx.N, "lib", lambda: self)
        monkeypatch.setattr(mx, "_on", self.on)
        monkeypatch.setattr(mx, "_watched", {})

    def on(self, device):
        self.current = device.index
        return mx._STAY

    def rt_last_error(self):
        return b"no device"

    def rt_mx_wait_faults(self, count):
        self.asked.append(self.current)
        ctypes.cast(count, ctypes.POINTER(ctypes.c_uint32))[0] = self.counts.get(self.current, 0)
        return 0


def test_waits_that_ran_out_raise_once(monkeypatch):
    lib = Library(monkeypatch)
    mx.check_faults()
    assert lib.asked == []                       # no device had products
    mx._watched.update({0: 0, 3: 0})
    mx.check_faults()
    assert lib.asked == [0, 3]
    lib.counts[3] = 5
    mx.check_faults(0)
    with pytest.raises(RuntimeError, match=r"5 wait\(s\).*cuda:3"):
        mx.check_faults()
    mx.check_faults()                            # told
    lib.counts[3] = 6
    with pytest.raises(RuntimeError, match=r"1 wait\(s\)"):
        mx.check_faults(torch.device("cuda", 3))
    mx.check_faults("cuda:3")
    with pytest.raises(ValueError):
        monkeypatch.setattr(lib, "rt_mx_wait_faults", lambda count: -5, raising=False)
        mx.check_faults()


@pytest.mark.gpu
def test_products_are_watched_and_the_step_asks(monkeypatch):
    from ramtorch_b200 import AdamW
    monkeypatch.setattr(mx, "_watched", {})
    x = torch.randn(40, 64, device="cuda").bfloat16()
    p = torch.nn.Parameter(torch.randn(64, 64, device="cuda").bfloat16())
    opt = AdamW([p], lr=1e-3, storage_device="cuda")
    asked = []
    real = mx.check_faults
    monkeypatch.setattr(mx, "check_faults", lambda device=None: asked.append(device) or real(device))
    p.grad = torch.randn_like(p)
    opt.step()
    assert asked == [] and mx._watched == {}     # nothing to ask where no product ran
    for call in (lambda: mx.weight_grad(x, mx.quantize_mxint8(x)), lambda: mx.mxfp4_matmul(mx.quantize_mxfp4(x), mx.quantize_mxfp4(x))):
        mx._watched.clear()
        call()
        assert mx._watched == {0: 0}
    for _ in range(3):                           # the repeated step as well
        opt.step()
    assert asked == [0, 0, 0]
    count = ctypes.c_uint32()
    N.check(N.lib().rt_mx_wait_faults(ctypes.byref(count)))
    mx._watched[0] = count.value - 2             # as if two waits had run out since
    with pytest.raises(RuntimeError, match="ran out on cuda:0"):
        opt.step()
    opt.step()
    w = torch.nn.Parameter(torch.randn(64, 64).bfloat16().pin_memory())      # a streamed parameter
    w.grad = torch.randn_like(w)
    mx._watched[0] = count.value - 1
    with pytest.raises(RuntimeError, match="ran out"):
        AdamW([w], lr=1e-3).step()
