"""The weight gradient from an 8-bit checkpoint, on whole numbers.

Gradients and checkpoint values are small integers, so every partial sum is an integer below 2^24 and any order of
additions gives the same bits: the result has to EQUAL the 64-bit one.  A step of the sum that is lost, taken twice, or
meets the wrong tile of a ring shows at once, however long the sum."""
import numpy as np
import pytest
import torch

from ramtorch_b200 import microscaling as mx

gpu = pytest.mark.gpu
DEV = "cuda"
TORCH = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
PIECES = {"bf16": 1, "f16": 2, "f32": 3}      # bf16 numbers that add up to a value of the type


def integers(rows, cols, top, seed, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-top, top + 1, (rows, cols), generator=g, device=DEV).to(dtype)


def sums(tokens, n, k, kind, seed=0):
    """(gradient, checkpoint, exact sums): magnitudes up to 7 and 15, so that 2^24 is out of reach below 150,000 tokens."""
    assert tokens * 7 * 15 < 1 << 24
    x, g = integers(tokens, k, 15, seed), integers(tokens, n, 7, seed + 1, TORCH[kind])
    q = mx.quantize_mxint8(x)
    assert torch.equal(q.dequantize(torch.float32), x)      # 15 * 8 = 120: exact in 8 bits
    return g, q, g.double().t() @ x.double()


LONG = [(20000, 8, 32), (16384, 256, 512), (40000, 130, 200), (8302, 167, 133), (18172, 436, 40), (6208, 490, 6815), (2051, 1001, 4104),
        (5327, 2725, 322), (693, 298, 2210), (2048, 1024, 4096), (4099, 2100, 2500)]


@gpu
@pytest.mark.parametrize("kind", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("tokens,n,k", LONG)
def test_long_sums_of_whole_numbers_are_exact(tokens, n, k, kind):
    """Many turns of the ring of stages, an odd and an even number of stages, both groups of converting warps."""
    g, q, exact = sums(tokens, n, k, kind)
    for _ in range(2):
        got = mx.weight_grad(g, q, dtype=torch.float32)
        assert torch.equal(got.double(), exact)
    held = integers(n, k, 9, 5)
    assert torch.equal(mx.weight_grad(g, q, out=held.clone(), accumulate=True).double(), exact + held.double())
