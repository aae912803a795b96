"""The product of MXFP4 matrices, on whole numbers, in every tile shape and way of summing.

All values are integers of the 4-bit grid and all sums stay below 2^24, so the result has to EQUAL the 64-bit one."""
import ctypes
import math
import random

import pytest
import torch

from ramtorch_b200 import _native as N
from ramtorch_b200 import microscaling as mx

gpu = pytest.mark.gpu
DEV = "cuda"
TORCH = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
VARIANTS = [(32, "whole"), (32, "cluster"), (64, "whole"), (64, "cluster"), (128, "whole"), (128, "cluster"), (384, "whole")]


def plan_of(m, n, k):
    """(rows of a tile, how its sum is formed)"""
    p = N.MxPlan()
    N.check(N.lib().rt_mxfp4_matmul_plan(m, n, k, ctypes.byref(p)))
    assert p.ctas == (2 if p.rows == 384 else 1) and not p.joined
    return p.rows, "whole" if p.splits == 1 else "cluster"


@pytest.fixture(scope="module")
def shapes_of():
    """Small shapes for every variant, found by asking; both for one block of the sum and for many."""
    rng, found = random.Random(11), {v: [] for v in VARIANTS}
    draw = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))      # noqa: E731
    for _ in range(20000):
        m, n, k = draw(1, 3000), draw(1, 12000), draw(1, 9000)
        if m * n * k < 4e9 and m * n < 1.2e7:
            found[plan_of(m, n, k)].append((m * n * k, m, n, k))
    return {v: sorted(s)[:: max(1, len(s) // 4)][:4] for v, s in found.items()}


def integers(rows, cols, seed):
    """Values 0, 1, 2, 3, 4, 6 of either sign, and their quantisation, which is exact."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    grid = torch.tensor([0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6], dtype=torch.float32, device=DEV)
    x = grid[torch.randint(0, 11, (rows, cols), generator=g, device=DEV)]
    q = mx.quantize_mxfp4(x)
    assert torch.equal(q.dequantize(torch.float32), x)
    return x.double(), q


@gpu
@pytest.mark.parametrize("rows,how", VARIANTS)
def test_every_variant_is_exact(rows, how, shapes_of):
    """All output types, on and off 16-byte boundaries; what lies around the output stays."""
    assert shapes_of[rows, how]
    for _, m, n, k in shapes_of[rows, how]:
        assert plan_of(m, n, k) == (rows, how)
        (a, qa), (b, qb) = integers(m, k, m), integers(n, k, n + 1)
        exact = a @ b.t()
        for kind, dtype in TORCH.items():
            for aligned in (True, False):
                buf = torch.full((m + 2, (n + 15) // 8 * 8 + (0 if aligned else 3)), 7.0, dtype=dtype, device=DEV)
                out = buf[1:1 + m, :n] if aligned else buf[1:1 + m, 1:1 + n]
                mx.mxfp4_matmul(qa, qb, out=out)
                assert torch.equal(out, exact.to(dtype)), (m, n, k, kind, aligned)
                out.fill_(7)
                assert (buf == 7).all()


@gpu
@pytest.mark.parametrize("m,n,k,rows,how", [(8192, 11008, 4096, 384, "whole"), (512, 11008, 4096, 128, "whole"), (1, 11008, 4096, 32, "whole"), (1, 4096, 4096, 32, "cluster")])
def test_plans_of_sizes_that_figures_are_given_for(m, n, k, rows, how):
    assert plan_of(m, n, k) == (rows, how)
