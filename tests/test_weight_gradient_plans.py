"""The weight gradient from an 8-bit checkpoint, on whole numbers, in every tile shape and way of summing.

Gradients and checkpoint values are small integers, so every partial sum is an integer below 2^24 and any order of
additions gives the same bits: the result has to EQUAL the 64-bit one.  A step of the sum that is lost, taken twice, or
meets the wrong tile of a ring shows at once, however long the sum."""
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


# ---------------------------------------------------------------------------------------- every variant
VARIANTS = [(512, "whole"), (512, "joined"), (256, "whole"), (256, "cluster"), (256, "joined"), (128, "whole"), (128, "cluster"), (128, "joined"),
            (64, "whole"), (64, "cluster"), (64, "joined")]


def plan_of(tokens, n, k, kind):
    """(rows of a tile, how its sum is formed) of a gradient whose rows lie next to each other."""
    p = N.MxPlan()
    N.check(N.lib().rt_mx_weight_grad_plan(256, N.DTYPE_CODE[TORCH[kind]], n, tokens, n, k, ctypes.byref(p)))
    assert p.ctas == (2 if p.rows >= 256 else 1)
    return p.rows, "whole" if p.splits == 1 else "joined" if p.joined else "cluster"


@pytest.fixture(scope="module")
def shapes_of():
    """Small shapes for every variant, found by asking: a rule that changes moves the shapes, and one that gives a variant up fails here."""
    rng, found = random.Random(7), {v: [] for v in VARIANTS}
    draw = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))      # noqa: E731
    for _ in range(20000):
        kind = rng.choice(["bf16", "bf16", "f32", "f16"])
        t, n, k = draw(1, 20000), draw(1, 5000), draw(1, 9000)
        if t * n * k < 2.5e9 and n * k < 2e7:
            found[plan_of(t, n, k, kind)].append((t * n * k, t, n, k, kind))
    return {v: sorted(s)[:: max(1, len(s) // 4)][:4] for v, s in found.items()}


def view(rows, cols, kind, aligned):
    """An output inside a buffer of sevens, its rows on 16-byte boundaries or not."""
    buf = torch.full((rows + 2, (cols + 15) // 8 * 8 + (0 if aligned else 3)), 7.0, dtype=TORCH[kind], device=DEV)
    return buf, buf[1:1 + rows, :cols] if aligned else buf[1:1 + rows, 1:1 + cols]


def rest_is_sevens(buf, out):
    out.fill_(7)
    return bool((buf == 7).all())


@gpu
@pytest.mark.parametrize("rows,how", VARIANTS)
def test_every_variant_is_exact(rows, how, shapes_of):
    """Each tile shape and way of summing: all output types, on and off 16-byte boundaries, set and added."""
    assert shapes_of[rows, how]
    for _, tokens, n, k, kind in shapes_of[rows, how]:
        assert plan_of(tokens, n, k, kind) == (rows, how)
        g, q, exact = sums(tokens, n, k, kind, seed=tokens)
        held = integers(n, k, 9, 5)
        for out_kind in TORCH:
            for aligned in (True, False):
                for accumulate in (False, True):
                    buf, out = view(n, k, out_kind, aligned)
                    out.copy_(held)
                    mx.weight_grad(g, q, out=out, accumulate=accumulate)
                    want = (exact + held.double() if accumulate else exact).to(TORCH[out_kind])
                    assert torch.equal(out, want), (tokens, n, k, kind, out_kind, aligned, accumulate)
                    assert rest_is_sevens(buf, out)


@gpu
@pytest.mark.parametrize("tokens,n,k,kind,rows,how", [(2051, 1001, 4104, "bf16", 256, "whole"), (2048, 1024, 4096, "bf16", 256, "whole"), (8192, 4096, 11008, "bf16", 512, "whole"),
                                                     (16384, 256, 512, "bf16", 128, "joined")])
def test_plans_of_sizes_that_figures_are_given_for(tokens, n, k, kind, rows, how):
    assert plan_of(tokens, n, k, kind) == (rows, how)


def test_plan_queries_refuse():
    p = N.MxPlan(1, 1, 1, 1)
    lib = N.lib()
    assert lib.rt_mx_weight_grad_plan(256, 0, 8, 2, 8, 8, None) == -1 and lib.rt_mxfp4_matmul_plan(2, 8, 8, None) == -1
    assert lib.rt_mx_weight_grad_plan(256, 7, 8, 2, 8, 8, ctypes.byref(p)) == -2
    assert lib.rt_mx_weight_grad_plan(256, 0, 8, -1, 8, 8, ctypes.byref(p)) == -3 and lib.rt_mxfp4_matmul_plan(2, -8, 8, ctypes.byref(p)) == -3
    for call in (lambda: lib.rt_mx_weight_grad_plan(None, 0, 8, 0, 8, 8, ctypes.byref(p)), lambda: lib.rt_mxfp4_matmul_plan(2, 8, 0, ctypes.byref(p))):
        p.rows = p.ctas = p.splits = p.joined = 1
        assert call() == 0 and (p.rows, p.ctas, p.splits, p.joined) == (0, 0, 0, 0)      # nothing is launched
