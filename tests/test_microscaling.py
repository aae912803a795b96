"""Microscaled formats, 8-bit checkpoints and 4-bit products: refusals on the CPU, kernels on the GPU
against plain 64-bit statements.

Codes, scales and dequantised values are exact.  The gated activation is held to half a step of the
result's type plus a few fp32 roundings; the products to half a step plus, for each of the `depth`
additions of the sum, one fp32 step (2^-23: the tensor core may cut instead of round) of the sum of
magnitudes."""
import ctypes

import numpy as np
import pytest
import torch

import mx_util as U
import oracle
from ramtorch_b200 import _native as N
from ramtorch_b200 import checkpointing as ck
from ramtorch_b200 import helpers
from ramtorch_b200 import microscaling as mx

gpu = pytest.mark.gpu
DEV = "cuda"
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def np64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def same(a, b):
    return a.shape == b.shape and bool(((a == b) | (np.isnan(a) & np.isnan(b))).all())


# ------------------------------------------------------------------------------------------ CPU
def test_sizes_of_the_two_arrays():
    lib = N.lib()
    for rows, cols in [(1, 1), (1, 32), (5, 33), (128, 128), (129, 127), (7, 4096), (0, 5), (5, 0)]:
        wide, blocks = U.pad(cols, 32), U.pad(U.pad(cols, 32) // 32, 4)
        assert lib.rt_mx_codes_bytes(0, rows, cols) == rows * wide
        assert lib.rt_mx_codes_bytes(1, rows, cols) == rows * wide // 2
        assert lib.rt_mx_scales_bytes(0, rows, cols) == rows * blocks
        assert lib.rt_mx_scales_bytes(1, rows, cols) == U.pad(rows, 128) * blocks
    assert lib.rt_mx_codes_bytes(2, 1, 1) == -6
    assert lib.rt_mx_codes_bytes(0, -1, 1) == -3
    assert lib.rt_mx_codes_bytes(0, 1 << 20, 1 << 20) == -3
    assert lib.rt_mx_scales_bytes(0, 1 << 31, 1) == -3


def test_calls_are_refused_before_any_launch():
    lib = N.lib()
    buf = (ctypes.c_uint8 * 4096)()
    p = (ctypes.addressof(buf) + 255) & ~255
    q = lambda **k: lib.rt_mx_quantize(*[{**dict(x=p, dt=0, r=2, c=8, ld=8, f=0, t=0, co=p, sc=p, d=None, s=None), **k}[n]   # noqa: E731
                                         for n in ("x", "dt", "r", "c", "ld", "f", "t", "co", "sc", "d", "s")])
    assert q(x=None) == -1 and q(co=None) == -1 and q(sc=None) == -1
    assert q(dt=3) == -2
    assert q(r=-1) == -3 and q(c=-1) == -3 and q(ld=7) == -3 and q(r=1 << 31) == -3
    assert q(x=p + 1) == -4 and q(co=p + 8) == -4 and q(sc=p + 4) == -4
    assert q(f=2) == -6 and q(t=1) == -6 and q(d=ctypes.byref(N.MxDraws(1, 0, 0))) == -6
    assert lib.rt_mx_dequantize(0, p, p, 2, 8, None, 0, 8, None) == -1
    assert lib.rt_mx_dequantize(0, p, p, 2, 8, p, 5, 8, None) == -2
    assert lib.rt_mx_dequantize(1, p + 2, p, 2, 8, p, 0, 8, None) == -4
    assert lib.rt_mx_gated_act(p, 8, p, 8, 0, 2, 8, 3, p, 8, p, p, p, p, None) == -6
    assert lib.rt_mx_gated_act(p, 8, None, 8, 0, 2, 8, 0, p, 8, p, p, p, p, None) == -1
    assert lib.rt_mx_gated_act(p, 8, p, 7, 0, 2, 8, 0, p, 8, p, p, p, p, None) == -3
    assert lib.rt_mx_gated_act_backward(p, 8, 0, 2, 8, 0, p, p, p, None, p, 8, p, 8, None) == -1
    assert lib.rt_mx_gated_act_backward(p, 8, 0, 2, 8, 0, p, p, p, p, p, 8, p + 1, 8, None) == -4
    assert lib.rt_mx_weight_grad_workspace(p, 7, 8, 2, 8, 8) == -2
    assert lib.rt_mx_weight_grad(None, 0, 8, p, p, 2, 8, 8, p, 0, 8, 0, None, 0, None) == -1
    assert lib.rt_mx_weight_grad(p, 0, 8, p, p, 2, 8, 8, p, 0, 7, 0, None, 0, None) == -3
    assert lib.rt_mx_weight_grad(p, 0, 8, p, p, 2, 8, 8, p, 9, 8, 0, None, 0, None) == -2
    need = lib.rt_mx_weight_grad_workspace(p, 1, 8, 2, 8, 8)
    if need:
        assert lib.rt_mx_weight_grad(p, 1, 8, p, p, 2, 8, 8, p, 0, 8, 0, None, 0, None) == -6
        assert lib.rt_mx_weight_grad(p, 1, 8, p, p, 2, 8, 8, p, 0, 8, 0, p, need - 1, None) == -6
        assert lib.rt_mx_weight_grad(p, 1, 8, p, p, 2, 8, 8, p, 0, 8, 0, p + 4, need, None) == -4
    assert lib.rt_mxfp4_matmul(p, p, p, None, 2, 2, 8, p, 0, 2, None) == -1
    assert lib.rt_mxfp4_matmul(p, p, p + 4, p, 2, 2, 8, p, 0, 2, None) == -4
    assert lib.rt_mxfp4_matmul(p, p, p, p, 2, -2, 8, p, 0, 2, None) == -3


def test_empty_calls_do_nothing():
    lib = N.lib()
    assert lib.rt_mx_quantize(None, 0, 0, 8, 8, 0, 0, None, None, None, None) == 0
    assert lib.rt_mx_dequantize(1, None, None, 3, 0, None, 0, 0, None) == 0
    assert lib.rt_mx_gated_act(None, 8, None, 8, 0, 0, 8, 0, None, 8, None, None, None, None, None) == 0
    assert lib.rt_mx_weight_grad(None, 0, 0, None, None, 4, 0, 8, None, 0, 8, 0, None, 0, None) == 0
    assert lib.rt_mxfp4_matmul(None, None, None, None, 0, 8, 8, None, 0, 8, None) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 32)
    for call in (lambda: mx.quantize_mxint8(x), lambda: mx.quantize_mxfp4(x), lambda: mx.gated_act(x, x),
                 lambda: ck.linear(x, torch.zeros(4, 32)),
                 lambda: mx.MxTensor("mxint8", torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 4, dtype=torch.uint8), (4, 32))):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    with pytest.raises(ValueError):
        mx.MxTensor("mxfp8", x, x, (4, 32))


def test_the_plain_statements_themselves():
    """The 64-bit statements on values whose codes are known."""
    x = np.zeros((1, 32)); x[0, :8] = [6, 5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25]
    code, byte, v = U.quantize_fp4(x)
    assert byte[0, 0] == 127
    assert v[0, :8].tolist() == [6, 4, 4, 2, 2, 1, 1, 0] and code[0, :8].tolist() == [7, 6, 6, 4, 4, 2, 2, 0]
    x[0, 0] = 6.0001
    assert U.quantize_fp4(x)[1][0, 0] == 128
    y = np.zeros((1, 32)); y[0, :4] = [127 / 64, -1, 1 / 128, 3 / 128]
    q, byte, v = U.quantize_int8(y)
    assert byte[0, 0] == 127 and q[0, :4].tolist() == [127, -64, 0, 2]
    y[0, 0] = 128 / 64
    assert U.quantize_int8(y)[1][0, 0] == 128


# ------------------------------------------------------------------------------------------ formats
SHAPES = [(1, 1), (1, 31), (3, 32), (2, 33), (7, 100), (33, 127), (128, 128), (129, 264), (5, 4096), (300, 72), (1, 11008), (257, 65)]
KINDS = ["bf16", "f32", "f16"]
VIEWS = {"whole": lambda c: dict(), "strided": lambda c: dict(ld=U.pad(c, 8) + 24), "odd": lambda c: dict(ld=c + 3, offset=1)}


def check_int8(q, want):
    codes, byte, values = want
    assert (q.codes.cpu().numpy() == codes).all()
    scales = q.scales.cpu().numpy()
    assert (scales[:, :byte.shape[1]] == byte).all() and (scales[:, byte.shape[1]:] == 0).all()


def check_fp4(q, want):
    codes, byte, values = want
    packed = q.codes.cpu().numpy()
    got = np.stack([packed & 15, packed >> 4], -1).reshape(codes.shape)
    assert (got == codes).all()
    scales = U.untile(q.scales.cpu().numpy())
    r, b = byte.shape
    assert (scales[:r, :b] == byte).all() and (scales[r:] == 0).all() and (scales[:, b:] == 0).all()


@gpu
@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_and_back(rows, cols, kind, view):
    x = U.matrix(rows, cols, kind, rows * 1000 + cols, device=DEV, **VIEWS[view](cols))
    x64 = np64(x)
    i8, f4 = U.quantize_int8(x64), U.quantize_fp4(x64)
    q = mx.quantize_mxint8(x)
    check_int8(q, i8)
    p = mx.quantize_mxfp4(x)
    check_fp4(p, f4)
    s = mx.quantize_mxfp4(x, seed=(5 << 33) | 77, tensor_id=3, step=9)
    check_fp4(s, U.quantize_fp4(x64, U.draws(rows, cols, (5 << 33) | 77, 3, 9)))
    for t, want in ((q, i8[2]), (p, f4[2])):
        assert t.dequantize().dtype == x.dtype and t.dequantize().shape == x.shape
        for dt in (torch.bfloat16, torch.float32):
            assert same(np64(t.dequantize(dt)), want)
        assert same(np64(t.dequantize(torch.float16)), np64(torch.from_numpy(want).to(torch.float16)))
        out = torch.full((rows, cols + 5), 7.0, dtype=torch.bfloat16, device=DEV)
        t.dequantize(out=out[:, 2:2 + cols])
        assert same(np64(out[:, 2:2 + cols]), want)
        assert (out[:, :2] == 7).all() and (out[:, 2 + cols:] == 7).all()


@gpu
@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (31, 3), (32, 64), (33, 65), (128, 64), (130, 100), (257, 129), (64, 1000), (700, 8)])
def test_quantize_transposed(rows, cols, kind, view):
    x = U.matrix(rows, cols, kind, rows * 999 + cols, device=DEV, **VIEWS[view](cols))
    q = mx.quantize_mxfp4(x, transpose=True)
    assert q.shape == (cols, rows)
    check_fp4(q, U.quantize_fp4(np64(x).T))
    q = mx.quantize_mxfp4(x, transpose=True, seed=12345, tensor_id=1, step=2)
    check_fp4(q, U.quantize_fp4(np64(x).T, U.draws(cols, rows, 12345, 1, 2)))


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_special_values(kind):
    """Blocks of zeros, of the type's extremes and smallest values, ties, and blocks with infinities or NaN."""
    info = torch.finfo(U.TORCH[kind])
    x = torch.zeros(16, 64, dtype=torch.float64)
    x[1] = info.max; x[2] = -info.max; x[3, ::2] = info.tiny; x[4] = info.smallest_normal / 2
    x[5] = torch.arange(64) / 8 - 3                      # ties of the grid
    x[6, 5] = float("inf"); x[7, 40] = float("nan"); x[8, 3] = -float("inf")
    x[9, 0] = 1.984375; x[10, 0] = 1.9921875; x[11, 0] = 6; x[12, 0] = 6.03125
    x[13] = torch.linspace(-6, 6, 64); x[14] = -0.0; x[15, 31] = info.max
    x = x.to(U.TORCH[kind])
    x64 = np64(x)
    for t in (x, torch.nn.functional.pad(x, (3, 2))[:, 3:67]):
        t = t.to(DEV) if t.is_contiguous() else torch.nn.functional.pad(x, (3, 2)).to(DEV)[:, 3:67]
        i8, f4 = U.quantize_int8(x64), U.quantize_fp4(x64)
        q, p = mx.quantize_mxint8(t), mx.quantize_mxfp4(t)
        check_int8(q, i8)
        check_fp4(p, f4)
        check_fp4(mx.quantize_mxfp4(t, seed=1), U.quantize_fp4(x64, U.draws(16, 64, 1)))
        check_fp4(mx.quantize_mxfp4(t.t().contiguous(), transpose=True, seed=1), U.quantize_fp4(x64, U.draws(16, 64, 1)))
        assert same(np64(q.dequantize(torch.bfloat16)), i8[2]) and same(np64(p.dequantize(torch.bfloat16)), f4[2])
        half = np64(q.dequantize(torch.float16))         # finite values stay finite
        assert (np.isnan(half) == np.isnan(i8[2])).all() and np.isfinite(half[~np.isnan(half)]).all()


@gpu
def test_every_scale_byte_and_code_reads_back():
    """All 256 scale bytes against all codes, also those that quantisation never writes."""
    codes8 = torch.arange(-128, 128, dtype=torch.int16).to(torch.int8).repeat(256, 1).to(DEV)
    scales8 = torch.arange(256, dtype=torch.int16).to(torch.uint8)[:, None].repeat(1, 8).to(DEV)
    v = np64(mx.MxTensor("mxint8", codes8, scales8, (256, 256)).dequantize(torch.float32))
    byte = np.arange(256)[:, None]
    want = np.where(byte == 255, np.nan, np.ldexp(np.arange(-128, 128)[None, :].astype(np.float64), byte - 133))
    with np.errstate(over="ignore"):
        want = want.astype(np.float32).astype(np.float64)
    assert same(v, want)
    codes4 = torch.tensor([(2 * i) % 16 | (2 * i + 1) % 16 << 4 for i in range(16)], dtype=torch.uint8).repeat(256, 1).to(DEV)
    tiled = torch.zeros(256, 4, dtype=torch.uint8)
    tiled[:, 0] = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    tiled = tiled.view(2, 4, 32, 1, 4).permute(0, 3, 2, 1, 4).contiguous().to(DEV)
    v = np64(mx.MxTensor("mxfp4", codes4, tiled, (256, 32)).dequantize(torch.float32))
    code = np.arange(32) % 16
    grid = np.where(code & 8, -U.GRID[code & 7], U.GRID[code & 7])
    with np.errstate(over="ignore"):
        want = np.where(byte == 255, np.nan, np.ldexp(grid[None, :], byte - 127)).astype(np.float32).astype(np.float64)
    assert same(v, want)


@gpu
def test_stochastic_rounding_is_unbiased_and_repeats():
    x = torch.full((64, 4096), 0.0, device=DEV)
    x[:, 0::32] = 6.0                                    # fixes the scale at 1
    x[:, 1::32], x[:, 2::32], x[:, 3::32] = 0.3, -2.8, 5.1
    q = mx.quantize_mxfp4(x, seed=5, step=1)
    v = q.dequantize(torch.float32)
    n = 64 * 128
    for col, value, low, high in ((1, 0.3, 0.0, 0.5), (2, -2.8, -3.0, -2.0), (3, 5.1, 4.0, 6.0)):
        got = v[:, col::32]
        assert ((got == low) | (got == high)).all()
        p = (value - low) / (high - low)
        assert abs(float(got.double().mean()) - value) < 4 * (high - low) * (p * (1 - p) / n) ** 0.5
    again = mx.quantize_mxfp4(x, seed=5, step=1)
    assert torch.equal(q.codes, again.codes)
    for other in (dict(seed=6, step=1), dict(seed=5, step=2), dict(seed=5, step=1, tensor_id=1)):
        assert not torch.equal(q.codes, mx.quantize_mxfp4(x, **other).codes)


# ------------------------------------------------------------------------------------------ gated
def act_relative(kind, g, act):
    """Relative error of act(g): half a step of the result's type, and of fp32 the error of a function whose argument
    was rounded up to four times.  A relative error r of the argument changes exp(z) by |z| r and erfc(g / sqrt 2), for
    negative g, by up to (g^2 + 1) r; the functions and the few products after them are off by up to 32 * 2^-24 (the quick
    exponential and reciprocal, used for 16-bit results, by 2^-22 each)."""
    sens = {"silu": np.abs(g), "gelu": g * g + 1, "gelu_tanh": 1.6 * np.abs(g) * (1 + 0.0448 * g * g)}[act]
    return HALF[kind] * 1.01 + (4 * sens + 32) * 2.0 ** -24


@gpu
@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 40), (129, 77), (64, 1024), (17, 2749)])
def test_gated_activation(rows, cols, kind, act, view):
    v = VIEWS[view](cols)
    gate = U.matrix(rows, cols, kind, 1, 1.5, DEV, loud=False, **v)
    up = U.matrix(rows, cols, kind, 2, 1.0, DEV, **v)
    grad = U.matrix(rows, cols, kind, 3, 1e-2, DEV, loud=False, **v)
    h, g8, u8 = mx.gated_act(gate, up, act)
    check_int8(g8, U.quantize_int8(np64(gate)))
    check_int8(u8, U.quantize_int8(np64(up)))
    tiny = torch.finfo(U.TORCH[kind]).smallest_normal
    exact = U.act(np64(gate), act)[0].numpy() * np64(up)
    assert (np.abs(np64(h) - exact) <= np.abs(exact) * act_relative(kind, np64(gate), act) + tiny).all()
    dgate, dup = mx.gated_act_backward(grad, g8, u8, act)
    gv, uv = np64(g8.dequantize(torch.float32)), np64(u8.dequantize(torch.float32))
    a, d = (t.numpy() for t in U.act(gv, act))
    exact = np64(grad) * a
    assert (np.abs(np64(dup) - exact) <= np.abs(exact) * act_relative(kind, gv, act) + tiny).all()
    # act' is a sum of terms no larger than 1 + |g| / 2.  |z| exp(-|z|) is below 0.37, so each term's absolute error is
    # below (4 * 0.37 + 32) * 2^-24 < 2^-18 of that.
    dterm = np.abs(d) + np.abs(gv) * 0.5 + 1.0
    err = np.abs(np64(dgate) - np64(grad) * uv * d)
    assert (err <= np.abs(np64(grad) * uv) * (np.abs(d) * HALF[kind] * 1.01 + dterm * 2.0 ** -18) + tiny).all()
    # into the two halves of one gradient
    both = torch.full((rows, 2 * cols + 2), 3.0, dtype=U.TORCH[kind], device=DEV)
    mx.gated_act_backward(grad, g8, u8, act, out=(both[:, :cols], both[:, cols:2 * cols]))
    assert torch.equal(both[:, :cols], dgate) and torch.equal(both[:, cols:2 * cols], dup) and (both[:, 2 * cols:] == 3).all()


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gated_gradient_against_differences(act):
    """act' against central differences of the forward's own definition, at the kept values."""
    g = torch.linspace(-9, 9, 4096, device=DEV).view(64, 64)
    one = torch.ones_like(g)
    _, g8, u8 = mx.gated_act(g, one, act)
    dgate, dup = mx.gated_act_backward(one, g8, u8, act)
    gv = np64(g8.dequantize(torch.float32))
    step = 1e-5
    diff = (U.act(gv + step, act)[0] - U.act(gv - step, act)[0]).numpy() / (2 * step)
    # third derivatives of all three are below 3: the difference quotient is off by step^2 / 2, its roundings by 1e-10
    assert np.abs(np64(dgate) - diff).max() < 2e-6
    assert np.abs(np64(dup) - U.act(gv, act)[0].numpy()).max() < 9 * 2.0 ** -20


@gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_gated_extremes(kind, act):
    big = float(torch.finfo(U.TORCH[kind]).max)
    vals = [0.0, -0.0, 1e4, -1e4, 1e20, -1e20, big, -big, 88.0, -88.0, 200.0, -200.0, 1e-30]
    g = torch.zeros(len(vals), 32, dtype=U.TORCH[kind], device=DEV)
    g[:, 0] = torch.tensor(vals)
    one = torch.ones_like(g)
    h, g8, u8 = mx.gated_act(g, one, act)
    dgate, dup = mx.gated_act_backward(one, g8, u8, act)
    for t in (h, dgate, dup):
        assert torch.isfinite(t).all()
    gv = np64(g8.dequantize(torch.float32))[:, 0]
    assert (np64(dgate)[gv > 50, 0] == 1).all() and (np.abs(np64(dgate)[gv < -100, 0]) < 1e-30).all()
    g[3, 1], g[5, 2] = float("nan"), float("inf")
    h, g8, u8 = mx.gated_act(g, one, act)
    dgate, dup = mx.gated_act_backward(one, g8, u8, act)
    assert torch.isnan(h[3, 1]) and torch.isnan(dgate[3]).all() and torch.isnan(dup[5]).all()
    assert torch.isfinite(dgate[4]).all() and torch.isfinite(h[3, 3:]).all()


# ----------------------------------------------------------------------------------------- products
def sum_bound(kind, depth, exact, magnitudes):
    """Half a step of the result, and one fp32 step of the sum of magnitudes for each addition."""
    return np.abs(exact) * HALF[kind] * 1.01 + magnitudes * (depth + 2) * 2.0 ** -23 + torch.finfo(U.TORCH[kind]).smallest_normal


def guarded(rows, cols, kind, ld):
    """An output view inside a buffer of sevens."""
    buf = torch.full((rows + 2, ld), 7.0, dtype=U.TORCH[kind], device=DEV)
    return buf, buf[1:1 + rows, 3:3 + cols]


def untouched(buf, rows, cols):
    inside = torch.zeros_like(buf, dtype=torch.bool)
    inside[1:1 + rows, 3:3 + cols] = True
    return bool((buf[~inside] == 7).all())


WGRAD = [(1, 1, 1), (1, 16, 32), (17, 256, 256), (64, 128, 128), (65, 130, 129), (200, 31, 300), (2051, 100, 72), (130, 1001, 264),
         (16, 8, 2080), (1000, 257, 520), (4096, 8, 40)]


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,n,k", WGRAD)
def test_weight_gradient(tokens, n, k, kind):
    x = U.matrix(tokens, k, "bf16", 5, 1.0, DEV)
    g = U.matrix(tokens, n, kind, 6, 1e-2, DEV, loud=False)
    q = mx.quantize_mxint8(x)
    xv, gv = np64(q.dequantize(torch.float32)), np64(g)
    exact, mags = gv.T @ xv, np.abs(gv).T @ np.abs(xv)
    for out_kind in ("bf16", "f32"):
        got = mx.weight_grad(g, q, dtype=U.TORCH[out_kind])
        assert got.shape == (n, k)
        assert (np.abs(np64(got) - exact) <= sum_bound(out_kind, tokens, exact, mags)).all()
    assert mx.weight_grad(g, q).dtype == g.dtype
    # strided gradient, output inside a larger buffer, added to what is there
    wide = U.matrix(tokens, n, kind, 6, 1e-2, DEV, loud=False, ld=n + 5, offset=1)
    buf, out = guarded(n, k, "f32", k + 9)
    out.fill_(0.25)
    mx.weight_grad(wide, q, out=out, accumulate=True)
    assert (np.abs(np64(out) - (exact + 0.25)) <= sum_bound("f32", tokens + 1, exact + 0.25, mags + 0.25)).all()
    assert untouched(buf, n, k)
    buf, out = guarded(n, k, "bf16", k + 9)
    out.fill_(0.25)
    mx.weight_grad(wide, q, out=out, accumulate=True)
    assert (np.abs(np64(out) - (exact + 0.25)) <= sum_bound("bf16", tokens + 1, exact + 0.25, mags + 0.25)).all()
    assert untouched(buf, n, k)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,n,k", [(1, 1, 1), (5, 33, 8), (17, 257, 129), (64, 600, 135), (300, 40, 1000), (77, 1030, 4103), (700, 64, 65)])
def test_weight_gradient_added_to_aligned_rows(tokens, n, k, kind):
    """Rows on 16-byte boundaries, ends inside and at the end of 16 bytes; what lies around stays."""
    q = mx.quantize_mxint8(U.matrix(tokens, k, "bf16", 15, 1.0, DEV))
    g = U.matrix(tokens, n, "bf16", 16, 1e-2, DEV, loud=False)
    held = U.matrix(n, k, kind, 17, 1.0, DEV)
    buf = torch.full((n + 2, (k + 15) // 8 * 8), 7.0, dtype=U.TORCH[kind], device=DEV)
    out = buf[1:1 + n, :k]
    out.copy_(held)
    mx.weight_grad(g, q, out=out, accumulate=True)
    xv, gv, hv = np64(q.dequantize(torch.float32)), np64(g), np64(held)
    exact, mags = gv.T @ xv + hv, np.abs(gv).T @ np.abs(xv) + np.abs(hv)
    assert (np.abs(np64(out) - exact) <= sum_bound(kind, tokens + 1, exact, mags)).all()
    assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, k:] == 7).all()
    again = torch.empty_like(held)
    again.copy_(held)
    mx.weight_grad(g, q, out=again, accumulate=True)      # the same sum wherever it lies
    if k % 8 == 0:
        assert torch.equal(again, out)


@gpu
def test_weight_gradient_of_nothing_and_of_nan():
    g, x = torch.ones(0, 24, device=DEV, dtype=torch.bfloat16), torch.ones(0, 40, device=DEV, dtype=torch.bfloat16)
    q = mx.quantize_mxint8(x)
    assert (mx.weight_grad(g, q) == 0).all()
    out = torch.full((24, 40), 2.0, device=DEV)
    mx.weight_grad(g, q, out=out, accumulate=True)
    assert (out == 2).all()
    x = torch.ones(70, 100, device=DEV, dtype=torch.bfloat16)
    x[69, 40] = float("inf")                              # block 1 of the last token
    dw = mx.weight_grad(torch.ones(70, 8, device=DEV, dtype=torch.bfloat16), mx.quantize_mxint8(x))
    assert torch.isnan(dw[:, 32:64]).all() and (dw[:, :32] == 70).all() and (dw[:, 64:] == 70).all()
    g = torch.ones(70, 8, device=DEV, dtype=torch.bfloat16)
    g[3, 2] = float("nan"); g[5, 4] = float("inf")
    dw = mx.weight_grad(g, mx.quantize_mxint8(torch.ones(70, 100, device=DEV, dtype=torch.bfloat16)))
    assert torch.isnan(dw[2]).all() and torch.isinf(dw[4]).all() and torch.isfinite(dw[[0, 1, 3, 5, 6, 7]]).all()


@gpu
def test_weight_gradient_over_the_whole_exponent_range():
    """Checkpoint blocks from the smallest to large exponents enter the product exactly."""
    x = torch.ones(40, 64, device=DEV) * torch.exp2(torch.arange(-118, 122, 6, device=DEV, dtype=torch.float32))[:, None]
    g = torch.zeros(40, 40, device=DEV)
    g.fill_diagonal_(1.0)
    q = mx.quantize_mxint8(x)
    assert torch.equal(mx.weight_grad(g.bfloat16(), q, dtype=torch.float32), q.dequantize(torch.float32))
    assert torch.equal(mx.weight_grad(g, q, dtype=torch.float32), q.dequantize(torch.float32))
    assert torch.equal(mx.weight_grad(g.half(), q, dtype=torch.float32), q.dequantize(torch.float32))


@gpu
def test_weight_gradient_against_differences():
    """The loss <grad, x8 @ w.T> is linear in w: along any direction v its difference quotient is <dw, v>, in 64 bits exactly."""
    x, g = U.matrix(300, 136, "bf16", 31, 1.0, DEV), U.matrix(300, 72, "bf16", 32, 1e-2, DEV, loud=False)
    q = mx.quantize_mxint8(x)
    dw = mx.weight_grad(g, q, dtype=torch.float32).double()
    x8, loss = q.dequantize(torch.float32).double(), lambda w: (g.double() * (x8 @ w.t())).sum()
    gen = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(72, 136, generator=gen, device=DEV, dtype=torch.float64)
    for _ in range(4):
        v = torch.randn(72, 136, generator=gen, device=DEV, dtype=torch.float64)
        quotient = (loss(w + v) - loss(w - v)) / 2
        bound = (v.abs() * (g.double().abs().t() @ x8.abs())).sum() * 302 * 2.0 ** -23
        assert abs(quotient - (dw * v).sum()) <= bound


@gpu
def test_weight_gradient_at_the_top_of_the_range():
    """Scale bytes 253 and 254, next to ordinary blocks and to a block of zeros in the same warp's share."""
    x = torch.randn(70, 200, device=DEV)
    x[::3, :32] *= 2.0 ** 126 / 4
    x[::3, 0] = 1.5 * 2.0 ** 126                         # fixes the scale byte at 253
    x[1::3, 32:64] = torch.sign(x[1::3, 32:64]) * torch.finfo(torch.float32).max
    x[5, 64:96] = 0
    g = (torch.randn(70, 24, device=DEV) * 2.0 ** -60).bfloat16()
    q = mx.quantize_mxint8(x)
    assert set(q.scales[:, :2].unique().tolist()) & {253, 254} == {253, 254}
    xv, gv = np64(q.dequantize(torch.float32)), np64(g)
    assert np.isfinite(xv).all()
    exact, mags = gv.T @ xv, np.abs(gv).T @ np.abs(xv)
    got = np64(mx.weight_grad(g, q, dtype=torch.float32))
    assert (np.abs(got - exact) <= sum_bound("f32", 70, exact, mags)).all()


MATMUL = [(1, 1, 1), (1, 128, 128), (1, 300, 2080), (2, 64, 33), (8, 1001, 256), (17, 129, 64), (33, 40, 4096), (128, 128, 256), (130, 257, 520),
          (300, 100, 96), (257, 513, 1000), (64, 8, 11008)]


@gpu
@pytest.mark.parametrize("m,n,k", MATMUL)
def test_fp4_product(m, n, k):
    a = mx.quantize_mxfp4(U.matrix(m, k, "bf16", 7, 1.0, DEV))
    b = mx.quantize_mxfp4(U.matrix(n, k, "bf16", 8, 0.02, DEV))
    av, bv = np64(a.dequantize(torch.float32)), np64(b.dequantize(torch.float32))
    exact, mags = av @ bv.T, np.abs(av) @ np.abs(bv).T
    for kind in KINDS:
        got = mx.mxfp4_matmul(a, b, dtype=U.TORCH[kind])
        assert got.shape == (m, n)
        assert (np.abs(np64(got) - exact) <= sum_bound(kind, k, exact, mags)).all()
        buf, out = guarded(m, n, kind, n + 9)
        mx.mxfp4_matmul(a, b, out=out)
        assert torch.equal(out, got) and untouched(buf, m, n)


@gpu
def test_fp4_product_of_nothing_and_of_nan():
    z = torch.zeros(5, 0, device=DEV, dtype=torch.bfloat16)
    assert (mx.mxfp4_matmul(mx.quantize_mxfp4(z), mx.quantize_mxfp4(torch.zeros(7, 0, device=DEV))) == 0).all()
    assert mx.mxfp4_matmul(mx.quantize_mxfp4(torch.zeros(0, 64, device=DEV)), mx.quantize_mxfp4(torch.zeros(7, 64, device=DEV))).shape == (0, 7)
    a, b = torch.ones(140, 200, device=DEV), torch.ones(150, 200, device=DEV)
    a[139, 199] = float("nan"); b[2, 0] = float("inf")
    y = mx.mxfp4_matmul(mx.quantize_mxfp4(a), mx.quantize_mxfp4(b))
    assert torch.isnan(y[139]).all() and torch.isnan(y[:, 2]).all()
    y[139] = 200; y[:, 2] = 200
    assert (y == 200).all()


@gpu
def test_fp4_product_keeps_every_scale_apart():
    """One block of one row at a time, each with a scale of its own: a scale that went to another row or block would show."""
    for m, n, k in ((130, 70, 416), (40, 300, 160)):
        nb = U.pad(k, 32) // 32
        a = torch.exp2(((torch.arange(m)[:, None] * 7 + torch.arange(nb)[None] * 5) % 23 - 11).double()).repeat_interleave(32, 1)[:, :k]
        b = torch.exp2(((torch.arange(n)[:, None] * 3 + torch.arange(nb)[None] * 11) % 19 - 9).double()).repeat_interleave(32, 1)[:, :k]
        y = mx.mxfp4_matmul(mx.quantize_mxfp4(a.float().to(DEV)), mx.quantize_mxfp4(b.float().to(DEV)), dtype=torch.float32)
        assert torch.allclose(y.double().cpu(), a @ b.t(), rtol=k * 2.0 ** -23, atol=0)


# ------------------------------------------------------------------------------- how a user has them
@gpu
def test_refusals():
    x = torch.zeros(8, 64, device=DEV, dtype=torch.bfloat16)
    q, p = mx.quantize_mxint8(x), mx.quantize_mxfp4(x)
    bad = [lambda: mx.quantize_mxint8(x.int()), lambda: mx.quantize_mxint8(x.t()), lambda: mx.quantize_mxint8(x.view(8, 2, 32).transpose(0, 1)),
           lambda: mx.quantize_mxint8(torch.tensor(1.0, device=DEV)), lambda: mx.quantize_mxint8(x[:1].expand(4, 64)),
           lambda: mx.quantize_mxfp4(x.view(2, 4, 64), transpose=True), lambda: mx.quantize_mxfp4(x, seed=1, step=-1),
           lambda: q.dequantize(torch.float64), lambda: q.dequantize(out=x[:4]), lambda: q.dequantize(torch.float32, out=x),
           lambda: mx.mxfp4_matmul(p, q), lambda: mx.mxfp4_matmul(p, mx.quantize_mxfp4(x[:, :32])),
           lambda: mx.mxfp4_matmul(p, p, out=x), lambda: mx.mxfp4_matmul(p, p, dtype=torch.int8),
           lambda: mx.weight_grad(x, p), lambda: mx.weight_grad(x[:4], q), lambda: mx.weight_grad(x, q, accumulate=True),
           lambda: mx.weight_grad(x, q, out=x), lambda: mx.gated_act(x, x[:4]), lambda: mx.gated_act(x, x.float()),
           lambda: mx.gated_act(x, x, "relu"), lambda: mx.gated_act_backward(x[:4], q, q), lambda: mx.gated_act_backward(x, p, q),
           lambda: mx.gated_act_backward(x, q, q, out=(x, x[:4])), lambda: ck.linear(x, x[:, :32]), lambda: ck.linear(x, x.float()),
           lambda: ck.linear(x, x, product="fp4"), lambda: mx.MxTensor("mxint8", q.codes[:, :32], q.scales, (8, 64)),
           lambda: mx.MxTensor("mxint8", q.codes, q.scales[1:], (8, 64)), lambda: mx.MxTensor("mxfp4", q.codes, q.scales, (8, 64)),
           lambda: mx.MxTensor("mxint8", q.codes, q.scales, (8, 64), torch.int32)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    flat = torch.zeros(8 * 64 + 1, device=DEV, dtype=torch.int8)
    with pytest.raises(ValueError, match="16-byte"):
        mx.MxTensor("mxint8", flat[1:].view(8, 64), q.scales, (8, 64))
    assert torch.equal(mx.quantize_mxint8(x.view(2, 4, 64)).codes, q.codes)      # leading dimensions are rows
    assert mx.quantize_mxint8(x[0]).shape == (64,)


@gpu
@pytest.mark.parametrize("product", [None, "mxfp4"])
def test_a_block_trains_like_its_plain_form(product):
    """A gated MLP with a bias: outputs and every gradient against the same sums written out in 64 bits from the 8- and 4-bit values."""
    torch.manual_seed(3)
    t, d, f = 70, 96, 136
    x = torch.randn(2, t // 2, d, device=DEV).bfloat16().requires_grad_()
    w1 = (torch.randn(2 * f, d, device=DEV) * 0.1).bfloat16().requires_grad_()
    w2 = (torch.randn(d, f, device=DEV) * 0.1).bfloat16().requires_grad_()
    b2 = torch.randn(d, device=DEV).bfloat16().requires_grad_()
    kw = dict(product=product, seed=11, step=4) if product else {}
    proj = ck.linear(x, w1, **kw)
    h = ck.gated_act(*proj.chunk(2, -1))
    y = ck.linear(h, w2, b2, tensor_id=1, **kw)
    gy = torch.randn_like(y)
    # what is kept is 8 bits: the layers' inputs, and the two inputs of the activation
    assert [t.dtype for t in proj.grad_fn.saved_tensors] == [torch.int8, torch.uint8, torch.bfloat16]
    assert [t.dtype for t in h.grad_fn.saved_tensors] == [torch.int8, torch.uint8] * 2
    gx, g1, g2, gb, gproj, gh = torch.autograd.grad(y, (x, w1, w2, b2, proj, h), gy)

    def v64(a):
        return np64(a).reshape(-1, a.shape[-1])

    def values(a, **k):
        q = mx.quantize_mxfp4(a, **k) if product else a
        return v64(q.dequantize(torch.float32)) if product else v64(a)

    close = lambda a, b, depth, mags: (np.abs(v64(a) - b) <= sum_bound("bf16", depth, b, mags) + np.abs(b) * 2.0 ** -8).all()   # noqa: E731
    for name, got, a, b in (("proj", proj, values(x), values(w1)), ("y", y - b2, values(h), values(w2))):
        slack = 2.0 ** -7 * np.abs(v64(y)).max() if name == "y" else 0.0       # y is rounded, b2 added, rounded, taken off, rounded
        assert (np.abs(v64(got) - a @ b.T) <= sum_bound("bf16", 200, a @ b.T, np.abs(a) @ np.abs(b).T) + slack).all(), name
    h8 = v64(mx.quantize_mxint8(h).dequantize(torch.float32))
    x8 = v64(mx.quantize_mxint8(x).dequantize(torch.float32))
    assert close(g2, v64(gy).T @ h8, t, np.abs(v64(gy)).T @ np.abs(h8))
    assert close(g1, v64(gproj).T @ x8, t, np.abs(v64(gproj)).T @ np.abs(x8))
    a, b = values(gy, **({"seed": 11, "tensor_id": 1, "step": 4} if product else {})), (values(w2, transpose=True).T if product else v64(w2))
    assert close(gh, a @ b, d, np.abs(a) @ np.abs(b))
    a, b = values(gproj, **({"seed": 11, "step": 4} if product else {})), (values(w1, transpose=True).T if product else v64(w1))
    assert close(gx, a @ b, 2 * f, np.abs(a) @ np.abs(b))
    assert np.abs(np64(gb) - v64(gy).sum(0)).max() <= 2.0 ** -8 * np.abs(v64(gy).sum(0)).max() + 1e-4


@gpu
def test_gradients_reach_the_optimizer_in_hbm():
    """CPU-resident weights: two micro-batches add up in rt_device_grad, AdamW.step takes them."""
    from ramtorch_b200 import AdamW
    torch.manual_seed(0)
    w = torch.nn.Parameter((torch.randn(40, 72) * 0.1).bfloat16().pin_memory())
    w.is_ramtorch = True
    xs = [torch.randn(33, 72, device=DEV).bfloat16() for _ in range(2)]
    gs = [torch.randn(33, 40, device=DEV).bfloat16() for _ in range(2)]
    for x, g in zip(xs, gs):
        ck.linear(x, w).backward(g)
    assert w.grad is None
    held = w.__dict__[helpers.DEVICE_GRAD_ATTR]
    first = mx.weight_grad(gs[0], mx.quantize_mxint8(xs[0]))
    want = mx.weight_grad(gs[1], mx.quantize_mxint8(xs[1]), out=first, accumulate=True)
    assert torch.equal(held, want)
    before = w.detach().clone()
    opt = AdamW([w], lr=1e-2)
    opt.step()
    assert not torch.equal(before, w.detach())
    opt.zero_grad()
    assert w.__dict__.get(helpers.DEVICE_GRAD_ATTR) is None
    # a hook sees the fresh gradient of each micro-batch
    seen = []
    helpers.register_ramtorch_hook(w, lambda t: seen.append(t.clone()) or t * 2, helpers.ZERO2_HOOK_NAME)
    for x, g in zip(xs, gs):
        ck.linear(x, w).backward(g)
    assert len(seen) == 2 and torch.equal(w.__dict__[helpers.DEVICE_GRAD_ATTR], seen[0] * 2 + seen[1] * 2)


@gpu
def test_captured_and_replayed_and_on_another_stream():
    g = torch.randn(200, 264, device=DEV).bfloat16()
    x = torch.randn(200, 520, device=DEV).bfloat16()
    w = torch.randn(264, 520, device=DEV).bfloat16()
    gf = g.float()

    def everything():
        q = mx.quantize_mxint8(x)
        h, g8, u8 = mx.gated_act(x, x)
        return (mx.weight_grad(g, q), mx.weight_grad(gf, q), mx.mxfp4_matmul(mx.quantize_mxfp4(x, seed=3), mx.quantize_mxfp4(w)), h,
                *mx.gated_act_backward(x, g8, u8), mx.quantize_mxfp4(x, transpose=True, seed=1).dequantize())

    want = everything()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = everything()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(everything())
        graphs.append(graph)
    x.mul_(2)
    graphs[0].replay()
    x.mul_(0.5)
    for graph in graphs:
        graph.replay()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in (other, *outs):
        for a, b in zip(want, got):
            assert torch.equal(a, b)


@gpu
def test_a_training_step_captured_into_a_graph():
    """Forward and backward of the layers inside one CUDA graph (leaves that no eager graph holds), replayed on new data."""
    torch.manual_seed(5)
    x = torch.randn(96, 128, device=DEV).bfloat16()
    gy = torch.randn(96, 128, device=DEV).bfloat16()
    shapes = [(2 * 160, 128), (128, 160)]
    first = [torch.randn(*s, device=DEV).bfloat16() for s in shapes]

    def step(ws):
        h = ck.gated_act(*ck.linear(x, ws[0], product="mxfp4", seed=3, step=1).chunk(2, -1), "gelu_tanh")
        y = ck.linear(h, ws[1], product="mxfp4", seed=3, tensor_id=1, step=1)
        return torch.autograd.grad(y, ws, gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step([w.clone().requires_grad_() for w in first])
    torch.cuda.current_stream().wait_stream(side)
    leaves = [w.clone().requires_grad_() for w in first]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step(leaves)
    for _ in range(2):
        x.copy_(torch.randn(96, 128, device=DEV))
        gy.copy_(torch.randn(96, 128, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, step([w.clone().requires_grad_() for w in first])):
            assert torch.equal(a, b)


@gpu
def test_repeated_calls_give_the_same_bits():
    g, x = torch.randn(3000, 300, device=DEV).bfloat16(), torch.randn(3000, 200, device=DEV).bfloat16()
    q = mx.quantize_mxint8(x)
    a, b = mx.quantize_mxfp4(x[:40]), mx.quantize_mxfp4(x)
    first = mx.weight_grad(g, q), mx.mxfp4_matmul(a, b)
    for _ in range(3):
        assert torch.equal(first[0], mx.weight_grad(g, q)) and torch.equal(first[1], mx.mxfp4_matmul(a, b))


@gpu
@pytest.mark.parametrize("tokens,n,k", [(64, 256, 256), (100, 300, 130), (700, 2100, 2500), (2000, 500, 4096), (320, 4000, 4500), (9000, 130, 301), (20000, 8, 32), (6000, 250, 600)])
def test_weight_gradient_of_many_tiles(tokens, n, k):
    """Enough tiles, or tokens, for every tile shape and split; the last tiles of both sides are cut."""
    x = U.matrix(tokens, k, "bf16", 15, 1.0, DEV)
    g = U.matrix(tokens, n, "bf16", 16, 1e-2, DEV, loud=False)
    q = mx.quantize_mxint8(x)
    xv, gv = q.dequantize(torch.float32).double(), g.double()
    exact, mags = np64(gv.T @ xv), np64(gv.T.abs() @ xv.abs())
    buf, out = guarded(n, k, "f32", k + 9)
    mx.weight_grad(g, q, out=out)
    assert (np.abs(np64(out) - exact) <= sum_bound("f32", tokens, exact, mags)).all()
    assert untouched(buf, n, k)
    assert (np.abs(np64(mx.weight_grad(g, q)) - exact) <= sum_bound("bf16", tokens, exact, mags)).all()


@gpu
@pytest.mark.parametrize("m,n,k", [(129, 300, 700), (700, 2100, 512), (2000, 500, 1024), (320, 4000, 300), (1, 20000, 4096), (60, 5000, 2080), (384, 256, 256),
                                   (385, 257, 1300), (3000, 9000, 160), (1000, 20000, 4100)])
def test_fp4_product_of_many_tiles(m, n, k):
    a = mx.quantize_mxfp4(U.matrix(m, k, "bf16", 17, 1.0, DEV))
    b = mx.quantize_mxfp4(U.matrix(n, k, "bf16", 18, 0.02, DEV))
    av, bv = a.dequantize(torch.float32).double(), b.dequantize(torch.float32).double()
    exact, mags = np64(av @ bv.T), np64(av.abs() @ bv.abs().T)
    buf, out = guarded(m, n, "f32", n + 9)
    mx.mxfp4_matmul(a, b, out=out)
    assert (np.abs(np64(out) - exact) <= sum_bound("f32", k, exact, mags)).all()
    assert untouched(buf, m, n)


@gpu
def test_both_host_sides_give_the_same(monkeypatch):
    """With the C++ host side and through ctypes: the same results and the same refusals."""
    x = torch.randn(3, 50, 264, device=DEV).bfloat16()
    g = torch.randn(3, 50, 72, device=DEV).bfloat16()
    w = torch.randn(72, 264, device=DEV).bfloat16()

    def everything():
        q, p = mx.quantize_mxint8(x), mx.quantize_mxfp4(x, seed=2**40 + 3, tensor_id=5, step=6)
        t = mx.quantize_mxfp4(w, transpose=True)
        h, g8, u8 = mx.gated_act(x[..., :130], x[..., 132:262])
        out = torch.ones(72, 264, device=DEV)
        found = [q.codes, q.scales, p.codes, p.scales, t.codes, t.scales, q.dequantize(), p.dequantize(torch.float32), t.dequantize(torch.float16),
                 h, g8.codes, u8.scales, *mx.gated_act_backward(h, g8, u8), mx.weight_grad(g, q), mx.weight_grad(g.float(), q),
                 mx.weight_grad(g, q, out=out, accumulate=True), mx.mxfp4_matmul(p, mx.quantize_mxfp4(w)), mx.mxfp4_matmul(p, mx.quantize_mxfp4(w), dtype=torch.float32)]
        assert p.shape == (3, 50, 264) and t.shape == (264, 72) and found[-1].shape == (3, 50, 72) and found[9].shape == (3, 50, 130)
        with pytest.raises(ValueError):
            mx.quantize_mxint8(torch.empty(0, device=DEV).as_strided((0, 1 << 31), (1, 1)))
        return found

    a = everything()
    monkeypatch.setattr(mx, "_fast", False)
    for s, t in zip(a, everything()):
        assert s.dtype == t.dtype and torch.equal(s, t)


@gpu
def test_outputs_may_not_lie_where_inputs_do():
    x = torch.zeros(16, 64, device=DEV, dtype=torch.bfloat16)
    q = mx.quantize_mxint8(x)
    pool = torch.zeros(64, 256, device=DEV, dtype=torch.bfloat16)
    g = pool[:16, :64]
    for out in ((g, torch.zeros_like(x)), (torch.zeros_like(x), g), (x, x), (pool[20:36, :64], pool[21:37, :64]), (pool[20:36, :64], pool[20:36, 32:96])):
        with pytest.raises(ValueError, match="overlap"):
            mx.gated_act_backward(g, q, q, out=out)
    mx.gated_act_backward(g, q, q, out=(pool[20:36, :64], pool[20:36, 64:128]))
    mx.gated_act_backward(g, q, q, out=(pool[20:36, 128:192], pool[20:36, 64:128]))
    mx.gated_act_backward(g, q, q, out=(pool[20:36, :64], pool[40:56, :64]))
    with pytest.raises(ValueError, match="overlap"):
        mx.weight_grad(pool[:16, :64], q, out=pool[:64, :64])
    raw = q.codes.view(-1)[:16 * 64].view(torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        mx.MxTensor("mxint8", q.codes[:8], q.scales[:8], (8, 64)).dequantize(out=raw.view(8, 64))


@gpu
def test_layers_take_inputs_of_any_strides():
    """Transposed and expanded inputs, weights and gradients, one vector, and an empty batch."""
    torch.manual_seed(1)
    w = torch.randn(48, 64, device=DEV).bfloat16()
    xt = torch.randn(64, 33, device=DEV).bfloat16()
    for product in (None, "mxfp4"):
        for x in (xt.t(), xt.t()[:1].expand(5, 64), xt.t()[3], xt.t()[:0], xt.t().contiguous().view(3, 11, 64).transpose(0, 1)):
            for weight in (w, w.t().contiguous().t()):
                a, b = x.detach().requires_grad_(), weight.detach().requires_grad_()
                y = ck.linear(a, b, product=product)
                assert y.shape == x.shape[:-1] + (48,)
                y.sum().backward()                      # an expanded gradient
                plain = ck.linear(x.contiguous(), weight.contiguous(), product=product)
                assert torch.equal(y.detach(), plain) or product is None
                assert a.grad.shape == x.shape and b.grad.shape == w.shape
                want = np.ones((48, 1)) * np64(mx.quantize_mxint8(x.reshape(-1, 64).contiguous()).dequantize(torch.float32)).sum(0)[None]
                assert np.allclose(np64(b.grad), want, rtol=2.0 ** -7, atol=1e-3)
    g, u = torch.randn(20, 30, device=DEV).t(), torch.randn(30, 20, device=DEV)
    assert torch.equal(ck.gated_act(g, u), ck.gated_act(g.contiguous(), u))


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements, and rows further apart than 2^31 bytes: the last rows are those of the same rows alone."""
    rows, cols = 66000, 32800
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x.fill_(1.0)
    tail = U.matrix(300, cols, "bf16", 21, 1.0, DEV)
    x[-300:] = tail
    q, t = mx.quantize_mxint8(x), mx.quantize_mxint8(tail)
    assert torch.equal(q.codes[-300:], t.codes) and torch.equal(q.scales[-300:], t.scales) and (q.codes[:-300:997] == 64).all()
    back = q.dequantize()
    assert torch.equal(back[-300:], t.dequantize()) and (back[:-300:997] == 1).all()
    del back
    h, g8, u8 = mx.gated_act(x, x)
    h2, g2, _ = mx.gated_act(tail, tail)
    assert torch.equal(h[-300:], h2) and torch.equal(g8.codes[-300:], g2.codes)
    dg, du = mx.gated_act_backward(x, g8, u8)
    dg2, du2 = mx.gated_act_backward(tail, g2, g2)
    assert torch.equal(dg[-300:], dg2) and torch.equal(du[-300:], du2)
    del h, dg, du, g8, u8
    p = mx.quantize_mxfp4(x)
    assert torch.equal(p.dequantize(torch.bfloat16)[-300:], mx.quantize_mxfp4(tail).dequantize(torch.bfloat16))
    p = mx.quantize_mxfp4(x, transpose=True)            # 32800 x 66000
    cut = mx.quantize_mxfp4(x[:, -40:], transpose=True)
    assert torch.equal(p.codes[-40:], cut.codes)
    del p, x
    # rows 2^31 bytes apart, at a misaligned start
    far = torch.empty(4 * (1 << 30) + 4096, dtype=torch.bfloat16, device=DEV)
    for ld in (1 << 30, (1 << 30) + 3):
        v = far[1:].as_strided((4, 1000), (ld, 1))
        v.copy_(U.matrix(4, 1000, "bf16", 22, 1.0, DEV))
        w = v.contiguous()
        assert torch.equal(mx.quantize_mxint8(v).codes, mx.quantize_mxint8(w).codes)
        assert torch.equal(mx.quantize_mxfp4(v, transpose=True).codes, mx.quantize_mxfp4(w, transpose=True).codes)
        g = torch.randn(4, 24, device=DEV).bfloat16()
        out = mx.weight_grad(v, mx.quantize_mxint8(g))
        assert torch.equal(out, mx.weight_grad(w, mx.quantize_mxint8(g)))
        mx.quantize_mxint8(w).dequantize(out=v)
        assert torch.equal(v, mx.quantize_mxint8(w).dequantize())


@gpu
def test_products_with_outputs_beyond_32_bits():
    n, k = 48000, 46000
    g = U.matrix(70, n, "bf16", 23, 1e-2, DEV, loud=False)
    x = U.matrix(70, k, "bf16", 24, 1.0, DEV)
    q = mx.quantize_mxint8(x)
    dw = mx.weight_grad(g, q)
    xv, gv = q.dequantize(torch.float32).double(), g.double()
    for i, j in ((0, 0), (n - 300, k - 400), (n - 300, 0), (0, k - 400)):
        a, b = gv[:, i:i + 300], xv[:, j:j + 400]
        exact, mags = np64(a.T @ b), np64(a.T.abs() @ b.abs())
        assert (np.abs(np64(dw[i:i + 300, j:j + 400]) - exact) <= sum_bound("bf16", 70, exact, mags)).all()
    del dw
    a4, b4 = mx.quantize_mxfp4(U.matrix(n, 96, "bf16", 25, 1.0, DEV)), mx.quantize_mxfp4(U.matrix(k, 96, "bf16", 26, 1.0, DEV))
    y = mx.mxfp4_matmul(a4, b4)
    av, bv = a4.dequantize(torch.float32).double(), b4.dequantize(torch.float32).double()
    for i, j in ((0, 0), (n - 300, k - 400), (n - 300, 0), (0, k - 400)):
        a, b = av[i:i + 300], bv[j:j + 400]
        exact, mags = np64(a @ b.T), np64(a.abs() @ b.abs().T)
        assert (np.abs(np64(y[i:i + 300, j:j + 400]) - exact) <= sum_bound("bf16", 96, exact, mags)).all()


@gpu
def test_no_wait_ran_out():
    torch.cuda.synchronize()
    count = ctypes.c_uint32(99)
    assert N.lib().rt_mx_wait_faults(ctypes.byref(count)) == 0 and count.value == 0
