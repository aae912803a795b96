"""Plain 64-bit statements of the microscaled formats (numpy), for the tests."""
import math

import numpy as np
import torch

import oracle

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
TORCH = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}


def pad(n, to):
    return -(-n // to) * to


def _blocks(x):
    x = np.asarray(x, np.float64)
    return np.pad(x, ((0, 0), (0, pad(x.shape[1], 32) - x.shape[1]))).reshape(x.shape[0], -1, 32)


def _exponent(amax, top, low, high):
    """Smallest e with amax <= top * 2^e, in [low, high]."""
    m, k = np.frexp(amax)                  # amax = m 2^k, 1/2 <= m < 1
    mt, kt = math.frexp(top)
    return np.clip(k - kt + (m > mt), low, high)


def quantize_int8(x):
    """(codes, scale bytes, values) of a float64 matrix."""
    b = _blocks(x)
    finite = np.isfinite(b).all(-1, keepdims=True)
    b = np.where(finite, b, 0.0)
    f = _exponent(np.abs(b).max(-1, keepdims=True), 127.0, -126, 121)       # f = e - 6
    f = np.where(np.abs(b).max(-1, keepdims=True) == 0, -126, f)
    q = np.clip(np.rint(np.ldexp(b, -f)), -127, 127)
    v = np.where(finite, np.ldexp(q, f), np.nan)
    byte = np.where(finite, f + 6 + 127, 255)[..., 0]
    return q.reshape(len(b), -1).astype(np.int8), byte.astype(np.uint8), v.reshape(len(b), -1)[:, :np.shape(x)[1]]


def quantize_fp4(x, draws=None):
    """(codes one per byte, scale bytes, values); draws: 16-bit integers (rows, padded columns)."""
    b = _blocks(x)
    finite = np.isfinite(b).all(-1, keepdims=True)
    b = np.where(finite, b, 0.0)
    amax = np.abs(b).max(-1, keepdims=True)
    e = np.where(amax == 0, -126, _exponent(amax, 6.0, -126, 126))
    y = np.ldexp(b, -e)
    y = np.where(e == 126, np.clip(y, -3, 3), y)         # 4 * 2^126 is beyond fp32 and bf16
    a = np.abs(y)
    if draws is None:
        # nearest by looking at all eight grid values; a tie goes to the even code
        d = np.abs(a[..., None] - GRID)
        k = np.where(d == d.min(-1, keepdims=True), np.arange(8) + 8 * (np.arange(8) & 1), 99).min(-1) & 7
    else:
        s = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
        v = np.floor(a / s + np.asarray(draws, np.float64).reshape(b.shape) / 65536) * s
        k = np.searchsorted(GRID, np.minimum(v, 6.0))
    sign = np.signbit(y) if draws is None else np.signbit(y) & (k > 0)       # a zero that was drawn is +0
    code = np.where(finite, k | (sign << 3), 0)
    v = np.where(finite, np.ldexp(np.where(np.signbit(y), -GRID[k], GRID[k]), e), np.nan)
    byte = np.where(finite, e + 127, 255)[..., 0]
    return code.reshape(len(b), -1).astype(np.uint8), byte.astype(np.uint8), v.reshape(len(b), -1)[:, :np.shape(x)[1]]


def draws(rows, cols, seed, tensor_id=0, step=0):
    wide = pad(cols, 32)
    return oracle.draws_np(seed, tensor_id, step, 3, 0, rows * wide).reshape(rows, wide)


def untile(scales):
    """(row tiles, block tiles, 32, 4, 4) -> (rows, blocks), written out index by index."""
    rt, kt = scales.shape[:2]
    out = np.empty((rt * 128, kt * 4), np.uint8)
    for r in range(rt * 128):
        for b in range(kt * 4):
            out[r, b] = scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]
    return out


def act(g, kind):
    """act(g), act'(g) in 64 bits."""
    g = torch.as_tensor(g, dtype=torch.float64)
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if kind == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    # (1 + tanh(z)) / 2 as the sigmoid of 2 z, which does not cancel for negative z
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(c * (g + 0.044715 * g ** 3))
    return g * s, s + g * s * (1 - s) * c * (1 + 3 * 0.044715 * g * g)


def matrix(rows, cols, kind, seed, scale=1.0, device="cpu", ld=None, offset=0, loud=True):
    """A seeded matrix, as a strided and shifted view of a larger buffer of NaNs when asked for."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64) * scale
    if loud:
        x = x * (1 + 20 * (torch.rand(1, cols, generator=g) > 0.95))
    x = x.to(TORCH[kind])
    ld = cols if ld is None else ld
    buf = torch.full((offset + max(rows, 1) * ld,), float("nan"), dtype=TORCH[kind], device=device)
    view = buf[offset:].as_strided((rows, cols), (ld, 1), offset)
    view.copy_(x)
    return view
