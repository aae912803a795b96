"""The microscaled operators as they are measured: cases, inputs, plain forms.

Five operators: the 8-bit checkpoint of an activation (store, restore), the gated activation that keeps its
inputs in 8 bits (forward, backward), the weight gradient from an 8-bit checkpoint, quantisation to 4-bit
microscaled floating point, and the product with 4-bit weights.

Formats (OCP microscaling): 32 consecutive values of a row share one scale 2^e, stored as the byte e + 127.
MXINT8 values are q * 2^(e-6) with |q| <= 127; MXFP4 values are +-{0, .5, 1, 1.5, 2, 3, 4, 6} * 2^e.  e is the
smallest exponent at which the largest magnitude of the block does not saturate.
"""
import math
from functools import reduce

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one short sequence's layer input: the call itself is what costs
        {"name": "checkpoint_short", "op": "checkpoint", "rows": 16, "cols": 4096, "dtype": "bf16"},
        # the input of a linear layer for 16 sequences of 1024 tokens
        {"name": "checkpoint_long", "op": "checkpoint", "rows": 16384, "cols": 4096, "dtype": "bf16"},
        # an odd width and an odd count of rows, other gate, other type
        {"name": "gated_odd", "op": "gated", "rows": 1001, "cols": 2749, "dtype": "fp16", "act": "gelu"},
        # the MLP of a decoder layer, 8192 tokens
        {"name": "gated_large", "op": "gated", "rows": 8192, "cols": 11008, "dtype": "bf16", "act": "silu"},
        # a small projection (adapter, router) over one long sequence: few outputs, a long sum
        {"name": "wgrad_narrow", "op": "wgrad", "tokens": 16384, "n": 256, "k": 512, "dtype": "bf16"},
        # a batch cut to its real tokens, and a head with an odd number of outputs
        {"name": "wgrad_ragged", "op": "wgrad", "tokens": 2051, "n": 1001, "k": 4104, "dtype": "bf16"},
        # the down projection of a decoder layer, 8192 tokens
        {"name": "wgrad_large", "op": "wgrad", "tokens": 8192, "n": 4096, "k": 11008, "dtype": "bf16"},
        # a gradient rounded stochastically along its tokens, odd in both directions
        {"name": "quant4_across", "op": "quant4", "rows": 4097, "cols": 2749, "dtype": "bf16", "stochastic": True, "transpose": True},
        # the gradient of a decoder layer's MLP, rounded stochastically along its features
        {"name": "quant4_large", "op": "quant4", "rows": 8192, "cols": 11008, "dtype": "bf16", "stochastic": True, "transpose": False},
        # one token against the weights of an MLP projection
        {"name": "linear4_token", "op": "linear4", "rows": 1, "n": 11008, "k": 4096, "dtype": "bf16"},
        # a small ragged batch, odd output width
        {"name": "linear4_ragged", "op": "linear4", "rows": 333, "n": 1001, "k": 2080, "dtype": "bf16"},
        # the up projection of a decoder layer, 8192 tokens
        {"name": "linear4_large", "op": "linear4", "rows": 8192, "n": 11008, "k": 4096, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["checkpoint", "gated", "wgrad", "quant4", "linear4"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "checkpoint":
        return {"op": op, "rows": _log(rng, 1, 8192), "cols": _log(rng, 32, 8192), "dtype": dtype}
    if op == "gated":
        return {"op": op, "rows": _log(rng, 1, 4096), "cols": _log(rng, 32, 11008), "dtype": dtype,
                "act": rng.choice(["silu", "gelu", "gelu_tanh"])}
    if op == "quant4":
        return {"op": op, "rows": _log(rng, 1, 4096), "cols": _log(rng, 32, 11008), "dtype": dtype,
                "stochastic": rng.random() < 0.5, "transpose": rng.random() < 0.5}
    if op == "wgrad":
        return {"op": op, "tokens": _log(rng, 1, 8192), "n": _log(rng, 16, 4096), "k": _log(rng, 32, 8192), "dtype": dtype}
    return {"op": op, "rows": _log(rng, 1, 8192), "n": _log(rng, 16, 8192), "k": _log(rng, 32, 4096), "dtype": dtype}


# ----------------------------------------------------------------------------------------- inputs
def _normal(gen, rows, cols, scale):
    return torch.randn(rows, cols, generator=gen, device=DEV) * scale


def _activation(gen, rows, cols, dtype):
    """Activations as a decoder's blocks see them: normal, with a few channels an order of magnitude larger."""
    loud = 1.0 + 15.0 * (torch.rand(1, cols, generator=gen, device=DEV) > 0.99)
    return (_normal(gen, rows, cols, 1.0) * loud).to(dtype)


def _gradient(gen, rows, cols, dtype):
    """Gradients of a mean loss: small, of another size from token to token."""
    return (_normal(gen, rows, cols, 1e-3) * torch.exp(_normal(gen, rows, 1, 1.0))).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype, op = DTYPES[case["dtype"]], case["op"]
    s = {"case": dict(case)}
    if op == "checkpoint":
        s["x"] = _activation(gen, case["rows"], case["cols"], dtype)
    elif op == "gated":
        s["gate"] = _activation(gen, case["rows"], case["cols"], dtype)
        s["up"] = _activation(gen, case["rows"], case["cols"], dtype)
        s["grad_h"] = _gradient(gen, case["rows"], case["cols"], dtype)
    elif op == "wgrad":
        s["x"] = _activation(gen, case["tokens"], case["k"], dtype)
        s["grad_out"] = _gradient(gen, case["tokens"], case["n"], dtype)
    elif op == "quant4":
        s["x"] = _gradient(gen, case["rows"], case["cols"], dtype)
        s["seed"] = seed * 7919 + 1
    else:
        s["x"] = _activation(gen, case["rows"], case["k"], dtype)
        # the weights as a program keeps them: 4-bit codes, two to a byte, and their scales
        e, q = _mxfp4(_blocks(_normal(gen, case["n"], case["k"], 0.02)))
        s["w_codes"], s["w_scales"] = _pack4(q), _tile_scales(e)
    return s


# ------------------------------------------------------------------------------------ plain forms
def _pad(n, to):
    return -(-n // to) * to


def _blocks(x):
    """fp32, the columns filled up to whole blocks with zeros: (rows, blocks, 32)."""
    x = x.float()
    return torch.nn.functional.pad(x, (0, _pad(x.shape[1], 32) - x.shape[1])).view(x.shape[0], -1, 32)


def _power(e):
    """2^e as fp32, -126 <= e <= 127."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _mxint8(b):
    """Exponents and integers of blocks of finite values."""
    m, k = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (k - 1 + (m > 127 / 128).int()).clamp(-120, 127)
    return e, torch.round(b / _power(e - 6)).clamp(-127, 127)


def _mxfp4(b, draws=None):
    """Exponents and values on the grid of blocks of finite values; `draws`: 16-bit integers that round instead of nearest."""
    m, k = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (k - 3 + (m > 0.75).int()).clamp(-126, 126)
    y = b * _power(-e)
    a = y.abs().double()
    step = 0.5 + 0.5 * (a >= 2) + 1.0 * (a >= 4)
    t = a / step
    t = torch.round(t) if draws is None else torch.floor(t + draws.double() / 65536)
    return e, torch.copysign((t * step).clamp(max=6).float(), y)


def _pack4(q):
    """Codes of 4 bits (sign, two of exponent, one of mantissa), the even column in the low half of a byte."""
    a = q.abs()
    code = ((a * 2).int() - (a > 2).int() - (a > 3).int() * 1 - (a > 4).int() * 3) | (torch.signbit(q).int() << 3)
    code = code.view(q.shape[0], -1, 2)
    return (code[..., 0] | (code[..., 1] << 4)).to(torch.uint8)


def _tile_scales(e):
    """Scale bytes of (rows, blocks, 1) exponents in tiles of 128 rows x 4 blocks, each 32 x 4 x 4: byte
    (r % 32) * 16 + (r // 32) * 4 + block % 4 of a tile; rows and blocks beyond the last are 0."""
    s = (e[..., 0] + 127).to(torch.uint8)
    r, n = _pad(s.shape[0], 128), _pad(s.shape[1], 4)
    s = torch.nn.functional.pad(s, (0, n - s.shape[1], 0, r - s.shape[0]))
    return s.view(r // 128, 4, 32, n // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _untile(codes, scales, rows, cols):
    """fp32 values of 4-bit codes and tiled scales."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = grid[torch.stack((codes & 15, codes >> 4), -1).view(rows, -1).int()]
    e = scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows, : v.shape[1] // 32].int() - 127
    return (v.view(rows, -1, 32) * _power(e)[..., None]).view(rows, -1)[:, :cols]


def _round_of(c, keys):
    """One round of Philox4x32 on 32-bit words held in 64-bit integers."""
    low = 0xFFFFFFFF
    p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    return ((p1 >> 32) & low ^ c[1] ^ keys[0], p1 & low, (p0 >> 32) & low ^ c[3] ^ keys[1], p0 & low)


def _draws(seed, rows, cols, device):
    """The 16-bit draws of a (rows, cols) matrix, cols a multiple of 8: Philox4x32-10, key = seed, counter =
    (index // 8, tensor 0, step 0, stream 3); eight draws to a counter."""
    low = 0xFFFFFFFF
    keys = [((seed + r * 0x9E3779B9) & low, ((seed >> 32) + r * 0xBB67AE85) & low) for r in range(10)]
    i = torch.arange(rows * cols // 8, device=device, dtype=torch.int64)
    w = torch.stack(reduce(_round_of, keys, (i, torch.zeros_like(i), torch.zeros_like(i), torch.full_like(i, 3))), -1)
    return torch.stack((w & 0xFFFF, w >> 16), -1).view(rows, cols)


def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        p = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


def _read8(x):
    """The values that an 8-bit checkpoint of x stands for, fp32."""
    e, q = _mxint8(_blocks(x))
    return (q * _power(e - 6)).view(x.shape[0], -1)[:, : x.shape[1]]


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "checkpoint":
        return {"restored": _read8(s["x"]).to(s["x"].dtype)}
    if op == "gated":
        dtype = s["gate"].dtype
        h = _act(s["gate"].float(), case["act"])[0] * s["up"].float()
        a, d = _act(_read8(s["gate"]), case["act"])
        dh = s["grad_h"].float()
        return {"h": h.to(dtype), "grad_gate": (dh * _read8(s["up"]) * d).to(dtype), "grad_up": (dh * a).to(dtype)}
    if op == "wgrad":
        return {"grad_weight": (s["grad_out"].float().t() @ _read8(s["x"])).bfloat16()}
    if op == "quant4":
        x = s["x"].t() if case["transpose"] else s["x"]
        b = _blocks(x)
        draws = _draws(s["seed"], x.shape[0], b.shape[1] * 32, x.device).view(b.shape) if case["stochastic"] else None
        e, q = _mxfp4(b, draws)
        return {"values": (q * _power(e)).view(x.shape[0], -1)[:, : x.shape[1]].bfloat16()}
    e, q = _mxfp4(_blocks(s["x"]))
    x = (q * _power(e)).view(case["rows"], -1)[:, : case["k"]]
    return {"y": (x @ _untile(s["w_codes"], s["w_scales"], case["n"], case["k"]).t()).bfloat16()}


# ---------------------------------------------------------------------------------- the framework's
def _own(s):
    from ramtorch_b200 import microscaling as mx
    case, op = s["case"], s["case"]["op"]
    if op == "checkpoint":
        return {"restored": mx.quantize_mxint8(s["x"]).dequantize()}
    if op == "gated":
        h, gate8, up8 = mx.gated_act(s["gate"], s["up"], case["act"])
        grad_gate, grad_up = mx.gated_act_backward(s["grad_h"], gate8, up8, case["act"])
        return {"h": h, "grad_gate": grad_gate, "grad_up": grad_up}
    if op == "wgrad":
        return {"grad_weight": mx.weight_grad(s["grad_out"], mx.quantize_mxint8(s["x"]), dtype=torch.bfloat16)}
    if op == "quant4":
        q = mx.quantize_mxfp4(s["x"], transpose=case["transpose"], seed=s["seed"] if case["stochastic"] else None)
        return {"values": q.dequantize(torch.bfloat16)}
    w = mx.MxTensor("mxfp4", s["w_codes"], s["w_scales"], (case["n"], case["k"]), torch.bfloat16)
    return {"y": mx.mxfp4_matmul(mx.quantize_mxfp4(s["x"]), w, dtype=torch.bfloat16)}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------- the floor
def work(case):
    """Bytes: inputs and outputs once, and the 8- or 4-bit form once each way where a program keeps it between
    two calls (the checkpoint between forward and backward); flops of the products."""
    size, op = DTYPES[case["dtype"]].itemsize, case["op"]
    c8, c4 = 1 + 1 / 32, 0.5 + 1 / 32
    if op == "checkpoint":
        return {"bytes": case["rows"] * case["cols"] * (2 * size + 2 * c8), "flops": 0}
    if op == "gated":
        return {"bytes": case["rows"] * case["cols"] * (6 * size + 4 * c8), "flops": 0}
    if op == "quant4":
        return {"bytes": case["rows"] * case["cols"] * (size + 2 * c4 + 2), "flops": 0}
    if op == "wgrad":
        t, n, k = case["tokens"], case["n"], case["k"]
        return {"bytes": t * n * size + t * k * (size + 2 * c8) + 2 * n * k, "flops": 2 * t * n * k}
    m, n, k = case["rows"], case["n"], case["k"]
    return {"bytes": m * k * size + n * k * c4 + 2 * m * n, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------- the definition, 64 bits
def _two(e):
    """2^e, read from a table: the device's pow and exp2 are not exact, and ties hang on the last bit."""
    return torch.tensor([2.0 ** i for i in range(-300, 300)], dtype=torch.float64, device=e.device)[e.long() + 300]


def _exact_scale(b, top):
    """The exponent of the smallest power of two at which `top` times it is no less than the block's largest magnitude."""
    a = b.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(a > 0, a, torch.full_like(a, 1e-45)) / top))
    e = torch.where(a > top * _two(e), e + 1, e)      # the logarithm may be off by one step either way
    return torch.where(a <= top * _two(e - 1), e - 1, e)


def _exact8(x):
    b = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    p = _two(_exact_scale(b, 127).clamp(-126, 121))
    return (torch.round(b / p).clamp(-127, 127) * p).flatten(1)[:, : x.shape[1]]


def _exact4(x, draws=None):
    b = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % 32)).unflatten(1, (-1, 32))
    p = _two(_exact_scale(b, 6).clamp(-126, 126))
    y = b / p
    a = y.abs()
    step = _two(torch.frexp(a.clamp(min=1))[1] - 2)
    t = torch.round(a / step) if draws is None else torch.floor(a / step + draws.unflatten(1, (-1, 32)) * 2.0 ** -16)
    return (torch.sign(y) * torch.clamp(t * step, max=6) * p).flatten(1)[:, : x.shape[1]]


def _exact_act(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if act == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) * (2 * math.pi) ** -0.5
    z = 2 * (2 / math.pi) ** 0.5 * (g + 0.044715 * g * g * g)
    s = torch.sigmoid(z)
    return g * s, s + g * s * (1 - s) * 2 * (2 / math.pi) ** 0.5 * (1 + 0.134145 * g * g)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "checkpoint":
        return {"restored": _exact8(s["x"])}
    if op == "gated":
        g8, u8, dh = _exact8(s["gate"]), _exact8(s["up"]), s["grad_h"].double()
        a, d = _exact_act(g8, case["act"])
        return {"h": _exact_act(s["gate"].double(), case["act"])[0] * s["up"].double(), "grad_gate": dh * u8 * d, "grad_up": dh * a}
    if op == "wgrad":
        return {"grad_weight": s["grad_out"].double().t() @ _exact8(s["x"])}
    if op == "quant4":
        x = s["x"].t() if case["transpose"] else s["x"]
        wide = _pad(x.shape[1], 32)
        return {"values": _exact4(x, _draws(s["seed"], x.shape[0], wide, x.device).double() if case["stochastic"] else None)}
    grid = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12], dtype=torch.float64, device=DEV) / 2
    codes = torch.stack((s["w_codes"] % 16, s["w_codes"] // 16), -1).flatten(1).long()
    w = grid[codes % 8] * (1 - 2 * (codes // 8)).double()
    e = s["w_scales"].permute(0, 3, 2, 1, 4).flatten(0, 2).flatten(1)[: w.shape[0], : w.shape[1] // 32].double() - 127
    w = (w.unflatten(1, (-1, 32)) * _two(e)[..., None]).flatten(1)[:, : case["k"]]
    return {"y": _exact4(s["x"]) @ w.t()}
