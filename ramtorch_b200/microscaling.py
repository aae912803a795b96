"""Microscaled block formats: 8-bit activation checkpoints and 4-bit floating point.

32 consecutive values of a row share one power-of-two scale (MXINT8 and MXFP4 of the OCP microscaling
specification; exact rules and layouts in ``include/rt_b200.h``).  Every stored value is exactly a
bf16 number and every rounding is defined bit for bit.

    x8 = quantize_mxint8(x)                      # 1.03 bytes per value instead of 2 or 4
    x  = x8.dequantize()
    dw = weight_grad(grad_out, x8)               # grad_out^T @ x8, straight from the codes
    h, g8, u8 = gated_act(gate, up, "silu")      # SwiGLU, and what its backward needs, in 8 bits
    dgate, dup = gated_act_backward(grad_h, g8, u8, "silu")
    w4 = quantize_mxfp4(w)                       # 0.53 bytes per value
    y  = mxfp4_matmul(quantize_mxfp4(x), w4)     # x @ w^T on the 4-bit tensor cores
    d4 = quantize_mxfp4(grad, seed=7, step=t)    # stochastic rounding from the framework's Philox streams

Functions that record for autograd are in ``ramtorch_b200.checkpointing``.  All calls enqueue on the
current stream of the inputs' device and allocate only through torch, so they can be captured into
CUDA graphs (after one uncaptured call that loads the kernels).  ``seed``, ``tensor_id`` and ``step`` are values
of the call: every replay of a captured stochastic rounding draws the same bits.  Rounding that is to be
unbiased over the steps of a run has to be called anew, outside the graph, with a new ``step``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N

BLOCK = 32
_FORMATS = {"mxint8": N.MXINT8, "mxfp4": N.MXFP4}
_CODES_DTYPE = {"mxint8": torch.int8, "mxfp4": torch.uint8}


_fast = None        # the C++ host side: a module, or False where it is not built


def _helper():
    """``_mxcall.so`` with the library's entry points handed to it, or ``False``."""
    global _fast
    if _fast is None:
        try:
            from . import _mxcall
        except ImportError:
            _fast = False
        else:
            L = N.lib()
            _mxcall.init({name: ctypes.cast(getattr(L, name), ctypes.c_void_p).value
                          for name in ("rt_last_error", "rt_mx_quantize", "rt_mx_dequantize", "rt_mx_gated_act", "rt_mx_gated_act_backward",
                                       "rt_mx_weight_grad_workspace", "rt_mx_weight_grad", "rt_mxfp4_matmul")})
            _fast = _mxcall
    return _fast


def _pad(n: int, to: int) -> int:
    return (n + to - 1) // to * to


def _layout(fmt: str, rows: int, cols: int):
    """Shapes of codes and scales."""
    wide = _pad(cols, BLOCK)
    blocks = wide // BLOCK
    if fmt == "mxint8":
        return (rows, wide), (rows, _pad(blocks, 4))
    return (rows, wide // 2), (_pad(rows, 128) // 128, _pad(blocks, 4) // 4, 32, 4, 4)


class MxTensor:
    """A tensor in a microscaled format: ``codes`` and ``scales`` on the GPU, the ``shape`` it stands for
    (blocks run along the last dimension) and the ``dtype`` that ``dequantize`` gives by default.

    ``codes``: (rows, padded columns) int8 for ``"mxint8"``, (rows, padded columns / 2) uint8 for
    ``"mxfp4"``, two codes to a byte.  ``scales``: uint8, (rows, blocks padded to 4) for ``"mxint8"``;
    (row tiles of 128, block tiles of 4, 32, 4, 4) for ``"mxfp4"``, where scale (r, b) is at
    ``[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]``.  What fills up the last block of a row, and the
    scales of rows and blocks that do not exist, are 0: products read them."""

    __slots__ = ("format", "codes", "scales", "shape", "dtype")

    def __init__(self, format: str, codes: torch.Tensor, scales: torch.Tensor, shape, dtype=torch.bfloat16):
        if format not in _FORMATS:
            raise ValueError(f"format must be 'mxint8' or 'mxfp4', not {format!r}")
        shape = tuple(shape)
        if not shape or min(shape) < 0:
            raise ValueError("shape needs at least one dimension and no negative sizes")
        if dtype not in N.DTYPE_CODE:
            raise ValueError(f"unsupported dtype {dtype} (bf16, fp32, fp16 only)")
        if not (codes.is_cuda and scales.is_cuda):
            raise RuntimeError("codes and scales must be CUDA tensors: ramtorch_b200 has no CPU implementation")
        rows, cols = _split(shape)
        want_codes, want_scales = _layout(format, rows, cols)
        if codes.dtype != _CODES_DTYPE[format] or codes.shape != want_codes or not codes.is_contiguous():
            raise ValueError(f"codes must be a contiguous {_CODES_DTYPE[format]} tensor of shape {want_codes}")
        if scales.dtype != torch.uint8 or scales.shape != want_scales or not scales.is_contiguous():
            raise ValueError(f"scales must be a contiguous torch.uint8 tensor of shape {want_scales}")
        if (codes.data_ptr() | scales.data_ptr()) & 15:
            raise ValueError("codes and scales must start on 16-byte boundaries")
        if codes.get_device() != scales.get_device():
            raise ValueError("codes and scales are on different devices")
        self.format, self.codes, self.scales, self.shape, self.dtype = format, codes, scales, shape, dtype

    @classmethod
    def _of(cls, fmt, codes, scales, shape, dtype):
        """From arrays that this module laid out itself."""
        t = object.__new__(cls)
        t.format, t.codes, t.scales, t.shape, t.dtype = fmt, codes, scales, shape, dtype
        return t

    @classmethod
    def _new(cls, fmt, shape, rows, cols, dtype, device):
        codes, scales = _layout(fmt, rows, cols)
        return cls._of(fmt, torch.empty(codes, dtype=_CODES_DTYPE[fmt], device=device),
                       torch.empty(scales, dtype=torch.uint8, device=device), shape, dtype)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def __repr__(self):
        return f"MxTensor({self.format}, shape={self.shape}, dtype={self.dtype}, device={self.device})"

    def record_stream(self, stream) -> None:
        """``torch.Tensor.record_stream`` of both arrays."""
        self.codes.record_stream(stream)
        self.scales.record_stream(stream)

    def dequantize(self, dtype=None, *, out: torch.Tensor | None = None) -> torch.Tensor:
        """The values as ``dtype`` (default: the source's)."""
        rows, cols = _split(self.shape)
        if out is None:
            dtype = dtype or self.dtype
            if dtype not in N.DTYPE_CODE:
                raise ValueError(f"unsupported dtype {dtype} (bf16, fp32, fp16 only)")
            fast = _fast or _helper()
            if fast:
                return fast.dequantize(_FORMATS[self.format], self.codes, self.scales, rows, cols, self.shape, N.DTYPE_CODE[dtype])
            out = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
            ld = cols
        else:
            if dtype is not None and out.dtype != dtype:
                raise ValueError("out and dtype disagree")
            if tuple(out.shape) != self.shape or out.device != self.codes.device:
                raise ValueError("out has another shape or device")
            ld = _rows(out, "out")[2]
            _apart(out, self)
        with _on(out.device):
            N.check(N.lib().rt_mx_dequantize(_FORMATS[self.format], self.codes.data_ptr(), self.scales.data_ptr(), rows, cols,
                                             out.data_ptr(), N.DTYPE_CODE[out.dtype], ld, N.stream_ptr(out.device.index)),
                    "rt_mx_dequantize")
        return out


class _Stay:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_STAY = _Stay()


def _on(device):
    """Make `device` current for a launch; free when it already is."""
    return _STAY if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _split(shape):
    """(rows, cols) of a shape whose leading dimensions count as rows."""
    rows = 1
    for n in shape[:-1]:
        rows *= n
    return rows, shape[-1]


def _rows(x: torch.Tensor, name: str):
    """(rows, cols, row stride in elements) of x with its leading dimensions taken as rows."""
    if not x.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: ramtorch_b200 has no CPU implementation")
    if x.dtype not in N.DTYPE_CODE:
        raise ValueError(f"{name}: unsupported dtype {x.dtype} (bf16, fp32, fp16 only)")
    if x.dim() == 0:
        raise ValueError(f"{name} needs at least one dimension")
    rows, cols = _split(x.shape)
    if x.is_contiguous():
        return rows, cols, cols
    if rows == 0 or cols == 0:
        return rows, cols, cols
    if cols > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name}: the values of a row must be consecutive")
    ld = None                        # leading dimensions have to step evenly
    for size, stride in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if size == 1:
            continue
        if ld is None:
            ld, step = stride, stride * size
        elif stride != step:
            raise ValueError(f"{name}: rows must be evenly spaced")
        else:
            step = stride * size
    ld = cols if ld is None else ld
    if ld < cols:
        raise ValueError(f"{name}: rows overlap")
    return rows, cols, ld


def _span(t):
    """First byte of a tensor, and one past its last."""
    if t.numel() == 0:
        return 0, 0
    first = t.data_ptr()
    return first, first + (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) * t.element_size()


def _apart(out, *inputs):
    """The kernels read ahead of what they write: an output must not lie where an input does."""
    a, b = _span(out)
    for t in inputs:
        for part in ((t.codes, t.scales) if isinstance(t, MxTensor) else (t,)):
            c, d = _span(part)
            if a < d and c < b:
                raise ValueError("out overlaps an input")


def _same_place(t, device, name):
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")


def _check_draws(tensor_id, step):
    if not (0 <= tensor_id < 2**32 and 0 <= step < 2**32):
        raise ValueError("tensor_id and step must fit 32 bits")


def _quantize(x, fmt, transpose, seed, tensor_id, step):
    rows, cols, ld = _rows(x, "x")
    if transpose and x.dim() != 2:
        raise ValueError("transpose needs a matrix")
    shape = (cols, rows) if transpose else tuple(x.shape)
    if seed is not None:
        _check_draws(tensor_id, step)
    fast = _fast or _helper()
    if fast:
        codes, scales = fast.quantize(x, rows, cols, ld, _FORMATS[fmt], transpose, seed is not None, (seed or 0) & (2**64 - 1), tensor_id, step)
        return MxTensor._of(fmt, codes, scales, shape, x.dtype)
    q = MxTensor._new(fmt, shape, cols if transpose else rows, rows if transpose else cols, x.dtype, x.device)
    draws = None if seed is None else ctypes.byref(N.MxDraws(seed & (2**64 - 1), tensor_id, step))
    with _on(x.device):
        N.check(N.lib().rt_mx_quantize(x.data_ptr(), N.DTYPE_CODE[x.dtype], rows, cols, ld, _FORMATS[fmt], transpose,
                                       q.codes.data_ptr(), q.scales.data_ptr(), draws, N.stream_ptr(x.device.index)), "rt_mx_quantize")
    return q


def quantize_mxint8(x: torch.Tensor) -> MxTensor:
    """``x`` (bf16, fp32 or fp16; leading dimensions count as rows, rows may be strided) in MXINT8, rounded
    to nearest: at most half of 2^-6 of the block's scale off."""
    return _quantize(x, "mxint8", False, None, 0, 0)


def quantize_mxfp4(x: torch.Tensor, *, transpose: bool = False, seed: int | None = None, tensor_id: int = 0,
                   step: int = 0) -> MxTensor:
    """``x`` in MXFP4, rounded to nearest, or with ``seed`` stochastically with the Philox draws
    ``(seed, tensor_id, step)``: unbiased, the same bits on every run.  ``transpose=True`` quantises
    ``x.T`` of a matrix, in blocks along x's rows, without forming it."""
    return _quantize(x, "mxfp4", bool(transpose), seed, tensor_id, step)


def mxfp4_matmul(a: MxTensor, b: MxTensor, *, dtype=None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ b.T`` of two MXFP4 tensors, ``a`` (..., k) and ``b`` (n, k): fp32 sums, rounded once to
    ``dtype`` (default: a's)."""
    for t, name in ((a, "a"), (b, "b")):
        if not isinstance(t, MxTensor) or t.format != "mxfp4":
            raise ValueError(f"{name} must be an mxfp4 MxTensor")
    if len(b.shape) != 2:
        raise ValueError("b must be a matrix")
    (m, k), (n, kb) = _split(a.shape), b.shape
    if k != kb:
        raise ValueError(f"a has {k} columns and b {kb}")
    _same_place(b, a.device, "b")
    _watched.setdefault(a.device.index, 0)
    shape = a.shape[:-1] + (n,)
    if out is None:
        dtype = _out_dtype(dtype or a.dtype)
        fast = _fast or _helper()
        if fast:
            return fast.matmul(a.codes, a.scales, b.codes, b.scales, m, n, k, shape, N.DTYPE_CODE[dtype])
        out = torch.empty(shape, dtype=dtype, device=a.device)
        ld = n
    else:
        ld = _check_out(out, shape, dtype, a.device)
        _apart(out, a, b)
    with _on(a.device):
        N.check(N.lib().rt_mxfp4_matmul(a.codes.data_ptr(), a.scales.data_ptr(), b.codes.data_ptr(), b.scales.data_ptr(), m, n, k,
                                        out.data_ptr(), N.DTYPE_CODE[out.dtype], ld, N.stream_ptr(a.device.index)),
                "rt_mxfp4_matmul")
    return out


_watched: dict = {}        # devices that products ran on -> waits that had run out there when it was last asked


def check_faults(device=None) -> None:
    """Raise ``RuntimeError`` if a wait inside a product's kernel (:func:`mxfp4_matmul`, :func:`weight_grad`) has run out since
    the last look, on `device` or on every device that had products.  Each wait is bounded by two seconds, so that a fault ends
    the kernel instead of hanging the GPU; what such a call did not form holds NaN.  Waits for the device.
    ``AdamW.step`` looks by itself where it waits anyway (``sync=True``)."""
    if device is None:
        asked = list(_watched)
    else:
        index = device if isinstance(device, int) else torch.device(device).index
        asked = [torch.cuda.current_device() if index is None else index]
    for index in asked:
        count = ctypes.c_uint32()
        with _on(torch.device("cuda", index)):
            N.check(N.lib().rt_mx_wait_faults(ctypes.byref(count)), "rt_mx_wait_faults")
        new, _watched[index] = count.value - _watched.get(index, 0), count.value
        if new:
            raise RuntimeError(f"{new} wait(s) inside the tensor-core kernels ran out on cuda:{index}: results of calls since the last look hold NaN")


def _out_dtype(dtype):
    if dtype not in N.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {dtype} (bf16, fp32, fp16 only)")
    return dtype


def _check_out(out, shape, dtype, device):
    if dtype is not None and out.dtype != dtype:
        raise ValueError("out and dtype disagree")
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"out must have shape {tuple(shape)}")
    _same_place(out, device, "out")
    return _rows(out, "out")[2]


def weight_grad(grad_out: torch.Tensor, x8: MxTensor, *, dtype=None, out: torch.Tensor | None = None,
                accumulate: bool = False) -> torch.Tensor:
    """The weight gradient of ``y = x @ w.T`` from an 8-bit checkpoint of ``x``: ``grad_out.T @ x8``, leading
    dimensions taken as tokens.  The 8-bit values enter the product exactly, sums are fp32, rounded
    once to ``dtype`` (default: grad_out's).  ``accumulate=True`` adds to ``out`` before that rounding.
    The sums are the tensor core's, which cuts what does not fit: an fp32 result of normal data is 3e-6 off at 8192 tokens
    (relative norm; as a bf16 matrix product with fp32 results is), a 16-bit result by its rounding alone."""
    if not isinstance(x8, MxTensor) or x8.format != "mxint8":
        raise ValueError("x8 must be an mxint8 MxTensor")
    tokens, n, ld = _rows(grad_out, "grad_out")
    rows, k = _split(x8.shape)
    if rows != tokens:
        raise ValueError(f"grad_out has {tokens} tokens and x8 {rows}")
    _same_place(x8, grad_out.device, "x8")
    _watched.setdefault(grad_out.device.index, 0)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        dtype, ld_out = _out_dtype(dtype or grad_out.dtype), k
    else:
        ld_out = _check_out(out, (n, k), dtype, grad_out.device)
        _apart(out, grad_out, x8)
        dtype = out.dtype
    fast = _fast or _helper()
    if fast:
        return fast.weight_grad(grad_out, ld, x8.codes, x8.scales, tokens, n, k, out, ld_out, N.DTYPE_CODE[dtype], accumulate)
    if out is None:
        out = torch.empty((n, k), dtype=dtype, device=grad_out.device)
    L, code, g = N.lib(), N.DTYPE_CODE[grad_out.dtype], grad_out.data_ptr()
    with _on(grad_out.device):
        need = L.rt_mx_weight_grad_workspace(g, code, ld, tokens, n, k)
        if need < 0:
            N.check(int(need), "rt_mx_weight_grad_workspace")
        space = torch.empty(need, dtype=torch.uint8, device=grad_out.device) if need else None
        N.check(L.rt_mx_weight_grad(g, code, ld, x8.codes.data_ptr(), x8.scales.data_ptr(), tokens, n, k, out.data_ptr(),
                                    N.DTYPE_CODE[out.dtype], ld_out, accumulate, None if space is None else space.data_ptr(),
                                    need, N.stream_ptr(grad_out.device.index)), "rt_mx_weight_grad")
    return out


def _act_code(act):
    try:
        return N.ACT_CODE[act]
    except KeyError:
        raise ValueError(f"act must be one of {sorted(N.ACT_CODE)}, not {act!r}") from None


def gated_act(gate: torch.Tensor, up: torch.Tensor, act: str = "silu"):
    """``(act(gate) * up, gate8, up8)``: the gated activation from the exact inputs, and both inputs in
    MXINT8 for :func:`gated_act_backward`, in one pass.  ``act``: ``"silu"``, ``"gelu"`` or ``"gelu_tanh"``.
    Rows may be strided: ``proj.chunk(2, -1)`` needs no copy."""
    code = _act_code(act)
    rows, cols, ld_gate = _rows(gate, "gate")
    _, _, ld_up = _rows(up, "up")
    if up.shape != gate.shape or up.dtype != gate.dtype:
        raise ValueError("gate and up differ in shape or dtype")
    _same_place(up, gate.device, "up")
    shape, device = tuple(gate.shape), gate.device
    fast = _fast or _helper()
    if fast:
        h, gc, gs, uc, us = fast.gated_act(gate, ld_gate, up, ld_up, rows, cols, code)
        return h, MxTensor._of("mxint8", gc, gs, shape, gate.dtype), MxTensor._of("mxint8", uc, us, shape, gate.dtype)
    h = torch.empty(shape, dtype=gate.dtype, device=device)
    g8 = MxTensor._new("mxint8", shape, rows, cols, gate.dtype, device)
    u8 = MxTensor._new("mxint8", shape, rows, cols, gate.dtype, device)
    with _on(device):
        N.check(N.lib().rt_mx_gated_act(gate.data_ptr(), ld_gate, up.data_ptr(), ld_up, N.DTYPE_CODE[gate.dtype], rows, cols, code,
                                        h.data_ptr(), cols, g8.codes.data_ptr(), g8.scales.data_ptr(), u8.codes.data_ptr(),
                                        u8.scales.data_ptr(), N.stream_ptr(device.index)), "rt_mx_gated_act")
    return h, g8, u8


def gated_act_backward(grad_h: torch.Tensor, gate8: MxTensor, up8: MxTensor, act: str = "silu", *, out=None):
    """``(grad_gate, grad_up)`` of :func:`gated_act` from what it kept: ``grad_h * up8 * act'(gate8)`` and
    ``grad_h * act(gate8)``.  ``out``: a pair of tensors to write to, e.g. the halves of one gradient; as with
    every ``out`` here, not where an input lies."""
    code = _act_code(act)
    rows, cols, ld = _rows(grad_h, "grad_h")
    for t, name in ((gate8, "gate8"), (up8, "up8")):
        if not isinstance(t, MxTensor) or t.format != "mxint8":
            raise ValueError(f"{name} must be an mxint8 MxTensor")
        if t.shape != tuple(grad_h.shape):
            raise ValueError(f"grad_h and {name} differ in shape")
        _same_place(t, grad_h.device, name)
    fast = out is None and (_fast or _helper())
    if fast:
        return fast.gated_act_backward(grad_h, ld, rows, cols, code, gate8.codes, gate8.scales, up8.codes, up8.scales)
    if out is None:
        dgate, dup = torch.empty_like(grad_h, memory_format=torch.contiguous_format), torch.empty_like(grad_h, memory_format=torch.contiguous_format)
        ld_gate = ld_up = cols
    else:
        dgate, dup = out
        ld_gate, ld_up = (_check_out(t, grad_h.shape, grad_h.dtype, grad_h.device) for t in (dgate, dup))
        for t in (dgate, dup):
            _apart(t, grad_h, gate8, up8)
        (a, b), (c, d) = _span(dgate), _span(dup)
        if a < d and c < b:              # two tensors whose rows take turns, as the halves of one gradient do
            off = abs(a - c) // dgate.element_size() % max(ld_gate, 1)
            if ld_gate != ld_up or not cols <= off <= ld_gate - cols:
                raise ValueError("the two outputs overlap")
    with _on(grad_h.device):
        N.check(N.lib().rt_mx_gated_act_backward(grad_h.data_ptr(), ld, N.DTYPE_CODE[grad_h.dtype], rows, cols, code,
                                                 gate8.codes.data_ptr(), gate8.scales.data_ptr(), up8.codes.data_ptr(),
                                                 up8.scales.data_ptr(), dgate.data_ptr(), ld_gate, dup.data_ptr(), ld_up,
                                                 N.stream_ptr(grad_h.device.index)), "rt_mx_gated_act_backward")
    return dgate, dup
