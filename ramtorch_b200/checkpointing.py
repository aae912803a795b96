"""Layers that keep what their backward pass needs in 8 bits.

    y = linear(x, weight, bias)                     # keeps x as MXINT8, weight by reference
    h = gated_act(gate, up, "silu")                 # keeps gate and up as MXINT8
    y = linear(x, weight, product="mxfp4", seed=7, step=t)   # 4-bit products forward and for grad_x

Both take part in autograd like their torch counterparts.  The weight gradient comes straight from
the 8-bit codes (``microscaling.weight_grad``); for a CPU-resident ``is_ramtorch`` parameter it is added to
``weight.rt_device_grad`` in HBM, where ``AdamW.step`` takes it (``helpers.accumulate_weight_grad``).
"""
from __future__ import annotations

import torch

from . import helpers
from . import microscaling as mx


def _rowed(t: torch.Tensor) -> torch.Tensor:
    """`t` itself where its rows are evenly spaced runs of memory, else a copy that is."""
    try:
        mx._rows(t, "t")
        return t
    except ValueError:
        return t.contiguous()


def _product(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """``a @ b`` in their own type, also where autocast is on when the backward pass is called."""
    if torch.is_autocast_enabled("cuda"):
        with torch.autocast("cuda", enabled=False):
            return a @ b
    return a @ b


def _flagged(p: torch.Tensor | None):
    """`p` if it is an ``is_ramtorch`` parameter itself, else None.  What was made of a parameter (a cast, a slice) has to
    pass its gradient on through autograd."""
    return p if p is not None and p.is_leaf and getattr(p, "is_ramtorch", False) else None


def _asked(ctx, i: int):
    """Whether this backward pass wants the gradient of tensor input `i`: ``"added"`` to the parameter, ``"returned"``
    (``torch.autograd.grad`` for the parameter itself), or None (``autograd.grad`` or ``backward(inputs=...)`` for others)."""
    node = ctx.next_functions[i][0]
    if node is None:
        return None
    try:
        return "added" if torch._C._will_engine_execute_node(node) else None
    except RuntimeError:                # a leaf whose gradient autograd.grad captures
        return "returned"


def _ready_for_caller(held: torch.Tensor) -> None:
    """What autograd does for ``.grad``: when this backward pass is over, the stream it was called on is ordered after the stream
    that `held` was written on (the forward pass's)."""
    index = held.get_device()
    written_on = mx.N.stream_ptr(index)

    def order():
        if mx.N.stream_ptr(index) != written_on:
            caller = torch.cuda.current_stream(index)
            caller.wait_stream(torch.cuda.ExternalStream(written_on, index))
            held.record_stream(caller)
    torch.autograd.Variable._execution_engine.queue_callback(order)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, product, seed, tensor_id, step):
        x = _rowed(x)
        w = weight if weight.is_cuda else weight.detach().to(x.device, non_blocking=True)
        if product == "mxfp4":
            y = mx.mxfp4_matmul(mx.quantize_mxfp4(x), mx.quantize_mxfp4(_rowed(w)), dtype=x.dtype)
        else:
            y = _product(x, w.to(x.dtype).t())
        if bias is not None:
            y = y + bias.to(x.device, x.dtype)
        keep = mx.quantize_mxint8(x) if ctx.needs_input_grad[1] else None
        ctx.save_for_backward(*((keep.codes, keep.scales) if keep is not None else (None, None)), weight)
        # the parameters themselves: what is saved comes back as another tensor after recomputation or through saved-tensor hooks
        ctx.flagged = _flagged(weight), _flagged(bias)
        ctx.x_shape, ctx.x_dtype, ctx.args = tuple(x.shape), x.dtype, (product, seed, tensor_id, step)
        ctx.bias_like = None if bias is None else {"dtype": bias.dtype, "device": bias.device}
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        codes, scales, weight = ctx.saved_tensors
        product, seed, tensor_id, step = ctx.args
        grad = _rowed(grad)
        gx = gw = gb = None
        if ctx.needs_input_grad[0]:
            w = weight if weight.is_cuda else weight.detach().to(grad.device, non_blocking=True)
            if product == "mxfp4":
                d4 = mx.quantize_mxfp4(grad, seed=seed, tensor_id=tensor_id, step=step)
                gx = mx.mxfp4_matmul(d4, mx.quantize_mxfp4(_rowed(w), transpose=True), dtype=ctx.x_dtype)
            else:
                gx = _product(grad, w.to(grad.dtype))
        if codes is not None and (asked := _asked(ctx, 1)):
            x8 = mx.MxTensor("mxint8", codes, scales, ctx.x_shape, ctx.x_dtype)
            if asked == "added" and ctx.flagged[0] is not None and not weight.is_cuda:
                _ready_for_caller(helpers.accumulate_weight_grad(ctx.flagged[0], grad, x8))
            else:
                gw = mx.weight_grad(grad, x8, dtype=weight.dtype)
                if asked == "added":
                    gw = helpers.invoke_ramtorch_hooks(ctx.flagged[0], gw)
                gw = gw.to(weight.device)
        if ctx.bias_like is not None and ctx.needs_input_grad[2] and (asked := _asked(ctx, 2)):
            gb = grad.reshape(mx._split(grad.shape)).sum(0, dtype=torch.float32).to(ctx.bias_like["dtype"])
            if asked == "added":
                gb = helpers.invoke_ramtorch_hooks(ctx.flagged[1], gb)
            gb = gb.to(ctx.bias_like["device"])
        return gx, gw, gb, None, None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, product: str | None = None,
           seed: int | None = None, tensor_id: int = 0, step: int = 0) -> torch.Tensor:
    """``x @ weight.T + bias`` that keeps ``x`` in MXINT8 for the weight gradient.

    ``product=None``: the product and ``grad_x`` in x's own type.  ``product="mxfp4"``: both in 4-bit
    microscaled floating point; the incoming gradient is rounded to 4 bits stochastically when
    ``seed`` is given (Philox draws ``(seed, tensor_id, step)``: pass another ``tensor_id`` for each layer
    and count ``step`` with every call, micro-batches too; inside a CUDA graph each replay draws the same), else to
    nearest.  The weight gradient always takes the gradient unrounded.

    Every call keeps a copy of its own: projections of one input (q, k, v; gate, up) keep it once as one call with their
    weights stacked, and once each as several.

    A weight in host memory is copied to x's device for the product, asynchronously where it is pinned.  The gradient of an ``is_ramtorch``
    parameter stays there as ``weight.rt_device_grad``; that of any other host weight (a leaf without the
    flag, a cast or a slice of a parameter) goes to host memory through autograd.  ``AdamW.step`` takes
    ``rt_device_grad`` in place of ``grad`` and ``AdamW.zero_grad`` clears it: a flagged parameter should get all of its gradient
    from one of the two, and ``Module.zero_grad``, ``clip_grad_norm_`` and ``GradScaler``, which know ``grad`` alone, want it unflagged.
    ZeRO-2 hooks of flagged parameters see the fresh gradient, of a weight and of a bias, before it is added anywhere.

    Under ``torch.autocast`` x is cast to its type, and y has that type; weight and bias may be of any of the three types,
    and their gradients are formed in their own."""
    if product not in (None, "mxfp4"):
        raise ValueError(f"product must be None or 'mxfp4', not {product!r}")
    if product and seed is not None:
        mx._check_draws(tensor_id, step)
    if weight.dim() != 2 or x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must have shape {tuple(weight.shape[:1])}, not {tuple(bias.shape)}")
    autocast = torch.is_autocast_enabled("cuda")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and (t.dtype not in mx.N.DTYPE_CODE if autocast else t.dtype != x.dtype):
            raise ValueError(f"x is {x.dtype} and {name} {t.dtype}")
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor: ramtorch_b200 has no CPU implementation")
    if autocast and x.dtype in mx.N.DTYPE_CODE:
        x = x.to(torch.get_autocast_dtype("cuda"))
    return _Linear.apply(x, weight, bias, product, seed, tensor_id, step)


class _GatedAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, act):
        h, g8, u8 = mx.gated_act(_rowed(gate), _rowed(up), act)
        ctx.save_for_backward(g8.codes, g8.scales, u8.codes, u8.scales)
        ctx.shape, ctx.dtype, ctx.act = tuple(gate.shape), gate.dtype, act
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        gc, gs, uc, us = ctx.saved_tensors
        g8 = mx.MxTensor("mxint8", gc, gs, ctx.shape, ctx.dtype)
        u8 = mx.MxTensor("mxint8", uc, us, ctx.shape, ctx.dtype)
        dgate, dup = mx.gated_act_backward(_rowed(grad), g8, u8, ctx.act)
        return dgate, dup, None


def gated_act(gate: torch.Tensor, up: torch.Tensor, act: str = "silu") -> torch.Tensor:
    """``act(gate) * up`` that keeps its two inputs in MXINT8 (``act``: ``"silu"``, ``"gelu"``, ``"gelu_tanh"``)."""
    return _GatedAct.apply(gate, up, act)
