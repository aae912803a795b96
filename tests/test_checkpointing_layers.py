"""The layers of ramtorch_b200.checkpointing as training programs call them: host weights of every kind, recomputation,
ZeRO-2 hooks, automatic mixed precision, and what they refuse."""
import numpy as np
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from ramtorch_b200 import checkpointing as ck
from ramtorch_b200 import helpers
from ramtorch_b200 import microscaling as mx

gpu = pytest.mark.gpu
DEV = "cuda"
T, N, K = 33, 40, 72


def np64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def randn(*shape, seed, dtype=torch.bfloat16, device=DEV):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(device=device, dtype=dtype)


def held(p):
    return p.__dict__.get(helpers.DEVICE_GRAD_ATTR)


def host_parameter(seed=1, flagged=True, dtype=torch.bfloat16, shape=(N, K)):
    p = torch.nn.Parameter(randn(*shape, seed=seed, dtype=dtype, device="cpu").mul_(0.1).pin_memory())
    if flagged:
        p.is_ramtorch = True
    return p


def dw_of(x, g, dtype=torch.bfloat16):
    return mx.weight_grad(g, mx.quantize_mxint8(x), dtype=dtype)


# ------------------------------------------------------------------------------------- host weights
@gpu
@pytest.mark.parametrize("flagged", [False, True])
def test_a_cast_or_a_part_of_a_host_parameter_gets_its_gradient(flagged):
    """What autograd made of a parameter hands the gradient on to the parameter."""
    x, g = randn(T, K, seed=2), randn(T, N, seed=3)
    master = host_parameter(flagged=flagged, dtype=torch.float32)
    ck.linear(x, master.bfloat16()).backward(g)
    want = dw_of(x, g)
    assert held(master) is None and torch.equal(master.grad, want.float().cpu())
    both = host_parameter(flagged=flagged, shape=(2 * N, K))
    part = both[N:]
    part.is_ramtorch = True                  # a flag on what is no leaf changes nothing
    ck.linear(x, part).backward(g)
    assert held(both) is None and held(part) is None
    assert torch.equal(both.grad[N:], want.cpu()) and (both.grad[:N] == 0).all()


@gpu
def test_a_host_leaf_without_the_flag_gets_an_ordinary_gradient():
    w = host_parameter(flagged=False)
    xs, gs = [randn(T, K, seed=s) for s in (2, 3)], [randn(T, N, seed=s) for s in (4, 5)]
    ck.linear(xs[0], w).backward(gs[0])
    assert held(w) is None and torch.equal(w.grad, dw_of(xs[0], gs[0]).cpu())
    ck.linear(xs[1], w).backward(gs[1])
    assert torch.equal(w.grad, dw_of(xs[0], gs[0]).cpu() + dw_of(xs[1], gs[1]).cpu())
    got, = torch.autograd.grad(ck.linear(xs[0], w), (w,), gs[0])
    assert torch.equal(got, dw_of(xs[0], gs[0]).cpu())
    before = w.detach().clone()
    torch.optim.SGD([w], lr=1.0).step()
    assert torch.equal(w.detach(), before - w.grad)


@gpu
@pytest.mark.parametrize("way", ["recomputed", "recomputed, reentrant", "saved on the host"])
def test_a_host_parameter_keeps_its_gradient_when_saved_tensors_are_packed(way):
    """Recomputation and saved-tensor hooks hand other tensors to the backward pass than the forward saved."""
    w, x, g = host_parameter(), randn(T, K, seed=2).requires_grad_(), randn(T, N, seed=3)
    if way == "saved on the host":
        with torch.autograd.graph.save_on_cpu(pin_memory=True):
            y = ck.linear(x, w)
    else:
        y = checkpoint(lambda a: ck.linear(a, w), x, use_reentrant="reentrant" in way)
    y.backward(g)
    assert torch.equal(held(w), dw_of(x, g)) and w.grad is None
    plain, = torch.autograd.grad(ck.linear(x, w), (x,), g)
    assert torch.equal(x.grad, plain)


@gpu
def test_a_held_gradient_in_any_order_of_memory_is_added_to():
    """A gradient that another producer left on the parameter, its rows not runs of memory."""
    w, x, g = host_parameter(), randn(T, K, seed=2), randn(T, N, seed=3)
    first = randn(K, N, seed=4).t()
    helpers.accumulate_device_grad(w, first.clone())
    assert not held(w).is_contiguous()
    want = first + dw_of(x, g)
    ck.linear(x, w).backward(g)
    assert torch.equal(held(w), want)


# -------------------------------------------------------------------------------------- ZeRO-2 hooks
@gpu
def test_zero2_hooks_see_the_gradient_of_a_bias_and_of_a_weight_in_hbm():
    """The hook dict of a flagged parameter runs on every fresh gradient: autograd itself knows nothing of it."""
    w, b = host_parameter(), torch.nn.Parameter(randn(N, seed=9, device="cpu"))
    b.is_ramtorch = True
    seen = []
    helpers.register_ramtorch_hook(b, lambda t: seen.append(t.clone()) or t * 4, helpers.ZERO2_HOOK_NAME)
    x, gs = randn(T, K, seed=2), [randn(T, N, seed=s) for s in (4, 5)]
    for g in gs:
        ck.linear(x, w, b).backward(g)
    assert [t.is_cuda for t in seen] == [True, True]
    for s, g in zip(seen, gs):
        assert torch.equal(s, g.sum(0, dtype=torch.float32).bfloat16())
    assert torch.equal(b.grad, (seen[0] * 4).cpu() + (seen[1] * 4).cpu())
    v = torch.nn.Parameter(randn(N, K, seed=1))
    v.is_ramtorch = True
    helpers.register_ramtorch_hook(v, lambda t: t * 2, helpers.ZERO2_HOOK_NAME)
    ck.linear(x, v).backward(gs[0])
    assert torch.equal(v.grad, dw_of(x, gs[0]) * 2)


# ------------------------------------------------------------------------------------------- refusals
@gpu
def test_a_bias_of_another_type_or_shape_is_refused():
    x, w = randn(T, K, seed=2), randn(N, K, seed=1)
    for bias in (torch.zeros(N, device=DEV), torch.zeros(1, device=DEV, dtype=torch.bfloat16), torch.zeros(T, N, device=DEV, dtype=torch.bfloat16),
                 torch.zeros(N + 1, device=DEV, dtype=torch.bfloat16), torch.zeros((), device=DEV, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="bias"):
            ck.linear(x, w, bias)


@gpu
def test_draws_that_do_not_fit_are_refused_before_the_forward_pass():
    x, w = randn(T, K, seed=2), randn(N, K, seed=1).requires_grad_()
    for kw in (dict(step=-1), dict(step=2 ** 32), dict(tensor_id=-1), dict(tensor_id=2 ** 32)):
        with pytest.raises(ValueError, match="32 bits"):
            ck.linear(x, w, product="mxfp4", seed=1, **kw)


@gpu
@pytest.mark.parametrize("product", [None, "mxfp4"])
def test_a_layer_without_outputs(product):
    x = randn(T, K, seed=2).requires_grad_()
    w, b = torch.zeros(0, K, device=DEV, dtype=torch.bfloat16).requires_grad_(), torch.zeros(0, device=DEV, dtype=torch.bfloat16).requires_grad_()
    y = ck.linear(x, w, b, product=product)
    y.backward(torch.zeros_like(y))
    assert y.shape == (T, 0) and (x.grad == 0).all() and w.grad.shape == (0, K) and b.grad.shape == (0,)


# --------------------------------------------------------------------------- automatic mixed precision
@gpu
@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("product", [None, "mxfp4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_under_autocast(dtype, product, inside):
    """As torch's linear: inputs are cast, fp32 weights and biases get fp32 gradients.  Those come from the gradient of the cast
    output and the checkpoint of the cast input, straight in fp32.  Two layers, the second on the first one's output."""
    x = randn(T, K, seed=2, dtype=torch.float32).requires_grad_()
    w1 = torch.nn.Parameter(randn(2 * N, K, seed=1, dtype=torch.float32) * 0.1)
    w2 = torch.nn.Parameter(randn(K, N, seed=4, dtype=torch.float32) * 0.1)
    b2 = torch.nn.Parameter(randn(K, seed=5, dtype=torch.float32))
    gy = randn(T, K, seed=6, dtype=dtype)
    with torch.autocast("cuda", dtype=dtype):
        proj = ck.linear(x, w1, product=product)
        h = ck.gated_act(*proj.chunk(2, -1))
        y = ck.linear(h, w2, b2, product=product)
        if inside:
            grads = torch.autograd.grad(y, (x, w1, w2, b2, proj, h), gy)
    assert proj.dtype == h.dtype == y.dtype == dtype
    if not inside:
        grads = torch.autograd.grad(y, (x, w1, w2, b2, proj, h), gy)
    gx, g1, g2, gb, gproj, gh = grads
    assert [t.dtype for t in grads] == [torch.float32] * 4 + [dtype] * 2
    assert torch.equal(g2, dw_of(h, gy, torch.float32)) and torch.equal(g1, dw_of(x.to(dtype), gproj, torch.float32))
    assert torch.equal(gb, gy.sum(0, dtype=torch.float32))
    if product:
        q = mx.quantize_mxfp4
        assert torch.equal(proj, mx.mxfp4_matmul(q(x.to(dtype)), q(w1))) and torch.equal(gh, mx.mxfp4_matmul(q(gy), q(w2, transpose=True)))
        assert torch.equal(gx, mx.mxfp4_matmul(q(gproj), q(w1, transpose=True)).float())
    else:
        assert torch.equal(proj, x.to(dtype) @ w1.to(dtype).t()) and torch.equal(gh, gy @ w2.to(dtype))
        assert torch.equal(gx, (gproj @ w1.to(dtype)).float())


@gpu
def test_under_autocast_with_a_host_weight():
    w, x, g = host_parameter(dtype=torch.float32), randn(T, K, seed=2, dtype=torch.float32), randn(T, N, seed=3)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = ck.linear(x, w)
    assert torch.equal(y, x.bfloat16() @ w.detach().to(DEV).bfloat16().t())
    y.backward(g)
    assert torch.equal(held(w), dw_of(x.bfloat16(), g, torch.float32))


@gpu
def test_an_fp32_layer_whose_backward_pass_alone_is_under_autocast():
    x, w, g = randn(T, K, seed=2, dtype=torch.float32).requires_grad_(), randn(N, K, seed=1, dtype=torch.float32).requires_grad_(), randn(T, N, seed=3, dtype=torch.float32)
    y = ck.linear(x, w)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        gx, = torch.autograd.grad(y, (x,), g)
    assert torch.equal(gx, g @ w)


@gpu
def test_types_that_differ_are_refused_without_autocast():
    x, w = randn(T, K, seed=2), randn(N, K, seed=1, dtype=torch.float32)
    with pytest.raises(ValueError):
        ck.linear(x, w)
    with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(ValueError):
        ck.linear(x, w.double())


@gpu
def test_a_gradient_that_is_not_asked_for_is_not_added():
    """``torch.autograd.grad`` and ``backward(inputs=...)`` add to nothing else, host parameters included."""
    w, b, x, g = host_parameter(), torch.nn.Parameter(randn(N, seed=9, device="cpu")), randn(T, K, seed=2).requires_grad_(), randn(T, N, seed=3)
    b.is_ramtorch, seen = True, []
    helpers.register_ramtorch_hook(b, lambda t: seen.append(t), helpers.ZERO2_HOOK_NAME)
    layer = lambda: ck.linear(x, w, b)      # noqa: E731
    torch.autograd.grad(layer(), (x,), g)
    layer().backward(g, inputs=[x])
    assert held(w) is None and w.grad is None and b.grad is None and not seen
    got, = torch.autograd.grad(layer(), (w,), g)
    assert torch.equal(got, dw_of(x, g).cpu()) and held(w) is None and w.grad is None and not seen
    layer().backward(g, inputs=[w])
    assert torch.equal(held(w), dw_of(x, g)) and w.grad is None and b.grad is None
    layer().backward(g)
    assert len(seen) == 1 and torch.equal(b.grad, g.sum(0, dtype=torch.float32).bfloat16().cpu())


@gpu
@pytest.mark.parametrize("reentrant", [None, True])
def test_a_held_gradient_is_ready_where_backward_was_called(reentrant):
    """As of ``.grad``: a forward pass on another stream, whose work is late, and a reader on the stream that called backward."""
    w, x, g = host_parameter(), randn(T, K, seed=2), randn(T, N, seed=3)
    want = dw_of(x, g)
    ck.linear(x, w).backward(g)                       # what is there before is another gradient
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    for add in (False, True):
        if not add:
            w.rt_device_grad = None
        side.wait_stream(main)
        with torch.cuda.stream(side):
            y = ck.linear(x, w)
            if reentrant:
                a = x.detach().requires_grad_()
                y = checkpoint(lambda a: ck.linear(a, w), a, use_reentrant=True)
            torch.cuda._sleep(200_000_000)            # a tenth of a second before the backward pass can run there
        y.backward(g)
        got = held(w).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, mx.weight_grad(g, mx.quantize_mxint8(x), out=want.clone(), accumulate=True) if add else want)
