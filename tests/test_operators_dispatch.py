"""The native operators under what stands between a call and its kernels:
tracers, fake tensors, torch.compile and dispatch modes see operators with
shapes of their own, never the memory behind them. On the CPU with meta
tensors; on the GPU the traced calls against the plain ones."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from naju_amd import _lib
from naju_amd.gated import gated_linear
from naju_amd.layernorm import layer_norm, layer_norm_fork
from naju_amd.linear_xent import linear_cross_entropy

BF16 = _lib.DT_BF16


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta", requires_grad=dtype.is_floating_point)


def _names(g):
    return [str(n.target) for n in g.graph.nodes if n.op == "call_function"]


# ------------------------------------------------------------ meta tensors, no GPU

@pytest.mark.parametrize("shape", [(72,), (5, 72), (2, 3, 72), (0, 72), (5, 71)])
def test_shapes_without_memory(shape):
    o, d = _lib.ops(), shape[-1]
    x, w = _meta(*shape), _meta(10, d)
    wf = _meta(d, dtype=torch.float32)
    y = o.layer_norm(x, wf, wf, 1e-5, _lib.DT_F32)
    assert y.shape == x.shape and y.dtype == torch.float32
    dx, dw = torch.autograd.grad(y.sum(), (x, wf))
    assert dx.shape == x.shape and dx.dtype == x.dtype and dw.shape == (d,) and dw.dtype == torch.float32
    res, y = o.layer_norm_fork(x, None, None, 1e-5, BF16)
    assert torch.autograd.grad((res + y).sum(), x)[0].shape == x.shape
    h = o.gated_linear(x, w, w, None, 0)
    assert h.shape == (*shape[:-1], 10) and h.dtype == x.dtype
    dx, dw = torch.autograd.grad(h.sum(), (x, w))
    assert dx.shape == x.shape and dw.shape == w.shape and dw.dtype == w.dtype
    t = torch.empty(shape[:-1], dtype=torch.int64, device="meta")
    w32 = _meta(10, d, dtype=torch.float32)
    for reduction, want in ((0, ()), (1, ()), (2, shape[:-1])):
        loss = o.linear_cross_entropy(x, w32, t, None, -100, reduction)
        assert loss.shape == want and loss.dtype == torch.float32
        dx, dw = torch.autograd.grad(loss.sum(), (x, w32))
        assert dx.shape == x.shape and dw.shape == w32.shape and dw.dtype == torch.float32
    with torch.no_grad():
        assert o.layer_norm(x, None, None, 1e-5, BF16).shape == x.shape
        assert o.gated_linear(x, w, w, None, 1).shape == (*shape[:-1], 10)
        assert o.linear_cross_entropy(x, w, t, None, -100, 2).shape == shape[:-1]


def _step(x, w, t):
    o = _lib.ops()
    r, y = o.layer_norm_fork(x, None, None, 1e-5, BF16)
    h = o.gated_linear(y, w, w, None, 0)
    loss = o.linear_cross_entropy(r + y, w, t, None, -100, 0)
    return torch.autograd.grad(h.sum() + loss, (x, w))


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_a_trace_holds_the_operators(mode):
    x, w, t = _meta(4, 6, 72), _meta(10, 72), torch.empty(4, 6, dtype=torch.int64, device="meta")
    g = make_fx(_step, tracing_mode=mode)(x, w, t)
    names = _names(g)
    for op in ("_layer_norm_fwd", "_layer_norm_bwd", "_gated_fwd", "_gated_bwd", "_linear_xent_fwd",
               "_linear_xent_bwd"):
        assert names.count(f"naju.{op}.default") == 1
    # nothing that the kernels write is made outside them
    assert not any("empty" in n for n in names)
    if mode == "symbolic":
        x, t = _meta(3, 9, 72), torch.empty(3, 9, dtype=torch.int64, device="meta")
    with torch.no_grad():
        assert [v.shape for v in g(x, w, t)] == [x.shape, w.shape]


def test_a_trace_without_a_graph_holds_the_operators():
    o = _lib.ops()

    def score(x, w, t):
        return o.linear_cross_entropy(o.layer_norm(x, None, None, 1e-5, BF16), w, t, None, -100, 2)

    x, w, t = _meta(4, 72), _meta(10, 72), torch.empty(4, dtype=torch.int64, device="meta")
    with torch.no_grad():
        assert _names(make_fx(score)(x, w, t)) == ["naju.layer_norm.default", "naju.linear_cross_entropy.default"]


def test_a_steps_derivative_is_refused():
    """A traced step holds the backward as an operator; a derivative of that raises."""
    x, w, t = _meta(4, 6, 72), _meta(10, 72), torch.empty(4, 6, dtype=torch.int64, device="meta")
    dx, dw = make_fx(_step)(x, w, t)(x, w, t)
    with pytest.raises(RuntimeError, match="naju.*not implemented"):
        torch.autograd.grad(dw.float().pow(2).sum(), x)


def test_derivatives_are_refused_on_meta_tensors_too():
    o = _lib.ops()
    x, w, t = _meta(4, 72), _meta(10, 72), torch.empty(4, dtype=torch.int64, device="meta")
    calls = (lambda x: o.layer_norm(x, None, None, 1e-5, BF16), lambda x: o.layer_norm_fork(x, None, None, 1e-5, BF16)[1],
             lambda x: o.gated_linear(x, w, w, None, 0), lambda x: o.linear_cross_entropy(x, w, t, None, -100, 0))
    for call in calls:
        for grad in (True, False):
            with torch.set_grad_enabled(grad), forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp"):
                call(forward_ad.make_dual(x, torch.empty_like(x)))
        z = x * 2
        (dx,) = torch.autograd.grad(call(z).float().sum(), z, create_graph=True)
        with pytest.raises(RuntimeError, match="naju: .*second"):
            torch.autograd.grad(dx.float().sum(), x)


def test_cpu_tensors_are_refused():
    with pytest.raises(NotImplementedError, match="naju::layer_norm"):
        _lib.ops().layer_norm(torch.randn(2, 8), None, None, 1e-5, _lib.DT_F32)


# ------------------------------------------------------------ GPU

def _inputs(d, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(d)
    x = torch.randn(3, 7, d, generator=g).to(dtype).cuda()
    w = torch.randn(20, d, generator=g).mul_(d ** -0.5).to(dtype).cuda()
    t = torch.randint(0, 20, (3, 7), generator=g).cuda()
    t[0, 1] = -100
    return x, w, t


def _user_step(x, w, t):
    res, y = layer_norm_fork(x)
    h = gated_linear(layer_norm(y), w, w)
    return linear_cross_entropy(res + y, w, t) + h.float().square().mean()


def _with_grads(fn, x, w, t):
    x, w = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        loss = fn(x, w, t)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w)))


# 72: operands as they lie; 71: copied to aligned rows by the functions or by the kernels' side
@pytest.mark.gpu
@pytest.mark.parametrize("d", [72, 71])
def test_traced_step_equals_the_call(gpu, d):
    x, w, t = _inputs(d)
    want = _with_grads(_user_step, x, w, t)
    x.requires_grad_(True), w.requires_grad_(True)

    def step(x, w, t):
        loss = _user_step(x, w, t)
        return (loss, *torch.autograd.grad(loss, (x, w)))

    g = make_fx(step)(x, w, t)
    x2, w2, t2 = _inputs(d)
    with torch.no_grad():
        x2.mul_(0.5)
        for _ in range(2):
            for a, b in zip(g(x2, w2, t2), _with_grads(_user_step, x2, w2, t2)):
                assert torch.equal(a, b)
        for a, b in zip(g(x, w, t), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [72, 71])
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_step_equals_the_call(gpu, d, dynamic):
    x, w, t = _inputs(d)
    torch._dynamo.reset()
    fn = torch.compile(_user_step, backend="aot_eager", dynamic=dynamic, fullgraph=True)
    for k in (3, 2):
        ins = (x[:k], w, t[:k])
        for a, b in zip(_with_grads(fn, *ins), _with_grads(_user_step, *ins)):
            assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(fn(x, w, t), _user_step(x, w, t))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [72, 71])
def test_operator_checks(gpu, d):
    """torch's own checks of an operator's schema, shapes and autograd, static and dynamic."""
    x, w, t = _inputs(d)
    wf = torch.randn(d, device=gpu)
    o = _lib.ops()
    for grad in (True, False):
        xr, wr, wfr = (v.clone().requires_grad_(grad) for v in (x, w, wf))
        for op, args in ((o.layer_norm, (xr, wfr, None, 1e-5, BF16)), (o.layer_norm, (xr, None, wfr, 1e-5, _lib.DT_F32)),
                         (o.gated_linear, (xr, wr, wr, None, 1)),
                         (o.linear_cross_entropy, (xr, wr, t, None, -100, 0)),
                         (o.linear_cross_entropy, (xr, wr, t, None, -100, 2))):
            torch.library.opcheck(op, args)


@pytest.mark.gpu
def test_dispatch_modes_change_nothing(gpu):
    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.ops = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.ops.append(str(func))
            return func(*args, **(kwargs or {}))

    for d in (72, 71):
        ins = _inputs(d)
        want = _with_grads(_user_step, *ins)
        with Seen() as seen:
            got = _with_grads(_user_step, *ins)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert "naju._gated_fwd.default" in seen.ops and "naju._gated_bwd.default" in seen.ops


@pytest.mark.gpu
def test_forward_inside_a_mode_backward_outside(gpu):
    """Operands kept by a forward under a mode serve a backward without it, and the other way round."""
    class Idle(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, w, t = _inputs(71)
    want = _with_grads(_user_step, x, w, t)
    for inside in (0, 1):
        xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        with Idle() if inside == 0 else torch.enable_grad():
            loss = _user_step(xr, wr, t)
        with Idle() if inside == 1 else torch.enable_grad():
            got = torch.autograd.grad(loss, (xr, wr))
        for a, b in zip(got, want[1:]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_vmap_without_a_graph(gpu):
    """Each slice as a call of its own; transforms that differentiate are refused."""
    x, w, _ = _inputs(72)
    with torch.no_grad():
        assert torch.equal(torch.vmap(lambda v: gated_linear(v, w, w))(x), gated_linear(x, w, w))
        assert torch.equal(torch.vmap(lambda v: layer_norm(v))(x), layer_norm(x))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: layer_norm(v).float().sum())(x)
    with pytest.raises(RuntimeError, match="jvp"):
        torch.func.jvp(lambda v: layer_norm(v), (x,), (x,))


@pytest.mark.gpu
def test_in_place_changes_of_what_is_kept_are_noticed(gpu):
    for d in (72, 71):
        x, w, t = _inputs(d)
        x.requires_grad_(True)
        for flat in (False, True):
            xi = x.flatten(0, 1) if flat else x
            xi = xi.clone()
            loss = layer_norm(xi).float().sum()
            with torch.no_grad():
                xi.add_(1)
            with pytest.raises(RuntimeError, match="inplace"):
                loss.backward()


@pytest.mark.gpu
def test_inference_mode(gpu):
    for d in (72, 71):
        x, w, t = _inputs(d)
        with torch.no_grad():
            want = (layer_norm(x), *layer_norm_fork(x), gated_linear(x, w, w), linear_cross_entropy(x, w, t))
        x.requires_grad_(True), w.requires_grad_(True)
        with torch.inference_mode():
            got = (layer_norm(x), *layer_norm_fork(x), gated_linear(x, w, w), linear_cross_entropy(x, w, t))
            again = (layer_norm(x.clone()), *layer_norm_fork(x.clone()), gated_linear(x.clone(), w, w),
                     linear_cross_entropy(x.clone(), w, t))
        for a, b, c in zip(got, want, again):
            assert torch.equal(a, b) and torch.equal(c, b)
        # (the fork's stream is x's view, of which torch says what it says of x)
        assert not any(a.requires_grad for i, a in enumerate(got) if i != 1)


@pytest.mark.gpu
def test_jit_trace_holds_the_operators(gpu):
    x, w, t = _inputs(72)
    with torch.no_grad():
        g = torch.jit.trace(lambda x, w, t: (layer_norm(x), gated_linear(x, w, w), linear_cross_entropy(x, w, t)), (x, w, t))
        x2 = x * 0.5
        for a, b in zip(g(x2, w, t), (layer_norm(x2), gated_linear(x2, w, w), linear_cross_entropy(x2, w, t))):
            assert torch.equal(a, b)
    assert "naju::gated_linear" in str(g.graph)


@pytest.mark.gpu
def test_recomputed_and_selectively_kept_steps(gpu):
    """Activation checkpointing, and its selective form, which keeps results by operator under a mode of its own."""
    from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts
    keep = {torch.ops.naju._gated_fwd.default, torch.ops.naju._layer_norm_fwd.default}

    def policy(ctx, op, *args, **kwargs):
        return CheckpointPolicy.MUST_SAVE if op in keep else CheckpointPolicy.PREFER_RECOMPUTE

    for d in (72, 71):
        ins = _inputs(d)
        want = _with_grads(_user_step, *ins)
        for kw in ({}, {"context_fn": lambda: create_selective_checkpoint_contexts(policy)}):
            got = _with_grads(lambda *a: checkpoint(_user_step, *a, use_reentrant=False, **kw), *ins)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
