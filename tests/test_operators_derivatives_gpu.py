"""Derivatives that the native operators (layer norm and its fork, the gated
product, the head's loss) do not have are refused, not taken as zero:
forward-mode tangents of any operand, and second derivatives by any way to
what they depend on."""
import pytest
import torch
from torch.autograd import forward_ad

from naju_amd.gated import gated_linear
from naju_amd.layernorm import layer_norm, layer_norm_fork
from naju_amd.linear_xent import linear_cross_entropy

pytestmark = pytest.mark.gpu
ROWS, D, F = 12, 32, 24


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _ops():
    """name: (function of the floating operands, those operands in float32)"""
    t = torch.arange(ROWS, device="cuda") % F
    t[3] = -100
    h = lambda v: v.bfloat16()  # noqa: E731
    x, w, b = _rand(ROWS, D, seed=1), _rand(D, seed=2), _rand(D, seed=3)
    wg, wu = _rand(F, D, seed=4), _rand(F, D, seed=5)
    return {
        "layer_norm": (lambda x, w, b: layer_norm(x, w, b), (x, w, b)),
        "layer_norm_fork": (lambda x, w, b: layer_norm_fork(x, w, b)[1], (x, w, b)),
        "gated_linear": (lambda x, g, u: gated_linear(h(x), h(g), h(u)).float(), (x, wg, wu)),
        "linear_cross_entropy": (lambda x, w: linear_cross_entropy(h(x), h(w), t), (x, wg)),
        "linear_cross_entropy_none": (lambda x, w: linear_cross_entropy(h(x), h(w), t, reduction="none"), (x, wg)),
    }


NAMES = ["layer_norm", "layer_norm_fork", "gated_linear", "linear_cross_entropy", "linear_cross_entropy_none"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(gpu, name):
    op, ins = _ops()[name]
    for i in range(len(ins)):
        for grad in (True, False):
            with torch.set_grad_enabled(grad), forward_ad.dual_level():
                duals = [forward_ad.make_dual(v, torch.ones_like(v)) if j == i else v for j, v in enumerate(ins)]
                with pytest.raises(RuntimeError, match="jvp"):
                    op(*duals)
    # a level without tangents, and a tangent after it, change nothing
    want = op(*ins)
    with forward_ad.dual_level():
        assert torch.equal(op(*ins), want)
    assert torch.equal(op(*ins), want)


def test_forward_mode_of_the_forks_stream_is_refused(gpu):
    x = _rand(ROWS, D)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        layer_norm_fork(forward_ad.make_dual(x, torch.ones_like(x)))


def _behind_a_layer(name):
    """(op's value of z = x m, x, m, the other operands), all leaves."""
    op, ins = _ops()[name]
    x = ins[0].requires_grad_(True)
    m = _rand(D, D, seed=9).mul_(D ** -0.5).requires_grad_(True)
    rest = [v.requires_grad_(True) for v in ins[1:]]
    return op(x @ m, *rest), x, m, rest


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("how", ["backward", "grad m", "grad x", "grad weight"])
def test_penalty_on_a_gradient_is_refused(gpu, name, how):
    """dx depends on m, on x and on the weights through the operator's
    backward; none of those shares may be left out."""
    y, x, m, rest = _behind_a_layer(name)
    (dx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    penalty = dx.pow(2).sum()
    with pytest.raises(RuntimeError, match="naju: .*second"):
        if how == "backward":
            penalty.backward()
        else:
            torch.autograd.grad(penalty, {"grad m": m, "grad x": x, "grad weight": rest[0]}[how])


@pytest.mark.parametrize("name", NAMES)
def test_penalty_on_a_weight_gradient_is_refused(gpu, name):
    y, x, m, rest = _behind_a_layer(name)
    for dw in torch.autograd.grad(y.sum(), rest, create_graph=True):
        with pytest.raises(RuntimeError, match="naju: .*second"):
            torch.autograd.grad(dw.pow(2).sum(), m, retain_graph=True)


@pytest.mark.parametrize("name", NAMES)
def test_through_the_incoming_gradient_is_refused(gpu, name):
    """A gradient is linear in the incoming one, which may have a graph."""
    y, x, m, rest = _behind_a_layer(name)
    s = torch.ones_like(y).requires_grad_(True)
    (dx,) = torch.autograd.grad(y, x, s, create_graph=True)
    with pytest.raises(RuntimeError, match="naju: .*second"):
        torch.autograd.grad(dx.sum(), s)


@pytest.mark.parametrize("name", NAMES)
def test_create_graph_alone_changes_no_gradient(gpu, name):
    y, x, m, rest = _behind_a_layer(name)
    a = torch.autograd.grad(y.sum(), (x, m, *rest), retain_graph=True)
    b = torch.autograd.grad(y.sum(), (x, m, *rest), create_graph=True)
    for p, q in zip(a, b):
        assert torch.equal(p, q.detach())


def test_the_forks_stream_alone_is_differentiable(gpu):
    """Where only the stream is used, its gradient passes through and keeps its graph."""
    x = _rand(ROWS, D).requires_grad_(True)
    res, _ = layer_norm_fork(x)
    (dx,) = torch.autograd.grad((res ** 3).sum(), x, create_graph=True)
    (ddx,) = torch.autograd.grad(dx.sum(), x)
    assert torch.allclose(ddx, 6 * x.detach())


def test_tied_weight_under_create_graph(gpu):
    """The tied weight's gradient hand-over keeps the refusal."""
    from naju_amd.embed import TiedGrad, embedding
    w = _rand(97, D).requires_grad_(True)
    ids, y = (torch.randint(0, 97, (40,), generator=torch.Generator().manual_seed(s)).cuda() for s in (1, 2))

    def grads(create):
        tied = TiedGrad(w)
        loss = linear_cross_entropy(embedding(ids, w, tied).bfloat16(), w, y, tied=tied)
        return torch.autograd.grad(loss, w, create_graph=create)[0]

    with torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = grads(False), grads(True)
    assert float((a - b).detach().norm()) <= 1e-6 * float(a.norm())
    with pytest.raises(RuntimeError, match="naju: .*second"):
        torch.autograd.grad(b.pow(2).sum(), w)
