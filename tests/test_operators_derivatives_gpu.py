"""Derivatives that the native operators (layer norm and its fork, the gated
product, the head's loss) do not have are refused, not taken as zero:
forward-mode tangents of any operand."""
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
