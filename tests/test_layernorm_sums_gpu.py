"""Layer norm's sums of the weight's and the bias's gradients: rows wider than
one launch of the fold."""
import pytest
import torch

from naju_amd.layernorm import layer_norm

pytestmark = pytest.mark.gpu


def test_fold_of_a_wide_row(gpu):
    """One row of more than 2^26 columns: db is dy, and dw is dy y with neither
    weight nor bias."""
    g = torch.Generator(device=gpu).manual_seed(2)
    d = (1 << 26) + 3
    x = torch.randn(1, d, generator=g, device=gpu)
    w = torch.ones(d, device=gpu, requires_grad=True)
    b = torch.zeros(d, device=gpu, requires_grad=True)
    dy = torch.randn(1, d, generator=g, device=gpu)
    y = layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(db, dy[0])
    assert float((dw - dy[0] * y.detach()[0]).abs().max()) <= 2.0 ** -22 * float(dw.abs().max())
