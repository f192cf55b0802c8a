"""Layer norm's sums over many rows and wide rows: the weight's and the bias's
gradients where every term has the same sign, so that a running sum rounds
the same way row after row, and rows wider than one launch of the fold."""
import pytest
import torch

from naju_amd.layernorm import layer_norm

pytestmark = pytest.mark.gpu


# below and above the widths that registers hold (8 and 16384 columns), and a
# count of rows that is no multiple of any slice
@pytest.mark.parametrize("rows, d", [
    ((1 << 24) + 5, 4), ((1 << 24) + 5, 1), ((1 << 22) + 1, 7), ((1 << 26) + 3, 8), ((1 << 23) + 11, 40),
    ((1 << 15) + 9, 16400)])
@pytest.mark.parametrize("value, out", [
    (0.298828125, torch.bfloat16), (0.33203125, torch.bfloat16), (0.3469262401991873, torch.float32)])
def test_constant_gradient(gpu, rows, d, value, out):
    """db is rows * value and dw value * sum(xh) with xh of one sign in a
    column. A float32 sum of n terms of one sign is off by n 2^-24 at most
    and the longest chain is 1024 rows (6.1e-5); xh itself, from float32
    statistics of values up to d, adds its own 1e-5."""
    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn(rows, d, generator=g, device=gpu, dtype=torch.bfloat16).mul_(0.125)
    # columns apart by their number (in steps of a small period, so that wide rows stay small)
    x += (torch.arange(d, device=gpu) % 8).to(x.dtype)
    w = torch.ones(d, device=gpu, requires_grad=True)
    b = torch.zeros(d, device=gpu, requires_grad=True)
    value = float(torch.tensor(value))
    y = layer_norm(x, w, b, out_dtype=out)
    dw, db = torch.autograd.grad(y, (w, b), torch.full((1, d), value, dtype=y.dtype, device=gpu).expand(rows, d))
    want = torch.zeros(d, dtype=torch.float64, device=gpu)
    for part in x.split(max(1, (1 << 26) // d)):
        p = part.double()
        want += ((p - p.mean(1, keepdim=True)) * (p.var(1, correction=0, keepdim=True) + 1e-5).rsqrt()).sum(0)
    rel = lambda a, r: float((a.double() - r).norm() / r.norm().clamp_min(1e-300))  # noqa: E731
    assert rel(db, torch.full_like(want, rows * value)) <= 6.1e-5
    if d > 1:
        assert rel(dw, want * value) <= 6.1e-5 + 1e-5


def test_statistics_of_a_wide_row(gpu):
    """One row of more than 2^26 columns: its statistics and the backward's row
    sums against float64."""
    g = torch.Generator(device=gpu).manual_seed(2)
    d = (1 << 26) + 3
    x = torch.randn(1, d, generator=g, device=gpu).requires_grad_(True)
    w = torch.ones(d, device=gpu, requires_grad=True)
    b = torch.zeros(d, device=gpu, requires_grad=True)
    dy = torch.randn(1, d, generator=g, device=gpu)
    dx, dw, db = torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    assert torch.equal(db, dy[0])
    xt = x.detach().double()
    xh = (xt - xt.mean()) * (xt.var(correction=0) + 1e-5).rsqrt()
    rel = lambda a, r: float((a.double() - r).norm() / r.norm())  # noqa: E731
    assert rel(dw, (dy * xh)[0]) <= 1e-5
    gt = dy.double()
    want = (xt.var(correction=0) + 1e-5).rsqrt() * (gt - gt.mean() - xh * (gt * xh).mean())
    assert rel(dx, want) <= 1e-5


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
