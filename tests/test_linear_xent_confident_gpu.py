"""The head's loss where one class takes nearly all: the loss is what is left of
two large numbers, and keeps its precision whatever they are."""
import pytest
import torch

from naju_amd.linear_xent import linear_cross_entropy

pytestmark = pytest.mark.gpu


# rows of each forward (few rows, small and large tiles, several tiles a row)
@pytest.mark.parametrize("rows, v", [(1, 300), (16, 5000), (60, 300), (200, 700), (3000, 9000)])
@pytest.mark.parametrize("scale", [2.0 ** -1, 1.0, 2.0 ** 4, 2.0 ** 9])
def test_confident_rows(gpu, rows, v, scale):
    """x is a multiple of its class's own row of W, whose rows are of one length,
    with entries of +-1 (products and their sums are exact in float32): the
    logits are whole multiples of `scale`, up to 2^16, and what is left is the
    error of log(1 + sum exp(l - l_t)) in float32. An exponent is off by 2^-24 of
    itself, in the mean over the terms log2(v) < 14 at most; a power of two by
    2^-23; 32 roundings of partial sums come on top: below 2^-18, whatever the
    logits, and 2^-18 of a large loss."""
    d = 128
    g = torch.Generator().manual_seed(rows + v)
    w = (torch.randint(0, 2, (v, d), generator=g) * 2 - 1).to(torch.bfloat16)
    t = torch.randint(0, v, (rows,), generator=g)
    x = w[t] * scale
    flip = torch.rand(rows, d, generator=g) < 0.25  # of differing distance to the class
    x = torch.where(flip, -x, x).to(torch.bfloat16)
    logits = x.double() @ w.double().t()
    gap = logits - logits.gather(1, t[:, None])
    want = torch.log(torch.exp(gap).sum(1)) if float(gap.max()) < 600 else torch.logsumexp(gap, 1)
    got = linear_cross_entropy(x.to(gpu), w.to(gpu), t.to(gpu), reduction="none").double().cpu()
    assert ((got - want).abs() <= 2.0 ** -18 * (1 + want)).all(), float((got - want).abs().max())


@pytest.mark.parametrize("rows, v", [(16, 300), (200, 700), (3000, 9000)])
@pytest.mark.parametrize("scale", [3.0, 296.0])
def test_gradient_of_rows_without_doubt(gpu, rows, v, scale):
    """Where every other class is exp(-64) or less, dl is 0 up to float32's
    rounding of p near 1 (2^-23), however large the logits (up to 2^15): dx and
    dw, its products with entries of 1 and `scale`, are below 2^-21 of those."""
    d = 128
    g = torch.Generator().manual_seed(rows + v)
    w = (torch.randint(0, 2, (v, d), generator=g) * 2 - 1).to(torch.bfloat16)
    t = torch.randint(0, v, (rows,), generator=g)
    x = (w[t] * scale).to(torch.bfloat16)
    x[:, : 5] *= -1  # logits that no power of two divides
    logits = x.double() @ w.double().t()
    gap = logits - logits.gather(1, t[:, None])
    gap[torch.arange(rows), t] = -1e9
    keep = gap.max(1).values <= -64
    assert keep.sum() > rows // 2
    x, t = x[keep].to(gpu).requires_grad_(True), t[keep].to(gpu)
    wr = w.to(gpu).requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_cross_entropy(x, wr, t, reduction="sum"), (x, wr))
    assert float(dx.abs().max()) <= 2.0 ** -21
    assert float(dw.abs().max()) <= 2.0 ** -21 * scale * float(torch.bincount(t).max())
