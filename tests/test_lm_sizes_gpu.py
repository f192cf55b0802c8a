"""The native operators through the model at sizes that reach their large tiles,
several pieces of the vocabulary, the paired 16-bit weight copies and float32
weight gradients: NajuLM.loss against the head's logits and their loss, and the
feed-forward sublayer against float64."""
import pytest
import torch
import torch.nn.functional as F

from naju_amd import wcast
from naju_amd.mixer import GatedFFN, NajuLM

pytestmark = pytest.mark.gpu
U = 2.0 ** -8  # bfloat16


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


@pytest.mark.parametrize("tie", [True, False])
def test_loss_of_the_lms_batch(gpu, tie):
    """8 x 2048 tokens over 50257 classes (three pieces). The logits' path rounds
    the logits and their gradient to 16 bits, the loss alone its gradient: the
    paths differ by the rounding of logits below 2 (2^-8 of the loss's share) and
    by at most 2 u in a gradient's terms, 3 u with sums that cancel."""
    torch.manual_seed(0)
    m = NajuLM(50257, d_model=256, n_layers=1, dropout=0.0, d_state=4, norm="layer", ffn_dim=704, tie_weights=tie,
               scan_backend="hip").to(gpu)
    ids, y = (torch.randint(0, 50257, (8, 2048), device=gpu) for _ in range(2))
    y[:, -100:] = -100
    grads = []
    for way in ("loss", "logits"):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = (m.loss(ids, y) if way == "loss" else
                    F.cross_entropy(m(ids).float().view(-1, 50257), y.view(-1)))
        grads.append((loss.detach(), dict(zip((n for n, _ in m.named_parameters()),
                                              torch.autograd.grad(loss, list(m.parameters()))))))
        del loss
    (la, a), (lb, b) = grads
    assert abs(float(la - lb)) <= U * float(lb)
    for n in a:
        assert a[n].dtype == torch.float32 and _rel(a[n], b[n]) <= 3 * U, n


def test_feed_forward_of_the_lms_batch(gpu):
    """16384 tokens, 768 x 2048, float32 weights with their paired 16-bit copies.
    Roundings to 16 bits on the way: h and the result (2 u); for a weight's
    gradient those of dh and of dg or du, or of h (2 u), for dx dh, dg, du and
    itself (3 u); u more where sums cancel."""
    torch.manual_seed(1)
    ffn = GatedFFN(768, 2048).to(gpu)
    x = torch.randn(16384, 768, device=gpu).bfloat16().requires_grad_(True)
    dy = torch.randn(16384, 768, device=gpu).bfloat16()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        with wcast.active(wcast.WeightCopies(), ffn.cast_groups(), torch.bfloat16):
            assert wcast.lookup((ffn.gate_proj.weight, ffn.up_proj.weight), torch.bfloat16) is not None
            y = ffn(x)
    ps = [ffn.gate_proj.weight, ffn.up_proj.weight, ffn.down_proj.weight]
    got = torch.autograd.grad(y, [x, *ps], dy)
    ws = [p.detach().bfloat16().double().requires_grad_(True) for p in ps]
    xs = x.detach().double().requires_grad_(True)
    ref = (F.silu(xs @ ws[0].t()) * (xs @ ws[1].t())) @ ws[2].t()
    want = torch.autograd.grad(ref, [xs, *ws], dy.double())
    assert y.dtype == torch.bfloat16 and _rel(y, ref) <= 3 * U
    for g, r, k in zip(got, want, (4, 3, 3, 3)):
        assert _rel(g, r) <= k * U
    assert all(g.dtype == torch.float32 for g in got[1:])
