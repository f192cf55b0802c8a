"""NajuLM.loss against the loss over its logits where no kernel runs: the
logits' precision is kept."""
import pytest
import torch
import torch.nn.functional as F

from naju_amd import scan as scan_mod
from naju_amd.mixer import NajuLM
from oracle.scan_ref import scan_loop_torch

VOCAB = 61


@pytest.fixture(autouse=True)
def oracle_backend(monkeypatch):
    monkeypatch.setitem(scan_mod._BACKEND_CACHE, "oracle_loop", scan_loop_torch)


def _model(**kw):
    torch.manual_seed(0)
    return NajuLM(VOCAB, d_model=16, n_layers=1, dropout=0.0, d_state=2, scan_backend="oracle_loop", **kw)


def _batch():
    g = torch.Generator().manual_seed(1)
    ids, y = (torch.randint(0, VOCAB, (2, 7), generator=g) for _ in range(2))
    y[1, 3] = -100
    return ids, y


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_double_model_keeps_its_precision(reduction):
    m = _model(norm="layer", ffn_dim=24).double()
    ids, y = _batch()
    a = m.loss(ids, y, reduction=reduction)
    b = F.cross_entropy(m(ids).view(-1, VOCAB), y.view(-1), reduction=reduction)
    assert a.dtype == torch.float64 and torch.equal(a.reshape(-1), b.reshape(-1))
    ga, gb = (torch.autograd.grad(v.sum(), list(m.parameters())) for v in (a, b))
    for p, q in zip(ga, gb):
        assert p.dtype == torch.float64 and torch.equal(p, q)


def test_16_bit_logits_are_taken_in_float32():
    """CPU autocast leaves bfloat16 logits: the loss over them is formed in float32."""
    m = _model()
    ids, y = _batch()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        logits = m(ids)
        loss = m.loss(ids, y)
    assert logits.dtype == torch.bfloat16 and loss.dtype == torch.float32
    assert torch.equal(loss, F.cross_entropy(logits.float().view(-1, VOCAB), y.view(-1)))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_targets_have_the_ids_shape(device):
    """The same targets are taken and refused on every path: ids' shape, class
    indices of any integer type."""
    m = _model() if device == "cpu" else NajuLM(VOCAB, d_model=16, n_layers=1, dropout=0.0, d_state=2).cuda()
    ids, y = (t.to(device) for t in _batch())
    for auto in (False, True):
        with torch.autocast(device, dtype=torch.bfloat16, enabled=auto):
            want = m.loss(ids, y)
            assert torch.equal(m.loss(ids, y.int()), want)
            for bad in (y.reshape(-1), y[:, :6], y.t(), y[None]):
                with pytest.raises(ValueError, match="targets must be"):
                    m.loss(ids, bad)
            for bad in (y.float(), y == 3):
                with pytest.raises(TypeError, match="class indices"):
                    m.loss(ids, bad)
            with pytest.raises(ValueError, match="reduction"):
                m.loss(ids, y, reduction="median")
