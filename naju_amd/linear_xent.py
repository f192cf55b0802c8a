"""Cross-entropy of a vocabulary head without its logits, on the HIP kernels
of include/naju_loss.h.

``linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean")``

is ``F.cross_entropy(F.linear(x, weight), target)`` for x [..., d], weight
[V, d] and int64 target [...]: the head's product and the loss of
evals/lm/train.py:70-74 in one, where naju_amd.linear.lm_head followed by
naju_amd.xent.cross_entropy holds 16-bit logits and their gradient (3.3 GB at
16384 tokens and 50257 classes). The logits stay in registers, float32 and
unrounded; the forward keeps one float32 per row, and the backward forms them
again by pieces of the vocabulary, in a workspace of at most 1 GiB (512 bytes
a row above 2^21 rows) for a piece's gradient, 6 bytes for each element of x
and the parts of split products. It computes in x's 16-bit dtype, or in the
autocast dtype under autocast (a weight of another dtype is cast, from
naju_amd.wcast where it is active there).

The loss is float32: the mean over the rows whose target is not
ignore_index ("mean"), their sum ("sum"), or a loss for every row with 0 for
ignored ones ("none", in target's shape). A target outside [0, V) that is
not ignore_index gives NaN. The weight's gradient comes in its dtype (in
float32, unrounded, for a float32 weight). Deterministic.

The kernels read 16-byte aligned rows a multiple of 8 elements apart;
operands of an odd width, stride or offset are copied once into such rows.
CUDA tensors computed in float16 / bfloat16 only: there is no other
implementation behind this function.
"""
import torch

from naju_amd import _lib, wcast
from naju_amd.linear import compute_dtype

REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}


class _ToTied(torch.autograd.Function):
    """weight, whose gradient goes to `tied` (naju_amd.embed.TiedGrad) as in
    naju_amd.linear's head: the tied embedding's backward adds its rows into
    it and returns the sum."""

    @staticmethod
    def forward(ctx, weight, tied):
        ctx.tied = tied
        return weight.view_as(weight)

    @staticmethod
    def backward(ctx, dw):
        # (one with a graph of its own, create_graph, keeps it only on autograd's way)
        if dw.dtype != torch.float32 or dw.requires_grad:
            return dw, None
        ctx.tied.put(dw)
        return None, None


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean", tied=None):
    """Cross-entropy of x weight^T against target in compute_dtype(x), which
    must not be None; see the module's docstring. tied: a
    naju_amd.embed.TiedGrad that takes the weight's gradient for the tied
    embedding's backward, as in naju_amd.linear.lm_head."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(REDUCTIONS)}, got {reduction!r}")
    dt = compute_dtype(x)
    if dt is None or not x.is_floating_point():
        raise ValueError("naju_amd.linear_xent.linear_cross_entropy serves CUDA tensors computed in float16 / "
                         "bfloat16")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be [classes, d], got {tuple(weight.shape)}")
    if x.dim() == 0 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., {weight.shape[1]}], got {tuple(x.shape)}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target must be {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    if target.is_floating_point() or target.is_complex() or target.dtype == torch.bool:
        raise TypeError(f"target must hold class indices, got {target.dtype}")
    if not weight.is_floating_point():
        raise TypeError("weight must be a floating-point tensor")
    if weight.device != x.device:
        raise ValueError("x and weight must be on one device")
    target = target.to(device=x.device, dtype=torch.int64).contiguous()
    # the LM's padded 16-bit copy serves as it is: its first V rows
    w16 = wcast.lookup((weight,), dt)
    if tied is not None:
        weight = _ToTied.apply(weight, tied)
    return _lib.ops().linear_cross_entropy(x if x.dtype == dt else x.to(dt), weight, target, w16, int(ignore_index),
                                           REDUCTIONS[reduction])
