"""
The relation driver's two losses as one autograd node (round 6).

Reference models/train_rels.py:140-141:
    losses['class_loss'] = F.cross_entropy(result.rm_obj_dists, result.rm_obj_labels)
    losses['rel_loss'] = F.cross_entropy(result.rel_dists, result.rel_labels[:, -1])
The framework evaluates each as log_softmax + nll_loss and their two backward kernels plus fills: ~25 launches of a few
microseconds on the main stream between the relation tail and the first product of the backward pass.  `relation_losses`
returns both means as ONE [2] tensor from csrc/exact_ops.hip ce_pair_* (two launches forward, one backward); the script
sums (or weights) that tensor.  MOTIFS_FUSED_LOSS=0, CPU tensors and anything but fp32 logits / int64 labels take the
framework's own functions.
"""
import collections
import os

import torch
import torch.nn.functional as F

from lib import _hip

FUSED = os.environ.get('MOTIFS_FUSED_LOSS', '1') != '0'


class _CrossEntropyPairFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits_a, labels_a, logits_b, labels_b):
        la, lb = logits_a.contiguous(), logits_b.contiguous()
        losses, lse = _hip.ce_pair_fwd(la, labels_a, lb, labels_b)
        ctx.save_for_backward(la, labels_a, lb, labels_b, lse)
        return losses

    @staticmethod
    def backward(ctx, g):
        la, labels_a, lb, labels_b, lse = ctx.saved_tensors
        ga, gb = _hip.ce_pair_bwd(la, labels_a, lb, labels_b, lse, g.contiguous(), ctx.needs_input_grad[0], ctx.needs_input_grad[2])
        return ga, None, gb, None


def relation_losses(result):
    """[class_loss, rel_loss] of a training `Result` (mean cross-entropy over the object rows / the sampled relation rows)"""
    a, la = result.rm_obj_dists, result.rm_obj_labels
    b, lb = result.rel_dists, result.rel_labels[:, -1]
    if (FUSED and a.is_cuda and a.dtype == torch.float32 and b.dtype == torch.float32 and la.dtype == torch.int64 and lb.dtype == torch.int64
            and a.shape[0] > 0 and b.shape[0] > 0 and la.dim() == 1):
        return _CrossEntropyPairFn.apply(a, la, b, lb)
    return torch.stack((F.cross_entropy(a, la), F.cross_entropy(b, lb)))


# ---- learning from another model's rows (csrc/label_dist.hip) -------------------------------------------------------------------
TopLogits = collections.namedtuple('TopLogits', ('values', 'indices', 'rest'))
TopLogits.__doc__ = """A teacher's record of its rows: values [R,k] (its k largest logits, descending), indices [R,k] (their classes, int32 or
int64; -1 leaves an entry out) and rest [R] fp32 (log-sum-exp of all other logits / temperature) or None."""


def _temperature(temperature):
    if not (isinstance(temperature, (int, float)) and 1e-30 <= temperature <= 1e30):
        raise ValueError('temperature must be a number above 0 (1e-30 to 1e30), got %r' % (temperature,))
    return float(temperature)


def top_logits(logits, k, temperature=1.0):
    """The record of a teacher's rows [R,V] (fp32, fp16 or bf16) that `distill_loss` learns from: the first k classes of every row in
    descending order (ties: the lowest class; NaN first) and the log-sum-exp of the others at the temperature of the later loss.
    k is at most the number of classes and 1024.  No gradient."""
    if not isinstance(k, int) or not 1 <= k <= logits.shape[-1]:
        raise ValueError('k must be a whole number between 1 and the %d classes, got %r' % (logits.shape[-1], k))
    return TopLogits(*_hip.top_logits(logits.detach(), k, _temperature(temperature)))


class _DistillFn(torch.autograd.Function):
    """The gradient at an upstream of 1 is made by the forward pass where the kernels have it in the same pass over memory; the backward pass
    then only looks at the upstream on the device, and computes anew where it is another (never a product of the rounded gradient: a loss
    scale would come too late for what fp16 has lost).  A second backward pass of the same node computes its own, and so does one that is captured
    into a graph, or run, apart from its forward pass: the one may then be replayed without the other.  The gradient is saved like the inputs, so
    that a checkpoint drops it with them and hooks that move saved tensors away move it too."""
    @staticmethod
    def forward(ctx, logits, values, indices, rest, temperature, row_weight, reduction, scale, graded):
        args = _hip.distill_args(logits, values, indices, rest, temperature, row_weight, scale)
        rows, total, stats, grad = _hip.distill_run_fwd(args, logits.device, reduction, logits.dtype if graded else None)
        ctx.unused = grad is not None
        ctx.capture = None if grad is None else _hip.capture_id(logits.device)
        ctx.save_for_backward(logits, values, indices, rest, row_weight, stats, grad)
        ctx.temperature, ctx.scale, ctx.reduced = temperature, scale, total is not None
        return total if ctx.reduced else rows

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        # (the saved tensors may be others than forward's: offloaded ones, a checkpoint's second run)
        logits, values, indices, rest, row_weight, stats, grad = ctx.saved_tensors
        args = _hip.distill_args(logits, values, indices, rest, ctx.temperature, row_weight, ctx.scale)
        unused, ctx.unused = ctx.unused, False
        if unused and ctx.capture == _hip.capture_id(logits.device):
            grad = grad.data             # (the caller may change it in place: a retained node's saved tensor is not asked about that)
        else:
            grad = None
        return (_hip.distill_run_bwd(args, logits.device, logits.dtype, stats, ctx.reduced, g.reshape(-1).contiguous(), grad),
                None, None, None, None, None, None, None, None)


def distill_loss(logits, teacher, temperature=1.0, row_weight=None, reduction='mean', scale=1.0):
    """scale T^2 KL(teacher || student) of a student's rows [R,V] (fp32, fp16 or bf16) against a teacher's record, with the gradient of the
    student's logits.  With teacher.rest the classes outside the record are one more bin on both sides; without, the teacher's mass is
    that of its k entries.  The record's temperature must be this one.  row_weight [R] fp32: a row of weight 0 counts for nothing,
    whatever it holds.  reduction: 'mean' (over the sum of the weights, or the rows), 'sum', 'none' ([R]).  A row whose logits are
    all -inf, or whose record is, has loss and gradient 0; a class the student excludes (-inf) and the teacher does not makes the loss inf.
    Neither the teacher nor row_weight gets a gradient; a row_weight that asks for one is refused.  A weight of this loss among others belongs into `scale`: the gradient is made with the loss for an upstream of
    1, and any other upstream costs a second pass over the rows."""
    if not (isinstance(scale, (int, float)) and abs(scale) <= 1e30):
        raise ValueError('scale must be a finite number, got %r' % (scale,))
    if reduction not in ('mean', 'sum', 'none'):
        raise ValueError("reduction must be 'mean', 'sum' or 'none', got %r" % (reduction,))
    if row_weight is not None and row_weight.requires_grad and torch.is_grad_enabled():
        raise ValueError('row_weight gets no gradient from this loss: give it detached')
    values, indices, rest = (t if t is None or (t.is_contiguous() and not t.requires_grad) else t.detach().contiguous() for t in teacher)
    if values.dim() != 2 or not 1 <= values.shape[1] <= _hip.MAX_TOP:
        raise ValueError('a record holds 1 to %d entries a row, got values of shape %s' % (_hip.MAX_TOP, tuple(values.shape)))
    return _DistillFn.apply(logits, values, indices, rest, _temperature(temperature), row_weight, reduction, float(scale),
                            logits.requires_grad and torch.is_grad_enabled())
