"""
Drawing labels from rows of class logits (csrc/label_dist.hip) -- what the label decoder does instead of its arg-max when it is asked
for a draw (reference lib/lstm/decoder_rnn.py:205-227 commits the arg-max).
"""
import math

import torch

from lib import _hip


def sample_labels(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One label of every row [R,V] (fp32, fp16 or bf16) from the numbers u [R] (fp32, uniform in [0, 1)): int64 [R].

    The classes stand in descending order (ties: the lowest class) with weights exp(logit / temperature).  Of these the first top_k (0: all)
    are left, of their weight the shortest head with at least top_p, of that the classes with at least min_p times the best one's weight;
    never fewer than one.  The label is the first class at which the running weight exceeds u times what is left: the same
    inputs give the same labels.  temperature 0 is the arg-max.  Every parameter is a number or a [R] tensor (fp32, top_k int32) with a value
    for each row; in a tensor, values outside the range mean what include/motifs_hip.h says.  A row whose logits are all -inf, or hold a
    NaN, gives -1.  Nothing is read back to the host."""
    for v, name, lo, hi in ((temperature, 'temperature', 0.0, math.inf), (top_p, 'top_p', 0.0, 1.0), (min_p, 'min_p', 0.0, 1.0)):
        if not torch.is_tensor(v) and not (isinstance(v, (int, float)) and lo <= v <= hi and v < math.inf):
            raise ValueError('%s must be a number between %g and %g or a tensor, got %r' % (name, lo, hi, v))
    if not torch.is_tensor(top_k) and not (isinstance(top_k, int) and 0 <= top_k < 2 ** 31):
        raise ValueError('top_k must be a whole number of at least 0 or a tensor, got %r' % (top_k,))
    return _hip.sample_labels(logits.detach(), u, temperature, top_k, top_p, min_p)
