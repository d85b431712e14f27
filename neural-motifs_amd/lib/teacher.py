"""
A trained relation model as the teacher of another one (models/train_rels.py -distill): its top logits for the SAME object and relation
rows as the student's, and the student's loss against them (lib/losses.py top_logits, distill_loss).
"""
import collections

import numpy as np
import torch

from lib.losses import distill_loss, top_logits
from lib.pytorch_misc import has_host, host_np

Records = collections.namedtuple('Records', ('obj', 'rel', 'rel_labels'))


class RelTeacher(object):
    """model: a RelModel (GT-box modes) that is not trained on: it runs as in training -- sampled relation rows, labels fed to the decoder --
    with dropout off and its BatchNorms' running statistics, and without gradients.
    k_obj, k_rel: entries of a row's record; temperature: of the loss that learns from it."""

    def __init__(self, model, k_obj=16, k_rel=8, temperature=2.0):
        if model.mode not in ('sgcls', 'predcls'):
            raise ValueError('a teacher needs the same rows as its student: GT-box modes (sgcls, predcls), not %r' % (model.mode,))
        self.model, self.temperature = model, temperature
        self.k_obj, self.k_rel = min(k_obj, model.num_classes), min(k_rel, model.num_rels)
        for p in model.parameters():
            p.requires_grad = False
        self._as_in_training()

    def _as_in_training(self):
        m = self.model
        m.eval()                                        # dropout off, running statistics; then only what decides about the rows
        context = getattr(m, 'context', None)           # (the message-passing baseline has none)
        for part in (m, m.detector, context):
            if part is not None:
                part.training = True
        decoder = getattr(context, 'decoder_rnn', None)
        if decoder is not None:
            decoder.training = True                     # labels are fed back, not its own answers
            decoder.recurrent_dropout_probability = 0.0

    def records(self, batch, sampler_rs):
        """the teacher's records of a dataloader blob; sampler_rs: a numpy RandomState in the state the student's sampler will start from"""
        self.model.sampler_rs = sampler_rs
        with torch.no_grad():
            result = self.model[batch]
            obj = None if self.model.mode == 'predcls' else top_logits(result.rm_obj_dists, self.k_obj, self.temperature)
            return Records(obj, top_logits(result.rel_dists, self.k_rel, self.temperature), result.rel_labels)

    def losses(self, result, records, scale=1.0):
        """[objects, relations]: the student's mean divergences from the records, times `scale`; objects is 0 where labels are given
        (predcls).  `result`: the student's, of the same blob and the same sampler state"""
        mine, theirs = result.rel_labels, records.rel_labels
        same = mine.shape == theirs.shape
        if same and has_host(mine) and has_host(theirs):
            same = bool(np.array_equal(host_np(mine), host_np(theirs)))
        if not same:
            raise RuntimeError("the teacher's relation rows are not the student's: give both the same sampler state")
        rel = distill_loss(result.rel_dists, records.rel, self.temperature, scale=scale)
        obj = torch.zeros_like(rel) if records.obj is None else distill_loss(result.rm_obj_dists, records.obj, self.temperature, scale=scale)
        return obj, rel
