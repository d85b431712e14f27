"""
The label-distribution operators and the calls that are timed: a teacher's top logits, distillation from them with its gradient,
and drawing labels with temperature, top-k, top-p and min-p.

A case is a dict of plain values:
  op       'top' | 'distill' | 'sample'
  rows, classes, dtype ('f32' | 'f16' | 'bf16'), offset (leading columns of the stored rows that the call leaves out, as the
  label decoder leaves out the background class), mask (1: about a third of the classes of a row are excluded with -inf, and
  every 64th row has none left)
  top:     k, temperature
  distill: k, temperature, rest (1: the record holds the mass of the other classes), weight (1: a weight for each row, some of them 0),
           grad (1: a training step's loss and gradient, 0: a validation pass that keeps the loss of every row)
  sample:  temperature, top_k, top_p, min_p, per_row (1: every row has parameters of its own around these)
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}


def _top(name, rows, classes, dtype, k, temperature=1.0, offset=0, mask=0):
    return dict(name=name, op='top', rows=rows, classes=classes, dtype=dtype, offset=offset, mask=mask, k=k, temperature=temperature)


def _distill(name, rows, classes, dtype, k, temperature=1.0, rest=1, weight=0, grad=1, offset=0, mask=0):
    return dict(name=name, op='distill', rows=rows, classes=classes, dtype=dtype, offset=offset, mask=mask, k=k, temperature=temperature,
                rest=rest, weight=weight, grad=grad)


def _sample(name, rows, classes, dtype, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, per_row=0, offset=0, mask=0):
    return dict(name=name, op='sample', rows=rows, classes=classes, dtype=dtype, offset=offset, mask=mask, temperature=temperature,
                top_k=top_k, top_p=top_p, min_p=min_p, per_row=per_row)


def listed():
    return [
        # the record of one batch's relation rows (6 images x 256 sampled pairs, 50 predicates + background)
        _top('top_relations', 1536, 51, 'f32', 8, 2.0),
        # the record of a batch over an open vocabulary
        _top('top_words', 2048, 32000, 'bf16', 32),
        # one row of an odd, large vocabulary: latency
        _top('top_one', 1, 100003, 'f32', 64),
        # the object rows of a batch of 6 images (about 20 boxes each)
        _distill('distill_objects', 120, 151, 'f32', 16, 2.0),
        # its relation rows
        _distill('distill_relations', 1536, 51, 'f32', 8, 2.0),
        # a training step over an open vocabulary, the largest case
        _distill('distill_words', 4096, 32000, 'bf16', 64),
        # an odd vocabulary, padded rows of weight 0, a record without the others' mass
        _distill('distill_padded', 777, 50021, 'f16', 33, 1.5, rest=0, weight=1),
        # validation: the loss of every row, no gradient
        _distill('distill_validate', 2048, 32000, 'f32', 32, grad=0),
        # label decoding: rows of 151 classes without the background column, parameters for each row
        _sample('sample_objects', 384, 150, 'f32', 0.9, 20, 0.9, 0.01, per_row=1, offset=1),
        # one row a step, the usual settings: latency
        _sample('sample_one', 1, 32000, 'f32', 0.8, 50, 0.95),
        # a batch of answers over an odd vocabulary, masked classes, no top-k
        _sample('sample_batch', 64, 100003, 'bf16', 1.0, 0, 0.9, 0.001, mask=1),
        # many rows, top-p alone
        _sample('sample_many', 1024, 65536, 'f16', 1.0, 0, 0.95),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(('top', 'distill', 'sample'))
    dtype = rng.choice(('f32', 'f16', 'bf16'))
    most = {'top': 2048 * 32000, 'distill': 4096 * 32000, 'sample': 1024 * 65536}[op] // (2 if dtype == 'f32' else 1)
    classes = _spread(rng, 2, 131072)
    rows = _spread(rng, 1, min(4096, most // classes))
    more = dict(offset=rng.choice((0, 0, 1, 3)), mask=rng.choice((0, 1)))
    temperature = round(rng.uniform(0.5, 2.5), 3)
    if op == 'top':
        case = _top('', rows, classes, dtype, _spread(rng, 1, min(classes, 256)), temperature, **more)
    elif op == 'distill':
        case = _distill('', rows, classes, dtype, _spread(rng, 1, min(classes, 256)), temperature, rest=rng.choice((0, 1)),
                        weight=rng.choice((0, 1)), grad=rng.choice((0, 1, 1)), **more)
    else:
        case = _sample('', rows, classes, dtype, rng.choice((0.0, 1.0, temperature, temperature, temperature)),
                       rng.choice((0, _spread(rng, 1, min(classes, 1024)))), rng.choice((1.0, round(rng.uniform(0.5, 0.99), 3))),
                       rng.choice((0.0, round(10 ** rng.uniform(-4, -0.7), 5))), per_row=rng.choice((0, 1)), **more)
    del case['name']
    return case


def _logits(g, case, like=None, noise=1.0):
    """rows as a trained head gives them: a broad bulk and a few classes well above it.  like: another model's rows of the same images"""
    R, V = case['rows'], case['classes'] + case['offset']
    x = torch.randn(R, V, generator=g, device='cuda')
    if like is None:
        hot = min(V, 12)
        at = (torch.randint(0, V, (R, 1), generator=g, device='cuda') + torch.arange(hot, device='cuda') * (V // hot)) % V      # no class twice
        up = torch.rand(R, hot, generator=g, device='cuda') * 8 + 2
        x = (x * 2).scatter_add_(1, at, up)
    else:
        x = like.float() + noise * x
    return x.to(_TYPES[case['dtype']])


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    R, V, off = case['rows'], case['classes'], case['offset']
    state = dict(case)
    x = _logits(g, case)
    out = None
    if case['mask']:
        out = torch.rand(x.shape, generator=g, device='cuda') < 0.3
        out[63::64] = True
        x = x.masked_fill_(out, -math.inf)
    state['logits'] = x[:, off:]
    if case['op'] == 'distill':
        T, k = case['temperature'], case['k']
        teacher = _logits(g, case, like=torch.where(torch.isfinite(x), x, 0.0))
        if out is not None:
            teacher = teacher.masked_fill_(out, -math.inf)
        teacher = teacher[:, off:].float()
        values, indices = teacher.topk(k, 1)
        state['values'], state['indices'] = values.to(x.dtype), indices.int()
        state['rest'] = (teacher / T).scatter_(1, indices, -math.inf).logsumexp(1) if case['rest'] else None
        state['row_weight'] = None
        if case['weight']:
            w = torch.rand(R, generator=g, device='cuda') + 0.5
            state['row_weight'] = w * (torch.rand(R, generator=g, device='cuda') < 0.8)
        state['logits'] = state['logits'].detach().requires_grad_(bool(case['grad']))
    if case['op'] == 'sample':
        state['u'] = torch.rand(R, generator=g, device='cuda')
        if case['per_row']:
            f = lambda: torch.rand(R, generator=g, device='cuda')  # noqa: E731
            state['temperature'] = case['temperature'] * (f() + 0.5)
            state['top_k'] = torch.randint(0, 2 * case['top_k'] + 1, (R,), generator=g, device='cuda', dtype=torch.int32)
            state['top_p'] = case['top_p'] + (1 - case['top_p']) * f()
            state['min_p'] = case['min_p'] * f()
    return state


# ---- the plain forms ------------------------------------------------------------------------------------------------------

def _plain_top(s):
    x, order = s['logits'].float().sort(dim=1, descending=True, stable=True)
    k = s['k']
    others = x[:, k:] / s['temperature']
    if others.shape[1] == 0:
        rest = x.new_full((x.shape[0],), -math.inf)
    else:
        m = others.amax(1)
        safe = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
        rest = torch.log(torch.exp(others - safe[:, None]).sum(1)) + safe
    return {'values': x[:, :k].to(s['logits'].dtype), 'indices': order[:, :k].int(), 'rest': rest}


def _plain_distill(s):
    x, T, k = s['logits'].detach().float(), s['temperature'], s['k']
    idx, t = s['indices'].long(), s['values'].float()
    zero = torch.zeros((), device=x.device)
    # the teacher: softmax over its k logits (and the others' mass)
    top = t.amax(1, keepdim=True)
    y = (t - top) / T
    if s['rest'] is not None:
        y = torch.cat((y, (s['rest'][:, None] - top / T)), 1)
    shift = y.amax(1, keepdim=True)
    ey = torch.exp(y - shift)
    logp = y - shift - torch.log(ey.sum(1, keepdim=True))
    p = torch.exp(logp)
    # the student
    m = x.amax(1, keepdim=True)
    e = torch.exp((x - m) / T)
    S = e.sum(1, keepdim=True)
    logq = (x.gather(1, idx) - m) / T - torch.log(S)
    others = e.scatter(1, idx, 0.0)
    O = others.sum(1, keepdim=True)
    if s['rest'] is not None:
        logq = torch.cat((logq, torch.log(O) - torch.log(S)), 1)
    live = (torch.isfinite(m) & torch.isfinite(top))[:, 0]
    rows = T * T * torch.where(p > 0, p * (logp - logq), zero).sum(1)
    rows = torch.where(live, rows, zero)
    w = s['row_weight']
    rows = rows if w is None else torch.where(w != 0, rows * w, zero)
    if not s['grad']:
        return {'rows': rows}
    total = torch.tensor(float(x.shape[0]), device=x.device) if w is None else w.sum()
    total = torch.where(total == 0, torch.ones_like(total), total)
    grad = e / S
    if s['rest'] is not None:
        share = torch.where(O > 0, p[:, k:] / O, zero)
        grad = grad - others * share
    grad.scatter_add_(1, idx, -p[:, :k])
    scale = T / total if w is None else T * w / total
    grad = torch.where(live[:, None], grad * scale.reshape(-1, 1), zero)
    return {'loss': rows.sum() / total, 'grad': grad.to(s['logits'].dtype)}


def _column(v, R, like, dtype):
    return (v if torch.is_tensor(v) else torch.full((R,), v, device=like.device, dtype=dtype))[:, None]


def _plain_sample(s):
    x = s['logits'].double()
    R, V = x.shape
    T = _column(s['temperature'], R, x, torch.float32).double()
    top_k = _column(s['top_k'], R, x, torch.int32).long()
    top_p = _column(s['top_p'], R, x, torch.float32).double()
    min_p = _column(s['min_p'], R, x, torch.float32).double()
    u = s['u'][:, None].double().clamp(0.0, 1.0 - 2.0 ** -24)
    x, order = x.sort(dim=1, descending=True, stable=True)
    head = x[:, :1]
    d = torch.where(x == head, torch.zeros_like(x), x - head)
    w = torch.exp(d / torch.where(T > 0, T, torch.ones_like(T)))
    cum = w.cumsum(1)
    n_k = torch.where((top_k <= 0) | (top_k > V), V, top_k)
    mass = cum.gather(1, n_k - 1)
    before = torch.cat((torch.zeros_like(cum[:, :1]), cum[:, :-1]), 1)
    n_p = torch.where(top_p < 1, (before < top_p * mass).sum(1, keepdim=True), V)
    n_m = torch.where(min_p > 0, (w >= min_p).sum(1, keepdim=True), V)
    n = torch.minimum(torch.minimum(n_k, n_p), n_m).clamp(min=1)
    target = u * cum.gather(1, n - 1)
    at = torch.minimum((cum <= target).sum(1, keepdim=True), n - 1)
    at = torch.where(T > 0, at, torch.zeros_like(at))
    label = order.gather(1, at)[:, 0]
    return torch.where(torch.isnan(head[:, 0]) | (head[:, 0] == -math.inf), torch.full_like(label, -1), label)


def run(state):
    op = state['op']
    if own:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'neural-motifs_amd')
        if root not in sys.path:
            sys.path.insert(0, root)
        from lib.losses import TopLogits, distill_loss, top_logits
        from lib.sampling import sample_labels
        if op == 'top':
            got = top_logits(state['logits'], state['k'], state['temperature'])
            return {'values': got.values, 'indices': got.indices, 'rest': got.rest}
        if op == 'distill':
            teacher = TopLogits(state['values'], state['indices'], state['rest'])
            if not state['grad']:
                return {'rows': distill_loss(state['logits'], teacher, state['temperature'], state['row_weight'], reduction='none')}
            loss = distill_loss(state['logits'], teacher, state['temperature'], state['row_weight'], reduction='mean')
            return {'loss': loss.detach(), 'grad': torch.autograd.grad(loss, state['logits'])[0]}
        return {'labels': sample_labels(state['logits'], state['u'], state['temperature'], state['top_k'], state['top_p'], state['min_p'])}
    if op == 'top':
        return _plain_top(state)
    if op == 'distill':
        return _plain_distill(state)
    return {'labels': _plain_sample(state)}


def work(case):
    R, V, b = case['rows'], case['classes'], 4 if case['dtype'] == 'f32' else 2
    n = R * V
    if case['op'] == 'top':         # a comparison, a subtraction, a scaling, an exponential and a sum for each class
        return {'bytes': n * b + R * case['k'] * (b + 4) + R * 4, 'flops': 5 * n}
    if case['op'] == 'distill':
        extra = R * case['k'] * (b + 4) + R * 4 * (case['rest'] + case['weight'])
        if case['grad']:
            return {'bytes': 2 * n * b + extra + 4, 'flops': 9 * n}
        return {'bytes': n * b + extra + R * 4, 'flops': 5 * n}
    return {'bytes': n * b + R * 12 + 16 * R * case['per_row'], 'flops': 5 * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def _exact_top(s):
    x = s['logits'].double().cpu().numpy()
    k, T = s['k'], s['temperature']
    order = np.argsort(-x, axis=1, kind='stable')
    ranked = np.take_along_axis(x, order, 1)
    others = ranked[:, k:] / T
    with np.errstate(all='ignore'):
        rest = np.full(x.shape[0], -np.inf)
        if others.shape[1]:
            m = others[:, 0]
            rest = np.where(np.isneginf(m), -np.inf, m + np.log(np.exp(others - m[:, None]).sum(1)))
    return {'values': ranked[:, :k], 'indices': order[:, :k].astype(np.int32), 'rest': rest}


def _exact_distill_rows(x, t, idx, rest, T):
    """KL(teacher || student) of every row, by torch's own differentiation in 64 bits"""
    k = t.shape[1]
    live = torch.isfinite(x).any(1) & torch.isfinite(t).any(1)
    x = torch.where(live[:, None], x, torch.zeros_like(x))
    t = torch.where(live[:, None], t, torch.zeros_like(t))
    logits = [t / T]
    logq = torch.log_softmax(x / T, 1)
    student = [logq.gather(1, idx)]
    if rest is not None:
        logits.append(rest[:, None])
        taken = torch.zeros_like(x, dtype=torch.bool).scatter_(1, idx, True)
        kept = torch.where(taken, torch.full_like(logq, -math.inf), logq)
        some = torch.isfinite(kept).any(1, keepdim=True)
        student.append(torch.where(some, torch.where(some, kept, torch.zeros_like(kept)).logsumexp(1, keepdim=True), torch.full_like(kept[:, :1], -math.inf)))
    p = torch.softmax(torch.cat(logits, 1), 1)
    q = torch.cat(student, 1)
    q = torch.where(p > 0, q, torch.zeros_like(q))
    rows = (torch.special.xlogy(p, p) - p * q).sum(1) * T * T
    return torch.where(live, rows, torch.zeros_like(rows))


def _exact_distill(s):
    R, V = s['logits'].shape
    step = max(1, (1 << 25) // V)
    w = torch.ones(R, dtype=torch.float64, device='cuda') if s['row_weight'] is None else s['row_weight'].double()
    total = float(w.sum()) or 1.0
    rows, grads = [], []
    for a in range(0, R, step):
        x = s['logits'][a:a + step].detach().double().requires_grad_(True)
        rest = None if s['rest'] is None else s['rest'][a:a + step].double()
        r = _exact_distill_rows(x, s['values'][a:a + step].double(), s['indices'][a:a + step].long(), rest, s['temperature']) * w[a:a + step]
        if s['grad']:
            grads.append((torch.autograd.grad(r.sum(), x)[0] / total).nan_to_num(nan=0.0))
        rows.append(r.detach())
    rows = torch.cat(rows)
    return {'loss': rows.sum() / total, 'grad': torch.cat(grads)} if s['grad'] else {'rows': rows}


def _exact_sample(s):
    R = s['logits'].shape[0]
    val = lambda k: (s[k].double().cpu().numpy() if torch.is_tensor(s[k]) else np.full(R, np.float32(s[k]), dtype=np.float64))  # noqa: E731
    T, top_k, top_p, min_p, u = val('temperature'), val('top_k').astype(np.int64), val('top_p'), val('min_p'), val('u')
    labels = np.full(R, -1, dtype=np.int64)
    logits = s['logits'].double().cpu().numpy()
    for r in range(R):
        x = logits[r]
        best = x.max()
        if np.isnan(best) or best == -np.inf:
            continue
        if not T[r] > 0:
            labels[r] = int(np.argmax(x))
            continue
        order = np.argsort(-x, kind='stable')
        w = np.exp((x[order] - best) / T[r])
        n = len(x) if not 0 < top_k[r] <= len(x) else int(top_k[r])
        first = np.cumsum(w[:n])
        keep = n
        if top_p[r] < 1:
            keep = min(keep, int(np.searchsorted(first, top_p[r] * first[-1], side='left')) + 1)
        if min_p[r] > 0:
            keep = min(keep, int((w >= min_p[r]).sum()))
        keep = max(keep, 1)
        labels[r] = order[min(int(np.searchsorted(first[:keep], u[r] * first[keep - 1], side='right')), keep - 1)]
    return {'labels': labels}


def exact(case, seed):
    if case['op'] != 'distill' and case['rows'] * case['classes'] > 70_000_000:
        return None          # sorting every row on the host takes too long
    state = prepare(case, seed)
    if case['op'] == 'top':
        return _exact_top(state)
    if case['op'] == 'distill':
        return _exact_distill(state)
    return _exact_sample(state)
