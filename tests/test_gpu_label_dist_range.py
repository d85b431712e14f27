"""Label distributions where the classes outside a record stand far below (or above) those inside it, at the ends of the number range, and what a
call keeps until its backward pass (csrc/label_dist.hip: lib/losses.py top_logits / distill_loss).

Bounds.  u = 2^-24.  A side of a row is its classes inside the record or those outside it; d_i = (largest of the side - logit) / T.  A weight
exp(-d_i) is off by u (8 d_i + 32) of itself: the difference, the constant log2(e) / T and the product round once each, a partial sum's lowering
to the side's maximum as often again, the exponential by two steps, and its argument holds rounded logarithms of at most log V.  A sum of positive
terms adds its depth, at most V / 512 + 32 additions.  So a side's sum is off by delta = u (mean of 8 d_i + 32 under the weights + V / 512 + 32), the sum of
all by the larger of the two sides', and with log q_rest and log q from them a row's loss by T^2 w (p_rest (delta_out + delta_all) + (1 - p_rest)
delta_all), and by two roundings of the loss itself.  An outside class has the gradient T w share (q_rest - p_rest), share = exp(-d_i) over the
side's sum; an inside one T w (q - p) with p in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def side(x, T):
    """(largest logit, sum of the weights below it, bound of that sum's relative error, the weights, the bounds of each) of some classes of a row"""
    top = x.max() if x.size else -np.inf
    if top == -np.inf:
        return top, 0.0, 0.0, np.zeros(x.size), np.zeros(x.size)
    d = (top - x) / T
    w = np.exp(-d)
    each = U * (8 * np.where(w > 0, d, 0.0) + 32)
    return top, w.sum(), (w * each).sum() / w.sum() + U * (x.size / 512 + 32), w, each


def divergence(x, t, idx, rest, T, w):
    """loss, its bound, gradient and its bound of one row, in 64 bits, with a maximum of its own for either side"""
    V = len(x)
    y = t / T if rest is None else np.append(t / T, rest)
    p = np.exp(y - y.max())
    logp = y - y.max() - math.log(p.sum())
    p = p / p.sum()
    out = np.ones(V, bool)
    if rest is not None:
        out[idx] = False
    mo, so, eo, wo, each = side(x[out], T)
    mi, si, ei, _, _ = side(x[~out], T)
    m, e = max(mo, mi), max(eo, ei)
    logs = math.log((so * math.exp((mo - m) / T) if so else 0.0) + (si * math.exp((mi - m) / T) if si else 0.0))
    logq = (x[idx] - m) / T - logs
    logqr = (mo - m) / T + math.log(so) - logs if so else -math.inf
    pr = 0.0 if rest is None else p[-1]
    if rest is not None:
        logq = np.append(logq, logqr)
    on = p > 0
    loss = T * T * w * np.sum(p[on] * (logp[on] - logq[on]))
    tol = T * T * w * (pr * (eo + e) + (1 - pr) * e) + 2 * U * abs(loss) + 1e-37
    grad, bound = np.zeros(V), np.zeros(V)
    qr = math.exp(logqr) if rest is not None else 1.0
    if so:
        share = wo / so
        grad[out] = T * w * share * (qr - pr)
        bound[out] = T * w * share * ((qr + pr) * (each + eo) + qr * (e + eo))
    if rest is not None:
        q = np.exp((x[idx] - m) / T - logs)
        np.add.at(grad, idx, T * w * (q - p[:-1]))
        np.add.at(bound, idx, T * w * q * (e + 4 * U) + 2.0 ** -40 * T * w * p[:-1])
    else:
        np.subtract.at(grad, idx, T * w * p)
        np.add.at(bound, idx, 2.0 ** -40 * T * w * p)
    return loss, tol, grad, bound


def check(x, values, indices, rest, T, reduction='mean', upstream=1.0):
    from lib.losses import TopLogits, distill_loss
    R, V = x.shape
    n = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    rows = [divergence(n(x)[r], n(values)[r], indices[r].cpu().numpy(), None if rest is None else float(rest[r]), T, 1.0) for r in range(R)]
    loss, tol = np.array([r[0] for r in rows]), np.array([r[1] for r in rows])
    grad, bound = np.stack([r[2] for r in rows]), np.stack([r[3] for r in rows])
    assert np.isfinite(loss).all()
    leaf = x.detach().requires_grad_(True)
    got = distill_loss(leaf, TopLogits(values, indices, rest), T, reduction=reduction)
    g = n(got)
    if reduction == 'none':
        assert np.all(np.abs(g - loss) <= tol), (g, loss, tol)
        up = torch.linspace(0.5, 1.5, R, device=x.device) * upstream
        got.backward(up)
        up = n(up)[:, None]
    else:
        over = R if reduction == 'mean' else 1
        assert abs(g - loss.sum() / over) <= (tol.sum() + U * (R / 1024 + 12) * np.abs(loss).sum()) / over, (g, loss, tol)
        (got * upstream).backward()
        up = upstream / over
    got, want = n(leaf.grad), grad * up
    step = torch.finfo(x.dtype).eps / 2
    lim = np.abs(bound * up) * 1.01 + (step + 4 * U) * np.abs(want) + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)
    bad = ~(np.abs(got - want) <= lim)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], lim[bad][:5])


def rows_with_gaps(V, dtype, T, gaps, sure, seed):
    """a row for each gap: the student's largest class, in the record, stands `gap` nats above the largest class outside.  sure: the teacher is
    the student itself, else it leaves the classes outside a share of 5 to 50 %"""
    g = torch.Generator().manual_seed(seed)
    R, k = len(gaps), 6
    x = torch.randn(R, V, generator=g, dtype=torch.float64) * 2.5 * min(T, 1.0)
    idx = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(R)])
    out = torch.ones(R, V, dtype=torch.bool).scatter_(1, idx, False)
    top = x.masked_fill(~out, -math.inf).amax(1)
    x[torch.arange(R), idx[:, 2]] = top + torch.tensor(gaps, dtype=torch.float64) * T
    x = x.to(dtype)
    if sure:
        values = x.gather(1, idx)
        rest = (x.double() / T).masked_fill(~out, -math.inf).logsumexp(1).float()
    else:
        values = torch.randn(R, k, generator=g, dtype=torch.float64).mul_(T).to(dtype)
        rest = ((values.double() / T).logsumexp(1) + torch.linspace(-3, 0, R, dtype=torch.float64)).float()
    return x.cuda(), values.cuda(), idx.int().cuda(), rest.cuda()


GAPS = [20.0, 60.0, 80.0, 88.0, 95.0, 104.0, 120.0, 300.0, 400.0, 740.0, 800.0, 2000.0]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T', [0.1, 0.5, 1.0, 2.0])
@pytest.mark.parametrize('V', [51, 2048, 2049, 5000, 70001])
def test_classes_outside_the_record_far_below(V, T, dtype):
    for sure in (False, True):
        rows = rows_with_gaps(V, dtype, T, GAPS, sure, V + int(10 * T))
        check(*rows, T)
        check(*rows, T, reduction='sum', upstream=-3.0)
        check(*rows, T, reduction='none')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [51, 2049, 70001])
def test_classes_outside_the_record_far_above(V, dtype):
    """the record's classes hold next to nothing of the student's mass"""
    x, values, idx, rest = rows_with_gaps(V, dtype, 1.0, [-90.0] * 3, False, V)
    for r, gap in enumerate((90.0, 300.0, 2000.0)):
        low = x[r].double().min() - gap
        x[r, idx[r].long()] = (low + torch.randn(6, device='cuda', dtype=torch.float64, generator=torch.Generator('cuda').manual_seed(r))).to(dtype)
    check(x, values, idx, rest, 1.0)
    check(x, values, idx, rest, 1.0, reduction='none')
    check(x, values, idx, None, 1.0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T', [0.5, 1.0, 1.4426950408889634, 2.0])
@pytest.mark.parametrize('V', [51, 2049, 5000, 70001])
def test_classes_masked_with_the_lowest_value(V, T, dtype):
    """a student whose classes outside the record, some or all of them, stand at the type's lowest value, and a teacher that gives them mass"""
    lowest = float(torch.finfo(dtype).min)
    x, values, idx, rest = rows_with_gaps(V, dtype, T, [3.0] * 5, False, V)
    kept = x.clone()
    x[:2] = lowest
    x[2, ::2] = lowest
    x[3, :V * 2 // 3] = lowest
    x.scatter_(1, idx.long(), kept.gather(1, idx.long()))
    rest = (values.double() / T).logsumexp(1).float() - 3.0
    if T == 2.0 and dtype == torch.float32:
        rest = rest - 1.0            # (T p_rest times the lowest value has to stay a 32-bit number)
    check(x, values, idx, rest, T)
    check(x, values, idx, rest, T, reduction='none')
    check(x, values, idx, None, T, reduction='none')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [51, 2049, 5000, 70001])
def test_every_class_at_the_lowest_value(V, dtype):
    """equal classes, wherever they stand; T = log2(e) makes the exponent's constant 1"""
    for T in (1.4426950408889634, 1.0, 1.4426951, 1.4426949, 0.3, 5.0):
        x, values, idx, rest = rows_with_gaps(V, dtype, T, [3.0] * 2, False, V)
        x.fill_(float(torch.finfo(dtype).min))
        check(x, values, idx, rest, T)
        check(x, values, idx, None, T)
        check(x, values, idx, rest, T, reduction='none')


@pytest.mark.parametrize('shift', [1e6, 2e8, 1e9, 2e10, 1e13, -2e8, -1e9, -1e13, 3e38, -3e38])
@pytest.mark.parametrize('V', [51, 5000, 70001])
def test_logits_far_from_zero(V, shift):
    """the row's own size cancels: differences of its classes are what counts"""
    for T in (1.0, 2.0, 0.01):
        x, values, idx, rest = rows_with_gaps(V, torch.float32, 1.0, [3.0, 100.0], False, V)
        x = x.double() * T + shift * torch.tensor([[1.0], [0.5]], device='cuda', dtype=torch.float64)
        rest = (values.double() / T).logsumexp(1).float() - 2.0
        for t in (torch.float32, torch.bfloat16):
            check(x.to(t), values, idx, rest, T)
            check(x.to(t), values, idx, None, T, reduction='none')


@pytest.mark.parametrize('V', [40, 300, 5000, 70001])
def test_rest_of_a_record_with_nan_and_infinity_outside(V):
    """a NaN among the classes outside the record makes their sum a NaN, whatever else stands there; +inf alone makes it +inf"""
    from lib.losses import top_logits
    for dtype in TYPES:
        x = torch.randn(4, V, generator=torch.Generator().manual_seed(V)).to(dtype)
        x[0, 5:25] = math.nan                  # more NaNs than entries, and an infinity behind or before them
        x[0, V - 1] = math.inf
        x[1, 5:25] = math.nan
        x[1, 0] = math.inf
        x[2, 5:25] = math.inf
        x[3, 5:13] = math.nan                  # all of them inside: the infinity is the largest outside
        x[3, 30] = math.inf
        rest = top_logits(x.cuda(), 8).rest.cpu()
        assert math.isnan(rest[0]) and math.isnan(rest[1])
        assert rest[2] == math.inf and rest[3] == math.inf


# ---- the longest row --------------------------------------------------------------------------------------------------------------------

def test_drawing_from_the_longest_row():
    """2^31 - 1 classes, cut over workgroups and not: four of them weigh anything, the ends among them"""
    from lib import _hip
    from lib.sampling import sample_labels
    n = 2 ** 31 - 1
    x = torch.full((1, n), -math.inf, dtype=torch.bfloat16, device='cuda')
    at = [n - 1, 0, 2 ** 30 + 1, n - 9]
    x[0, at] = torch.tensor([3.0, 2.0, 1.0, 0.5], dtype=torch.bfloat16, device='cuda')
    w = np.exp(np.array([3.0, 2.0, 1.0, 0.5]))
    cum = np.cumsum(w) / w.sum()
    assert _hip.lib().mh_sample_ws_bytes(1, n) > 0
    for u in (0.1, 0.7, 0.9, 0.999):
        want = at[int(np.sum(cum <= u))]
        assert sample_labels(x, torch.full((1,), u, device='cuda')).tolist() == [want]
    assert sample_labels(x, torch.full((1,), 0.99, device='cuda'), top_p=0.9).tolist() == [at[2]]
    assert sample_labels(x, torch.full((1,), 0.99, device='cuda'), top_k=2).tolist() == [at[1]]


# ---- what a call keeps until its backward pass ------------------------------------------------------------------------------------------

R, V = 2048, 4000            # (a gradient of 33 MB)


def growth(call):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    kept = call()
    torch.cuda.synchronize()
    return kept, torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before


def student_and_record():
    from lib.losses import top_logits
    g = torch.Generator('cuda').manual_seed(4)
    x = torch.randn(R, V, generator=g, device='cuda', requires_grad=True)
    return x, top_logits(torch.randn(R, V, generator=g, device='cuda'), 8)


def test_no_gradient_is_made_where_none_can_be_asked_for():
    from lib.losses import distill_loss
    x, rec = student_and_record()
    with torch.no_grad():
        _, _, most = growth(lambda: distill_loss(x, rec))
    assert most < R * V
    with torch.inference_mode():
        _, _, most = growth(lambda: distill_loss(x, rec))
    assert most < R * V


def test_checkpoints_and_offloading_hold_no_gradient():
    """a checkpoint drops what the forward pass saved, and hooks that move saved tensors away move all of them"""
    from torch.utils.checkpoint import checkpoint
    from lib.losses import distill_loss
    x, rec = student_and_record()
    (want,) = torch.autograd.grad(distill_loss(x * 1.0, rec), x)
    loss, held, _ = growth(lambda: checkpoint(lambda x: distill_loss(x * 1.0, rec), x, use_reentrant=False))
    assert held < R * V
    assert torch.equal(torch.autograd.grad(loss, x)[0], want)

    def offloaded():
        with torch.autograd.graph.save_on_cpu():
            return distill_loss(x * 1.0, rec)
    loss, held, _ = growth(offloaded)
    assert held < R * V
    assert torch.equal(torch.autograd.grad(loss, x)[0], want)


def test_a_gradient_that_was_handed_out_is_the_callers():
    """changed in place, it is not what a second backward pass gives, and that pass is not refused"""
    from lib.losses import distill_loss
    x, rec = student_and_record()
    loss = distill_loss(x, rec)
    (first,) = torch.autograd.grad(loss, x, retain_graph=True)
    want = first.clone()
    first.zero_()
    (second,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(second, want)
    second.zero_()
    (third,) = torch.autograd.grad(loss * 1.0, x)
    assert torch.equal(third, want)
