"""Label distributions (csrc/label_dist.hip: lib/losses.py top_logits / distill_loss, lib/sampling.py sample_labels) against plain
implementations in 64 bits on the host.

Bounds.  u = 2^-24 is fp32's largest relative rounding error; L = (range of the finite logits / T) + log V + 2 bounds every exponent and
logarithm of a row.  A log-probability is a difference of rounded terms of at most L: (logit - max), its product with 1/T, the exponential's
argument (its rounding, L u, is the sum's relative error), the logarithm, two differences -- 8 of them on the teacher's side and 8 on the
student's: 16 L u; a probability is off by 8 L u of itself, against a difference of logs of at most L.  So a row's loss is within
T^2 u (16 L + 8 L^2).  A gradient T w (q f - p) has q, f = 1 - p_rest / q_rest and p within 16 L u of their own sizes: u 16 L T w (q + q p_rest /
q_rest + p), then the rounding to the logits' type, half a step: eps / 2 of the value, or half of fp16's smallest subnormal 2^-24.
The rest of a record: log-sum-exp with one division: u (16 L + |rest|)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def dev(t):
    return t.cuda()


def make(R, V, dtype, seed, offset=0, kind='spread'):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V + offset, generator=g, dtype=torch.float64) * 2.5
    if kind == 'masked':
        x[torch.rand(x.shape, generator=g) < 0.4] = -math.inf
        x[1::3] = -math.inf
    elif kind == 'lowest':
        x[torch.rand(x.shape, generator=g) < 0.4] = float(torch.finfo(dtype).min)
        x[1::3] = float(torch.finfo(dtype).min)
    elif kind == 'ties':
        x = x.round().clamp(-2, 2)
    elif kind == 'equal':
        x = torch.full_like(x, 1.5)
    elif kind == 'far':
        x = x + 900.0
    elif kind == 'peaked':
        x[torch.arange(x.shape[0]), torch.arange(x.shape[0]) % x.shape[1]] += 60.0
    elif kind == 'sorted':
        x = x.sort(1)[0]
    return x.to(dtype)


def order_of(x):
    """the classes of every row in the operators' order: descending, ties to the lowest class, NaN in front"""
    key = np.where(np.isnan(x), np.inf, x)
    return np.stack([np.lexsort((np.arange(x.shape[1]), -key[r], ~np.isnan(x[r]))) for r in range(x.shape[0])]) if len(x) else np.zeros(x.shape, np.int64)


def span(x, T):
    f = x[np.isfinite(x) & (np.abs(x) < 1e30)]
    return ((f.max() - f.min()) if f.size else 0.0) / T + math.log(max(x.shape[1], 1)) + 2.0


# ---- top logits ---------------------------------------------------------------------------------------------------------------

def check_top(x, k, T):
    from lib.losses import top_logits
    got = top_logits(x, k, T)
    xd = x.detach().double().cpu().numpy()
    order = order_of(xd)
    want = np.take_along_axis(xd, order, 1)
    np.testing.assert_array_equal(got.indices.cpu().numpy(), order[:, :k])
    np.testing.assert_array_equal(got.values.double().cpu().numpy(), want[:, :k])
    assert got.values.dtype == x.dtype and got.indices.dtype == torch.int32 and got.rest.dtype == torch.float32
    rest = got.rest.double().cpu().numpy()
    others = want[:, k:] / T
    for r in range(xd.shape[0]):
        o = others[r]
        if o.size == 0 or np.all(np.isneginf(o)):
            assert rest[r] == -np.inf
        elif np.isnan(o).any():
            assert np.isnan(rest[r])
        else:
            m = o.max()
            if m == np.inf:
                assert rest[r] == np.inf
                continue
            ref = m + math.log(np.exp(o - m).sum())
            with np.errstate(over='ignore'):
                if np.isinf(np.float32(ref)):
                    assert rest[r] == np.float32(ref)
                    continue
            assert abs(rest[r] - ref) <= U * (16 * span(xd[r:r + 1], T) + abs(ref)), (r, rest[r], ref)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('R,V,k,T', [(1, 1, 1, 1.0), (3, 2, 1, 0.5), (5, 3, 3, 2.0), (7, 51, 8, 2.0), (66, 64, 64, 1.0), (9, 65, 33, 1.0), (4, 151, 151, 4.0),
                                     (3, 257, 100, 1.0), (5, 512, 9, 1.0), (6, 513, 1, 1.0), (2, 1023, 1000, 1.5), (2, 1024, 1024, 1.0), (3, 1025, 1024, 0.7),
                                     (2, 2049, 64, 1.0), (3, 5001, 17, 1.0), (2, 33333, 256, 3.0), (1, 131073, 64, 1.0), (1, 262147, 1024, 1.0), (300, 4100, 20, 1.0)])
def test_top_logits(R, V, k, T, dtype):
    check_top(dev(make(R, V, dtype, 7 * R + V)), k, T)


@pytest.mark.parametrize('kind', ['masked', 'lowest', 'ties', 'equal', 'far', 'peaked', 'sorted'])
@pytest.mark.parametrize('V,k', [(151, 20), (900, 31), (6000, 40), (6000, 1000), (70001, 5)])
def test_top_logits_hard_rows(V, k, kind):
    for dtype in TYPES:
        check_top(dev(make(4, V, dtype, 3, kind=kind)), k, 0.9)


def test_top_logits_nan_and_infinities():
    for V in (40, 300, 5000):
        for dtype in TYPES:
            x = make(6, V, dtype, 5)
            x[0, V // 2] = math.nan
            x[1, 1] = math.inf
            x[1, V - 1] = math.inf
            x[2, 3] = -math.inf
            x[3, ::2] = math.nan
            x[4, ::2] = math.inf
            x[4, 1] = -math.inf
            x[5, 0], x[5, 2] = 0.0, -0.0
            check_top(dev(x), 7, 1.0)


def test_top_logits_views():
    x = dev(make(40, 152, torch.bfloat16, 2))
    check_top(x[:, 1:], 10, 1.0)
    check_top(x[::3, 2:150], 10, 1.0)
    check_top(x[:1].expand(9, 152), 5, 1.0)
    y = dev(make(3, 7003, torch.float16, 2))
    for off in (1, 2, 3, 5):
        check_top(y[:, off:], 10, 1.0)
    check_top(x[:0], 3, 1.0)


# ---- distillation ----------------------------------------------------------------------------------------------------------------

def plain_distill(x, values, indices, rest, T, w, V):
    """loss, gradient and gradient bound of every row, in 64 bits, one row after the other from the formulas"""
    R = x.shape[0]
    loss, grad, bound = np.zeros(R), np.zeros((R, V)), np.zeros((R, V))
    tol = np.zeros(R)
    for r in range(R):
        wr = 1.0 if w is None else w[r]
        use = (indices[r] >= 0) & (indices[r] < V)
        t, idx = values[r][use], indices[r][use]
        if wr == 0 or not use.any() or np.all(np.isneginf(t)) or np.all(np.isneginf(x[r])):
            continue
        y = t / T
        if rest is not None:
            y = np.append(y, rest[r])
        p = np.exp(y - y.max())
        logp = y - y.max() - math.log(p.sum())
        p = p / p.sum()
        e = np.exp((x[r] - x[r].max()) / T)
        q = e / e.sum()
        with np.errstate(divide='ignore'):
            logq = np.log(q[idx])
        out = np.ones(V, bool)
        out[idx] = False
        if rest is not None:
            qr = q[out].sum()
            with np.errstate(divide='ignore'):
                logq = np.append(logq, np.log(qr))
        on = p > 0
        loss[r] = T * T * wr * np.sum(p[on] * (logp[on] - logq[on]))
        g = q.copy()
        b = q.copy()
        if rest is not None and qr > 0:
            g[out] -= q[out] * p[-1] / qr
            b[out] += q[out] * p[-1] / qr
        np.subtract.at(g, idx, p[:len(idx)])
        np.add.at(b, idx, p[:len(idx)])
        grad[r] = T * wr * g
        L = max(span(x[r:r + 1], T), span(values[r:r + 1].astype(np.float64), T))
        if rest is not None and np.isfinite(rest[r]):
            L += abs(rest[r])        # rest is a rounded number of its own size
        bound[r] = 16 * L * U * T * abs(wr) * b
        tol[r] = T * T * abs(wr) * U * (16 * L + 8 * L * L)
    return loss, grad, bound, tol


def check_distill(x, values, indices, rest, T, w=None, reduction='mean', upstream=1.0):
    from lib.losses import TopLogits, distill_loss
    x = x.detach().requires_grad_(True)
    R, V = x.shape
    n = lambda t: None if t is None else t.detach().double().cpu().numpy()  # noqa: E731
    loss, grad, bound, tol = plain_distill(n(x), n(values), indices.cpu().numpy(), n(rest), T, n(w), V)
    total = 1.0
    if reduction == 'mean':
        total = float(R) if w is None else float(n(w).sum())
        total = total or 1.0
    got = distill_loss(x, TopLogits(values, indices, rest), T, w, reduction)
    assert got.dtype == torch.float32
    g = got.detach().double().cpu().numpy()
    if reduction == 'none':
        assert got.shape == (R,)
        fine = np.isfinite(loss)
        np.testing.assert_array_equal(g[~fine], loss[~fine])
        assert np.all(np.abs(g - loss)[fine] <= tol[fine]), np.max((np.abs(g - loss) - tol)[fine])
        ups = torch.linspace(0.5, 1.5, R, device=x.device) * upstream if R else x.new_zeros(0, dtype=torch.float32)
        got.backward(ups)
        ups = ups.double().cpu().numpy()[:, None]
    else:
        # a sum of R rounded rows in 32 bits, at most R / 1024 + 10 additions deep
        assert abs(g - loss.sum() / total) <= (tol.sum() + U * (R / 1024 + 12) * np.abs(loss).sum()) / total or not np.isfinite(loss.sum()) and g == loss.sum()
        (got * upstream).backward()
        ups = upstream / total
    gx = x.grad
    assert gx.dtype == x.dtype and gx.shape == x.shape
    got_g, want = gx.double().cpu().numpy(), grad * ups
    step = torch.finfo(x.dtype).eps / 2
    lim = np.abs(bound * ups) * 1.01 + (step + 4 * U) * np.abs(want) + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)
    bad = ~(np.abs(got_g - want) <= lim)
    assert not bad.any(), (np.argwhere(bad)[:5], got_g[bad][:5], want[bad][:5], lim[bad][:5])


def record(x, k, T, rest=True, seed=0, noise=1.0):
    """a teacher's record near x, taken on the host: distinct classes, any order of the entries"""
    g = torch.Generator().manual_seed(seed + 11)
    xd = x.detach().double().cpu()
    t = torch.where(torch.isfinite(xd), xd, torch.zeros_like(xd)) + noise * torch.randn(xd.shape, generator=g, dtype=torch.float64)
    t = t.masked_fill(xd == -math.inf, -math.inf).to(x.dtype)
    v, i = t.double().sort(dim=1, descending=True, stable=True)
    others = (v[:, k:] / T).logsumexp(1) if k < xd.shape[1] else torch.full((xd.shape[0],), -math.inf, dtype=torch.float64)
    return dev(v[:, :k].to(x.dtype)), dev(i[:, :k].int()), dev(others.float()) if rest else None


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rest', [True, False])
@pytest.mark.parametrize('R,V,k,T', [(1, 1, 1, 1.0), (2, 2, 1, 1.0), (5, 3, 2, 2.0), (120, 151, 16, 2.0), (33, 51, 51, 1.0), (17, 64, 8, 4.0), (5, 65, 64, 1.0), (9, 1000, 65, 1.0),
                                     (3, 1024, 1024, 1.0), (4, 1025, 7, 0.5), (3, 4099, 300, 1.0), (2, 65537, 33, 1.5), (1, 200001, 64, 1.0)])
def test_distill(R, V, k, T, rest, dtype):
    x = dev(make(R, V, dtype, R + V))
    check_distill(x, *record(x, k, T, rest), T)


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_distill_reductions_and_weights(reduction):
    for V in (151, 3000):
        x = dev(make(37, V, torch.float32, 4))
        w = dev(torch.rand(37, generator=torch.Generator().manual_seed(1)))
        w[::4] = 0
        for rest in (True, False):
            check_distill(x, *record(x, 9, 1.3, rest), 1.3, w, reduction, upstream=0.37)
            check_distill(x, *record(x, 9, 1.3, rest), 1.3, None, reduction, upstream=-2.0)
            check_distill(x, *record(x, 9, 1.3, rest), 1.3, torch.zeros_like(w), reduction)


@pytest.mark.parametrize('kind', ['masked', 'lowest', 'ties', 'equal', 'far', 'peaked'])
@pytest.mark.parametrize('V,k', [(51, 8), (151, 140), (5000, 40)])
def test_distill_hard_rows(V, k, kind):
    for dtype in TYPES:
        x = dev(make(7, V, dtype, 9, kind=kind))
        if kind == 'lowest' and dtype == torch.float32:      # (range of the finite logits: the masked classes stand at the type's lowest value)
            check_distill(x, *record(x, k, 1.0, True, noise=0.0), 1.0)
            continue
        for rest in (True, False):
            check_distill(x, *record(x, k, 1.0, rest, noise=0.0 if kind == 'lowest' else 1.0), 1.0)


def test_distill_excluded_classes():
    """a class the student excludes and the teacher does not: the loss is inf, the gradient finite"""
    x = make(4, 30, torch.float32, 1)
    values, indices, rest = record(x, 6, 1.0)
    xs = x.clone()
    xs[1, indices[1, 2].item()] = -math.inf
    gone = torch.ones(30, dtype=torch.bool)
    gone[indices[2].cpu().long()] = False
    xs[2, gone] = -math.inf                                  # nothing left outside the record, the teacher has some mass there
    check_distill(dev(xs), values, indices, rest, 1.0, reduction='none')


def test_distill_entries():
    """left-out entries (-1, beyond the classes), int64 classes, a class named twice and three times, unordered entries, another type"""
    for V in (51, 700, 9000):
        x = dev(make(6, V, torch.float32, 1))
        values, indices, rest = record(x, 12, 2.0)
        indices = indices.long()
        indices[0, 3] = -1
        indices[1, :] = -1
        indices[2, 0] = V
        indices[2, 1] = 2 ** 40
        indices[3, 5] = indices[3, 0]
        indices[3, 7] = indices[3, 0]
        indices[4, 11] = indices[4, 3]
        indices[5] = indices[5].flip(0)
        values[5] = values[5].flip(0)
        for r in (rest, None):
            for reduction in ('mean', 'none'):
                check_distill(x, values, indices, r, 2.0, reduction=reduction)
                check_distill(x.bfloat16(), values.half(), indices, r, 2.0, reduction=reduction)


def test_distill_rows_of_weight_zero_may_hold_anything():
    from lib.losses import TopLogits, distill_loss
    for V in (51, 3001):
        x = make(5, V, torch.float32, 1)
        values, indices, rest = record(x, 4, 1.0)
        x[2] = math.nan
        values[2] = math.nan
        w = torch.tensor([1.0, 0.5, 0.0, 2.0, 0.0])
        keep = [0, 1, 3]
        xs = dev(x).requires_grad_(True)
        loss = distill_loss(xs, TopLogits(values, indices, rest), 1.0, dev(w))
        loss.backward()
        part = dev(x[keep]).requires_grad_(True)
        ref = distill_loss(part, TopLogits(values[keep], indices[keep], rest[keep]), 1.0, dev(w[keep]))
        ref.backward()
        assert abs(loss.item() - ref.item()) <= 8 * U * abs(ref.item())
        assert torch.equal(xs.grad[2], torch.zeros_like(xs.grad[2])) and torch.equal(xs.grad[4], torch.zeros_like(xs.grad[4]))
        assert torch.equal(xs.grad[keep], part.grad)
        nan = dev(x).requires_grad_(True)                       # and with a weight the NaN is seen
        assert math.isnan(distill_loss(nan, TopLogits(values, indices, rest), 1.0).item())


def test_distill_gradient_against_differences():
    """central differences of the kernel's own loss: with step h the loss of a row is off by h^2 / 6 of its third derivative (at most T^-1 here)
    and by its rounding over h"""
    from lib.losses import TopLogits, distill_loss
    x = dev(make(1, 40, torch.float32, 3))
    values, indices, rest = record(x, 6, 2.0)
    rec = TopLogits(values, indices, rest)
    xs = x.clone().requires_grad_(True)
    distill_loss(xs, rec, 2.0, reduction='sum').backward()
    h = 0.03125
    rows = x.repeat(80, 1)
    for c in range(40):
        rows[2 * c, c] += h
        rows[2 * c + 1, c] -= h
    many = TopLogits(values.repeat(80, 1), indices.repeat(80, 1), rest.repeat(80))
    f = distill_loss(rows, many, 2.0, reduction='none').double().view(40, 2)
    L = span(x.double().cpu().numpy(), 2.0)
    lim = h * h / 6 + 4 * U * (16 * L + 8 * L * L) / h
    assert float(((f[:, 0] - f[:, 1]) / (2 * h) - xs.grad[0].double()).abs().max()) <= lim


@pytest.mark.parametrize('dtype', TYPES)
def test_distill_scale_and_upstream(dtype):
    """a factor inside the loss, and an upstream other than 1 (computed anew, not multiplied): the same gradient, bit for bit, where the
    factor is a power of two; fp16 keeps what a loss scale is there to keep"""
    from lib.losses import TopLogits, distill_loss
    for V in (151, 3000, 70001):
        x = dev(make(6, V, dtype, 2))
        rec = TopLogits(*record(x, 9, 1.5))
        grads = []
        for scale, up in ((1024.0, 1.0), (1.0, 1024.0), (32.0, 32.0)):
            leaf = x.clone().requires_grad_(True)
            loss = distill_loss(leaf, rec, 1.5, scale=scale)
            (loss * up).backward()
            grads.append((leaf.grad, loss.detach() / scale))
        for g, l in grads[1:]:
            assert torch.equal(g, grads[0][0]) and torch.equal(l, grads[0][1])
        assert float(grads[0][0].double().abs().max()) > 0


def test_distill_views_and_second_backward():
    from lib.losses import TopLogits, distill_loss
    base = dev(make(20, 53, torch.bfloat16, 6))
    x = base[:, 1:52]
    check_distill(x, *record(x, 8, 1.0), 1.0)
    check_distill(x[::2], *record(x[::2], 8, 1.0), 1.0)
    one = base[:1].expand(7, 53)
    check_distill(one, *record(one, 8, 1.0), 1.0)
    wide = dev(make(4, 6002, torch.float16, 6))[:, 1:]
    check_distill(wide, *record(wide, 8, 1.0), 1.0)
    leaf = base.clone().requires_grad_(True)             # through a view, twice, accumulated
    rec = TopLogits(*record(x, 8, 1.0))
    loss = distill_loss(leaf[:, 1:52], rec)
    loss.backward(retain_graph=True)
    first = leaf.grad.clone()
    loss.backward()
    assert torch.equal(leaf.grad, first + first) and float(leaf.grad[:, 0].abs().max()) == 0.0
    scaled = distill_loss(leaf[:, 1:52], rec)            # a loss may be changed in place, as where gradients are accumulated
    scaled /= 4
    leaf.grad = None
    scaled.backward()
    assert torch.equal(leaf.grad * 4, first)
    rows = distill_loss(leaf[:, 1:52], rec, reduction='none')
    rows *= 0.25
    leaf.grad = None
    rows.sum().backward()
    assert float((leaf.grad.double() * 4 / 20 - first.double()).abs().max()) <= 2.0 ** -7 * float(first.abs().max())
    empty = x[:0].detach().requires_grad_(True)
    z = TopLogits(rec.values[:0], rec.indices[:0], rec.rest[:0])
    out = distill_loss(empty, z)
    out.backward()
    assert out.item() == 0.0 and empty.grad.shape == (0, 51)


# ---- sampling -------------------------------------------------------------------------------------------------------------------------

def plain_sample(x, u, T, k, p, m):
    """one row in 64 bits"""
    if np.isnan(x).any() or np.all(np.isneginf(x)):
        return -1
    order = np.lexsort((np.arange(len(x)), -x))
    if not T > 0:
        return int(order[0])
    s = x[order]
    with np.errstate(invalid='ignore'):
        w = np.exp(np.where(s == s[0], 0.0, s - s[0]) / T)
    n = len(x) if not 0 < k <= len(x) else int(k)
    cum = np.cumsum(w)
    keep = n
    if p < 1:
        before = np.concatenate(([0.0], cum[:-1]))
        keep = min(keep, int(np.sum(before[:n] < max(p, 0.0) * cum[n - 1])))
    if m > 0:
        keep = min(keep, int(np.sum(w >= m)))
    keep = max(keep, 1)
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)
    return int(order[min(int(np.sum(cum[:keep] <= u * cum[keep - 1])), keep - 1)])


def check_sample(x, u, T=1.0, k=0, p=1.0, m=0.0):
    from lib.sampling import sample_labels
    got = sample_labels(x, u, T, k, p, m)
    R = x.shape[0]
    assert got.dtype == torch.int64 and got.shape == (R,)
    f = lambda v: v.double().cpu().numpy() if torch.is_tensor(v) else np.full(R, float(np.float32(v)))  # noqa: E731
    xd, ud, Td, kd, pd, md = x.double().cpu().numpy(), f(u), f(T), f(k), f(p), f(m)
    want = np.array([plain_sample(xd[r], ud[r], Td[r], int(kd[r]), pd[r], md[r]) for r in range(R)], dtype=np.int64)
    np.testing.assert_array_equal(got.cpu().numpy(), want)


def numbers(R, seed):
    return dev(torch.rand(R, generator=torch.Generator().manual_seed(seed)))


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.95, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (2.0, 1500, 0.8, 0.001), (0.0, 5, 0.5, 0.5),
            (0.05, 0, 0.99, 0.0), (30.0, 0, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 3, 0.0, 0.0), (1.0, 0, 0.6, 1.0), (1.0, 40, 0.7, 0.02)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('R,V', [(1, 1), (6, 2), (64, 51), (40, 150), (9, 64), (9, 65), (20, 500), (10, 1024), (10, 1025), (8, 2050), (12, 9001), (3, 100003), (1, 262147)])
def test_sample(R, V, dtype):
    x = dev(make(R, V, dtype, R * 3 + V))
    for i, (T, k, p, m) in enumerate(SETTINGS):
        check_sample(x, numbers(R, i), T, k, p, m)


@pytest.mark.parametrize('kind', ['masked', 'lowest', 'ties', 'equal', 'far', 'peaked', 'sorted'])
@pytest.mark.parametrize('V', [40, 700, 5003, 70001])
def test_sample_hard_rows(V, kind):
    for dtype in TYPES:
        x = dev(make(7, V, dtype, 13, kind=kind))
        for i, (T, k, p, m) in enumerate(SETTINGS):
            if kind == 'equal' and p < 1:
                p = 0.6123            # (equal weights: a share of their number that is no whole number)
            check_sample(x, numbers(7, 50 + i), T, k, p, m)


def test_sample_rows_with_their_own_parameters():
    for V in (150, 3001):
        R = 48
        x = dev(make(R, V + 1, torch.float32, 21))[:, 1:]
        g = torch.Generator().manual_seed(2)
        T, p, m = torch.rand(R, generator=g) * 2, torch.rand(R, generator=g), torch.rand(R, generator=g) * 0.2
        k = torch.randint(-2, V + 3, (R,), generator=g, dtype=torch.int32)
        T[3], T[4], p[5], p[6], p[7], m[8], m[9], m[10] = 0.0, -1.0, 2.0, math.nan, -1.0, math.nan, 7.0, -1.0
        T[11] = math.nan
        u = torch.rand(R, generator=g)
        u[12], u[13], u[14], u[15], u[16] = 0.0, 1.0, math.nan, -3.0, 2.0
        k[17], k[18] = 2 ** 31 - 1, -2 ** 31
        check_sample(x, dev(u), dev(T), dev(k), dev(p), dev(m))
        check_sample(x, dev(u), dev(T), 7, dev(p), 0.0)


def test_sample_nan_infinities_and_ties():
    for V in (30, 3000):
        for dtype in TYPES:
            x = make(6, V, dtype, 1)
            x[0, V // 3] = math.nan
            x[1, 2] = math.inf
            x[2, 1] = math.inf
            x[2, V - 1] = math.inf
            x[3] = -math.inf
            x[4] = -math.inf
            x[4, V - 2] = -5.0
            x[5, 0], x[5, 1:] = 0.0, -0.0
            for i, (T, k, p, m) in enumerate(SETTINGS[:9]):
                check_sample(dev(x), numbers(6, i), T, k, 0.777 if p < 1 else p, m)


def test_sample_frequencies():
    """the draws of many numbers follow softmax: with u = (i + 1/2) / n the counts are n q to within one on either border"""
    from lib.sampling import sample_labels
    n = 4096
    x = dev(make(1, 20, torch.float32, 8))
    u = (torch.arange(n, device='cuda').float() + 0.5) / n
    got = torch.bincount(sample_labels(x.expand(n, 20), u), minlength=20).double().cpu()
    q = torch.softmax(x.double(), 1)[0].cpu()
    assert float((got - n * q).abs().max()) <= 2.0


# ---- together, streams, graphs ---------------------------------------------------------------------------------------------------------

def test_a_record_is_learned_and_answered_from():
    """teacher rows -> record -> a student's gradient step towards them -> labels, on a stream of its own"""
    from lib.losses import distill_loss, top_logits
    from lib.sampling import sample_labels
    teacher = dev(make(64, 151, torch.float32, 1))
    student = dev(make(64, 151, torch.float32, 2)).requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rec = top_logits(teacher, 10, 2.0)
        loss = distill_loss(student, rec, 2.0)
        loss.backward()
        labels = sample_labels(teacher[:, 1:], numbers(64, 1), top_k=5) + 1
    torch.cuda.current_stream().wait_stream(s)
    check_top(teacher, 10, 2.0)
    check_distill(student, *rec, 2.0)
    same = distill_loss(teacher, rec, 2.0, reduction='none')
    L = span(teacher.double().cpu().numpy(), 2.0) + float(rec.rest.abs().max())
    assert float(same.abs().max()) <= 4 * U * (16 * L + 8 * L * L)          # a student that is the teacher
    assert int(labels.min()) >= 1 and int(labels.max()) <= 150
    check_sample(teacher[:, 1:], numbers(64, 1), k=5)


@pytest.mark.parametrize('R,V', [(24, 151), (3, 70001)])
def test_captured_and_replayed(R, V):
    """all three in one graph, replayed on new inputs between eager work: equal to the eager calls, bit for bit"""
    from lib import _hip
    from lib.losses import TopLogits, top_logits, distill_loss
    from lib.sampling import sample_labels
    x, t, u = dev(make(R, V, torch.float32, 1)), dev(make(R, V, torch.float32, 2)), numbers(R, 3)
    one = torch.ones(1, device='cuda')

    def all_of_it():
        rec = top_logits(t, 8, 1.5)
        rows, total, stats = _hip.distill_fwd(x, *rec, 1.5, None, 'mean')
        grad = _hip.distill_bwd(x, *rec, 1.5, None, stats, total, one)
        return rec.values, rec.indices, rec.rest, total, grad, sample_labels(x, u, 0.9, 0, 0.9), sample_labels(x, u, 0.9, 30, 0.9, 0.01)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        all_of_it()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = all_of_it()
    for seed in (5, 6, 7):
        x.copy_(make(R, V, torch.float32, seed))
        t.copy_(make(R, V, torch.float32, seed + 10))
        u.copy_(numbers(R, seed))
        want = [o.clone() for o in all_of_it()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        leaf = x.clone().requires_grad_(True)
        distill_loss(leaf, TopLogits(*want[:3]), 1.5).backward()
        assert torch.equal(leaf.grad, want[4])


def test_the_same_inputs_give_the_same_bits():
    from lib.losses import TopLogits, distill_loss, top_logits
    from lib.sampling import sample_labels
    x, t, u = dev(make(5, 40001, torch.bfloat16, 1)), dev(make(5, 40001, torch.bfloat16, 2)), numbers(5, 3)
    runs = []
    for _ in range(3):
        rec = top_logits(t, 33, 1.0)
        leaf = x.clone().requires_grad_(True)
        loss = distill_loss(leaf, TopLogits(*rec))
        loss.backward()
        runs.append([*rec, loss.detach(), leaf.grad, sample_labels(x, u, 1.0, 0, 0.9)])
    for other in runs[1:]:
        for a, b in zip(runs[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize('V', [51, 5000, 70000])
def test_distill_backward_reads_what_autograd_unpacks(V):
    """saved tensors that were moved away, or made anew by a checkpoint, while the forward pass's memory holds something else"""
    from torch.utils.checkpoint import checkpoint
    from lib.losses import distill_loss, top_logits
    rec = top_logits(dev(make(37, V, torch.float32, 91)), 7, 1.5)
    weight = dev(torch.linspace(0.5, 2.0, 37))
    x = dev(make(37, V, torch.float32, 92))

    def loss_of(x):
        return distill_loss(x * 1.0, rec, 1.5, row_weight=weight * 1.0)

    def grad_of(make_loss):
        leaf = x.clone().requires_grad_()
        loss = make_loss(leaf)
        junk = [torch.full((37, V), 7.0, device='cuda') for _ in range(4)]
        (loss * 3.0).backward()
        del junk
        return leaf.grad

    def offloaded(leaf):
        with torch.autograd.graph.save_on_cpu():
            return loss_of(leaf)

    want = grad_of(loss_of)
    assert torch.equal(grad_of(offloaded), want)
    assert torch.equal(grad_of(lambda leaf: checkpoint(loss_of, leaf, use_reentrant=False)), want)


@pytest.mark.parametrize('R,V', [(24, 151), (9, 5000)])
def test_forward_in_a_graph_and_backward_outside(R, V):
    """a gradient that was handed out is the caller's: the next replay of the forward pass leaves it as it is"""
    from lib.losses import distill_loss, top_logits
    rec = top_logits(dev(make(R, V, torch.float32, 21)), 8, 1.5)
    x = dev(make(R, V, torch.float32, 22)).requires_grad_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        distill_loss(x, rec, 1.5)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = distill_loss(x, rec, 1.5)
    got, want = [], []
    for seed in (23, 24, 25):
        x.data.copy_(make(R, V, torch.float32, seed))
        graph.replay()
        got.append(torch.autograd.grad(loss, x, retain_graph=True)[0])
        eager = x.detach().clone().requires_grad_()
        want += torch.autograd.grad(distill_loss(eager, rec, 1.5), eager)
        torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize('R,V', [(24, 151), (9, 5000), (3, 70001)])
def test_graphed_callable(R, V):
    """forward and backward in graphs of their own, with upstreams of 1 and others, backward twice after one forward pass"""
    from lib.losses import distill_loss, top_logits
    rec = top_logits(dev(make(R, V, torch.float32, 21)), 8, 1.5)
    graphed = torch.cuda.make_graphed_callables(lambda x: distill_loss(x, rec, 1.5), (dev(make(R, V, torch.float32, 22)).requires_grad_(),))
    for seed, factors in ((23, (1.0,)), (24, (2.0, 1.0)), (25, (1.0, 0.5, 1.0))):
        x = dev(make(R, V, torch.float32, seed))
        for f in factors:
            a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
            mine, theirs = graphed(a), distill_loss(b, rec, 1.5)
            assert torch.equal(mine, theirs)
            for g in (f, 1.0):
                up = torch.full((), g, device='cuda')
                got, want = (torch.autograd.grad(l, t, up, retain_graph=True)[0].clone() for l, t in ((mine, a), (theirs, b)))
                torch.cuda.synchronize()
                assert torch.equal(got, want)


def test_more_rows_than_a_launch_holds():
    """refused by name, on rows that are one row of memory; one less is answered"""
    from lib._hip import HipKernelError
    from lib.losses import top_logits
    from lib.sampling import sample_labels
    row = dev(make(1, 51, torch.float32, 31))
    with pytest.raises(HipKernelError, match='range'):
        top_logits(row.expand(2 ** 23, 51), 2)
    with pytest.raises(HipKernelError, match='range'):
        sample_labels(row.expand(2 ** 23, 51), torch.zeros(2 ** 23, device='cuda'))
    most = 2 ** 23 - 1
    rec, one = top_logits(row.expand(most, 51), 2), top_logits(row, 2)
    for a, b in zip(rec, one):
        assert bool((a == b).all())
    long_row = dev(make(1, 300, torch.float32, 32))
    labels = sample_labels(long_row.expand(most, 300), torch.full((most,), 0.5, device='cuda'))
    assert bool((labels == sample_labels(long_row, torch.full((1,), 0.5, device='cuda'))).all())
