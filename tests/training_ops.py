"""Plain 64-bit forms of the training operators (embedding, token log probabilities, preference loss, AdamW) on the CPU, and
the error bounds that the tests of the kernels use.

Bounds count roundings: U = 2^-24 is half a step of fp32 relative to the value, `half(dtype)` half a step of an output type.  A
sum of n products formed in fp32 in any order is off by at most (n + 1) U times the sum of the absolute values."""
import torch

U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step of the type: what a value that is rounded to a subnormal is off by."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what=''):
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), torch.as_tensor(bound, dtype=torch.float64).cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), what + ': NaN in other places'
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), what + ': infinities'
    off = ((got - want).abs() - bound)[~(want.isnan() | inf)]
    assert off.numel() == 0 or off.max() <= 0, '%s: off by %.3g beyond the bound' % (what, off.max())


# ---------------------------------------------------------------- embedding
def embedding(table, ids, scale, combiner):
    """(out, sum of absolute values) in float64."""
    t, i = table.double().cpu(), ids.long().cpu()
    rows = torch.zeros(tuple(i.shape) + (t.shape[1],), dtype=torch.float64)
    inside = (i >= 0) & (i < t.shape[0])
    if inside.any():
        rows[inside] = t[i[inside]]
    rows[i >= t.shape[0]] = float('nan')
    if combiner is None:
        return rows * scale, rows.abs() * abs(scale)
    f = torch.full(i.shape[:-1], float(scale), dtype=torch.float64)
    if combiner == 'mean':
        f = f / (i >= 0).sum(-1).clamp(min=1)
    return rows.sum(-2) * f.unsqueeze(-1), rows.abs().sum(-2) * f.abs().unsqueeze(-1)


def embedding_gradient(grad, ids, rows, scale, combiner):
    """(gradient, sum of absolute values, occurrences of each row) in float64."""
    g, i = grad.double().cpu(), ids.long().cpu()
    dim = g.shape[-1]
    if combiner is not None:
        f = torch.full(i.shape[:-1], float(scale), dtype=torch.float64)
        if combiner == 'mean':
            f = f / (i >= 0).sum(-1).clamp(min=1)
        g = (g * f.unsqueeze(-1)).unsqueeze(-2).expand(tuple(i.shape) + (dim,))
    else:
        g = g * scale
    i, g = i.reshape(-1), g.reshape(-1, dim)
    ok = (i >= 0) & (i < rows)
    i, g = i[ok], g[ok]
    out = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, i, g)
    size = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, i, g.abs())
    return out, size, torch.bincount(i, minlength=rows).double()


# ---------------------------------------------------------------- token log probabilities
def log_probs(logits, targets, temperature):
    z = logits.double().cpu() / temperature
    z = z - z.amax(-1, keepdim=True)          # of logits as low as -3e38 fp64 keeps differences only
    t = targets.long().cpu()
    v = z.shape[-1]
    lse = torch.logsumexp(z, -1)
    out = z.gather(-1, t.clamp(0, v - 1).unsqueeze(-1)).squeeze(-1) - lse
    out = torch.where(t >= v, torch.nan, out)
    return torch.where(t < 0, 0.0, out)


def log_probs_gradient(grad, logits, targets, temperature):
    z = logits.double().cpu() / temperature
    t = targets.long().cpu().unsqueeze(-1)
    v = z.shape[-1]
    p = torch.softmax(z, -1)
    hot = torch.zeros_like(p).scatter_(-1, t.clamp(0, v - 1), 1.0)
    out = (hot - p) * grad.double().cpu().unsqueeze(-1) / temperature
    out = torch.where(t >= v, torch.nan, out)
    return torch.where(t < 0, 0.0, out), p


def log_probs_bounds(logits, targets, temperature):
    """(bound on log probabilities, relative bound on probabilities), one a row.

    An exponential's argument (x - max) / T is off by 3 U of itself (difference, factor, product) and the exponential by 2 U
    more; terms far below the maximum weigh e^-d, so that the sum's relative error from its arguments is at most
    3 U max(d e^-d) n <= 3 U (1 + log n).  Additions: a thread adds at most n / 64 + 24 terms and factors one after the other."""
    z = logits.double().cpu() / temperature
    n = z.shape[-1]
    size = torch.where(z.isfinite(), z, 0.0)
    top = size.amax(-1)
    log_n = torch.log(torch.tensor(float(n), dtype=torch.float64))
    total = (n / 64 + 32 + 3 * (1 + log_n)) * U
    at = size.gather(-1, targets.long().cpu().clamp(0, n - 1).unsqueeze(-1)).squeeze(-1)
    return total + 4 * U * ((at - top).abs() + 1 + log_n), total


# ---------------------------------------------------------------- preferences
def preference(labels, lp, reference, mask, weights, kind, beta, smoothing, normalize, scale=1.0):
    """(loss [B], gradient [B, L, T], sum of absolute log ratios [B, L]) in float64, the gradient by the formula."""
    lp = lp.double().cpu()
    b, l, t = lp.shape
    m = torch.ones(b, l, t, dtype=torch.bool) if mask is None else (mask.cpu() != 0)
    y = labels.double().cpu()
    m = m & (y >= 0).unsqueeze(-1)
    d = lp - (0 if reference is None else reference.double().cpu())
    d = torch.where(m, d, 0.0)
    f = torch.full((b, l), float(beta), dtype=torch.float64)
    if normalize:
        f = f / m.sum(-1).clamp(min=1)
    s = f * d.sum(-1)
    w = (torch.ones(b, dtype=torch.float64) if weights is None else weights.double().cpu().reshape(-1).expand(b)) * scale
    loss, slope = torch.zeros(b, dtype=torch.float64), torch.zeros(b, l, dtype=torch.float64)
    for n in range(b):
        pairs = [(i, j) for i in range(l) for j in range(l) if y[n, i] > y[n, j] >= 0]
        for i, j in pairs:
            h = s[n, i] - s[n, j]
            if kind == 'logistic':
                sp = torch.nn.functional.softplus
                value = (1 - smoothing) * sp(-h) + smoothing * sp(h)
                by = torch.sigmoid(h) - (1 - smoothing)
            elif kind == 'hinge':
                value, by = torch.clamp(1 - h, min=0), (-1.0 if h < 1 else 0.0)
            else:
                value, by = (h - 0.5) ** 2, 2 * h - 1
            loss[n] += value * w[n] / len(pairs)
            slope[n, i] += by * w[n] / len(pairs)
            slope[n, j] -= by * w[n] / len(pairs)
    return loss, torch.where(m, (slope * f).unsqueeze(-1), 0.0), d.abs().sum(-1)


# ---------------------------------------------------------------- AdamW
def adamw(p, g, m, v, step, lr, betas, eps, decay):
    """(p, m, v, bound on m, bound on v, bound on p without its own rounding) in float64."""
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    b1, b2 = betas
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    m_size, den = (b1 * m).abs() + ((1 - b1) * g).abs(), (v1 / (1 - b2 ** step)).sqrt() + eps
    rate = lr / (1 - b1 ** step)
    p1 = p * (1 - lr * decay) - rate * m1 / den
    # m: two factors and two products rounded, one sum; v one product more
    dm, dv = 4 * U * m_size + 2.0 ** -149, 5 * U * v1 + 2.0 ** -149
    # root: half of v's error and 2 U, product, eps, sum, quotient and rate: 12 U; where v underflows den is eps alone
    root = (v1 / (1 - b2 ** step)).sqrt()
    dden = torch.where(v1 < 2.0 ** -120, root + (dv / (1 - b2 ** step)).sqrt(), 0.0) / den
    dp = 3 * U * p.abs() + rate / den * dm + (rate * m1 / den).abs() * (12 * U + dden)
    return p1, m1, v1, dm, dv, dp


def adamw_codes(m1, v1, block=128):
    """Codes and scales of float64 moments, and where a code is certain (not next to a border)."""
    def pad(x):
        return torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % block)).view(-1, block)
    m1, v1 = pad(m1), pad(v1)
    sm = (m1.float().abs().amax(1).double() / 127).float()
    sv = (v1.float().amax(1).double().sqrt() / 255).float()
    ym = torch.where(sm > 0, 1.0 / sm.double(), 0.0).unsqueeze(1) * m1
    yv = torch.where(sv > 0, 1.0 / sv.double(), 0.0).unsqueeze(1) * v1.sqrt()
    sure = lambda y: ((y - y.floor() - 0.5).abs() > 1e-9).view(-1)            # noqa: E731
    cm = ym.round().clamp(-127, 127)
    cv = torch.where((v1 > 0) & (sv > 0).unsqueeze(1), yv.round().clamp(1, 255), 0.0)
    return cm.view(-1), cv.view(-1), sm, sv, sure(ym), sure(yv)
