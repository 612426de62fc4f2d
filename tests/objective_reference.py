"""The objectives over logits written out in extended precision (numpy longdouble), with a bound on the
rounding error of an implementation that works in `dtype`, to first order in its unit roundoff u (times
1.25 for the higher orders; exponentials and logarithms count two units in the last place, 4 u).

The bound of a row: with z the (scaled) logits, m their maximum, s the sum of exp(z - m) and p = exp(z - m) / s,
a computed exp(z_j - m) is off by u (2.3 |z_j - m| + 4) relatively: the difference is rounded, the exponent
of the power of two that stands for it is rounded (u each, times ln 2 log2 e = 1), and log2 e (or log2 e / T) as
a float is off by at most 0.3 u of it. It is off by 2 u (|z_j| + |m|) more where the logits were scaled first. s is off by the p-weighted mean of that plus u per addition on the longest path of
sums, `adds`. An exponential below the smallest normal number may be taken as 0, and so may the factor
between two parts of a row: 2 tiny of p (s is at least 1). From those follow the bounds of log s, lp, p and of what is computed from them.
"""
import numpy as np

L = np.longdouble


class Rows:
    """x (rows, V) and labels (rows,) of an objective's live rows."""

    def __init__(self, x, dtype, adds, temperature=1.0):
        self.u = np.finfo(dtype).eps / 2 * 1.25
        self.tiny = np.finfo(dtype).tiny
        with np.errstate(all="ignore"):
            z = x.astype(L) / L(temperature)
            self.z, self.m = z, z.max(-1, keepdims=True)
            e = np.exp(z - self.m)
            self.s = e.sum(-1, keepdims=True)
            self.p = e / self.s
            far = np.where(np.isfinite(z), np.abs(z - self.m), 0)
            scaled = 0 if temperature == 1.0 else 2 * (np.where(np.isfinite(z), np.abs(z), 0) + np.abs(self.m))
            self.rel_e = self.u * (2.3 * far + scaled + 4)
            self.rel_s = (self.p * self.rel_e).sum(-1, keepdims=True) + self.u * adds
            self.rel_p = self.rel_e + self.rel_s + 3 * self.u
            self.logs = np.log(self.s)

    def at(self, index):
        """log p at `index` (rows, k), and its bound."""
        with np.errstate(all="ignore"):
            z = np.take_along_axis(self.z, index, -1)
            lp = (z - self.m) - self.logs
            off = np.take_along_axis(self.rel_e, index, -1) - 4 * self.u + self.rel_s + 4 * self.u * np.abs(self.logs) + 2 * self.u * np.abs(lp) + self.u
        return lp, off

    def grad(self, label, c, dc):
        """c (onehot(label) - p) for columns c, dc (the bound of c) of (rows, 1), and its bound."""
        hot = np.zeros_like(self.p)
        np.put_along_axis(hot, label, 1, -1)
        d = hot - self.p
        return c * d, np.abs(c) * self.p * self.rel_p + 4 * self.u * np.abs(c * d) + dc * np.abs(d) + self.tiny * (1 + 2 * np.abs(c))


def _labels(labels, v):
    return np.clip(labels.astype(np.int64), 0, v - 1)[..., None]


def token_log_prob(x, labels, dlogp, dtype, adds):
    """(value, bound) of logp and of the gradient; x (rows, V)."""
    r = Rows(x, dtype, adds)
    at = _labels(labels, x.shape[-1])
    lp, off = r.at(at)
    g = r.grad(at, dlogp.astype(L)[..., None], L(0))
    return (lp[..., 0], off[..., 0]), g


def policy(x, labels, old, advantage, weight, ref, low, high, kl, dtype, adds):
    """(value, bound) of loss, terms, logp and gradient; rows with weight 0 give zeros."""
    n, v = x.shape
    live = weight != 0
    r = Rows(x[live], dtype, adds)
    u = r.u
    at = _labels(labels[live], v)
    lp, dlp = (a[..., 0] for a in r.at(at))
    a, w = advantage[live].astype(L), weight[live].astype(L)
    with np.errstate(all="ignore"):
        d = lp - old[live].astype(L)
        ratio = np.exp(d)
        rel = np.expm1(dlp + u * np.abs(d)) + 4 * u
        held = np.clip(ratio, 1 - L(low), 1 + L(high))
        term = -np.minimum(ratio * a, held * a)
        dterm = np.abs(a) * np.maximum(ratio * (rel + 2 * u), held * (2 * u + rel))
        active = np.where(a >= 0, ratio <= 1 + L(high), ratio >= 1 - L(low))
        c = np.where(active, -a * ratio, 0)
        dc = np.where(active, np.abs(a) * ratio * (rel + u), 0)
        if kl:
            k = ref[live].astype(L) - lp
            e = np.exp(k)
            dk = dlp + u * np.abs(k)
            de = e * (np.expm1(dk) + 4 * u)
            term = term + L(kl) * (e - k - 1)
            dterm = dterm + kl * (de + dk + 3 * u * (e + np.abs(k) + 1)) + u * np.abs(term)
            c = c + L(kl) * (1 - e)
            dc = dc + kl * (de + 2 * u * (1 + e)) + u * np.abs(c)
    term, dterm = w * term, np.abs(w) * dterm + 2 * u * np.abs(w * term)
    c, dc = w * c, np.abs(w) * dc + 2 * u * np.abs(w * c)
    g, dg = r.grad(at, c[:, None], dc[:, None])

    def spread(values, like):
        out = np.zeros(like, L)
        out[live] = values
        return out
    loss = term.sum()
    return ((loss, dterm.sum() + 2 * u * np.abs(loss)), (spread(term, n), spread(dterm, n)), (spread(lp, n), spread(dlp, n)),
            (spread(g, x.shape), spread(dg, x.shape)))


def preference(x, labels, weight, ref, beta, smoothing, dtype, adds):
    """(value, bound) of loss, margins, logp and gradient; x (2 n, T, V)."""
    b, t, v = x.shape
    n = b // 2
    u = np.finfo(dtype).eps / 2 * 1.25
    live = weight != 0
    lp, dlp = np.zeros((b, t), L), np.zeros((b, t), L)
    r = Rows(x[live], dtype, adds)
    at = _labels(labels[live], v)
    lp[live], dlp[live] = (q[..., 0] for q in r.at(at))
    w = weight.astype(L)
    total, dtotal = (w * lp).sum(1), (np.abs(w) * dlp).sum(1)
    gain = total - ref.astype(L)
    h = L(beta) * (gain[:n] - gain[n:])
    dh = abs(beta) * (dtotal[:n] + dtotal[n:])
    soft = np.log1p(np.exp(-np.abs(h)))
    eps = L(smoothing)
    term = (1 - eps) * (soft + np.maximum(-h, 0)) + eps * (soft + np.maximum(h, 0))
    loss = term.mean()
    slope = L(beta) * (eps / (1 + np.exp(-h)) - (1 - eps) / (1 + np.exp(h))) / n
    dslope = abs(beta) * dh / 4 / n + 2 * u * np.abs(slope)
    c = np.concatenate([slope, -slope])[:, None] * w
    dc = np.concatenate([dslope, dslope])[:, None] * np.abs(w) + 2 * u * np.abs(c)
    g, dg = np.zeros(x.shape, L), np.zeros(x.shape, L)
    g[live], dg[live] = r.grad(at, c[live][:, None], dc[live][:, None])
    return ((loss, dh.mean() + 3 * u * np.abs(loss)), (h, dh + 2 * u * np.abs(h)), (total, dtotal + 2 * u * np.abs(total)), (g, dg))


def distillation(x, index, teacher, weight, temperature, dtype, adds):
    """(value, bound) of loss, terms and gradient; x (rows, V), index and teacher (rows, k)."""
    n, v = x.shape
    k = index.shape[-1]
    live = (weight != 0) & ~np.all(teacher == -np.inf, -1)
    t = L(temperature)
    q = Rows(teacher[live], dtype, k + 40, temperature)
    r = Rows(x[live], dtype, adds, temperature)
    u = r.u
    at = np.clip(index[live].astype(np.int64), 0, v - 1)
    lp, dlp = r.at(at)
    with np.errstate(all="ignore"):
        some = q.p > 0
        logq = np.where(some, np.log(np.where(some, q.p, 1)), 0)
        gap = np.where(some, logq - np.where(some, lp, 0), 0)
        term = (q.p * gap).sum(-1)
        dterm = np.where(some, q.p * (np.abs(gap) * (q.rel_p + 2 * u) + q.rel_p + 4 * u * np.abs(logq) + np.where(some, dlp, 0)), 0).sum(-1)
    w = weight[live].astype(L)
    term, dterm = w * t * t * term, np.abs(w) * t * t * dterm + 6 * u * np.abs(w * t * t * term)
    g, dg = r.p.copy(), r.p * r.rel_p
    for row in range(g.shape[0]):
        np.subtract.at(g[row], at[row], q.p[row])
        np.add.at(dg[row], at[row], q.p[row] * (q.rel_p[row] + (k + 2) * u) + r.p[row][at[row]] * 2 * u)
    c = (w * t)[:, None]
    g, dg = c * g, np.abs(c) * dg + 4 * u * np.abs(c * g) + r.tiny * (1 + 2 * np.abs(c))

    def spread(values, like):
        out = np.zeros(like, L)
        out[live] = values
        return out
    loss = term.sum()
    return ((loss, dterm.sum() + 2 * u * np.abs(loss)), (spread(term, n), spread(dterm, n)), (spread(g, x.shape), spread(dg, x.shape)))


def assert_within(got, want, what):
    """`got` within the bound of `want` = (value, bound); non-finite values must agree."""
    value, bound = (np.asarray(v) for v in want)
    got = np.asarray(got).astype(L).reshape(value.shape)
    fine = np.isfinite(value)
    same = np.where(np.isnan(value), np.isnan(got), got == value)
    assert same[~fine].all(), f"{what}: non-finite values differ"
    off = np.abs(got - np.where(fine, value, 0))
    bad = fine & ~(off <= bound)
    if bad.any():
        k = np.unravel_index(np.argmax(np.where(bad, off / np.maximum(bound, 1e-300), 0)), bad.shape) if bad.shape else ()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} values off, worst at {tuple(int(i) for i in k)}: {got[k]!r} against {value[k]!r} "
                             f"(off {float(off[k]):.3g}, bound {float(np.broadcast_to(bound, bad.shape)[k]):.3g})")


# ---- inputs ----

KINDS = ["normal", "wide", "banned", "lowest", "peaked"]


def logits(rng, rows, v, kind, dtype):
    x = rng.normal(size=(rows, v)) * 2.5
    if kind == "wide":
        x *= 30
    if kind == "banned" and v > 1:
        x[:, rng.random(v) < 0.3] = -np.inf
        x[:, rng.integers(v)] = rng.normal(size=rows)
    if kind == "lowest" and v > 1:
        x[:, rng.random(v) < 0.5] = np.finfo(dtype).min
        x[:, rng.integers(v)] = rng.normal(size=rows)
        x[0] = np.finfo(dtype).min  # a row of nothing but the lowest value: uniform
    if kind == "peaked":
        x[np.arange(rows), rng.integers(0, v, rows)] += 30
    return x.astype(dtype)


def labels(rng, x):
    """A label per row with a finite, not the lowest logit where the row has one."""
    ok = x > np.finfo(x.dtype).min
    ok[~ok.any(-1)] = True
    return np.array([rng.choice(np.flatnonzero(r)) for r in ok], dtype=np.int32)


def log_prob(x, label):
    z = x.astype(L)
    m = z.max(-1, keepdims=True)
    return (np.take_along_axis(z, label.astype(np.int64)[:, None], -1) - m - np.log(np.exp(z - m).sum(-1, keepdims=True)))[:, 0]


def policy_inputs(rng, x, label, dtype, low=0.2, high=0.28):
    """old, advantage, weight, ref. Ratios within 0.002 of a clip bound move off it."""
    n = len(label)
    ratio = np.exp(rng.normal(size=n) * 0.25)
    for edge in (1 - low, 1 + high):
        ratio = np.where(np.abs(ratio - edge) < 0.002, edge + 0.004, ratio)
    lp = log_prob(x, label).astype(np.float64)
    return ((lp - np.log(ratio)).astype(dtype), rng.normal(size=n).astype(dtype), (np.where(rng.random(n) < 0.8, rng.random(n), 0) / n).astype(dtype),
            (lp + rng.normal(size=n) * 0.3).astype(dtype))


def teacher_inputs(rng, x, k, dtype):
    """index, teacher, weight: indices at finite logits, some twice, some rows short, one row without entries."""
    n, v = x.shape
    index = np.stack([rng.choice(np.flatnonzero(r > np.finfo(dtype).min) if (r > np.finfo(dtype).min).any() else np.arange(v), size=k) for r in x]).astype(np.int32)
    teacher = (rng.random((n, k)) * 9).astype(dtype)
    short = rng.random(n) < 0.3
    teacher[short, max(1, k // 2):] = -np.inf
    index[short, max(1, k // 2):] = -7
    if n > 2:
        teacher[n // 2] = -np.inf
    return index, teacher, (np.where(rng.random(n) < 0.8, rng.random(n), 0) / n).astype(dtype)
