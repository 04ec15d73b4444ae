"""Scoring, distillation and rotary positions in 64 bits, and the error that f32 sums may have.

Bounds, with u = 2^-24 (half an ulp of f32, relative), d = z - m, m the row's largest logit:
  an exponential of d / T: d rounds (u |d|), d / T rounds twice more (2 u |d| / T), a sum that is rescaled goes through
    one exponential more of a part of d; the exponential itself 4 ulps = 8 u: EXP(d) = (20 + 6 |d|) u relative, |d| at T.
  a row's sum: at most v / 64 + 64 terms follow one another, each with three roundings (a product, two sums):
    SUM(v) = 3 (v / 64 + 64) u relative to the sum of magnitudes.
  logarithms and log1p: 2 ulps of the value, 4 u.
  underflow: exponentials below 2^-126 may be 0: TINY each, relative to a sum of at least 1.
"""
import numpy as np

U = 2.0 ** -24
TINY = 2.0 ** -126


def _rows(z, rate=1.0):
    """m, d, e = exp(d rate), S and the relative error of S, for rows of finite largest logit."""
    z = z.astype(np.float64)
    m = z.max(-1, keepdims=True)
    d = z - m
    dr = np.where(d == -np.inf, -1e9, d) * rate
    e = np.exp(dr)
    s = e.sum(-1, keepdims=True)
    v = z.shape[-1]
    err = ((e * (20 + 6 * np.abs(dr)) * U).sum(-1, keepdims=True) / s) + 3 * (v / 64 + 64) * U + v * TINY
    return d, dr, e, s, err


def token_logprobs(z, targets, k):
    """(logprob, tol), (entropy, tol), (ids, (values, tol)) of rows of finite largest logit; targets may be None."""
    d, dr, e, s, err = _rows(z)
    v = z.shape[-1]
    rest = np.log(s)
    rest_tol = err * (s - (e == 1.0).any(-1, keepdims=True)) / s + 4 * U * rest  # (the largest term is exactly 1)
    dd = np.maximum(dr, -1e9)
    us = (e * dd).sum(-1, keepdims=True)
    us_tol = (e * np.abs(dd) * (22 + 6 * np.abs(dd)) * U).sum(-1, keepdims=True) + np.abs(us) * 3 * (v / 64 + 64) * U + 200 * v * TINY
    h = rest - us / s
    h_tol = rest_tol + us_tol / s + np.abs(us) / s * (err + 4 * U) + 2 * U * h

    def value(dj):
        lp = dj - rest
        return lp, rest_tol + 2 * U * (np.abs(dj) + np.abs(lp))

    lp = None
    if targets is not None:
        lp = tuple(x[:, 0] for x in value(np.take_along_axis(d, targets[:, None].astype(np.int64), 1)))
    # the largest first, lower ids first among equals
    ids = np.argsort(-(z.astype(np.float64) + 0.0), axis=-1, kind="stable")[:, :k]
    return lp, (h[:, 0], h_tol[:, 0]), (ids.astype(np.int32), value(np.take_along_axis(d, ids, 1)))


def token_logprobs_backward(z, targets, dl, dh):
    d, dr, e, s, err = _rows(z)
    _, (h, h_tol), _ = token_logprobs(z, None, 0)
    h, h_tol = h[:, None], h_tol[:, None]
    p, rest = e / s, np.log(s)
    dd = np.maximum(dr, -1e9)
    dl = np.zeros((len(z), 1)) if dl is None else dl.astype(np.float64)[:, None]
    dh = np.zeros((len(z), 1)) if dh is None else dh.astype(np.float64)[:, None]
    lnp = dd - rest
    g = p * (-dl - dh * (lnp + h))
    size = np.abs(dl) + np.abs(dh) * (np.abs(dd) + rest + h)
    tol = p * size * ((20 + 6 * np.abs(dd) + 8) * U + err) + p * np.abs(dh) * (h_tol + err + 4 * U * rest) + TINY * (1 + 200 * size)
    if targets is not None:
        rows = np.arange(len(z))
        g[rows, targets] += dl[:, 0]
        tol[rows, targets] += 2 * U * np.abs(dl[:, 0])
    return g, tol


def distillation(z, targets, ids, teacher, temperature, alpha, count):
    """(row losses, tol, dlogits, tol) of rows that count, `count` of them in the mean."""
    t, a = float(np.float32(temperature)), float(np.float32(alpha))
    rate = 1.0 / t
    n, v = z.shape
    d, dr, e, s, err = _rows(z, rate)
    d1, dr1, e1, s1, err1 = _rows(z)
    rest, rest1 = np.log(s), np.log(s1)
    rest_tol = err + 4 * U * rest
    filled = (ids >= 0) & (teacher > -np.inf)
    safe = np.where(filled, ids, 0).astype(np.int64)
    u = np.where(filled, teacher.astype(np.float64), -np.inf)
    top = u.max(-1, keepdims=True)
    none = top == -np.inf
    u = np.where(none | (u == -np.inf), -np.inf, u - np.where(none, 0.0, top))
    ur = np.where(u == -np.inf, -1e9, u) * rate
    q = np.where(none, 0.0, np.exp(ur))
    qs = np.where(none, 1.0, q.sum(-1, keepdims=True))
    k = ids.shape[-1]
    q = q / qs
    q_err = (20 + 6 * np.abs(np.maximum(ur, -1e4))) * U + ((q * (20 + 6 * np.abs(np.maximum(ur, -1e4)))).sum(-1, keepdims=True) + k + 16) * U
    dj = np.take_along_axis(d, safe, 1) * rate
    lq, lp = np.maximum(ur, -1e9) - np.log(qs), np.where(q > 0, dj, 0.0) - rest
    with np.errstate(invalid="ignore"):
        gap = np.where(q > 0, lq - lp, 0.0)
    size = np.abs(np.maximum(ur, -1e4)) + np.log(qs) + np.abs(np.where(q > 0, dj, 0.0)) + rest
    kl = (q * gap).sum(-1)
    kl_tol = (q * (np.abs(gap) * q_err + 8 * U * size + q_err.max(-1, keepdims=True) + rest_tol)).sum(-1) + k * U * (q * np.abs(gap)).sum(-1) + k * TINY * 1e4
    row, tol = a * t * t * kl, a * t * t * (kl_tol + 6 * U * np.abs(kl))
    soft, hard = np.where(none, 0.0, a * t / count), (1.0 - a) / count  # (a row of empty slots has no first term)
    p, p1 = e / s, e1 / s1
    g = soft * p + hard * p1
    g_tol = (soft * p * ((28 + 6 * np.abs(np.maximum(dr, -1e4))) * U + err) + hard * p1 * ((28 + 6 * np.abs(np.maximum(dr1, -1e4))) * U + err1)
             + 2 * TINY)
    rows = np.arange(n)
    if targets is not None:
        y = targets.astype(np.int64)
        ce = rest1[:, 0] - d1[rows, y]
        row = row + (1.0 - a) * ce
        tol = tol + (1.0 - a) * (err1[:, 0] + 4 * U * rest1[:, 0] + 6 * U * (np.abs(d1[rows, y]) + ce)) + 2 * U * np.abs(row)
        np.add.at(g, (rows, y), -hard)
        np.add.at(g_tol, (rows, y), 4 * U * hard)
    w = np.where(filled, soft * q, 0.0)
    np.add.at(g, (rows[:, None].repeat(k, 1), safe), -w)
    np.add.at(g_tol, (rows[:, None].repeat(k, 1), safe), w * (q_err + (k + 6) * U))
    return row, tol, g, g_tol


def frequencies(width, theta, scaling="none", factor=1.0, trained=0, low=1.0, high=32.0):
    theta, factor, low, high = (float(np.float32(x)) for x in (theta, factor, low, high))
    i = np.arange(width // 2, dtype=np.float64)
    base = theta * factor ** (width / (width - 2.0)) if scaling == "base" and width > 2 else theta
    w = base ** (-2.0 * i / width)
    if scaling == "linear":
        return w / factor
    if scaling == "parts":
        r = np.clip((trained * w / (2 * np.pi) - low) / (high - low), 0.0, 1.0)
        return w * (r + (1.0 - r) / factor)
    return w


def rotate(x, cos, sin, layout, width, back=False):
    """x [b, h, t, hd], cos and sin [b or 1, 1, t, width / 2] in the products' own rounding: f32 operations one by one."""
    s = -sin if back else sin
    out = x.copy()
    i0, i1 = (slice(0, width // 2), slice(width // 2, width)) if layout == "half" else (slice(0, width, 2), slice(1, width, 2))
    a, b = x[..., i0], x[..., i1]
    out[..., i0] = a * cos - b * s
    out[..., i1] = b * cos + a * s
    return out
