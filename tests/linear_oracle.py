"""The linear layer's operators in 64 bits, and the error that f32 sums may have.

Bounds, with u = 2^-24 (half an ulp of f32, relative):
  product over K: both product kernels round the running sum at most K / 2 + 24 times by 2 u of S = sum_p |a_p b_p|
    (the split tiles six times per 16 k, where the matrix core may truncate; the fp32 MFMA once per k by u; a K split adds
    its partials, one rounding each, and a split keeps at least 128 of K): product_bound.
  activations: a few ulps of |x| (|act(x)| <= |x|), their slopes are at most 1.13: 16 ulps = 32 u are allowed.
  derivatives: at most 1.13, evaluated to 16 ulps of 1.
  underflow: a value below 2^-126 may become 0 (exponentials of far logits): TINY for each.
"""
import math

import numpy as np

U = 2.0 ** -24
SLOPE = 1.13
TINY = 2.0 ** -126


def product_bound(k, s):
    return (k / 2 + 24) * 2 * U * s


def philox(counter, key):
    """Philox4x32-10 on arrays of counters (four words each) under one key of two words."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(x, np.uint64) for x in counter]
    k = [int(x) for x in key]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1)


def words(n, seed, offset):
    """The generator's words for the values 0..n-1 of an array."""
    j = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(offset)  # wraps at 2^64
    zero = np.zeros_like(j)
    w = philox((j & np.uint64(0xFFFFFFFF), j >> np.uint64(32), zero, zero), (seed & 0xFFFFFFFF, seed >> 32))
    return w.reshape(-1)[:n]


def kept(n, p, seed, offset):
    return words(n, seed, offset) >= np.uint64(math.floor(float(np.float32(p)) * 2.0 ** 32))


def drop(x, p, seed, offset):
    """dropout(x) in 64 bits: dropped values are 0 whatever they were."""
    p64 = float(np.float32(p))
    if p64 == 0.0:
        return x
    mask = kept(x.size, p, seed, offset).reshape(x.shape)
    return np.where(mask, x / (1.0 - p64) if p64 < 1.0 else 0.0, 0.0)


_erf = np.vectorize(math.erf, otypes=[np.float64])
C0, C1 = math.sqrt(2.0 / math.pi), 0.044715


def erf(x):
    try:
        from scipy.special import erf as f
        return f(x)
    except ImportError:
        return _erf(x)


def act(name, x):
    with np.errstate(over="ignore"):
        if name == "relu":
            return np.maximum(x, 0.0)
        if name == "gelu":
            return 0.5 * x * (1.0 + erf(x / math.sqrt(2.0)))
        if name == "gelu_tanh":
            return 0.5 * x * (1.0 + np.tanh(C0 * (x + C1 * x ** 3)))
        if name == "silu":
            return x / (1.0 + np.exp(-x))
    return x


def act_grad(name, x):
    with np.errstate(over="ignore"):
        if name == "relu":
            return (x > 0).astype(np.float64)
        if name == "gelu":
            return 0.5 * (1.0 + erf(x / math.sqrt(2.0))) + x * np.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi)
        if name == "gelu_tanh":
            t = np.tanh(C0 * (x + C1 * x ** 3))
            return 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * C0 * (1.0 + 3.0 * C1 * x * x)
        if name == "silu":
            g = 1.0 / (1.0 + np.exp(-x))
            return g * (1.0 + x * (1.0 - g))
    return np.ones_like(x)


def scale_of(p):
    return 1.0 / (1.0 - float(np.float32(p))) if float(np.float32(p)) < 1.0 else 0.0


def linear(x, w, bias, residual, name, p, seed, offset):
    """(out, its bound, pre, its bound) for w [k, n]."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    b = np.zeros(w.shape[1]) if bias is None else bias.astype(np.float64)
    pre = x @ w + b
    pre_tol = product_bound(x.shape[1], np.abs(x) @ np.abs(w)) + 2 * U * np.abs(pre)
    h = act(name, pre)
    out = drop(h, p, seed, offset)
    live = drop(np.ones_like(h), p, seed, offset) > 0 if p else np.ones(h.shape, bool)
    s = scale_of(p)
    tol = np.where(live, s * (SLOPE * pre_tol + 32 * U * np.abs(pre)), 0.0)
    if residual is not None:
        out = out + residual.astype(np.float64)
    return out, tol + 4 * U * np.abs(out), pre, pre_tol


def linear_backward(x, w, pre, dout, name, p, seed, offset):
    """{name: (value, bound)} of dx, dw [k, n], dbias for w [k, n]."""
    x, w, dout = x.astype(np.float64), w.astype(np.float64), dout.astype(np.float64)
    g = np.ones_like(dout) if pre is None else act_grad(name, pre.astype(np.float64))
    dpre = drop(dout, p, seed, offset) * g
    tol = np.abs(drop(dout, p, seed, offset)) * 40 * U
    rows, k, n = x.shape[0], x.shape[1], w.shape[1]
    size = np.abs(dpre) + tol
    return {"dx": (dpre @ w.T, product_bound(n, size @ np.abs(w).T) + tol @ np.abs(w).T),
            "dw": (x.T @ dpre, product_bound(rows, np.abs(x).T @ size) + np.abs(x).T @ tol),
            "dbias": (dpre.sum(0), rows * U * size.sum(0) + tol.sum(0))}


def cross_entropy(x, w, targets, ignore=-1, blocks=1):
    """{name: (value, bound)} of loss, dx, dw [d, V] for w [d, V]; blocks: parts that dw is added up from."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    n, d, V = x.shape[0], x.shape[1], w.shape[1]
    keep = np.flatnonzero(targets != ignore)
    dx, dx_tol = np.zeros((n, d)), np.zeros((n, d))
    if not len(keep):
        return {"loss": (0.0, 0.0), "dx": (dx, dx_tol), "dw": (np.zeros((d, V)), np.zeros((d, V)))}
    xk, t = x[keep], targets[keep]
    z = xk @ w
    ez = product_bound(d, np.abs(xk) @ np.abs(w))
    top = z.max(1, keepdims=True)
    e = np.exp(z - top)
    total = e.sum(1, keepdims=True)
    at = np.arange(len(keep))
    rows = (top + np.log(total))[:, 0] - z[at, t]
    # the sum of V exponentials: a lane adds V / 256 of them or less one after another, then lanes in pairs
    sums = (V / 256 + 40) * 2 * U
    ezm = ez.max(1, keepdims=True)
    row_tol = 2 * ezm[:, 0] + sums + 4 * U * (np.abs(top[:, 0]) + np.log(total[:, 0]) + np.abs(z[at, t]) + 4)
    s = 1.0 / len(keep)
    p = e / total
    dz = p * s
    dz_tol = dz * (2 * ezm + sums + U * (16 + 4 * np.abs(z - top))) + TINY
    dz[at, t] -= s
    dz_tol += 4 * U * np.abs(dz)
    dz_tol[at, t] += 4 * U * s
    size = np.abs(dz) + dz_tol
    dx[keep] = dz @ w.T
    dx_tol[keep] = product_bound(V, size @ np.abs(w).T) + dz_tol @ np.abs(w).T + V * TINY
    dw_tol = product_bound(len(keep) + 2 * blocks, np.abs(xk).T @ size) + np.abs(xk).T @ dz_tol + len(keep) * TINY
    loss = rows.mean()
    return {"loss": (loss, row_tol.mean() + 2 * U * abs(loss)), "dx": (dx, dx_tol), "dw": (xk.T @ dz, dw_tol)}
