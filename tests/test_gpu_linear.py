"""GPU checks of the linear layer's operators (linear.hip, linear_loss.hip) against 64-bit evaluations, within the bounds
that linear_oracle.py derives; every output lies between guard words, and every case is run at the alignments given."""
import ctypes

import numpy as np
import pytest

import linear_oracle as R
import midman_hip as mh

pytestmark = pytest.mark.gpu

GUARD = 64
MARK = np.float32(-7.25e33)


class Box:
    """An array of the device `shift` floats off a 256-byte boundary, between guard words."""

    def __init__(self, ctx, a, shift=0):
        self.shape, self.n = np.shape(a), int(np.size(a))
        self.at = GUARD + shift
        flat = np.full(self.at + self.n + GUARD, MARK, np.float32)
        flat[self.at:self.at + self.n] = np.ravel(a)
        self.dev = ctx.to_device(flat)
        self.ptr = self.dev.offset(self.at)

    def numpy(self):
        a = self.dev.numpy()
        assert (a[:self.at] == MARK).all() and (a[self.at + self.n:] == MARK).all(), "a write outside the output"
        return a[self.at:self.at + self.n].reshape(self.shape)


def empty(ctx, shape, shift=0):
    return Box(ctx, np.full(shape, np.nan, np.float32), shift)


def ptr(b):
    return None if b is None else b.ptr


def near(got, value, tol, what):
    err = np.abs(got.astype(np.float64) - value)
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(err / np.maximum(tol, 1e-300))), np.argwhere(bad)[:3].tolist())


def stored(w, form):
    """w [k, n] as the form stores it."""
    return np.ascontiguousarray(w.T) if form else w


# (rows, k, n): every product kernel (32x32 and 64x64 tiles, K split inside and over launches, large tiles whole and
# split), rows and columns and K that end inside a tile, one row, one column, one of K
SHAPES = [(1, 1, 1), (1, 5, 3), (2, 130, 1), (64, 64, 176), (33, 255, 31), (130, 96, 64), (7, 2048, 130), (515, 48, 301),
          (1003, 517, 770), (300, 5003, 301), (767, 1598, 1373), (2300, 50, 2301), (1000, 2050, 4100), (3900, 100, 4000),
          (4100, 31, 600), (32768, 40, 60)]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def operands(rows, k, n, seed, bias=True, residual=True):
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, k)).astype(np.float32)
    w = (r.standard_normal((k, n)) * (1.5 / np.sqrt(k))).astype(np.float32)
    b = r.standard_normal(n).astype(np.float32) if bias else None
    res = r.standard_normal((rows, n)).astype(np.float32) if residual else None
    return x, w, b, res


def run_linear(ctx, form, x, w, b, res, act, p, seed, offset, want_pre, shift=0, inplace=False):
    rows, k, n = x.shape[0], x.shape[1], w.shape[1]
    X, W = Box(ctx, x, shift), Box(ctx, stored(w, form), shift)
    B = None if b is None else Box(ctx, b, shift)
    S = None if res is None else Box(ctx, res, shift)
    P = empty(ctx, (rows, n), shift) if want_pre else None
    O = S if inplace else empty(ctx, (rows, n), shift)
    mh.check(mh.lib().mmh_linear(ctx.handle, form, X.ptr, W.ptr, ptr(B), ptr(S), rows, k, n, R_ACT[act], p, seed, offset,
                                 ptr(P), O.ptr))
    return O.numpy(), None if P is None else P.numpy()


R_ACT = mh.ACTIVATIONS


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear(ctx, i, form):
    rows, k, n = SHAPES[i]
    # the options turn with the shape, so that each meets several kernels
    for act, p, bias, residual, pre in [(ACTS[i % 5], (0.0, 0.1, 0.5)[i % 3], True, i % 2 == 0, i % 3 == 0),
                                        (ACTS[(i + 2 + form) % 5], (0.25, 0.0)[i % 2], i % 2 == 1, i % 4 < 2, i % 2 == form)]:
        print(f"\n[linear] {SHAPES[i]} form={form} act={act} p={p} bias={bias} residual={residual} pre={pre}", flush=True)
        x, w, b, res = operands(rows, k, n, 100 * i + form, bias, residual)
        seed, offset = 0x1234567890ABCDEF + i, 2 ** 33 + 5 * i
        out, got_pre = run_linear(ctx, form, x, w, b, res, act, p, seed, offset, pre)
        want, tol, want_pre, pre_tol = R.linear(x, w, b, res, act, p, seed, offset)
        near(out, want, tol, "out")
        if pre:
            near(got_pre, want_pre, pre_tol, "pre")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(64, 64, 176), (130, 1000, 515), (3000, 200, 2048)])
def test_linear_activations_dropout_in_place(ctx, act, shape):
    rows, k, n = shape
    print(f"\n[linear in place] {shape} {act}", flush=True)
    x, w, b, res = operands(rows, k, n, 7)
    out, _ = run_linear(ctx, 0, x, w, b, res, act, 0.3, 77, 0, False, inplace=True)
    want, tol, _, _ = R.linear(x, w, b, res, act, 0.3, 77, 0)
    near(out, want, tol, "out")


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("shape", [(66, 64, 176), (515, 301, 1004), (2300, 50, 2300)])
def test_linear_alignments(ctx, shape, shift):
    rows, k, n = shape
    print(f"\n[linear alignment] {shape} {shift}", flush=True)
    x, w, b, res = operands(rows, k, n, 8)
    for form in (0, 1):
        out, pre = run_linear(ctx, form, x, w, b, res, "silu", 0.4, 78, 3, True, shift=shift)
        want, tol, want_pre, pre_tol = R.linear(x, w, b, res, "silu", 0.4, 78, 3)
        near(out, want, tol, "out")
        near(pre, want_pre, pre_tol, "pre")


@pytest.mark.parametrize("shape", [(5, 64, 7), (64, 64, 176), (1003, 517, 770), (2300, 50, 2302), (256, 4096, 256)])
def test_linear_mask_is_dropouts(ctx, shape):
    """The epilogue drops the values that mmh_dropout drops of an array of that size; dropped ones are the residual."""
    rows, k, n = shape
    x, w, b, res = operands(rows, k, n, 9)
    seed, offset = 2 ** 64 - 3, 2 ** 64 - 7  # (the counter wraps inside the array)
    out, pre = run_linear(ctx, 0, x, w, b, res, "none", 0.5, seed, offset, True)
    ones = ctx.to_device(np.ones((rows, n), np.float32))
    mask = mh.dropout(ctx, ones, 0.5, seed, offset).numpy()
    assert np.array_equal(mask, np.where(R.kept(rows * n, 0.5, seed, offset).reshape(rows, n), 2.0, 0.0))
    assert np.array_equal(out[mask == 0], res[mask == 0])
    assert np.array_equal(out, np.where(mask > 0, res + np.float32(2.0) * pre, res))


def test_linear_dropped_values_and_special_values(ctx):
    # row 0 of x: NaN, row 1: an infinity; the others as they are alone
    rows, k, n = 70, 96, 136
    x, w, b, res = operands(rows, k, n, 10)
    x[0, 3], x[1, 5] = np.nan, np.inf
    out, pre = run_linear(ctx, 0, x, w, b, res, "gelu", 0.5, 3, 0, True)
    keep = R.kept(rows * n, 0.5, 3, 0).reshape(rows, n)
    assert np.array_equal(out[~keep], res[~keep])
    assert np.isnan(out[0][keep[0]]).all() and np.isnan(pre[0]).all()
    assert not np.isfinite(pre[1]).any()
    want, tol, _, _ = R.linear(x[2:], w, b, res[2:], "gelu", 0.0, 0, 0)
    alone = np.where(keep[2:], (want - res[2:]) * 2 + res[2:], res[2:])
    near(out[2:], alone, 2 * tol + 4 * R.U * np.abs(alone), "the finite rows")
    # p = 1: only the residual is left, whatever the product is
    out, _ = run_linear(ctx, 0, x, w, b, res, "none", 1.0, 3, 0, False)
    assert np.array_equal(out, res)
    out, _ = run_linear(ctx, 0, x, w, b, None, "relu", 1.0, 3, 0, False)
    assert (out == 0).all()


# every product kernel: 32x32 and 64x64 tiles, K split in the launch, large tiles whole and split over launches
@pytest.mark.parametrize("shape", [(64, 64, 176), (33, 300, 64), (520, 200, 515), (300, 5003, 301), (2300, 64, 2301),
                                   (3300, 70, 3000), (1000, 2050, 4100)])
@pytest.mark.parametrize("form", [0, 1])
def test_values_outside_the_split(ctx, shape, form):
    """Rows of x with an infinity, a NaN, values from 2^104 on and subnormal ones, beside ordinary rows: the ordinary ones
    keep their bounds, the others follow IEEE (row r of the result depends on row r of x alone)."""
    rows, k, n = shape
    print(f"\n[values outside the split] {shape} {form}", flush=True)
    x, w, b, res = operands(rows, k, n, 31)
    x[3, 1], x[7, 2] = np.inf, np.nan
    x[11, :4] = np.float32(2.0) ** 106 * np.array([1, -1, 2, 0.5], np.float32)
    x[15] *= np.float32(2.0) ** -120
    seed, offset = 8, 1
    out, pre = run_linear(ctx, form, x, w, b, res, "silu", 0.25, seed, offset, True)
    odd = [3, 7]
    rest = np.setdiff1d(np.arange(rows), odd)
    x0 = x.copy()
    x0[odd] = 0
    want, tol, want_pre, pre_tol = R.linear(x0, w, b, res, "silu", 0.25, seed, offset)
    # a subnormal product or input may be flushed by the fp32 kernels: one smallest normal value per term
    tiny = k * R.TINY
    near(pre[rest], want_pre[rest], pre_tol[rest] + tiny, "pre")
    near(out[rest], want[rest], tol[rest] + 2 * tiny, "out")
    with np.errstate(invalid="ignore"):
        sign = np.where(np.isnan(w[1]) | (w[1] == 0), np.nan, np.sign(w[1]) * np.inf)
    assert np.array_equal(pre[3], sign.astype(np.float32), equal_nan=True)
    assert np.isnan(pre[7]).all()
    keep = R.kept(rows * n, 0.25, seed, offset).reshape(rows, n)
    assert np.array_equal(out[7][~keep[7]], res[7][~keep[7]]) and np.isnan(out[7][keep[7]]).all()


def test_activations_far_out(ctx):
    """Large arguments of either sign: k = 1 products of 1 and the value itself."""
    v = np.array([0.0, -0.0, 1e-30, -1e-30, 0.5, -0.5, 3, -3, 6, -6, 9, -9, 20, -20, 88, -88, 104, -104, 1e4, -1e4, 1e20,
                  -1e20, 3e38, -3e38], np.float32)
    for act in ACTS:
        for rows in (1, 40):
            x = np.ones((rows, 1), np.float32)
            out, pre = run_linear(ctx, 0, x, v[None, :], None, None, act, 0.0, 0, 0, True)
            assert np.array_equal(pre, np.repeat(v[None], rows, 0))
            with np.errstate(over="ignore", invalid="ignore"):
                want = R.act(act, v.astype(np.float64))
            # relative too: gelu's far negative side is x * erfc, which the 1 + erf of the oracle cannot show beyond -5
            near(out, np.repeat(want[None], rows, 0), np.repeat((32 * R.U * np.abs(v.astype(np.float64)))[None], rows, 0), act)
            assert np.isfinite(out).all()
            dout = np.ones((rows, len(v)), np.float32)
            D, P, W, X = (Box(ctx, a) for a in (dout, pre, v[None, :], x))
            db = empty(ctx, (len(v),))
            mh.check(mh.lib().mmh_linear_backward(ctx.handle, 0, X.ptr, W.ptr, P.ptr, D.ptr, rows, 1, len(v), R_ACT[act], 0.0,
                                                  0, 0, None, None, db.ptr))
            with np.errstate(over="ignore", invalid="ignore"):
                g = np.nan_to_num(R.act_grad(act, np.clip(v.astype(np.float64), -1e6, 1e6)))
            near(db.numpy(), rows * g, np.full(len(v), rows * (40 + rows) * R.U * 1.2), act + " slope")


def run_backward(ctx, form, x, w, pre, dout, act, p, seed, offset, shift=0, outs=("dx", "dw", "dbias")):
    rows, k, n = x.shape[0], x.shape[1], w.shape[1]
    X, W, D = Box(ctx, x, shift), Box(ctx, stored(w, form), shift), Box(ctx, dout, shift)
    P = None if pre is None else Box(ctx, pre, shift)
    got = {"dx": (rows, k), "dw": stored(w, form).shape, "dbias": (n,)}
    got = {name: empty(ctx, shape, shift) for name, shape in got.items() if name in outs}
    mh.check(mh.lib().mmh_linear_backward(ctx.handle, form, X.ptr if "dw" in got else None, W.ptr if "dx" in got else None,
                                          ptr(P), D.ptr, rows, k, n, R_ACT[act], p, seed, offset, ptr(got.get("dx")),
                                          ptr(got.get("dw")), ptr(got.get("dbias"))))
    got = {name: b.numpy() for name, b in got.items()}
    if form and "dw" in got:
        got["dw"] = got["dw"].T
    return got


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear_backward(ctx, i, form):
    rows, k, n = SHAPES[i]
    act, p = ACTS[(i + 3 * form) % 5], (0.1, 0.0, 0.6)[(i + form) % 3]
    print(f"\n[linear_backward] {SHAPES[i]} form={form} act={act} p={p}", flush=True)
    x, w, _, dout = operands(rows, k, n, 200 * i + form)
    pre = None if act == "none" and i % 2 else np.random.default_rng(i).standard_normal((rows, n)).astype(np.float32) * 2
    seed, offset = 99 + i, 2 ** 40 + i
    got = run_backward(ctx, form, x, w, pre, dout, act, p, seed, offset)
    want = R.linear_backward(x, w, pre, dout, act, p, seed, offset)
    for name, (value, tol) in want.items():
        near(got[name], value, tol, name)


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("shape", [(40, 33, 70), (512, 384, 1500), (1003, 517, 770), (256, 1500, 5632), (1500, 3000, 768),
                                   (3000, 256, 2816)])
def test_backward_values_outside_the_split(ctx, shape, form):
    """A NaN and an infinity of dout, and values from 2^104 on, reach their row of dx and their column of dW alone, in
    products that run by themselves and together."""
    rows, k, n = shape
    print(f"\n[backward, values outside the split] {shape} {form}", flush=True)
    x, w, _, dout = operands(rows, k, n, 51)
    x[np.abs(x) < 1e-3] = 0.5  # (an infinity times 0 would be NaN)
    w[np.abs(w) < 1e-6] = 0.5
    clean = dout.copy()
    bad = [(5, 3), (9, 11)]
    for r, c in bad:
        clean[r, c] = 0
    dout = clean.copy()
    dout[5, 3], dout[9, 11] = np.nan, np.inf
    dout[20, 17] = clean[20, 17] = np.float32(2.0) ** 105
    got = run_backward(ctx, form, x, w, None, dout, "none", 0.0, 0, 0)
    want = R.linear_backward(x, w, None, clean, "none", 0.0, 0, 0)
    ok_rows, ok_cols = np.setdiff1d(np.arange(rows), [5, 9]), np.setdiff1d(np.arange(n), [3, 11])
    near(got["dx"][ok_rows], want["dx"][0][ok_rows], want["dx"][1][ok_rows], "dx")
    near(got["dw"][:, ok_cols], want["dw"][0][:, ok_cols], want["dw"][1][:, ok_cols], "dw")
    near(got["dbias"][ok_cols], want["dbias"][0][ok_cols], want["dbias"][1][ok_cols], "dbias")
    assert np.isnan(got["dx"][5]).all() and np.isnan(got["dw"][:, 3]).all() and np.isnan(got["dbias"][3])
    assert np.array_equal(got["dx"][9], np.sign(w[:, 11]) * np.float32(np.inf))
    assert np.array_equal(got["dw"][:, 11], np.sign(x[9]) * np.float32(np.inf)) and got["dbias"][11] == np.inf


@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("p", [0.0, 0.5])
def test_backward_of_infinite_and_missing_values(ctx, act, p):
    """One row, so that dbias is dpre: NaN and infinities of pre, and of dout, where the mask keeps them and where it drops
    them (0 there). The slope is 1 at inf and 0 at -inf, a NaN stays one."""
    n, seed, offset = 96, 31, 5
    keep = R.kept(n, p, seed, offset)
    pre = np.resize(np.array([np.nan, np.inf, -np.inf, 0.75], np.float32), n)
    dout = np.repeat(np.array([1.5, -2.0, np.nan], np.float32), n // 3)
    x, w = np.ones((1, 3), np.float32), np.ones((3, n), np.float32)
    got = run_backward(ctx, 0, x, w, pre[None], dout[None], act, p, seed, offset, outs=("dbias",))["dbias"]
    assert not p or 0 < keep.sum() < n
    assert (got[~keep] == 0).all()
    bad = keep & (np.isnan(pre) | (np.isnan(dout) & ((pre > 0) | (act != "relu"))))
    assert np.isnan(got[bad]).all()
    scale = np.float32(1.0 / (1.0 - p))
    for value, slope in ((np.inf, 1.0), (-np.inf, 0.0)):
        at = keep & (pre == np.float32(value)) & ~np.isnan(dout)
        assert np.array_equal(got[at], dout[at] * scale * np.float32(slope)), (act, value)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("outs", [("dx",), ("dw",), ("dbias",), ("dw", "dbias"), ("dx", "dw"), ()])
def test_linear_backward_outputs_and_alignments(ctx, act, outs):
    x, w, _, dout = operands(301, 70, 133, 5)
    pre = np.random.default_rng(1).standard_normal((301, 133)).astype(np.float32)
    for shift in (0, 1, 2):
        got = run_backward(ctx, 0, x, w, pre, dout, act, 0.2, 6, 7, shift, outs)
        want = R.linear_backward(x, w, pre, dout, act, 0.2, 6, 7)
        assert set(got) == set(outs)
        for name in outs:
            near(got[name], *want[name], name)


DROPOUTS = [1, 2, 3, 4, 5, 63, 255, 256, 1023, 4096, 4099, 262144 * 4 + 7, 5003 * 1021]


@pytest.mark.parametrize("n", DROPOUTS)
@pytest.mark.parametrize("p", [0.0, 2.0 ** -40, 0.1, 0.5, 0.9375, 1.0])
def test_dropout(ctx, n, p):
    r = np.random.default_rng(n)
    x, res = (r.standard_normal(n).astype(np.float32) for _ in range(2))
    seed, offset = int(r.integers(2 ** 63)), 2 ** 64 - n // 8 - 1
    keep = R.kept(n, p, seed, offset)
    scale = np.float32(1.0 / (1.0 - float(np.float32(p)))) if p < 1 else np.float32(0)
    want = np.where(keep, x * scale, np.float32(0))
    for shift in (0, 1, 3) if n < 5000 else (0, 2):
        X, S, O = Box(ctx, x, shift), Box(ctx, res, shift), empty(ctx, (n,), shift)
        call = mh.lib().mmh_dropout
        mh.check(call(ctx.handle, X.ptr, None, n, p, seed, offset, O.ptr))
        assert np.array_equal(O.numpy(), want)
        mh.check(call(ctx.handle, X.ptr, S.ptr, n, p, seed, offset, O.ptr))
        assert np.array_equal(O.numpy(), res + want)
        mh.check(mh.lib().mmh_dropout_backward(ctx.handle, X.ptr, n, p, seed, offset, O.ptr))
        assert np.array_equal(O.numpy(), want)
        # in place: over the residual, over x
        mh.check(call(ctx.handle, X.ptr, S.ptr, n, p, seed, offset, S.ptr))
        assert np.array_equal(S.numpy(), res + want)
        mh.check(mh.lib().mmh_dropout_backward(ctx.handle, X.ptr, n, p, seed, offset, X.ptr))
        assert np.array_equal(X.numpy(), want)


def test_dropout_special_values(ctx):
    n = 4096
    x = np.tile(np.array([np.nan, np.inf, -np.inf, 3e38], np.float32), n // 4)
    keep = R.kept(n, 0.25, 11, 0)
    out = mh.dropout(ctx, ctx.to_device(x), 0.25, 11).numpy()
    assert (out[~keep] == 0).all()
    with np.errstate(over="ignore"):
        assert np.array_equal(out[keep], (x * np.float32(1 / 0.75))[keep], equal_nan=True)
    # an array of x itself as its own residual
    one = np.arange(n, dtype=np.float32)
    X = ctx.to_device(one)
    out = mh.dropout(ctx, X, 0.25, 11, residual=X, out=X).numpy()
    assert np.array_equal(out, np.where(keep, one + one * np.float32(1 / 0.75), one))


def run_loss(ctx, form, x, w, targets, ignore=-1, grads=("dx", "dw"), shift=0, loss=True):
    n, d, V = x.shape[0], x.shape[1], w.shape[1]
    X, W = Box(ctx, x, shift), Box(ctx, stored(w, form), shift)
    got = {"dx": (n, d), "dw": stored(w, form).shape}
    got = {name: empty(ctx, shape, shift) for name, shape in got.items() if name in grads}
    value = ctypes.c_float(np.nan)
    t = np.ascontiguousarray(targets, np.int32).ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
    mh.check(mh.lib().mmh_linear_cross_entropy_backward(ctx.handle, form, X.ptr, W.ptr, t, n, d, V, ignore, ptr(got.get("dx")),
                                                        ptr(got.get("dw")), ctypes.byref(value) if loss else None))
    got = {name: b.numpy() for name, b in got.items()}
    if form and "dw" in got:
        got["dw"] = got["dw"].T
    if loss:
        got["loss"] = value.value
        mh.check(mh.lib().mmh_linear_cross_entropy(ctx.handle, form, X.ptr, W.ptr, t, n, d, V, ignore, ctypes.byref(value)))
        got["forward"] = value.value
    return got


# (n, d, vocab): stored logits of small products and folded ones of large tiles; a vocabulary of one, of less than a unit
# of 128 columns, odd ones, wider than a row's registers
HEADS = [(1, 1, 1), (1, 7, 2), (3, 16, 65), (24, 16, 12), (5, 33, 129), (130, 64, 256), (257, 48, 1001), (64, 300, 4099),
         (2048, 128, 4096), (1021, 770, 5003), (33, 40, 32769), (129, 24, 70001), (4100, 31, 2050), (1, 512, 40000), (64, 48, 131072), (65, 48, 32768), (40, 20, 8192)]


def head(n, d, V, seed, sharp=1.0):
    r = np.random.default_rng(seed)
    x = r.standard_normal((n, d)).astype(np.float32)
    w = (r.standard_normal((d, V)) * (sharp / np.sqrt(d))).astype(np.float32)
    return x, w, r.integers(0, V, n).astype(np.int32)


def check_loss(got, want, what=""):
    for name in got:
        value, tol = want["loss" if name == "forward" else name]
        near(np.asarray(got[name]), value, tol, what + name)


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("shape", HEADS)
def test_linear_cross_entropy(ctx, shape, form):
    print(f"\n[linear_cross_entropy] {shape} form={form}", flush=True)
    x, w, t = head(*shape, seed=sum(shape), sharp=3.0 if shape[0] % 2 else 1.0)
    check_loss(run_loss(ctx, form, x, w, t), R.cross_entropy(x, w, t))


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("shape", [(1, 7, 2), (24, 16, 12), (300, 64, 1001), (1021, 130, 4096), (2048, 40, 2050)])
@pytest.mark.parametrize("share", [0.1, 0.9, 1.0])
def test_ignored_rows_leave_no_trace(ctx, shape, form, share):
    print(f"\n[ignored rows] {shape} form={form} {share}", flush=True)
    x, w, t = head(*shape, seed=sum(shape) + 1)
    out = np.random.default_rng(3).random(shape[0]) < share
    t[out] = -100
    want = R.cross_entropy(x, w, t, -100)
    x[out] = np.resize(np.array([np.nan, np.inf, -np.inf, 3e38], np.float32), (out.sum(), shape[1]))
    got = run_loss(ctx, form, x, w, t, ignore=-100)
    check_loss(got, want)
    assert (got["dx"][out] == 0).all()


def test_ignored_class(ctx):
    # the ignored value may be a class: its rows are left out, the class stays in the softmax
    x, w, t = head(400, 32, 10, seed=5)
    check_loss(run_loss(ctx, 0, x, w, t, ignore=4), R.cross_entropy(x, w, t, 4))


@pytest.mark.parametrize("grads", [("dx",), ("dw",), ()])
def test_linear_cross_entropy_outputs(ctx, grads):
    x, w, t = head(257, 48, 1003, seed=6)
    t[::3] = -1
    want = R.cross_entropy(x, w, t)
    for shift in (0, 1, 2, 3):
        got = run_loss(ctx, 0, x, w, t, grads=grads, shift=shift)
        assert set(got) == set(grads) | {"loss", "forward"}
        check_loss(got, want)
    assert set(run_loss(ctx, 1, x, w, t, grads=grads, loss=False)) == set(grads)


def test_far_logits_and_special_rows(ctx):
    # logits of several hundred: most exponentials are 0, a lone top one is the loss of its row
    x, w, t = head(200, 32, 3001, seed=7, sharp=1.0)
    x *= 150.0
    check_loss(run_loss(ctx, 1, x, w, t), R.cross_entropy(x, w, t))
    # equal logits
    z = np.zeros((32, 3001), np.float32)
    check_loss(run_loss(ctx, 0, x, z, t), R.cross_entropy(x, z, t))
    # a NaN in a row that counts: the loss is NaN, and the row's gradient, not the others'
    x, w, t = head(300, 64, 515, seed=8)
    want = R.cross_entropy(x, w, t)
    x[17, 5] = np.nan
    got = run_loss(ctx, 1, x, w, t)
    assert np.isnan(got["loss"]) and np.isnan(got["forward"]) and np.isnan(got["dx"][17]).all()
    rest = np.arange(300) != 17
    near(got["dx"][rest], want["dx"][0][rest], want["dx"][1][rest], "dx")
    # a NaN in a lone column, the first, one inside, the last (alone in its unit of 128, at 4097), that is no row's target
    for V, d, n in ((515, 64, 300), (4097, 64, 1200), (40001, 24, 40), (40001, 24, 100)):
        for at in (0, 77, V - 1):
            x, w, t = head(n, d, V, seed=9)
            t[t == at] = 1
            w[3, at] = np.nan
            got = run_loss(ctx, 1, x, w, t)
            assert np.isnan(got["loss"]) and np.isnan(got["forward"]), (V, at)


def test_row_blocks(ctx):
    """More logits than the workspace holds: blocks of rows, the last a smaller one, gradients added up over blocks."""
    for n, d, V, share in ((1100, 16, 64003, 0.0), (2300, 12, 64003, 0.02)):
        print(f"\n[row blocks] {n} {d} {V}", flush=True)
        x, w, t = head(n, d, V, seed=n)
        t[np.random.default_rng(1).random(n) < share] = -1
        got = run_loss(ctx, 1, x, w, t)
        want = R.cross_entropy(x, w, t, blocks=2)
        check_loss(got, want, f"{n}: ")


@pytest.mark.parametrize("n,d,V,form,share", [(300, 520, 105001, 0, 0.0), (330, 1700, 32100, 1, 0.1), (260, 1664, 32768, 0, 0.0),
                                             (257, 500, 110001, 1, 0.0)])
def test_a_few_rows_past_the_last_tile(ctx, n, d, V, form, share):
    """Beside large weights the few rows past a block's last 256 are a part of their own."""
    print(f"\n[few rows past a tile] {n} {d} {V} {form}", flush=True)
    x, w, t = head(n, d, V, seed=n)
    t[np.random.default_rng(1).random(n) < share] = -1
    check_loss(run_loss(ctx, form, x, w, t), R.cross_entropy(x, w, t), f"{n}: ")


def test_row_blocks_of_the_loss_alone(ctx):
    """More partial sums than the workspace holds: the mean over all rows against that of calls on a few thousand each,
    which take one block. Both are within the bound of a row's term, which other tests hold to 64 bits."""
    n, d, V = 33001, 8, 131072
    x, w, t = head(n, d, V, seed=3)
    X, W = ctx.to_device(x), ctx.to_device(stored(w, 1))
    whole, parts = mh.linear_cross_entropy(ctx, X, W, t), []
    for at in range(0, n, 9000):
        part = ctx.to_device(x[at:at + 9000])
        parts.append(mh.linear_cross_entropy(ctx, part, W, t[at:at + 9000]) * len(t[at:at + 9000]))
        part.free()
    bound = 2 * R.product_bound(d, np.abs(x).sum(1).max() * np.abs(w).max()) + (V / 256 + 40) * 2 * R.U + 64 * R.U
    assert abs(whole - sum(parts) / n) <= 2 * bound


def test_gradients_against_differences(ctx):
    """Central differences of the calls' own values along random directions. The truncation is of third order in the step
    (1e-2 of it here), f32 values are 1e-7 of theirs off, and the sums are taken in 64 bits: 2e-3 of the directional
    derivative's own size is allowed."""
    r = np.random.default_rng(12)
    x, w, b, _ = operands(40, 24, 36, 13)
    dout = r.standard_normal((40, 36)).astype(np.float32)
    for act in ("gelu", "gelu_tanh", "silu"):
        args = (act, 0.3, 5, 6)
        _, pre = run_linear(ctx, 0, x, w, b, None, *args, True)
        g = run_backward(ctx, 0, x, w, pre, dout, *args)
        for name, at in (("dx", 0), ("dw", 1), ("dbias", 2)):
            v = r.standard_normal((x, w, b)[at].shape).astype(np.float32)
            side = []
            for s in (1e-2, -1e-2):
                a = [x, w, b]
                a[at] = (a[at] + np.float32(s) * v).astype(np.float32)
                o, _ = run_linear(ctx, 0, *a, None, *args, False)
                side.append((o.astype(np.float64) * dout).sum())
            along = float((g[name].astype(np.float64) * v).sum())
            size = float(np.linalg.norm(g[name].astype(np.float64)) * np.linalg.norm(v)) / np.sqrt(v.size)
            assert abs((side[0] - side[1]) / 2e-2 - along) <= 2e-3 * max(abs(along), size), (act, name)
    x, w, t = head(64, 24, 200, seed=14)
    g = run_loss(ctx, 0, x, w, t)
    for name, at in (("dx", 0), ("dw", 1)):
        # along the gradient itself, where the derivative is largest
        v = (g[name] / np.linalg.norm(g[name])).astype(np.float32)
        side = []
        for s in (0.05, -0.05):
            a = [x, w]
            a[at] = (a[at] + np.float32(s) * v).astype(np.float32)
            side.append(R.cross_entropy(a[0], a[1], t)["loss"][0])
            assert abs(run_loss(ctx, 0, *a, t)["forward"] - side[-1]) < 1e-5
        along = float((g[name].astype(np.float64) * v).sum())
        assert abs((side[0] - side[1]) / 0.1 - along) <= 2e-3 * abs(along), name


@pytest.mark.parametrize("rows,d,ff,V", [(96, 32, 80, 201), (700, 64, 176, 1009)])
def test_a_training_step_of_them_together(ctx, rows, d, ff, V):
    """dropout of the input, an MLP with dropout and the residual in its epilogues, the loss over a tied head, and all
    gradients back, against the same in 64 bits; the calls queue on one context with nothing waited for between."""
    r = np.random.default_rng(rows)
    x0 = r.standard_normal((rows, d)).astype(np.float32)
    w1, b1 = (r.standard_normal((d, ff)) / np.sqrt(d)).astype(np.float32), r.standard_normal(ff).astype(np.float32) * 0.1
    w2, b2 = (r.standard_normal((d, ff)) / np.sqrt(ff)).astype(np.float32), r.standard_normal(d).astype(np.float32) * 0.1
    e = (r.standard_normal((V, d)) / np.sqrt(d)).astype(np.float32)
    t = r.integers(0, V, rows).astype(np.int32)
    t[::5] = -1
    seed, o1 = 42, (rows * d + 3) // 4
    o2 = o1 + (rows * ff + 3) // 4
    X0, W1, B1, W2, B2, E = (ctx.to_device(a) for a in (x0, w1, b1, w2, b2, e))
    X = mh.dropout(ctx, X0, 0.1, seed)
    P1 = ctx.empty((rows, ff))
    H = mh.linear(ctx, X, W1, B1, activation="gelu_tanh", p=0.2, seed=seed, offset=o1, pre=P1)
    Y = mh.linear(ctx, H, W2, B2, residual=X, form="nt", p=0.1, seed=seed, offset=o2)
    loss, dY, dE = mh.linear_cross_entropy_backward(ctx, Y, E, t)
    dH, dW2, dB2 = mh.linear_backward(ctx, H, W2, dY, form="nt", p=0.1, seed=seed, offset=o2)
    dX, dW1, dB1 = mh.linear_backward(ctx, X, W1, dH, pre=P1, activation="gelu_tanh", p=0.2, seed=seed, offset=o1)
    mh.add(ctx, dX, dY, out=dX)
    dX0 = mh.dropout_backward(ctx, dX, 0.1, seed, out=dX)
    assert abs(mh.linear_cross_entropy(ctx, Y, E, t) - loss) < 1e-5

    # float64, by the chain rule
    x = R.drop(x0.astype(np.float64), 0.1, seed, 0)
    pre = x @ w1 + b1
    h = R.drop(R.act("gelu_tanh", pre), 0.2, seed, o1)
    y = x + R.drop(h @ w2.T + b2, 0.1, seed, o2)
    z = y @ e.T.astype(np.float64)
    z -= z.max(1, keepdims=True)
    prob = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    keep = np.flatnonzero(t >= 0)
    assert abs(-np.log(prob[keep, t[keep]]).mean() - loss) < 1e-5
    dz = np.zeros_like(prob)
    dz[keep] = prob[keep] / len(keep)
    dz[keep, t[keep]] -= 1.0 / len(keep)
    dy = dz @ e
    d2 = R.drop(dy, 0.1, seed, o2)
    d1 = R.drop(d2 @ w2, 0.2, seed, o1) * R.act_grad("gelu_tanh", pre)
    want = dict(dE=dz.T @ y, dW2=d2.T @ h, dB2=d2.sum(0), dW1=x.T @ d1, dB1=d1.sum(0),
                dX0=R.drop(d1 @ w1.T + dy, 0.1, seed, 0))
    for name, got in dict(dE=dE, dW2=dW2, dB2=dB2, dW1=dW1, dB1=dB1, dX0=dX0).items():
        # chained products of f32 sums: each is at most a few 1e-6 of its norm off, and there are eight
        off = np.linalg.norm(got.numpy() - want[name]) / np.linalg.norm(want[name])
        assert off < 1e-5, (name, off)


def test_the_same_bits_again_and_on_two_contexts(ctx):
    """Every call gives the same bits when it is repeated, and while another context runs its own."""
    x, w, t = head(600, 96, 4099, seed=21)
    t[::7] = -1
    a, wl, b, res = operands(520, 700, 391, 22)
    dout = np.random.default_rng(2).standard_normal((520, 391)).astype(np.float32)

    def all_of(c):
        out, pre = run_linear(c, 1, a, wl, b, res, "gelu", 0.3, 1, 2, True)
        g = run_backward(c, 1, a, wl, pre, dout, "gelu", 0.3, 1, 2)
        l = run_loss(c, 0, x, w, t)
        return [out, pre, *g.values(), *(np.float32(v) for v in l.values())]

    first = all_of(ctx)
    with mh.Context(0) as other:
        # two contexts' work in flight at once: queued by turns, read at the end
        X = [c.to_device(a) for c in (ctx, other)]
        W = [c.to_device(stored(wl, 1)) for c in (ctx, other)]
        R2 = [c.to_device(res) for c in (ctx, other)]
        O = [c.empty((520, 391)) for c in (ctx, other)]
        B = [c.to_device(b) for c in (ctx, other)]
        for _ in range(8):
            for i, c in enumerate((ctx, other)):
                mh.linear(c, X[i], W[i], B[i], R2[i], form="nt", activation="gelu", p=0.3, seed=1, offset=2, out=O[i])
        assert all(np.array_equal(o.numpy(), first[0]) for o in O)
        second = all_of(other)
        for arrays in (X, W, R2, O, B):
            for v in arrays:
                v.free()
    for u, v in zip(first, second):
        assert np.array_equal(u, v)
    for u, v in zip(first, all_of(ctx)):
        assert np.array_equal(u, v)


def test_a_refused_call_runs_nothing(ctx):
    x, w, t = head(40, 16, 70, seed=3)
    X, W = ctx.to_device(x), ctx.to_device(stored(w, 1))
    dx, dw = ctx.to_device(np.full((40, 16), 3, np.float32)), ctx.to_device(np.full((70, 16), 4, np.float32))
    for bad in (70, -1, 2 ** 31 - 1):
        t[33] = bad
        with pytest.raises(mh.IndexOutOfRange):
            mh.linear_cross_entropy_backward(ctx, X, W, t, ignore=-2, dx=dx, dw=dw)
        with pytest.raises(mh.IndexOutOfRange):
            mh.linear_cross_entropy(ctx, X, W, t, ignore=-2)
    with pytest.raises(mh.ArgumentError):
        mh.linear_cross_entropy_backward(ctx, X, W, np.zeros(40, np.int32), dx=X, dw=dw)
    with pytest.raises(mh.ArgumentError):
        mh.dropout(ctx, X, 1.5, 1, out=dx)
    with pytest.raises(mh.ArgumentError):
        mh.linear(ctx, X, W, form="nt", activation="gelu", p=-1.0, out=ctx.empty((40, 70)))
    assert (dx.numpy() == 3).all() and (dw.numpy() == 4).all() and np.array_equal(X.numpy(), x)


def test_a_failed_allocation_fails_no_later_call(ctx):
    """The runtime keeps the error of an allocation until it is asked for; the next call's launch is not that call."""
    X = ctx.to_device(np.arange(64, dtype=np.float32))
    with pytest.raises(mh.DeviceError):
        ctx.empty((1 << 45,))
    assert np.array_equal(mh.dropout(ctx, X, 0.0, 1).numpy(), np.arange(64, dtype=np.float32))


def test_two_threads_with_a_context_each(ctx):
    """Calls of two threads at once, each on its own context, give what they give alone."""
    import threading
    x, w, t = head(300, 64, 2050, seed=41)
    t[::9] = -1
    a, wl, b, res = operands(300, 200, 260, 42)
    pre = np.random.default_rng(1).standard_normal((300, 260)).astype(np.float32)

    def work(c, found, turns):
        for _ in range(turns):
            l = run_loss(c, 0, x, w, t)
            out, _ = run_linear(c, 1, a, wl, b, res, "gelu", 0.3, 1, 2, True)
            g = run_backward(c, 1, a, wl, pre, res, "silu", 0.3, 1, 2)
            found.append([l["dx"], l["dw"], np.float32(l["loss"]), np.float32(l["forward"]), out, *g.values()])

    alone = []
    work(ctx, alone, 1)
    with mh.Context(0) as c1, mh.Context(0) as c2:
        found = [[], []]
        threads = [threading.Thread(target=work, args=(c, f, 8)) for c, f in zip((c1, c2), found)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
    for f in found:
        assert len(f) == 8
        for got in f:
            assert all(np.array_equal(u, v) for u, v in zip(got, alone[0]))


def test_arrays_beyond_32_bits(ctx):
    """More than 2^32 values: dropout in place, and a linear layer's output, whose last rows are read back."""
    n, tail = 2 ** 32 + 4099, 8192
    seed, offset = 5, 77
    print("\n[beyond 32 bits] dropout", flush=True)
    try:
        buf = ctx.empty((n,))
    except mh.DeviceError:
        pytest.skip("needs 17 GB of free device memory")
    r = np.random.default_rng(0)
    x = r.standard_normal(tail).astype(np.float32)
    at = buf.offset(n - tail)
    mh.check(mh.lib().mmh_upload(ctx.handle, at, x.ctypes.data, x.nbytes))
    mh.check(mh.lib().mmh_dropout(ctx.handle, buf.ptr, None, n, 0.5, seed, offset, buf.ptr))
    got = np.empty(tail, np.float32)
    mh.check(mh.lib().mmh_download(ctx.handle, got.ctypes.data, at, got.nbytes))
    first = n - tail  # the mask from there on: whole blocks, and the values before the first one
    keep = R.kept(tail + first % 4, 0.5, seed, offset + first // 4)[first % 4:]
    assert np.array_equal(got, np.where(keep, x * np.float32(2), np.float32(0)))

    print("[beyond 32 bits] linear", flush=True)
    cols, k = 2047, 3
    rows = n // cols
    xs = r.standard_normal((rows, k)).astype(np.float32)
    w, b = r.standard_normal((k, cols)).astype(np.float32), r.standard_normal(cols).astype(np.float32)
    X, W, B = ctx.to_device(xs), ctx.to_device(w), ctx.to_device(b)
    mh.check(mh.lib().mmh_linear(ctx.handle, 0, X.ptr, W.ptr, B.ptr, None, rows, k, cols, R_ACT["silu"], 0.25, seed, offset,
                                 None, buf.ptr))
    last = 300
    got = np.empty((last, cols), np.float32)
    mh.check(mh.lib().mmh_download(ctx.handle, got.ctypes.data, buf.offset((rows - last) * cols), got.nbytes))
    want, tol, _, _ = R.linear(xs[-last:], w, b, None, "silu", 0.0, 0, 0)
    first = (rows - last) * cols
    keep = R.kept(last * cols + first % 4, 0.25, seed, offset + first // 4)[first % 4:].reshape(last, cols)
    scale = 1.0 / 0.75
    near(got, np.where(keep, want * scale, 0.0), np.where(keep, tol * scale + 2 * R.U * np.abs(want) * scale, 0.0), "out")

    # the column sums of its |values|, whole and in two parts: each call rounds at most 256 + 4 + 129 + 16 times
    print("[beyond 32 bits] bias gradient", flush=True)
    mh.check(mh.lib().mmh_linear(ctx.handle, 0, X.ptr, W.ptr, B.ptr, None, rows, k, cols, R_ACT["relu"], 0.0, 0, 0, None,
                                 buf.ptr))
    db = [ctx.empty((cols,)) for _ in range(3)]
    half = rows // 2
    for out, start, count in ((db[0], 0, rows), (db[1], 0, half), (db[2], half, rows - half)):
        mh.check(mh.lib().mmh_linear_backward(ctx.handle, 0, None, None, None, buf.offset(start * cols), count, k, cols, 0, 0.0,
                                              0, 0, None, None, out.ptr))
    whole, a, b2 = (v.numpy().astype(np.float64) for v in db)
    near(whole, a + b2, 2 * 405 * R.U * (a + b2), "dbias")
    for v in (buf, X, W, B, *db):
        v.free()
