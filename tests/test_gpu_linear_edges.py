"""GPU checks of what the linear layer's operators promise at their edges: what a call has done when it returns, values that
are not finite, several row blocks, very many rows, every tile that the products take, the activations' digits."""
import ctypes
import math

import numpy as np
import pytest

import linear_oracle as R
import midman_hip as mh
from test_gpu_linear import Box, check_loss, empty, head, near, operands, run_backward, run_linear, stored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grads", [("dx", "dw"), ("dx",), ("dw",)])
def test_a_loss_of_ignored_rows_alone_waits_for_its_zeros(ctx, grads):
    """With every row ignored the gradients are fills, and they too are there when the call returns: read at once through
    another context, whose stream does not wait for this one's, behind work that keeps this one's busy."""
    n, d, V, big = 300, 64, 1001, 8192
    r = np.random.default_rng(1)
    x, w = r.standard_normal((n, d)).astype(np.float32), r.standard_normal((V, d)).astype(np.float32)
    X, W = ctx.to_device(x), ctx.to_device(w)
    outs = {"dx": ctx.to_device(np.full((n, d), 3, np.float32)), "dw": ctx.to_device(np.full((V, d), 4, np.float32))}
    A, C = ctx.empty((big, big)), ctx.empty((big, big))
    mh.dropout(ctx, A, 1.0, 0, out=A)  # (zeros)
    t = np.full(n, -1, np.int32)
    at = {name: outs[name].ptr if name in grads else None for name in outs}
    with mh.Context(0) as other:
        ctx.synchronize()
        for _ in range(12):  # tens of milliseconds
            mh.gemm(ctx, "nn", A, A, C, big, big, big)
        mh.check(mh.lib().mmh_linear_cross_entropy_backward(
            ctx.handle, 1, X.ptr, W.ptr, t.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), n, d, V, -1, at["dx"], at["dw"],
            None))
        for name in grads:
            got = np.empty(outs[name].shape, np.float32)
            mh.check(mh.lib().mmh_download(other.handle, got.ctypes.data, outs[name].ptr, got.nbytes))
            assert (got == 0).all(), name
    for a in (A, C):
        a.free()


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("shift", [0, 1])
def test_relu_backward_is_the_product_with_its_slope(ctx, p, shift):
    """dout * (pre > 0) by IEEE: a NaN of dout stays one where the slope is 0 too, an infinity becomes one there, finite
    values become 0; the others' formula (dout times slope) has it the same way, and a dropped value is 0 whatever it was.
    One row, so that dbias is dpre."""
    n, seed, offset = 120, 41, 9
    pre = np.tile(np.array([-2, 0, -0.0, 3, -np.inf, np.inf], np.float32), n // 6)
    dout = np.repeat(np.array([np.nan, np.inf, -np.inf, 1.5, -2.5], np.float32), n // 5)
    keep = R.kept(n, p, seed, offset)
    with np.errstate(invalid="ignore"):
        want = np.where(keep, dout * (pre > 0).astype(np.float32) * np.float32(1 / (1 - p)), np.float32(0))
    x, w = np.ones((1, 3), np.float32), np.ones((3, n), np.float32)
    got = run_backward(ctx, 0, x, w, pre[None], dout[None], "relu", p, seed, offset, shift, outs=("dbias",))["dbias"]
    assert np.isnan(want).any() and np.array_equal(got, want, equal_nan=True)
    # a NaN of pre stays one beside any dout
    got = run_backward(ctx, 0, x, w, np.full((1, n), np.nan, np.float32), dout[None], "relu", p, seed, offset, shift,
                       outs=("dbias",))["dbias"]
    assert np.isnan(got[keep]).all() and (got[~keep] == 0).all()


def limit_blocks(ctx, limit):
    f = mh.lib().mmh_test_loss_block_bytes
    f.argtypes = [ctypes.c_int64, ctypes.c_int64]
    mh.check(f(ctx.handle, limit))


def block_sizes(n, row_bytes, limit):
    rows = ctypes.c_int64()
    f = mh.lib().mmh_test_loss_block_rows
    f.argtypes = [ctypes.c_int64] * 3 + [ctypes.POINTER(ctypes.c_int64)]
    mh.check(f(n, row_bytes, limit, ctypes.byref(rows)))
    return [min(rows.value, n - at) for at in range(0, n, rows.value)]


# kept rows, rows that the bytes hold, the blocks that this gives
BLOCKS = [(300, 128, [100, 100, 100]), (257, 128, [86, 86, 85]), (1072, 536, [512, 512, 48]), (514, 257, [256, 256, 2]),
          (513, 510, [256, 256, 1]), (769, 511, [385, 384]), (1300, 900, [768, 532])]


@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("ignored", [0, 37])
@pytest.mark.parametrize("d,V", [(40, 1003), (33, 8192), (12, 33001)])
@pytest.mark.parametrize("kept,most,blocks", BLOCKS)
def test_several_row_blocks(ctx, kept, most, blocks, d, V, ignored, form):
    """Blocks of equal sizes, ones cut down to whole tiles, a last one of 48 rows, of 2, of 1; the gradients' (logits) and
    the loss's own (partial sums where the tiles fold it), with every row kept and with some ignored."""
    print(f"\n[several row blocks] {kept} in {blocks}, d {d} V {V} ignored {ignored} form {form}", flush=True)
    x, w, t = head(kept + ignored, d, V, seed=kept + V)
    if ignored:
        t[np.random.default_rng(ignored).choice(kept + ignored, ignored, replace=False)] = -1
        x[t < 0] = np.nan
    want = R.cross_entropy(x if not ignored else np.nan_to_num(x), w, t, blocks=len(blocks))
    row = (V + 31) // 32 * 32 * 4
    folds = V > 32768 or V == 8192 and kept > 512  # (256 tiles of 128x128 and more)
    parts = (V + 127) // 128 * 8 if folds else row
    assert block_sizes(kept, row, most * row) == block_sizes(kept, parts, most * parts) == blocks
    X, W = Box(ctx, x), Box(ctx, stored(w, form))
    dx, dw = empty(ctx, x.shape), empty(ctx, stored(w, form).shape)
    tp = t.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))
    loss = ctypes.c_float(np.nan)
    try:
        limit_blocks(ctx, most * row)
        mh.check(mh.lib().mmh_linear_cross_entropy_backward(ctx.handle, form, X.ptr, W.ptr, tp, len(t), d, V, -1, dx.ptr,
                                                            dw.ptr, ctypes.byref(loss)))
        got = {"dx": dx.numpy(), "dw": dw.numpy().T if form else dw.numpy(), "loss": loss.value}
        limit_blocks(ctx, most * parts)
        mh.check(mh.lib().mmh_linear_cross_entropy(ctx.handle, form, X.ptr, W.ptr, tp, len(t), d, V, -1, ctypes.byref(loss)))
        got["forward"] = loss.value
    finally:
        limit_blocks(ctx, 0)
    check_loss(got, want)
    assert (got["dx"][t < 0] == 0).all()


@pytest.mark.parametrize("form", [0, 1])
def test_row_blocks_beside_large_weights(ctx, form):
    """Blocks whose few rows past the last 256 are a part of their own, in the first block and in later ones."""
    d, V, kept, most = 1700, 32100, 1600, 560
    row, parts = (V + 31) // 32 * 32 * 4, (V + 127) // 128 * 8
    print(f"\n[row blocks beside large weights] {form}", flush=True)
    assert d * V >= 52 << 20 and block_sizes(kept, row, most * row) == [512, 512, 512, 64]
    x, w, t = head(kept, d, V, seed=4)
    want = R.cross_entropy(x, w, t, blocks=4)
    X, W = ctx.to_device(x), ctx.to_device(stored(w, form))
    try:
        limit_blocks(ctx, most * row)
        loss, dx, dw = mh.linear_cross_entropy_backward(ctx, X, W, t, form=("nn", "nt")[form])
        limit_blocks(ctx, most * parts)
        forward = mh.linear_cross_entropy(ctx, X, W, t, form=("nn", "nt")[form])
    finally:
        limit_blocks(ctx, 0)
    dw = dw.numpy().T if form else dw.numpy()
    check_loss({"loss": loss, "forward": forward, "dx": dx.numpy(), "dw": dw}, want)


def test_the_loss_alone_over_more_rows_than_a_block(ctx):
    """The ordinary workspace holds the partial sums of 65536 rows of 131072 columns. The mean over more rows against that of
    calls of one block each, both within the bound of a row's term."""
    n, d, V = 70000, 8, 131072
    x, w, t = head(n, d, V, seed=5)
    t[::100] = -1
    x[::100] = np.nan
    keep = t >= 0
    blocks = block_sizes(int(keep.sum()), V // 128 * 8, 0)
    assert len(blocks) == 2
    print(f"\n[the loss of blocks of {blocks} rows]", flush=True)
    X, W = ctx.to_device(x), ctx.to_device(stored(w, 1))
    whole, parts = mh.linear_cross_entropy(ctx, X, W, t), []
    for at in range(0, n, 20000):
        part, ids = ctx.to_device(x[at:at + 20000]), t[at:at + 20000]
        parts.append(mh.linear_cross_entropy(ctx, part, W, ids) * (ids >= 0).sum())
        part.free()
    bound = 2 * R.product_bound(d, np.abs(x[keep]).sum(1).max() * np.abs(w).max()) + (V / 256 + 40) * 2 * R.U + 64 * R.U
    assert abs(whole - sum(parts) / keep.sum()) <= 2 * bound


def test_more_rows_than_the_smallest_tiles_cover(ctx):
    """A launch has less than 2^32 threads: 2^29 rows and more take larger tiles than 64x64. The rows repeat a pattern, so
    every output is known from one pass over it."""
    rows, p = 2 ** 29 + 77, 4099
    print(f"\n[many rows] {rows}", flush=True)
    x = np.random.default_rng(1).standard_normal(p).astype(np.float32)
    w, b = np.full((1, 1), 0.75, np.float32), np.full(1, 0.125, np.float32)
    try:
        X, O = ctx.empty((rows, 1)), ctx.empty((rows, 1))
    except mh.DeviceError:
        pytest.skip("needs 4.3 GB of free device memory")
    whole = np.resize(x, rows)[:, None]
    X.upload(whole)
    W, B = ctx.to_device(w), ctx.to_device(b)

    def repeats(first, tol):
        got = O.numpy()[:, 0]
        near(got[:p], first, tol, "the first rows")
        assert np.array_equal(got[:rows // p * p].reshape(-1, p), np.broadcast_to(got[:p], (rows // p, p)))
        assert np.array_equal(got[rows // p * p:], got[:rows % p])

    mh.linear(ctx, X, W, B, activation="silu", out=O)
    want, tol, _, _ = R.linear(x[:, None], w, b, None, "silu", 0.0, 0, 0)
    repeats(want[:, 0], tol[:, 0])
    print("[many rows] dx", flush=True)
    mh.check(mh.lib().mmh_linear_backward(ctx.handle, 0, None, W.ptr, None, X.ptr, rows, 1, 1, 0, 0.0, 0, 0, O.ptr, None, None))
    repeats(x.astype(np.float64) * 0.75, 2 * R.U * np.abs(x))
    for a in (X, O, W, B):
        a.free()


@pytest.mark.parametrize("ignored", [False, True])
def test_the_loss_of_very_many_rows(ctx, ignored):
    """2^26 rows of a narrow vocabulary, whose partial sums would all fit one block but not one launch. The rows repeat a
    pattern of 4096: the mean is the pattern's, a row's gradient its own divided by the repetitions (a power of two)."""
    p, times, V = 4096, 2 ** 14, 100
    n = p * times
    print(f"\n[very many rows] {n} {ignored}", flush=True)
    x, w, t = head(p, 1, V, seed=6)
    if ignored:
        t[5::17] = -1
    want = R.cross_entropy(x, w, t)
    try:
        X, dX = ctx.empty((n, 1)), ctx.empty((n, 1))
    except mh.DeviceError:
        pytest.skip("needs 0.6 GB of free device memory")
    X.upload(np.tile(x, (times, 1)))
    W = ctx.to_device(w)
    ids = np.tile(t, times)
    loss = mh.linear_cross_entropy(ctx, X, W, ids, form="nn")
    check_loss({"loss": loss}, want)
    value = ctypes.c_float()
    mh.check(mh.lib().mmh_linear_cross_entropy_backward(
        ctx.handle, 0, X.ptr, W.ptr, ids.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), n, 1, V, -1, dX.ptr, None,
        ctypes.byref(value)))
    got = dX.numpy().reshape(times, p)
    check_loss({"loss": value.value, "dx": got[0][:, None] * np.float32(times)}, want)
    assert np.array_equal(got, np.broadcast_to(got[0], (times, p)))
    X.free(), dX.free()


# (form, rows, k, n, tile rows and columns, K splits) of mmh_linear on 256 CUs: every tile, whole and split
FORWARD_PLANS = [
    (0, 1, 1, 1, (32, 32, 1)), (0, 1, 536, 1, (32, 32, 2)), (0, 68, 1817, 3274, (128, 128, 8)),
    (0, 177, 2534, 599, (64, 64, 8)), (0, 395, 1, 8778, (256, 128, 1)), (0, 397, 1126, 8553, (256, 256, 3)),
    (0, 576, 1, 11456, (128, 128, 1)), (0, 1192, 107, 9803, (256, 256, 1)), (0, 2436, 3342, 33, (128, 64, 12)),
    (0, 3205, 381, 220, (64, 64, 1)), (0, 10174, 1124, 90, (256, 128, 5)), (0, 11388, 1, 290, (128, 64, 1)),
    (1, 1, 1, 1, (32, 32, 1)), (1, 1, 225, 1, (32, 32, 2)), (1, 68, 1817, 3274, (128, 128, 8)),
    (1, 177, 2534, 599, (64, 64, 8)), (1, 395, 1, 8778, (256, 128, 1)), (1, 397, 1126, 8553, (256, 256, 3)),
    (1, 576, 1, 11456, (128, 128, 1)), (1, 1192, 107, 9803, (256, 256, 1)), (1, 2436, 3342, 33, (128, 64, 12)),
    (1, 3205, 381, 220, (64, 64, 1)), (1, 10174, 1124, 90, (256, 128, 5)), (1, 11388, 1, 290, (128, 64, 1))]
# the same with the splits of dx and dw, for the tiles that mmh_linear_backward takes for both in one launch: neither, either
# and both of them split, and for both the rows of either a multiple of four floats or not (the sums' 16-byte form)
BACKWARD_PLANS = [
    (0, 412, 667, 994, (64, 64, 1, 1)), (0, 5398, 57, 874, (64, 64, 1, 8)), (0, 531, 279, 1817, (64, 64, 2, 1)),
    (0, 4552, 22, 2718, (64, 64, 3, 6)), (0, 3741, 21, 3592, (64, 64, 2, 2)), (0, 2514, 52, 2134, (64, 64, 3, 4)),
    (0, 1152, 192, 1216, (64, 64, 2, 2)), (0, 177, 2534, 599, (128, 64, 1, 1)), (0, 4036, 250, 273, (128, 64, 1, 8)),
    (0, 214, 382, 3293, (128, 64, 8, 1)), (0, 1124, 315, 759, (128, 64, 2, 3)), (0, 168, 7170, 230, (128, 128, 1, 1)),
    (0, 2404, 1109, 102, (128, 128, 1, 8)), (0, 70, 1086, 3562, (128, 128, 8, 1)), (0, 2980, 78, 1185, (128, 128, 4, 8)),
    (0, 164, 9477, 233, (256, 128, 1, 1)), (0, 386, 8409, 85, (256, 128, 1, 3)), (0, 144, 2534, 817, (256, 128, 6, 1)),
    (0, 3010, 129, 1543, (256, 128, 4, 8)), (0, 305, 11253, 335, (256, 256, 1, 1)),
    (0, 1830, 4527, 138, (256, 256, 1, 6)), (0, 395, 4679, 1691, (256, 256, 3, 1)),
    (0, 7406, 137, 2947, (256, 256, 4, 8)), (1, 412, 667, 994, (64, 64, 1, 1)), (1, 5398, 57, 874, (64, 64, 1, 8)),
    (1, 270, 722, 1390, (64, 64, 2, 1)), (1, 2548, 43, 2854, (64, 64, 3, 3)), (1, 4921, 63, 976, (64, 64, 2, 6)),
    (1, 4108, 56, 1295, (64, 64, 2, 6)), (1, 1152, 64, 3776, (64, 64, 6, 2)), (1, 177, 2534, 599, (128, 64, 1, 1)),
    (1, 4036, 250, 273, (128, 64, 1, 8)), (1, 214, 382, 3293, (128, 64, 8, 1)), (1, 1124, 315, 759, (128, 64, 3, 4)),
    (1, 148, 7122, 259, (128, 128, 1, 1)), (1, 2404, 1109, 102, (128, 128, 1, 8)), (1, 171, 1009, 1570, (128, 128, 6, 1)),
    (1, 2980, 78, 1185, (128, 128, 4, 8)), (1, 157, 9065, 191, (256, 128, 1, 1)), (1, 733, 4402, 86, (256, 128, 1, 4)),
    (1, 144, 2534, 817, (256, 128, 6, 1)), (1, 3299, 78, 3227, (256, 128, 8, 8)), (1, 305, 11253, 335, (256, 256, 1, 1)),
    (1, 1830, 4527, 138, (256, 256, 1, 6)), (1, 341, 3231, 2633, (256, 256, 4, 1)),
    (1, 7406, 137, 2947, (256, 256, 4, 8))]


def plan(ctx, form, rows, k, n, backward):
    out, x = (ctypes.c_int32 * 4)(), ctx.empty((4,))
    f = mh.lib().mmh_test_linear_plan
    f.argtypes = [ctypes.c_int64, ctypes.c_int32, ctypes.c_void_p] + [ctypes.c_int64] * 3 + [
        ctypes.c_int32, ctypes.POINTER(ctypes.c_int32)]
    mh.check(f(ctx.handle, form, x.ptr, rows, k, n, backward, out))
    x.free()
    return tuple(out)


def on_256_cus(ctx):
    if ctx.device_info()[1] != 256:
        pytest.skip("the plans are those of 256 CUs")


@pytest.mark.parametrize("form,rows,k,n,want", FORWARD_PLANS)
def test_linear_on_every_tile(ctx, form, rows, k, n, want):
    on_256_cus(ctx)
    assert plan(ctx, form, rows, k, n, 0)[:3] == want
    print(f"\n[linear] {form} {rows} {k} {n} {want}", flush=True)
    x, w, b, res = operands(rows, k, n, rows + n)
    out, pre = run_linear(ctx, form, x, w, b, res, "gelu", 0.25, 3, 4, True)
    value, tol, want_pre, pre_tol = R.linear(x, w, b, res, "gelu", 0.25, 3, 4)
    near(out, value, tol, "out")
    near(pre, want_pre, pre_tol, "pre")


@pytest.mark.parametrize("form,rows,k,n,want", BACKWARD_PLANS)
def test_linear_backward_on_every_pair_of_tiles(ctx, form, rows, k, n, want):
    on_256_cus(ctx)
    assert plan(ctx, form, rows, k, n, 1) == want
    print(f"\n[linear_backward] {form} {rows} {k} {n} {want}", flush=True)
    x, w, _, dout = operands(rows, k, n, rows + k)
    pre = np.random.default_rng(k).standard_normal((rows, n)).astype(np.float32)
    assert x.shape == (rows, k) and w.shape == (k, n) and dout.shape == pre.shape == (rows, n)
    got = run_backward(ctx, form, x, w, pre, dout, "silu", 0.1, 5, 6)
    for name, (value, tol) in R.linear_backward(x, w, pre, dout, "silu", 0.1, 5, 6).items():
        near(got[name], value, tol, name)


def test_products_that_are_not_joined(ctx):
    """Small products and ones that two launches are estimated to take less time for."""
    on_256_cus(ctx)
    for form, rows, k, n in ((0, 64, 64, 176), (1, 64, 64, 176), (0, 4096, 1024, 2816), (1, 4096, 1024, 2816)):
        assert plan(ctx, form, rows, k, n, 1) == (0, 0, 0, 0)


def exact_activations(x):
    """{activation: (value, slope, the exponent whose rounding its far tail shows)} in 64 bits, by forms that do not cancel."""
    tail = 0.5 * np.vectorize(math.erfc)(np.abs(x) / math.sqrt(2.0))  # Phi(-|x|)
    cdf = np.where(x < 0, tail, 1.0 - tail)

    def sigmoid(y):
        e = np.exp(-np.abs(y))
        return np.where(y < 0, e, 1.0) / (1.0 + e)

    y = 2.0 * R.C0 * (x + R.C1 * x ** 3)
    return {"gelu": (x * cdf, cdf + x * np.exp(-0.5 * x * x) / math.sqrt(2.0 * math.pi), 0.0),
            "silu": (x * sigmoid(x), sigmoid(x) * (1.0 + x * sigmoid(-x)), 0.0),
            "gelu_tanh": (x * sigmoid(y),
                          sigmoid(y) + x * sigmoid(y) * sigmoid(-y) * 2.0 * R.C0 * (1.0 + 3.0 * R.C1 * x * x), np.abs(y))}


def test_activations_keep_their_digits(ctx):
    """Relative to the value itself, far tails too. In u = 2^-24: an exponential of a carried argument is off by 5 (the
    hardware's 2, three roundings); gelu's tail adds its polynomial's fit (1), argument (2), steps (2) and two products: 12,
    and 1 - tail and a product to that: 14; a sigmoid's small side is the exponential (4), over 1 + it (4), a product each:
    10; gelu_tanh's argument, six roundings, is 6 |y| more of it. The slopes, at most 1.13, are sums of such terms: 16 u.
    An exponential below 2^-126 is 0."""
    r = np.random.default_rng(7)
    v = np.concatenate([np.linspace(-13, 13, 400001), r.standard_normal(100000), 10.0 ** r.uniform(-30, 0, 20000),
                        -10.0 ** r.uniform(-30, 0, 20000)]).astype(np.float32)
    n, one = len(v), np.ones((1, 1), np.float32)
    for act, (value, slope, y) in exact_activations(v.astype(np.float64)).items():
        out, pre = run_linear(ctx, 0, one, v[None], None, None, act, 0.0, 0, 0, True)
        assert np.array_equal(pre[0], v)
        bound = {"gelu": 14, "silu": 10, "gelu_tanh": 10 + 6 * y}[act]
        near(out[0], value, bound * R.U * np.abs(value) + 2 * R.TINY * np.abs(v), act)
        got = run_backward(ctx, 0, one, v[None], v[None], np.ones((1, n), np.float32), act, 0.0, 0, 0, outs=("dbias",))
        near(got["dbias"], slope, np.full(n, 16 * R.U), act + " slope")
