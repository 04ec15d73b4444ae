"""The linear layer's operators without a device: the oracle's generator against its published vectors, the calls that
are refused before a context is looked up, and the host binding's shape checks."""
import ctypes

import numpy as np
import pytest

import linear_oracle as R
import midman_hip as mh

GOOD = 0  # no context has this handle: a call whose arguments pass ends there
BASE = 0x10000000  # addresses that no call reads


def test_generator_known_answers():
    # the authors' known-answer vectors of philox4x32-10
    for counter, key, want in [
        ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
        ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
        ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
         [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
    ]:
        got = R.philox([np.array([c]) for c in counter], key)[0]
        assert [int(x) for x in got] == want


def test_oracle_mask_rate_and_independence():
    for p in (0.1, 0.5, 0.9):
        m = R.kept(400000, p, 7, 0)
        assert abs(m.mean() - (1 - p)) < 5 * np.sqrt(p * (1 - p) / 400000)
    assert R.kept(1000, 1.0, 7, 0).sum() == 0 and R.kept(1000, 0.0, 7, 0).all()
    # the mask of values 4j.. from offset o is that of values 0.. from o + j
    assert np.array_equal(R.kept(100, 0.3, 5, 9)[40:], R.kept(60, 0.3, 5, 19))
    # the counter wraps
    assert np.array_equal(R.kept(16, 0.3, 5, 2 ** 64 - 2)[8:], R.kept(8, 0.3, 5, 0))


def call(name, *args):
    st = getattr(mh.lib(), "mmh_" + name)(GOOD, *args)
    return st, mh.last_error()


def ptr(i, null=()):
    return None if i in null else BASE + i * (1 << 24)


def linear(form=0, rows=4, k=8, n=12, act=0, p=0.5, null=(), **at):
    a = {name: at.get(name, ptr(i, null)) for i, name in enumerate(("x", "w", "bias", "residual", "pre", "out"))}
    return call("linear", form, a["x"], a["w"], a["bias"], a["residual"], rows, k, n, act, p, 1, 0, a["pre"], a["out"])


def linear_backward(form=0, rows=4, k=8, n=12, act=1, p=0.5, null=(), **at):
    a = {name: at.get(name, ptr(i, null)) for i, name in enumerate(("x", "w", "pre", "dout", "dx", "dw", "dbias"))}
    return call("linear_backward", form, a["x"], a["w"], a["pre"], a["dout"], rows, k, n, act, p, 1, 0, a["dx"], a["dw"],
                a["dbias"])


REACHES = (mh.ERR_ARGUMENT, "invalid context handle 0")


def test_good_calls_reach_the_context():
    assert linear() == REACHES
    assert linear(null=(2, 3, 4)) == REACHES
    assert linear(residual=BASE, out=BASE, x=BASE + (1 << 28)) == REACHES
    assert linear_backward() == REACHES
    assert linear_backward(act=0, null=(2,)) == REACHES
    assert linear_backward(null=(0, 5)) == REACHES       # no dw: no x
    assert linear_backward(null=(1, 4)) == REACHES       # no dx: no w
    assert linear_backward(null=(0, 1, 4, 5, 6)) == REACHES
    assert call("dropout", BASE, None, 7, 0.0, 1, 2, BASE) == REACHES
    assert call("dropout", BASE, BASE + 64, 7, 1.0, 1, 2, BASE + 64) == REACHES
    assert call("dropout_backward", BASE, 7, 0.3, 1, 2, BASE) == REACHES


@pytest.mark.parametrize("p", [-0.1, 1.0000001, float("nan"), float("inf")])
def test_probability_outside_the_unit_interval(p):
    for st, msg in (linear(p=p), linear_backward(p=p), call("dropout", BASE, None, 7, p, 1, 2, BASE),
                    call("dropout_backward", BASE, 7, p, 1, 2, BASE)):
        assert st == mh.ERR_ARGUMENT and "p must be in [0, 1]" in msg


@pytest.mark.parametrize("sizes", [dict(rows=0), dict(k=0), dict(n=0), dict(rows=-1), dict(rows=2 ** 31),
                                   dict(k=2 ** 31), dict(n=2 ** 62), dict(rows=2 ** 31 - 1, n=2 ** 31 - 1)])
def test_sizes(sizes):
    assert linear(**sizes)[0] == mh.ERR_SHAPE
    assert linear_backward(**sizes)[0] == mh.ERR_SHAPE


def test_dropout_sizes_and_nulls():
    for n in (0, -4, 2 ** 62):
        assert call("dropout", BASE, None, n, 0.5, 1, 2, BASE)[0] == mh.ERR_SHAPE
        assert call("dropout_backward", BASE, n, 0.5, 1, 2, BASE)[0] == mh.ERR_SHAPE
    assert call("dropout", None, None, 8, 0.5, 1, 2, BASE)[0] == mh.ERR_ARGUMENT
    assert "null" in call("dropout", BASE, None, 8, 0.5, 1, 2, None)[1]
    assert "null" in call("dropout_backward", None, 8, 0.5, 1, 2, BASE)[1]
    assert "null" in call("dropout_backward", BASE, 8, 0.5, 1, 2, None)[1]


def test_linear_nulls_forms_and_activations():
    for i in (0, 1, 5):
        assert "null" in linear(null=(i,))[1]
    assert "null" in linear_backward(null=(3,))[1]
    assert "null" in linear_backward(null=(2,))[1]  # an activation needs pre
    assert "null" in linear_backward(null=(0,))[1]
    assert "null" in linear_backward(null=(1,))[1]
    for form in (2, -1, 7):
        assert linear(form=form)[0] == mh.ERR_ARGUMENT and "form" in linear(form=form)[1]
        assert linear_backward(form=form)[0] == mh.ERR_ARGUMENT
    for act in (-1, 5):
        assert "activation" in linear(act=act)[1] and "activation" in linear_backward(act=act)[1]


def test_overlaps():
    x, w, pre = ptr(0), ptr(1), ptr(4)
    # one float of one buffer inside the other is an overlap, its neighbour is not
    assert "overlaps x" in linear(out=x + 4 * 8 * 4 - 4)[1]
    assert linear(out=x + 4 * 8 * 4) == REACHES
    assert "overlaps w" in linear(out=w - 4 * 12 * 4 + 4)[1]
    assert linear(out=w - 4 * 12 * 4) == REACHES
    assert "overlaps residual" in linear(out=ptr(3) + 4)[1]
    assert "overlaps out" in linear(pre=ptr(5))[1]
    assert "overlaps bias" in linear(pre=ptr(2) + 4)[1]
    assert "overlaps pre" in linear_backward(dx=ptr(2))[1]
    assert "overlaps dout" in linear_backward(dx=ptr(3))[1]
    assert "overlaps dbias" in linear_backward(dw=ptr(6))[1]
    assert "overlaps x" in linear_backward(dbias=x + 8)[1]
    assert "overlaps x" in call("dropout", BASE, None, 9, 0.5, 1, 2, BASE + 4)[1]
    assert "overlaps residual" in call("dropout", BASE, BASE + 64, 9, 0.5, 1, 2, BASE + 60)[1]
    assert "overlaps dout" in call("dropout_backward", BASE, 9, 0.5, 1, 2, BASE - 8)[1]


def head(n=4, d=8, vocab=6, form=1, targets=(0, 5, -1, 2), ignore=-1, null=(), backward=True, loss=True, **at):
    t = np.array(targets, np.int32)
    value = ctypes.c_float()
    a = {name: at.get(name, ptr(i, null)) for i, name in enumerate(("x", "w", "dx", "dw"))}
    out = ctypes.byref(value) if loss else None
    tp = t.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)) if len(t) else None
    if backward:
        return call("linear_cross_entropy_backward", form, a["x"], a["w"], tp, n, d, vocab, ignore, a["dx"], a["dw"], out)
    return call("linear_cross_entropy", form, a["x"], a["w"], tp, n, d, vocab, ignore, out)


def test_linear_cross_entropy_refusals():
    for b in (False, True):
        assert head(backward=b) == REACHES
        assert head(backward=b, targets=(0, 5, 99, 2), ignore=99) == REACHES
        assert head(backward=b, targets=(0, 5, 6, 2))[0] == mh.ERR_INDEX
        assert head(backward=b, targets=(0, 5, -1, 2), ignore=-100)[0] == mh.ERR_INDEX
        assert head(backward=b, form=2)[0] == mh.ERR_ARGUMENT
        for i in (0, 1):
            assert "null" in head(backward=b, null=(i,))[1]
        assert "null" in head(backward=b, targets=())[1]
        for sizes in (dict(n=0), dict(d=0), dict(vocab=0), dict(d=2 ** 31), dict(vocab=2 ** 31), dict(n=2 ** 40),
                      dict(d=2 ** 30, vocab=2 ** 30)):
            assert head(backward=b, **sizes)[0] == mh.ERR_SHAPE
    assert "null" in head(backward=False, loss=False)[1]
    assert head(loss=False) == REACHES
    assert head(null=(2, 3)) == REACHES
    assert "overlaps w" in head(dx=ptr(1) + 16)[1]
    assert "overlaps dw" in head(dx=ptr(3))[1]
    assert "overlaps x" in head(dw=ptr(0))[1]


class Shaped:
    """An array of the binding's checks: a shape and an address."""

    def __init__(self, *shape):
        self.shape, self.ptr = shape, BASE
        self.size = int(np.prod(shape))


class NoContext:
    handle = GOOD


def test_binding_checks_shapes():
    c, S = NoContext(), Shaped
    with pytest.raises(mh.ShapeError):
        mh.linear(c, S(2, 8), S(12, 8), form="nn", out=S(2, 12))
    with pytest.raises(mh.ShapeError):
        mh.linear(c, S(2, 8), S(8, 12), bias=S(8), out=S(2, 12))
    with pytest.raises(mh.ShapeError):
        mh.linear(c, S(2, 3, 8), S(8, 12), residual=S(6, 12), out=S(2, 3, 12))
    with pytest.raises(mh.ArgumentError):
        mh.linear(c, S(2, 8), S(8, 12), activation="tanh", out=S(2, 12))
    with pytest.raises(mh.ArgumentError):
        mh.linear(c, S(2, 8), S(8, 12), form="tn", out=S(2, 12))
    with pytest.raises(mh.ArgumentError):
        mh.dropout(c, S(8), 0.5, -1, out=S(8))
    with pytest.raises(mh.ArgumentError):
        mh.dropout(c, S(8), 0.5, 1, offset=2 ** 64, out=S(8))
    with pytest.raises(mh.ShapeError):
        mh.dropout(c, S(8), 0.5, 1, residual=S(4), out=S(8))
    with pytest.raises(mh.ShapeError):
        mh.linear_backward(c, S(2, 8), S(8, 12), S(2, 11), dx=S(2, 8), dw=S(8, 12), dbias=S(12))
    with pytest.raises(mh.ShapeError):
        mh.linear_cross_entropy(c, S(4, 8), S(6, 8), np.zeros(3, np.int32))
    with pytest.raises(mh.ShapeError):
        mh.linear_cross_entropy(c, S(4, 8), S(8, 6), np.zeros(4, np.int32))


def block_rows(n, row_bytes, limit=0):
    rows = ctypes.c_int64()
    f = mh.lib().mmh_test_loss_block_rows
    f.argtypes = [ctypes.c_int64] * 3 + [ctypes.POINTER(ctypes.c_int64)]
    assert f(n, row_bytes, limit, ctypes.byref(rows)) == mh.OK
    return rows.value


@pytest.mark.parametrize("limit", [0, 1, 64 << 20, 512 << 20])
def test_blocks_of_the_loss_keep_to_their_workspace(limit):
    """A block's rows fit the bytes given (128 rows always do) and a launch (2^22 rows); they are all there are, whole tiles of 256 or of one size, in
    a quarter more blocks at most than the bytes need."""
    bytes_ = limit or 512 << 20
    r = np.random.default_rng(limit)
    cases = [(8192, 152064 * 4), (1072, 250016 * 4), (514, 522016 * 4), (670, 400000 * 4), (4096, 200000 * 4), (1, 128),
             (4096, 32000 * 4), (817, 131072 * 4), (33001, 8192), (2 ** 31 - 1, 128), (2 ** 31 - 1, 8), (129, 2 ** 33)]
    cases += [(int(2 ** r.uniform(0, 24)), 128 * int(2 ** r.uniform(0, 14))) for _ in range(3000)]
    for n, row_bytes in cases:
        rows, most = block_rows(n, row_bytes, limit), min(2 ** 22, max(128, bytes_ // row_bytes))
        assert 1 <= rows <= min(n, most), (n, row_bytes, rows)
        need = -(-n // most)
        assert rows == n or rows % 256 == 0 or rows == -(-n // need), (n, row_bytes, rows)
        assert -(-n // rows) <= 1.25 * need + 1, (n, row_bytes, rows)


def test_binding_refuses_targets_that_do_not_fit_32_bits():
    c, x, w = NoContext(), Shaped(3, 8), Shaped(6, 8)
    calls = (lambda t, **a: mh.linear_cross_entropy(c, x, w, t, **a),
             lambda t, **a: mh.linear_cross_entropy_backward(c, x, w, t, dx=x, dw=w, **a))
    for f in calls:
        for bad in (np.array([0, 2 ** 32 + 1, 2]), np.array([0, 2 ** 32 - 1, 2], np.uint32), np.array([0.0, 1.5, 2.0]),
                    np.array([0.0, np.nan, 2.0]), np.array([0, 1, -2 ** 40])):
            with pytest.raises(mh.IndexOutOfRange):
                f(bad)
        with pytest.raises(mh.ArgumentError, match="ignore"):
            f([0, 1, 2], ignore=2 ** 32 - 1)
        for good in ([0, 1, 5], np.array([0, -1, 5]), np.array([0, 1, 5], np.uint8), np.array([[0], [1], [5]], np.int32)):
            with pytest.raises(mh.ArgumentError, match="invalid context|overlaps"):
                f(good)
