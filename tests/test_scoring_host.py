"""Scoring, distillation and rotary positions without a device: the oracle against differences, the calls that are refused
before a context is looked up, and the host binding's shape checks."""
import ctypes

import numpy as np
import pytest

import midman_hip as mh
import scoring_oracle as R

GOOD = 0  # no context has this handle: a call whose arguments pass ends there
BASE = 0x10000000  # addresses that no call reads
REACHES = (mh.ERR_ARGUMENT, "invalid context handle 0")
IDS = ctypes.POINTER(ctypes.c_int32)


def call(name, *args):
    args = [a.ctypes.data_as(IDS) if isinstance(a, np.ndarray) else a for a in args]
    st = getattr(mh.lib(), "mmh_" + name)(GOOD, *args)
    return st, mh.last_error()


def at(i):
    return BASE + i * (1 << 24)


T4 = np.array([0, 3, 5, 2], np.int32)


def logprobs(logits=at(0), targets=T4, n=4, vocab=6, ignore=-1, k=2, lp=at(1), h=at(2), ids=at(3), top=at(4)):
    return call("token_logprobs", logits, targets, n, vocab, ignore, k, lp, h, ids, top)


def logprobs_bwd(logits=at(0), targets=T4, n=4, vocab=6, ignore=-1, dl=at(1), dh=at(2), out=at(3)):
    return call("token_logprobs_backward", logits, targets, n, vocab, ignore, dl, dh, out)


def distill(logits=at(0), targets=T4, n=4, vocab=6, ignore=-1, ids=at(1), teacher=at(2), k=3, temperature=2.0, alpha=0.5, out=None,
            loss=True, grad=False):
    keep = ctypes.c_float()
    tail = [out if out is not None else at(3)] if grad else []
    return call("distillation" + ("_backward" if grad else ""), logits, targets, n, vocab, ignore, ids, teacher, k, temperature, alpha,
                *tail, ctypes.byref(keep) if loss else None)


def tables(width=8, positions=16, theta=1e4, scaling=3, factor=4.0, trained=64, low=1.0, high=32.0, amplitude=1.0, cos=at(0), sin=at(1)):
    return call("rotary_tables", width, positions, theta, scaling, factor, trained, low, high, amplitude, cos, sin)


def rotary(layout=0, q=at(0), k=at(1), pos=None, b=2, h=4, hkv=2, t=3, hd=8, width=6, table=5, cos=at(2), sin=at(3), qo=at(4), ko=at(5),
           back=False):
    return call("rotary" + ("_backward" if back else ""), layout, q, k, pos, b, h, hkv, t, hd, width, table, cos, sin, qo, ko)


def test_good_calls_reach_the_context():
    assert logprobs() == REACHES
    assert logprobs(targets=None, lp=None) == REACHES
    assert logprobs(k=0, ids=None, top=None) == REACHES
    assert logprobs(lp=None, h=None, k=0) == REACHES
    assert logprobs(k=6) == REACHES
    assert logprobs(targets=np.array([0, -7, 5, 2], np.int32), ignore=-7) == REACHES
    assert logprobs(targets=np.array([0, 100, 5, 2], np.int32), ignore=100) == REACHES
    assert logprobs_bwd() == REACHES
    assert logprobs_bwd(out=at(0)) == REACHES
    assert logprobs_bwd(targets=None, dl=None) == REACHES
    assert logprobs_bwd(dl=None, dh=None) == REACHES
    for grad in (False, True):
        assert distill(grad=grad) == REACHES
        assert distill(grad=grad, targets=None, alpha=1.0) == REACHES
        assert distill(grad=grad, alpha=0.0, k=256) == REACHES
        assert distill(grad=grad, temperature=1000.0) == REACHES
    assert distill(grad=True, out=at(0)) == REACHES
    assert distill(grad=True, loss=False) == REACHES
    assert tables() == REACHES
    assert tables(scaling=0, factor=float("nan"), trained=0, low=5.0, high=1.0) == REACHES
    for back in (False, True):
        assert rotary(back=back) == REACHES
        assert rotary(back=back, q=None, h=-1, qo=None) == REACHES
        assert rotary(back=back, k=None, hkv=0, ko=None) == REACHES
        assert rotary(back=back, qo=at(0), ko=at(1)) == REACHES
        assert rotary(back=back, pos=np.array([4, 4, 0, 1, 2, 3], np.int32)) == REACHES
        assert rotary(back=back, hd=7) == REACHES


def refused(result, status, words):
    assert result[0] == status and words in result[1], result


def test_logits_and_targets_that_are_refused():
    for f in (logprobs, logprobs_bwd, distill, lambda **a: distill(grad=True, **a)):
        refused(f(logits=None), mh.ERR_ARGUMENT, "logits is a null pointer")
        refused(f(n=0), mh.ERR_SHAPE, "rows must be at least 1")
        refused(f(n=1 << 31), mh.ERR_SHAPE, "rows must be below 2^31")
        refused(f(vocab=0), mh.ERR_SHAPE, "vocab must be at least 1")
        refused(f(vocab=1 << 31), mh.ERR_SHAPE, "vocab must be below 2^31")
        refused(f(targets=np.array([0, 1, 6, 2], np.int32)), mh.ERR_INDEX, "target 6 is out of range for 6")
        refused(f(targets=np.array([0, 1, -2, 2], np.int32)), mh.ERR_INDEX, "target -2 is out of range for 6")


def test_token_logprobs_refusals():
    refused(logprobs(k=-1), mh.ERR_SHAPE, "k must be 0 to 6")
    refused(logprobs(k=7), mh.ERR_SHAPE, "k must be 0 to 6")
    refused(logprobs(k=257, vocab=1000), mh.ERR_SHAPE, "k must be 0 to 256")
    refused(logprobs(targets=None), mh.ERR_ARGUMENT, "targets (of log probabilities)")
    refused(logprobs(ids=None), mh.ERR_ARGUMENT, "top_ids")
    refused(logprobs(top=None), mh.ERR_ARGUMENT, "top_logprobs")
    refused(logprobs(lp=at(0) + 92), mh.ERR_ARGUMENT, "logprobs overlaps logits")
    refused(logprobs(h=at(1) + 12), mh.ERR_ARGUMENT, "logprobs overlaps entropy")
    refused(logprobs(ids=at(2)), mh.ERR_ARGUMENT, "entropy overlaps top_ids")
    refused(logprobs(ids=at(4) + 28), mh.ERR_ARGUMENT, "top_ids overlaps top_logprobs")
    refused(logprobs(top=at(0)), mh.ERR_ARGUMENT, "top_logprobs overlaps logits")
    refused(logprobs_bwd(out=None), mh.ERR_ARGUMENT, "dlogits is a null pointer")
    refused(logprobs_bwd(targets=None), mh.ERR_ARGUMENT, "targets (of log probabilities)")
    refused(logprobs_bwd(out=at(0) + 4), mh.ERR_ARGUMENT, "dlogits overlaps logits")
    refused(logprobs_bwd(out=at(1) - 92), mh.ERR_ARGUMENT, "dlogits overlaps dlogprobs")
    refused(logprobs_bwd(out=at(2)), mh.ERR_ARGUMENT, "dlogits overlaps dentropy")


@pytest.mark.parametrize("grad", [False, True])
def test_distillation_refusals(grad):
    refused(distill(grad=grad, ids=None), mh.ERR_ARGUMENT, "teacher_ids is a null pointer")
    refused(distill(grad=grad, teacher=None), mh.ERR_ARGUMENT, "teacher_logits is a null pointer")
    for k in (0, -1, 257):
        refused(distill(grad=grad, k=k), mh.ERR_SHAPE, "k must be 1 to 256")
    for t in (0.0, -1.0, 0.0009, 1001.0, float("nan"), float("inf")):
        refused(distill(grad=grad, temperature=t), mh.ERR_ARGUMENT, "temperature must be in [0.001, 1000]")
    for a in (-0.001, 1.001, float("nan")):
        refused(distill(grad=grad, alpha=a), mh.ERR_ARGUMENT, "alpha must be in [0, 1]")
    refused(distill(grad=grad, targets=None), mh.ERR_ARGUMENT, "targets (of alpha below 1)")
    if grad:
        refused(distill(grad=True, out=0), mh.ERR_ARGUMENT, "dlogits is a null pointer")
        refused(distill(grad=True, out=at(0) + 4), mh.ERR_ARGUMENT, "dlogits overlaps logits")
        refused(distill(grad=True, out=at(1)), mh.ERR_ARGUMENT, "dlogits overlaps teacher_ids")
        refused(distill(grad=True, out=at(2) + 44), mh.ERR_ARGUMENT, "dlogits overlaps teacher_logits")
    else:
        refused(distill(loss=False), mh.ERR_ARGUMENT, "loss is a null pointer")


def test_rotary_refusals():
    refused(tables(width=7), mh.ERR_SHAPE, "width must be even")
    refused(tables(width=0), mh.ERR_SHAPE, "width must be at least 1")
    refused(tables(positions=0), mh.ERR_SHAPE, "positions must be at least 1")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        refused(tables(theta=bad), mh.ERR_ARGUMENT, "theta must be positive and finite")
        refused(tables(factor=bad), mh.ERR_ARGUMENT, "factor must be positive and finite")
        refused(tables(amplitude=bad), mh.ERR_ARGUMENT, "amplitude must be positive and finite")
    for scaling in (-1, 4):
        refused(tables(scaling=scaling), mh.ERR_ARGUMENT, "unknown scaling")
    refused(tables(trained=0), mh.ERR_SHAPE, "trained length must be at least 1")
    for low, high in ((2.0, 2.0), (-1.0, 2.0), (1.0, float("inf")), (float("nan"), 2.0)):
        refused(tables(low=low, high=high), mh.ERR_ARGUMENT, "low must be at least 0")
    refused(tables(cos=None), mh.ERR_ARGUMENT, "cos is a null pointer")
    refused(tables(sin=at(0) + 4 * 63), mh.ERR_ARGUMENT, "cos overlaps sin")
    for back in (False, True):
        def r(**a):
            return rotary(back=back, **a)
        refused(r(layout=2), mh.ERR_ARGUMENT, "unknown layout 2")
        refused(r(q=None, k=None), mh.ERR_ARGUMENT, "neither q nor k")
        refused(r(qo=None), mh.ERR_ARGUMENT, "q_out is a null pointer")
        refused(r(ko=None), mh.ERR_ARGUMENT, "k_out is a null pointer")
        refused(r(cos=None), mh.ERR_ARGUMENT, "cos is a null pointer")
        for name in ("b", "h", "hkv", "t", "hd", "table"):
            refused(r(**{name: 0}), mh.ERR_SHAPE, "must be at least 1")
        for width in (0, 1, 5, 10, -2):
            refused(r(width=width), mh.ERR_SHAPE, "width must be even and 2 to 8")
        refused(r(h=32768), mh.ERR_SHAPE, "at most 32767 heads")
        refused(r(b=1 << 16, t=1 << 15, table=1 << 15), mh.ERR_SHAPE, "positions must be below 2^31")
        refused(r(t=6), mh.ERR_SHAPE, "6 positions but tables of 5")
        refused(r(pos=np.array([0, 1, 2, 3, 4, 5], np.int32)), mh.ERR_INDEX, "rotary position 5 is out of range for 5")
        refused(r(pos=np.array([0, 1, 2, 3, -1, 4], np.int32)), mh.ERR_INDEX, "rotary position -1")
        refused(r(qo=at(0) + 4), mh.ERR_ARGUMENT, "q_out overlaps q")
        refused(r(qo=at(1)), mh.ERR_ARGUMENT, "q_out overlaps k")
        refused(r(ko=at(4)), mh.ERR_ARGUMENT, "q_out overlaps k_out")
        refused(r(ko=at(0)), mh.ERR_ARGUMENT, "k_out overlaps q")
        refused(r(qo=at(2)), mh.ERR_ARGUMENT, "q_out overlaps cos")


def test_oracle_gradients_are_the_differences():
    r = np.random.default_rng(0)
    z = (2 * r.standard_normal((3, 11))).astype(np.float64)
    y = np.array([0, 10, 4])
    dl, dh = r.standard_normal(3), r.standard_normal(3)
    ids = r.integers(0, 11, (3, 5)).astype(np.int32)
    ids[1, 3:] = -1
    ids[2, 1] = ids[2, 0]
    teacher = r.standard_normal((3, 5))

    def scores(v):
        (lp, _), (h, _), _ = R.token_logprobs(v, y, 1)
        return (lp * dl + h * dh).sum()

    def loss(v):
        return R.distillation(v, y, ids, teacher, 1.7, 0.6, 3)[0].sum() / 3

    for f, g in ((scores, R.token_logprobs_backward(z, y, dl, dh)[0]), (loss, R.distillation(z, y, ids, teacher, 1.7, 0.6, 3)[2])):
        for i in range(3):
            for j in range(11):
                s = np.zeros_like(z)
                s[i, j] = 1e-5
                assert abs((f(z + s) - f(z - s)) / 2e-5 - g[i, j]) < 1e-8


def test_binding_checks_shapes():
    class Fake:
        def __init__(self, shape, dtype=np.float32):
            self.shape, self.dtype, self.ptr = shape, np.dtype(dtype), BASE
            self.size = int(np.prod(shape))

    class Ctx:
        handle = 0

        def empty(self, shape, dtype=np.float32):
            return Fake(shape if isinstance(shape, tuple) else (shape,), dtype)

    c, z = Ctx(), Fake((2, 3, 9))
    y = np.zeros((2, 3), np.int32)
    for f in (lambda **a: mh.token_logprobs(c, z, **a), lambda **a: mh.token_logprobs_backward(c, z, **a)):
        with pytest.raises(mh.ShapeError):
            f(targets=np.zeros(5, np.int32))
        with pytest.raises(mh.IndexOutOfRange):
            f(targets=np.full((2, 3), 1 << 32))
        with pytest.raises(mh.ArgumentError):
            f(targets=y, ignore=1 << 31)
    for k in (-1, 10):
        with pytest.raises(mh.ShapeError):
            mh.token_logprobs(c, z, y, k=k)
    with pytest.raises(mh.ShapeError):
        mh.token_logprobs_backward(c, z, y, dlogprobs=Fake((6,)))
    with pytest.raises(mh.ArgumentError):
        mh.token_logprobs_backward(c, z, y, dentropy=Fake((2, 3), np.int32))
    for ids, teacher, error in ((Fake((2, 3, 4)), Fake((2, 3, 4)), mh.ArgumentError),
                                (Fake((2, 3, 4), np.int32), Fake((2, 3, 5)), mh.ShapeError),
                                (Fake((6, 4), np.int32), Fake((6, 4)), mh.ShapeError)):
        for f in (mh.distillation, mh.distillation_backward):
            with pytest.raises(error):
                f(c, z, ids, teacher, y)
    t = Fake((1, 1))
    t.cos = t.sin = Fake((16, 4))
    q, k = Fake((2, 4, 5, 8)), Fake((2, 2, 5, 8))
    for f in (mh.rotary, mh.rotary_backward):
        with pytest.raises(mh.ArgumentError):
            f(c, q, k, t, layout="rows")
        with pytest.raises(mh.ShapeError):
            f(c, None, None, t)
        with pytest.raises(mh.ShapeError):
            f(c, q, Fake((2, 2, 6, 8)), t)
        with pytest.raises(mh.ShapeError):
            f(c, q, k, t, positions=np.zeros(9, np.int32))
        with pytest.raises(mh.IndexOutOfRange):
            f(c, q, k, t, positions=np.full((2, 5), 1 << 33))
    with pytest.raises(mh.ArgumentError):
        mh.ScaledRotaryTables(c, 8, 4, scaling="other")
    with pytest.raises(mh.ShapeError):
        mh.ScaledRotaryTables(c, 7, 4)
