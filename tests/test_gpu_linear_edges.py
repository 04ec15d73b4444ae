"""GPU checks of what the linear layer's operators promise at their edges: what a call has done when it returns, values that
are not finite."""
import ctypes

import numpy as np
import pytest

import linear_oracle as R
import midman_hip as mh
from test_gpu_linear import run_backward

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
