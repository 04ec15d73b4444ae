"""GPU checks of rotary positions (rotary.hip): far angles, and more places than one launch takes, past 2^32 values."""
import numpy as np
import pytest

import midman_hip as mh
import scoring_oracle as R
from test_gpu_scoring import near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("factor", [1e-5, 1e-7, 1e-9])
def test_tables_of_far_angles(ctx, factor):
    # frequencies divided by a small factor: angles on both sides of 1e9, where another reduction takes over
    width, positions = 10, 20000
    t = mh.ScaledRotaryTables(ctx, width, positions, 1e4, "linear", factor)
    angle = np.outer(np.arange(positions), R.frequencies(width, 1e4, "linear", factor))
    assert angle.max() > 1e9
    # half a step of f32, and the angle's own f64 roundings
    for got, want in ((t.cos, np.cos(angle)), (t.sin, np.sin(angle))):
        near(got.numpy(), want, R.U * np.abs(want) + 16 * 2.0 ** -53 * (1 + angle), "table")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_more_places_than_a_launch(ctx, layout):
    # heads of 600 columns, a workgroup to each place: 2^23 of them are one launch. In place, 20 GB; looked at where the first
    # launch ends and at the last places.
    b, t, hd, width = (1 << 21) + 40, 4, 600, 8
    n = b * t
    X = ctx.empty((b, 1, t, hd))
    assert X.size > 1 << 32
    tables = mh.ScaledRotaryTables(ctx, width, t)
    r = np.random.default_rng(3)
    spots = {at: r.standard_normal((2, 1, t, hd)).astype(np.float32) for at in (0, (1 << 21) - 1, b - 2)}
    for at, x in spots.items():
        mh.check(mh.lib().mmh_upload(ctx.handle, X.offset(at * t * hd), x.ctypes.data, x.nbytes))
    mh.rotary(ctx, X, None, tables, layout, q_out=X)
    cos, sin = (a.numpy()[None, None] for a in (tables.cos, tables.sin))
    for at, x in spots.items():
        got = np.empty_like(x)
        mh.check(mh.lib().mmh_download(ctx.handle, got.ctypes.data, X.offset(at * t * hd), got.nbytes))
        assert np.array_equal(got, R.rotate(x, cos, sin, layout, width)), (n, at)
    X.free()
