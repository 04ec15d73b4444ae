"""GPU checks of token_logprobs and distillation (scoring.hip) against 64-bit evaluations, within the bounds that
scoring_oracle.py derives; every output lies between guard words, at the alignments given."""
import ctypes

import numpy as np
import pytest

import midman_hip as mh
import scoring_oracle as R

pytestmark = pytest.mark.gpu

GUARD = 64
IDS = ctypes.POINTER(ctypes.c_int32)


class Box:
    """An array of the device `shift` values off a 256-byte boundary, between guard words."""

    def __init__(self, ctx, a, shift=0):
        a = np.asarray(a)
        self.shape, self.n, self.at = a.shape, a.size, GUARD + shift
        self.mark = a.dtype.type(-7.25e33 if a.dtype == np.float32 else -1234567)
        flat = np.full(self.at + self.n + GUARD, self.mark, a.dtype)
        flat[self.at:self.at + self.n] = a.ravel()
        self.dev = ctx.to_device(flat)
        self.ptr = self.dev.offset(self.at)

    def numpy(self):
        a = self.dev.numpy()
        assert (a[:self.at] == self.mark).all() and (a[self.at + self.n:] == self.mark).all(), "a write outside the output"
        return a[self.at:self.at + self.n].reshape(self.shape)


def empty(ctx, shape, shift=0, dtype=np.float32):
    return Box(ctx, np.full(shape, 77, dtype), shift)


def ptr(a):
    return None if a is None else a.ctypes.data_as(IDS) if isinstance(a, np.ndarray) else a.ptr


def near(got, value, tol, what):
    with np.errstate(invalid="ignore"):
        _near(got, value, tol, what)


def _near(got, value, tol, what):
    err = np.abs(got.astype(np.float64) - value)
    bad = ~((err <= tol) | (got == value))
    assert not bad.any(), (what, int(bad.sum()), float(np.nanmax(err / np.maximum(tol, 1e-300))), np.argwhere(bad)[:3].tolist())


def run_logprobs(ctx, z, targets, k, ignore=-1, shift=0):
    n, v = z.shape
    Z = Box(ctx, z, shift)
    lp = None if targets is None else empty(ctx, n, shift)
    h, ids, top = empty(ctx, n, shift), empty(ctx, (n, k), shift, np.int32), empty(ctx, (n, k), shift)
    mh.check(mh.lib().mmh_token_logprobs(ctx.handle, Z.ptr, ptr(targets), n, v, ignore, k, ptr(lp), h.ptr, ids.ptr, top.ptr))
    out = [None if a is None else a.numpy() for a in (lp, h, ids, top)]
    assert np.array_equal(Z.numpy(), z, equal_nan=True)
    return out


def run_logprobs_bwd(ctx, z, targets, dl, dh, ignore=-1, shift=0, inplace=False):
    n, v = z.shape
    Z = Box(ctx, z, shift)
    L, H = (None if a is None else Box(ctx, a, shift) for a in (dl, dh))
    out = Z if inplace else empty(ctx, (n, v), shift)
    mh.check(mh.lib().mmh_token_logprobs_backward(ctx.handle, Z.ptr, ptr(targets), n, v, ignore, ptr(L), ptr(H), out.ptr))
    return out.numpy()


def run_distill(ctx, z, targets, ids, teacher, temperature, alpha, ignore=-1, shift=0, grad=True, inplace=False):
    """(loss, dlogits)"""
    n, v = z.shape
    Z, I, T = Box(ctx, z, shift), Box(ctx, ids, shift), Box(ctx, teacher, shift)
    out = None if not grad else Z if inplace else empty(ctx, (n, v), shift)
    loss = ctypes.c_float(99.0)
    args = [Z.ptr, ptr(targets), n, v, ignore, I.ptr, T.ptr, ids.shape[1], temperature, alpha]
    if grad:
        mh.check(mh.lib().mmh_distillation_backward(ctx.handle, *args, out.ptr, ctypes.byref(loss)))
        return loss.value, out.numpy()
    mh.check(mh.lib().mmh_distillation(ctx.handle, *args, ctypes.byref(loss)))
    return loss.value, None


def drawn(n, v, seed, std=2.0):
    r = np.random.default_rng(seed)
    z = (std * r.standard_normal((n, v))).astype(np.float32)
    z[np.arange(n), r.integers(0, v, n)] += np.float32(6.0)
    return z, r.integers(0, v, n).astype(np.int32), r


def teachers(r, z, k, noise=1.0):
    n, v = z.shape
    k = min(k, v)
    t = z + (noise * r.standard_normal((n, v))).astype(np.float32)
    ids = np.argsort(-t, axis=1, kind="stable")[:, :k].astype(np.int32)
    return ids, np.take_along_axis(t, ids.astype(np.int64), 1)


# (rows, vocab): one row and token, waves and strips that end inside, every width's kernel and its border, more rows than CUs
SHAPES = [(1, 1), (3, 2), (5, 63), (7, 64), (2, 65), (64, 256), (9, 1000), (4, 1023), (3, 1024), (6, 1025), (17, 4096), (5, 4097),
          (3, 8191), (2, 8193), (3, 16385), (2, 32000), (3, 32768), (2, 32769), (1, 50257), (300, 4099), (520, 9001), (1, 131071),
          (2, 262144), (5, 65537), (1030, 77), (260, 33000),
          # as many wide rows that a workgroup takes each whole: what its registers and LDS hold, borders of both, more
          (66, 32750), (70, 49153), (65, 65535), (66, 65600), (65, 98303), (66, 98400), (65, 131100), (65, 140001)]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_token_logprobs(ctx, i):
    n, v = SHAPES[i]
    z, y, _ = drawn(n, v, i)
    for k in sorted({min(v, x) for x in ((0, 5, 64), (1, 20, 256), (2, 33, 100))[i % 3]}):
        targets = None if (i + k) % 4 == 3 else y
        print(f"\n[token_logprobs] {(n, v)} k={k} targets={targets is not None}", flush=True)
        lp, h, ids, top = run_logprobs(ctx, z, targets, k, shift=i % 4)
        want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, targets, k)
        if targets is not None:
            near(lp, *want_lp, "logprobs")
        near(h, *want_h, "entropy")
        assert np.array_equal(ids, want_ids)
        near(top, *want_top, "top")


@pytest.mark.parametrize("v", [50, 700, 1500, 5000, 20000, 40000, 140000])
def test_top_of_equal_and_masked_logits(ctx, v):
    r = np.random.default_rng(v)
    rows = []
    rows.append(np.zeros(v))                                      # all equal
    rows.append(np.round(r.standard_normal(v)))                   # a handful of values
    rows.append(np.where(r.random(v) < 0.5, 0.0, -0.0))           # equal zeros of both signs
    masked = np.full(v, -np.inf)
    masked[r.integers(0, v, 3)] = [1.0, 2.0, 0.5]
    rows.append(masked)                                           # fewer tokens than alternatives
    rows.append(np.where(np.arange(v) % 2 == 0, -np.inf, np.round(4 * r.standard_normal(v)) / 4))
    rows.append(-np.arange(v) / 64.0)                             # falling
    rows.append(np.arange(v) / 64.0)                              # rising
    lowest = np.full(v, np.finfo(np.float32).min)
    lowest[v // 2:] = np.round(r.standard_normal(v - v // 2) * 2)
    rows.append(lowest)                                           # masks of the type's lowest value
    steps = np.zeros(v)                                           # the largest ones all within one thread's share
    for width in (1024, 2048, 4096):
        steps[::width] += 5.0
    rows.append(steps + np.arange(v) * 1e-6)
    wave = np.zeros(v)
    wave[(np.arange(v) // 4) % 512 < 16] = 3.0                    # many large ones, in few threads
    rows.append(wave + r.random(v))
    last = np.zeros(v)
    last[-1] = 1.0
    rows.append(last)
    z = np.stack(rows).astype(np.float32)
    y = np.full(len(z), v - 1, np.int32)
    y[3] = int(np.argmax(z[3]))
    y[4] = 1
    for k in sorted({1, 7, min(v, 50), min(v, 64), min(v, 255), min(v, 256)}):
        print(f"\n[top, equal values] {v} k={k}", flush=True)
        lp, h, ids, top = run_logprobs(ctx, z, y, k)
        want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, k)
        assert np.array_equal(ids, want_ids), [i for i in range(len(z)) if not np.array_equal(ids[i], want_ids[i])]
        near(lp, *want_lp, "logprobs")
        near(h, *want_h, "entropy")
        near(top, *want_top, "top")


@pytest.mark.parametrize("v", [3, 300, 9000, 33000, 140000])
def test_rows_without_a_distribution(ctx, v):
    z, y, r = drawn(6, v, 5)
    z[0] = -np.inf
    z[1, v // 2] = np.inf
    z[2, v - 1] = np.nan
    z[3, 0] = np.inf
    z[3, v - 1] = np.nan
    z[4, :] = -np.inf
    z[4, v // 3] = np.nan
    k = min(v, 4)
    print(f"\n[no distribution] {v}", flush=True)
    lp, h, ids, top = run_logprobs(ctx, z, y, k)
    assert np.isnan(lp[:5]).all() and np.isnan(h[:5]).all() and np.isnan(top[:5]).all()
    assert ids[0].tolist() == list(range(k)) and ids[1, 0] == v // 2 and ids[2, 0] == v - 1
    assert ids[3, :2].tolist() == [0, v - 1] and ids[4, 0] == v // 3
    want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z[5:], y[5:], k)
    near(lp[5:], *want_lp, "logprobs")
    near(top[5:], *want_top, "top")
    dl, dh = r.standard_normal(6).astype(np.float32), r.standard_normal(6).astype(np.float32)
    g = run_logprobs_bwd(ctx, z, y, dl, dh)
    assert np.isnan(g[:5]).all()
    near(g[5:], *R.token_logprobs_backward(z[5:], y[5:], dl[5:], dh[5:]), "dlogits")
    t_ids, t_logits = teachers(r, np.nan_to_num(z, posinf=0.0, neginf=0.0), 3)
    for temperature in (1.0, 2.0):
        loss, g = run_distill(ctx, z, y, t_ids, t_logits, temperature, 0.5)
        assert np.isnan(loss) and np.isnan(g[:5]).all()
        near(g[5:], *R.distillation(z[5:], y[5:], t_ids[5:], t_logits[5:], temperature, 0.5, 6)[2:], "dlogits")
        # left out, they do not count
        y2 = np.where(np.arange(6) < 5, -1, y).astype(np.int32)
        loss, g = run_distill(ctx, z, y2, t_ids, t_logits, temperature, 0.5)
        row, tol, want, g_tol = R.distillation(z[5:], y[5:], t_ids[5:], t_logits[5:], temperature, 0.5, 1)
        near(np.float32(loss), row.sum(), tol.sum() + R.U * abs(row.sum()), "loss")
        assert (g[:5] == 0).all()
        near(g[5:], want, g_tol, "dlogits")


def test_a_certain_token_keeps_its_small_values(ctx):
    # 1 - p down to 1e-38: the log probability and the entropy are as small, and right relative to themselves
    gaps = np.array([5.0, 20.0, 40.0, 80.0], np.float32)
    z = np.full((4, 5000), -np.inf, np.float32)
    z[:, 17] = 3.0
    z[:, 4000] = 3.0 - gaps
    lp, h, ids, top = run_logprobs(ctx, z, np.full(4, 17, np.int32), 2)
    x = np.exp(-gaps.astype(np.float64))
    assert np.abs(lp / -np.log1p(x) - 1).max() < 1e-5
    assert np.abs(h / (np.log1p(x) + gaps * x / (1 + x)) - 1).max() < 1e-5
    assert np.array_equal(ids, np.tile([17, 4000], (4, 1))) and np.array_equal(top[:, 0], lp)


@pytest.mark.parametrize("scale", [1e-30, 1e4, 1e37])
def test_logits_of_other_sizes(ctx, scale):
    r = np.random.default_rng(3)
    z = (scale * r.standard_normal((4, 6001))).astype(np.float32)
    y = r.integers(0, 6001, 4).astype(np.int32)
    y[0] = z[0].argmax()
    lp, h, ids, top = run_logprobs(ctx, z, y, 9)
    want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, 9)
    near(lp, *want_lp, "logprobs")
    near(h, *want_h, "entropy")
    assert np.array_equal(ids, want_ids)
    near(top, *want_top, "top")


def test_rows_left_out_are_not_read(ctx):
    z, y, r = drawn(40, 700, 9)
    y[::3] = 5
    z[y == 5] = np.nan
    lp, h, ids, top = run_logprobs(ctx, z, y, 6, ignore=5)
    out = y == 5
    assert (lp[out] == 0).all() and (h[out] == 0).all() and (ids[out] == -1).all() and (top[out] == -np.inf).all()
    want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z[~out], y[~out], 6)
    near(lp[~out], *want_lp, "logprobs")
    assert np.array_equal(ids[~out], want_ids)
    # every row left out
    all_out = np.full(40, -1, np.int32)
    lp, h, ids, top = run_logprobs(ctx, z, all_out, 6)
    assert (lp == 0).all() and (ids == -1).all()
    t_ids, t_logits = teachers(r, np.nan_to_num(z), 4)
    loss, g = run_distill(ctx, z, all_out, t_ids, t_logits, 2.0, 0.5)
    assert loss == 0 and (g == 0).all()
    assert run_distill(ctx, z, all_out, t_ids, t_logits, 2.0, 0.5, grad=False)[0] == 0
    assert (run_logprobs_bwd(ctx, z, all_out, np.ones(40, np.float32), None) == 0).all()


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_token_logprobs_backward(ctx, i):
    n, v = SHAPES[i]
    z, y, r = drawn(n, v, 50 + i)
    dl, dh = r.standard_normal(n).astype(np.float32), (0.1 * r.standard_normal(n)).astype(np.float32)
    if v > 4:
        z[:, v // 2] = -np.inf  # a masked token
        y[y == v // 2] = 0
    for dl_, dh_, targets in ((dl, dh, y), (dl, None, y), (None, dh, None))[:3 if n * v < 3e6 else 1]:
        print(f"\n[token_logprobs_backward] {(n, v)} dl={dl_ is not None} dh={dh_ is not None}", flush=True)
        g = run_logprobs_bwd(ctx, z, targets, dl_, dh_, shift=(i + 1) % 4, inplace=i % 2 == 0)
        near(g, *R.token_logprobs_backward(z, targets, dl_, dh_), "dlogits")
    assert (run_logprobs_bwd(ctx, z, None, None, None) == 0).all()


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_distillation(ctx, i):
    n, v = SHAPES[i]
    z, y, r = drawn(n, v, 90 + i)
    if n > 2:
        y[1] = -1
    kept = y != -1
    for temperature, alpha, k in (((1.0, 1.0, 5), (2.0, 0.5, 64)), ((3.0, 0.25, 256), (0.5, 1.0, 1)), ((1.0, 0.7, 20), (2.0, 0.0, 3)))[i % 3]:
        print(f"\n[distillation] {(n, v)} T={temperature} alpha={alpha} k={k}", flush=True)
        ids, teacher = teachers(r, z, k)
        if ids.shape[1] > 2:
            ids[0, 2:] = -1  # empty slots
            teacher[n - 1, 1] = -np.inf
        row, tol, want, g_tol = R.distillation(z[kept], y[kept], ids[kept], teacher[kept], temperature, alpha, int(kept.sum()))
        loss, g = run_distill(ctx, z, y, ids, teacher, temperature, alpha, shift=i % 4, inplace=i % 2 == 1)
        near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
        near(g[kept], want, g_tol, "dlogits")
        assert (g[~kept] == 0).all()
        assert run_distill(ctx, z, y, ids, teacher, temperature, alpha, shift=i % 4, grad=False)[0] == loss
        if alpha == 1.0 and n <= 2:
            loss, _ = run_distill(ctx, z, None, ids, teacher, temperature, alpha, grad=False)
            near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")


@pytest.mark.parametrize("v", [700, 5000, 30000, 40000, 140000])
def test_gradients_of_masked_rows(ctx, v):
    # few tokens left, whole stretches and parts of a row masked
    n = 5
    z, y, r = drawn(n, v, v)
    for i, left in enumerate(([0, 1], [v - 1], [v // 2, v - 2, 3], range(0, v, 5), range(v // 3, v // 3 + 40))):
        keep = np.zeros(v, bool)
        keep[list(left)] = True
        z[i, ~keep] = -np.inf if i != 2 else np.finfo(np.float32).min
        y[i] = list(left)[0]
    dl, dh = r.standard_normal(n).astype(np.float32), r.standard_normal(n).astype(np.float32)
    g = run_logprobs_bwd(ctx, z, y, dl, dh)
    near(g, *R.token_logprobs_backward(z, y, dl, dh), "dlogits")
    assert (g[z < -1e30] == 0).all()
    ids = np.tile(y[:, None], (1, 3))
    ids[:, 2] = -1
    teacher = r.standard_normal((n, 3)).astype(np.float32)
    for temperature, alpha in ((1.0, 0.5), (2.0, 0.5), (0.001, 0.5), (1000.0, 1.0)):
        loss, g = run_distill(ctx, z, y, ids, teacher, temperature, alpha)
        row, tol, want, g_tol = R.distillation(z, y, ids, teacher, temperature, alpha, n)
        near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
        near(g, want, g_tol, "dlogits")


def test_slots_of_every_kind(ctx):
    v = 5000
    z, y, r = drawn(9, v, 4)
    ids = r.integers(0, v, (9, 40)).astype(np.int32)
    teacher = (3 * r.standard_normal((9, 40))).astype(np.float32)
    ids[0] = 17                       # one token in every slot
    ids[1, ::2] = ids[1, 1::2]        # each token twice
    ids[2] = -1                       # nothing
    teacher[3] = -np.inf              # nothing either
    ids[4, :] = y[4]                  # the target itself
    ids[5, 20:] = -5
    teacher[6] = np.finfo(np.float32).min  # all equal, at the type's end
    teacher[7, 0] = 200.0             # one certain token
    z[8, ids[8, 3]] = -1e4            # a token that the model thinks impossible
    for temperature in (1.0, 4.0):
        for alpha in (1.0, 0.3):
            loss, g = run_distill(ctx, z, y, ids, teacher, temperature, alpha)
            row, tol, want, g_tol = R.distillation(z, y, ids, teacher, temperature, alpha, 9)
            near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
            near(g, want, g_tol, "dlogits")
    # an impossible token of the teacher: the loss is infinite, the gradient is not
    z[8, ids[8, 3]] = -np.inf
    loss, g = run_distill(ctx, z, y, ids, teacher, 1.0, 1.0)
    assert loss == np.inf
    with np.errstate(invalid="ignore"):
        near(g, *R.distillation(z, y, ids, teacher, 1.0, 1.0, 9)[2:], "dlogits")
    # a teacher without a distribution
    for bad in (np.nan, np.inf):
        t = teacher.copy()
        t[8, 5] = bad
        loss, g = run_distill(ctx, z, y, ids, t, 1.0, 0.5)
        assert np.isnan(loss) and np.isnan(g[8, ids[8, 5]])


@pytest.mark.parametrize("v", [60, 3000, 40000])
def test_a_teachers_id_beyond_the_vocabulary(ctx, v):
    z, y, r = drawn(5, v, 4)
    ids, teacher = teachers(r, z, 4)
    for bad in (v, v + 1, 2 ** 31 - 1):
        wrong = ids.copy()
        wrong[3, 2] = bad
        for grad in (False, True):
            with pytest.raises(mh.IndexOutOfRange, match="teacher's id"):
                run_distill(ctx, z, y, wrong, teacher, 1.0, 0.5, grad=grad)
    # the next call is not told of it; ids of a row that is left out are not looked at
    wrong[3, 2] = v
    y2 = y.copy()
    y2[3] = -1
    assert np.isfinite(run_distill(ctx, z, y, ids, teacher, 1.0, 0.5)[0])
    assert np.isfinite(run_distill(ctx, z, y2, wrong, teacher, 1.0, 0.5)[0])


def test_results_do_not_depend_on_the_run(ctx):
    z, y, r = drawn(300, 33001, 11)
    z = np.round(z * 8) / 8
    ids, teacher = teachers(r, z, 64)
    first = None
    for _ in range(3):
        out = run_logprobs(ctx, z, y, 64) + [run_logprobs_bwd(ctx, z, y, z[:, 0].copy(), z[:, 1].copy()),
                                            *run_distill(ctx, z, y, ids, teacher, 2.0, 0.5)]
        first = first or out
        for a, b in zip(first, out):
            assert np.array_equal(a, b)


def test_offsets_past_32_bits(ctx):
    # 2^31 logits and more: rows at the end, behind 2^33 bytes of others
    v, n = 262144, 8200
    free = ctx.empty((n, v))
    z, y, r = drawn(3, v, 12)
    targets = np.full(n, -1, np.int32)
    targets[n - 3:] = y
    mh.check(mh.lib().mmh_upload(ctx.handle, free.offset((n - 3) * v), z.ctypes.data, z.nbytes))
    s = mh.token_logprobs(ctx, free, targets, k=7)
    want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, 7)
    near(s.logprobs.numpy()[-3:], *want_lp, "logprobs")
    assert np.array_equal(s.top_ids.numpy()[-3:], want_ids) and (s.top_ids.numpy()[:-3] == -1).all()
    ids, teacher = teachers(r, z, 7)
    all_ids, all_teacher = np.full((n, 7), -1, np.int32), np.zeros((n, 7), np.float32)
    all_ids[-3:], all_teacher[-3:] = ids, teacher
    loss, out = mh.distillation_backward(ctx, free, ctx.to_device(all_ids), ctx.to_device(all_teacher), targets, 2.0, 0.5, out=free)
    row, tol, want, g_tol = R.distillation(z, y, ids, teacher, 2.0, 0.5, 3)
    near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
    tail = np.empty((4, v), np.float32)
    mh.check(mh.lib().mmh_download(ctx.handle, tail.ctypes.data, free.offset((n - 4) * v), tail.nbytes))
    near(tail[1:], want, g_tol, "dlogits")
    assert (tail[0] == 0).all()
    free.free()


@pytest.mark.parametrize("shape", [(5, 300), (3, 33001), (70, 33001), (300, 2000)])
def test_outputs_that_are_not_asked_for(ctx, shape):
    z, y, r = drawn(*shape, 17)
    n, v = shape
    Z = ctx.to_device(z)
    full = mh.token_logprobs(ctx, Z, y, k=9)
    lp, h, ids, top = (a.numpy() for a in full)
    some = mh.token_logprobs(ctx, Z, y, entropy=False)
    assert some.entropy is None and some.top_ids is None and np.array_equal(some.logprobs.numpy(), lp)
    some = mh.token_logprobs(ctx, Z)
    assert some.logprobs is None and np.array_equal(some.entropy.numpy(), h)
    some = mh.token_logprobs(ctx, Z, k=9, entropy=False)
    assert np.array_equal(some.top_ids.numpy(), ids) and np.array_equal(some.top_logprobs.numpy(), top)
    out = Box(ctx, np.zeros((n, 9), np.float32)), Box(ctx, np.zeros((n, 9), np.int32))
    y[0] = -1  # targets as a mask alone
    mh.check(mh.lib().mmh_token_logprobs(ctx.handle, Z.ptr, ptr(y), n, v, -1, 9, None, None, out[1].ptr, out[0].ptr))
    assert np.array_equal(out[1].numpy()[1:], ids[1:]) and (out[1].numpy()[0] == -1).all()
    # the loss not asked for; the teacher's log probabilities in its logits' place
    loss, g = mh.distillation_backward(ctx, Z, full.top_ids, full.top_logprobs, y, 2.0, 0.5)
    G = Box(ctx, np.zeros((n, v), np.float32))
    mh.check(mh.lib().mmh_distillation_backward(ctx.handle, Z.ptr, ptr(y), n, v, -1, full.top_ids.ptr, full.top_logprobs.ptr, 9, 2.0, 0.5,
                                                G.ptr, None))
    assert np.array_equal(G.numpy(), g.numpy())
    logits = np.take_along_axis(z, ids.astype(np.int64), 1)
    assert abs(mh.distillation(ctx, Z, full.top_ids, ctx.to_device(logits), y, 2.0, 0.5) - loss) <= 1e-5 * abs(loss) + 1e-6


def test_more_slots_than_tokens(ctx):
    for v, n in ((1, 4), (60, 7), (200, 300)):
        z, y, r = drawn(n, v, 18)
        ids = r.integers(-1, v, (n, 256)).astype(np.int32)
        teacher = r.standard_normal((n, 256)).astype(np.float32)
        row, tol, want, g_tol = R.distillation(z, y, ids, teacher, 1.5, 0.6, n)
        loss, g = run_distill(ctx, z, y, ids, teacher, 1.5, 0.6)
        near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
        near(g, want, g_tol, "dlogits")


def test_losses_that_share_pinned_memory(ctx):
    z, y, r = drawn(700, 501, 19)
    ids, teacher = teachers(r, z, 8)
    x, w = (r.standard_normal(s).astype(np.float32) for s in ((900, 32), (501, 32)))
    X, W, yy = ctx.to_device(x), ctx.to_device(w), r.integers(0, 501, 900).astype(np.int32)
    first = run_distill(ctx, z, y, ids, teacher, 2.0, 0.5)
    ce = mh.linear_cross_entropy(ctx, X, W, yy)
    for _ in range(3):
        again = run_distill(ctx, z, y, ids, teacher, 2.0, 0.5)
        assert again[0] == first[0] and np.array_equal(again[1], first[1])
        assert mh.linear_cross_entropy(ctx, X, W, yy) == ce


def test_more_lists_than_a_join_holds(ctx):
    # 16 parts with 256 entries each, equal values across them; a part that a row's place in its line leaves empty or short
    for v in (500001, 16 * 32768 - 31, 16 * 32768 - 30):
        z, y, _ = drawn(3, v, 16)
        z[1] = np.round(2 * z[1]) / 2
        z[2, :] = -1.0
        for k in (256, 200, 3):
            lp, h, ids, top = run_logprobs(ctx, z, y, k, shift=k % 32)
            want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, k)
            near(lp, *want_lp, "logprobs")
            near(h, *want_h, "entropy")
            assert np.array_equal(ids, want_ids)
            near(top, *want_top, "top")


def test_more_rows_than_a_launch(ctx):
    n, v = 2 ** 21 + 5, 3
    z, y, r = drawn(n, v, 15)
    lp, h, ids, top = run_logprobs(ctx, z, y, 2)
    want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, 2)
    near(lp, *want_lp, "logprobs")
    near(h, *want_h, "entropy")
    assert np.array_equal(ids, want_ids)
    dl = r.standard_normal(n).astype(np.float32)
    near(run_logprobs_bwd(ctx, z, y, dl, None), *R.token_logprobs_backward(z, y, dl, None), "dlogits")
    row, tol, want, g_tol = R.distillation(z, y, want_ids, z[:, :2].copy(), 2.0, 0.5, n)
    loss, g = run_distill(ctx, z, y, want_ids, z[:, :2].copy(), 2.0, 0.5)
    near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
    near(g, want, g_tol, "dlogits")


@pytest.mark.parametrize("shift", [0, 5, 31])
@pytest.mark.parametrize("v", [994, 1000, 1024, 32736, 32768, 98304])
def test_rows_at_every_place_of_a_line(ctx, v, shift):
    # rows and outputs that begin at other places of a cache line, lengths at the kernels' borders
    n = 70 if v > 32000 else 9
    z, y, r = drawn(n, v, v + shift)
    lp, h, ids, top = run_logprobs(ctx, z, y, 17, shift=shift)
    want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, 17)
    near(lp, *want_lp, "logprobs")
    near(h, *want_h, "entropy")
    assert np.array_equal(ids, want_ids)
    t_ids, teacher = teachers(r, z, 11)
    row, tol, want, g_tol = R.distillation(z, y, t_ids, teacher, 2.0, 0.5, n)
    for inplace in (False, True):
        loss, g = run_distill(ctx, z, y, t_ids, teacher, 2.0, 0.5, shift=shift, inplace=inplace)
        near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
        near(g, want, g_tol, "dlogits")
    # the output elsewhere in its line than the logits
    Z, out = Box(ctx, z, shift), empty(ctx, (n, v), (shift + 3) % 32)
    dl = r.standard_normal(n).astype(np.float32)
    L = Box(ctx, dl)
    mh.check(mh.lib().mmh_token_logprobs_backward(ctx.handle, Z.ptr, ptr(y), n, v, -1, L.ptr, None, out.ptr))
    near(out.numpy(), *R.token_logprobs_backward(z, y, dl, None), "dlogits")


def test_calls_that_follow_each_other_without_waiting(ctx):
    # targets change between queued calls: each call has its own
    n, v = 700, 900
    z, _, r = drawn(n, v, 13)
    Z = ctx.to_device(z)
    want, got = [], []
    for i in range(12):
        y = r.integers(0, v, n).astype(np.int32)
        want.append(np.take_along_axis(z, y[:, None].astype(np.int64), 1)[:, 0])
        got.append(mh.token_logprobs(ctx, Z, y, k=3))
        y[:] = 0
    base = R.token_logprobs(z, np.zeros(n, np.int32), 3)
    for w, g in zip(want, got):
        near(g.logprobs.numpy(), base[0][0] + w - z[:, 0], base[0][1] + 4e-6, "logprobs")


def test_two_contexts_in_two_threads(ctx):
    import threading
    z, y, r = drawn(400, 5001, 14)
    ids, teacher = teachers(r, z, 32)
    want = (run_logprobs(ctx, z, y, 32), run_distill(ctx, z, y, ids, teacher, 2.0, 0.5))
    errors = []

    def work():
        try:
            with mh.Context(0) as c:
                for _ in range(5):
                    a, b = run_logprobs(c, z, y, 32), run_distill(c, z, y, ids, teacher, 2.0, 0.5)
                    assert all(np.array_equal(x, w) for x, w in zip(a, want[0])) and b[0] == want[1][0]
                    assert np.array_equal(b[1], want[1][1])
        except BaseException as e:  # noqa: BLE001 (reported by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
