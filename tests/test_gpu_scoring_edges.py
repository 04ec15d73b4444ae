"""GPU checks of token_logprobs and distillation (scoring.hip) at the rows and sizes where a term, a column or a row is
easily lost, against 64-bit evaluations."""
import numpy as np
import pytest

import midman_hip as mh
import scoring_oracle as R
from test_gpu_scoring import Box, drawn, empty, near, ptr, run_distill, run_logprobs, run_logprobs_bwd, teachers

pytestmark = pytest.mark.gpu

# (rows, vocab) of every kernel: whole rows in registers, wide ones in registers and LDS, and few wide ones by parts
KERNELS = [(5, 300), (5, 3000), (5, 8000), (5, 16000), (5, 30000), (70, 32750), (70, 40000), (70, 70000), (70, 140000), (5, 40000),
           (5, 140000)]


@pytest.mark.parametrize("n,v", KERNELS)
def test_rows_without_a_teacher_have_no_gradient_of_it(ctx, n, v):
    z, y, r = drawn(n, v, v)
    ids, teacher = teachers(r, z, 6)
    ids[1] = -1                    # nothing
    teacher[2] = -np.inf           # nothing either
    ids[3, :4], teacher[3, 4:] = -7, -np.inf
    for temperature in (1.0, 2.0):
        for alpha in (1.0, 0.4):
            print(f"\n[no teacher] {(n, v)} T={temperature} alpha={alpha}", flush=True)
            row, tol, want, g_tol = R.distillation(z, y, ids, teacher, temperature, alpha, n)
            loss, g = run_distill(ctx, z, y, ids, teacher, temperature, alpha)
            near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
            near(g, want, g_tol, "dlogits")
            if alpha == 1.0:
                assert (g[1:4] == 0).all() and (row[1:4] == 0).all()
    # with no teacher in any row and no other term the loss and the gradient are 0
    ids[:] = -1
    loss, g = run_distill(ctx, z, None, ids, teacher, 2.0, 1.0)
    assert loss == 0 and (g == 0).all()


# Logits whose differences are exact, one large and the others 70 T to 80 T below it, so that their sum is 1 in f32. A
# far token's exponential is off by its exponent's rounding, half a step of the exponent d / T log2 e, at most |d| / T u
# of itself (u = 2^-24) to either side: over many tokens a mean within 6 / sqrt(3 M) of that. The hardware's 2^x, the
# gradient's factor (the mean's and the temperature's products and a quotient) and its product are within 7 u of 70.
@pytest.mark.parametrize("n,v", [(max(n, 70) if v < 32768 else n, v) for n, v in KERNELS])
def test_far_tokens_are_not_biased(ctx, n, v):
    r = np.random.default_rng(v)
    y = r.integers(0, v, n).astype(np.int32)
    m = min(v // 2, 2000)
    steps = -r.integers(70 << 12, 80 << 12, (n, m)) / 4096.0  # differences over T
    at = np.stack([r.choice(np.delete(np.arange(v), y[i]), m, replace=False) for i in range(n)])
    ids, teacher = y[:, None].copy(), np.zeros((n, 1), np.float32)
    rows = np.arange(n)[:, None]

    def check(got, want, what):
        err = (got / want - 1.0) / (-steps * R.U)
        assert np.abs(err).max() <= 1.0 + 7 / 70 and abs(err.mean()) <= 6 / np.sqrt(3 * n * m) + 7 / 70, (what, np.abs(err).max(), err.mean())

    for t in (1.0, 3.0, 7.0):
        z = np.full((n, v), -np.inf, np.float32)
        z[np.arange(n), y] = 3.0
        z[rows, at] = 3.0 + t * steps
        assert (z[rows, at] == 3.0 + t * steps).all()
        _, g = run_distill(ctx, z, None, ids, teacher, t, 1.0)
        check(g[rows, at].astype(np.float64), t / n * np.exp(steps), ("softened", t))
        z[rows, at] = 3.0 + steps
        if t == 1.0:
            g = run_logprobs_bwd(ctx, z, y, np.ones(n, np.float32), None)
            check(g[rows, at].astype(np.float64), -np.exp(steps), "log probabilities")
        else:  # the plain exponential beside the softened one
            _, g = run_distill(ctx, z, y, np.full_like(ids, -1), teacher, t, 0.5)
            check(g[rows, at].astype(np.float64), 0.5 / n * np.exp(steps), ("plain", t))


def test_log_probabilities_are_not_biased(ctx):
    # Log probabilities from -8 to -16 round by half a step of 2^-20 at most, either way, a standard deviation of 2.8e-7,
    # and their sums less; the mean of 4096 rows is then within 6 x 2.8e-7 / 64 = 2.6e-8 of nothing. (An exponential that is
    # too large by 2^-26 |d| moves it by 5e-8 or more.)
    n, v = 4096, 8000
    z, y, r = drawn(n, v, 21)
    d = z.astype(np.float64) - z.max(1, keepdims=True)
    want = d - np.log(np.exp(d).sum(1, keepdims=True))
    y = np.abs(want + 12.0).argmin(1).astype(np.int32)
    lp, h, ids, top = run_logprobs(ctx, z, y, 0)
    assert abs((lp - want[np.arange(n), y]).mean()) <= 2.6e-8


# One token far ahead of the others: 1 - p is as small as exp(-gap), and the target's gradient is right relative to itself.
# In steps of u: the small sum's exponential (3 + 2 gap) (d is exact here but for its exponent, which rounds), its sum and
# quotients 3 each, the factors 3; the entropy's has a product by the gap and one quotient more.
@pytest.mark.parametrize("n,v", KERNELS)
def test_a_certain_targets_gradient_keeps_its_bits(ctx, n, v):
    gaps = np.array([1.0, 5.0, 20.0, 40.0, 80.0])[np.arange(n) % 5]
    z = np.full((n, v), -np.inf, np.float32)
    at, y = np.full(n, v // 3), np.full(n, v - 2, np.int32)
    rows = np.arange(n)
    z[rows, y], z[rows, at] = 3.0, 3.0 - gaps
    x = np.exp(-gaps)
    tol = (20 + 2 * gaps) * R.U
    one = np.ones(n, np.float32)
    g = run_logprobs_bwd(ctx, z, y, one, None)
    assert (np.abs(g[rows, y] / (x / (1 + x)) - 1) <= tol).all()
    g = run_logprobs_bwd(ctx, z, y, None, one)
    assert (np.abs(g[rows, y] / (-gaps * x / (1 + x) ** 2) - 1) <= tol).all()
    # the cross entropy's, alone and beside a teacher's term that has nothing there
    ids = np.full((n, 2), -1, np.int32)
    for temperature, alpha in ((1.0, 0.0), (1.0, 0.5), (2.0, 0.5)):
        _, g = run_distill(ctx, z, y, ids, np.zeros((n, 2), np.float32), temperature, alpha)
        want = -(1 - alpha) / n * x / (1 + x)
        assert (np.abs(g[rows, y] / want - 1) <= tol).all(), (temperature, alpha)


# (rows, vocab): odd lengths, so that the rows begin at every place of a cache line, on both sides of each kernel's width;
# 33 rows wider than a workgroup's registers go by parts, 70 by a workgroup each
ODD = [(40, v) for v in (1, 3, 63, 991, 993, 995, 1025, 4063, 4065, 4067, 8159, 8161, 8163, 16353, 16355, 32735, 32737)]
ODD += [(n, v) for v in (32739, 32767, 32769, 65535, 65537, 98303, 98305, 131041, 131073, 140001) for n in (33, 70)] + [(33, 262143)]
HALF = float(np.float32(np.log(2.0)))  # exp(-HALF / T T) is 1/2 in f32, and sums of halves and quarters are exact


@pytest.mark.parametrize("n,v", ODD)
def test_every_column_counts_once(ctx, n, v):
    # Rows of equal logits, and of one with all the others log 2 (at T) below it: every sum is exact, so a column that is
    # lost or counted twice moves a gradient by 1 / v of itself, where its factor's roundings (the mean's, the temperature's,
    # a quotient, a sum of two terms, the hardware's 2^x) are within 16 u, and a log probability by 1 / v, where log1p and a
    # difference are within 2.5 steps of its value.
    assert 1.0 / v > 24 * R.U
    y, at = (np.arange(n) * 13 % v).astype(np.int32), (np.arange(n) * 7 + v // 2) % v
    rows, free = np.arange(n), np.ones((n, v), bool)
    free[rows, y] = free[rows, at] = False
    one, none = np.ones(n, np.float32), np.zeros((n, 1), np.float32)
    ids = y[:, None].copy()
    for low in (0.0, HALF):
        for t in (1.0, 2.0):
            z = np.full((n, v), -t * low, np.float32)
            z[rows, at] = 0.0
            x, x1 = (1.0, 1.0) if low == 0.0 else (0.5, 0.5 ** t)
            s, s1 = 1.0 + (v - 1) * x, 1.0 + (v - 1) * x1

            def factor(got, want, what):
                assert np.abs(got[free] / want - 1.0).max(initial=0.0) <= 16 * R.U, (what, low, t, np.abs(got[free] / want - 1.0).max() / R.U)

            if t == 1.0:
                lp, h, _, top = run_logprobs(ctx, z, y, 1, shift=n % 32)
                step = np.spacing(np.float32(max(np.log(s), 1e-30)))
                d = z[rows, y].astype(np.float64)
                assert np.abs(lp - (d - np.log(s))).max() <= 2.5 * max(step, float(np.spacing(np.float32(abs(lp).max()))))
                assert np.abs(top[:, 0] + np.log(s)).max() <= 2.5 * step
                factor(run_logprobs_bwd(ctx, z, y, one, None, shift=3), -x / s, "log probabilities")
            factor(run_distill(ctx, z, None, ids, none, t, 1.0, shift=1)[1], t / n * x / s, "softened")
            if t != 1.0:
                factor(run_distill(ctx, z, y, ids, none, t, 0.5, inplace=True)[1], (0.5 * t * x / s + 0.5 * x1 / s1) / n, "both")


@pytest.mark.parametrize("n,v", [(n, v) for n, v in ODD if v > 200])
def test_entropies_of_tokens_at_borders(ctx, n, v):
    # All but 48 tokens of a row masked: its ends, and others on both sides of cache lines, where strips, passes and parts
    # begin. Masked ones add 0 exactly, so 48 terms and 64 joins round, three times each.
    r = np.random.default_rng(v)
    f = 48
    z = np.full((n, v), -np.inf, np.float32)
    for i in range(n):
        shift = (5 + i * v) % 32
        line = 32 * r.integers(1, v // 32 + 1, 300) - shift - r.integers(0, 2, 300)
        line = np.unique(line[(line >= 2) & (line < v - 2)])
        cols = np.concatenate([[0, 1, v - 2, v - 1], r.permutation(line)[:f - 4]])
        z[i, cols] = r.integers(0, 64, len(cols)) / 64.0
    y = z.argmax(1).astype(np.int32)
    lp, h, ids, top = run_logprobs(ctx, z, y, 20, shift=5)
    d = z.astype(np.float64) - z.max(1, keepdims=True)
    e = np.exp(d)
    s = e.sum(1)
    want_h = np.log(s) - np.where(e > 0, e * np.maximum(d, -1e9), 0.0).sum(1) / s
    tol = 3 * (f + 64) * R.U
    assert np.abs(lp + np.log(s)).max() <= tol + 8 * R.U * np.log(s).max()
    assert np.abs(h - want_h).max() <= 3 * tol + 8 * R.U * want_h.max()
    want_ids = np.argsort(-z, axis=1, kind="stable")[:, :20]
    assert np.array_equal(ids, want_ids)


@pytest.mark.parametrize("v", [999, 4001, 8001, 16001, 32001, 32751, 49999, 90001, 120001, 140001])
def test_outputs_past_the_caches(ctx, v):
    # 256 MiB of gradients and more, rows by a workgroup each: 67 different ones over and over, at every place of a line
    base = 67
    reps = (1 << 26) // (base * v) + 1
    n = base * reps
    assert n * v * 4 >= 1 << 28
    z, y, r = drawn(base, v, v)
    y[5] = -1
    keep = y != -1
    dl, dh = r.standard_normal(base).astype(np.float32), (0.1 * r.standard_normal(base)).astype(np.float32)
    ids, teacher = teachers(r, z, 9)
    Z, yy = np.tile(z, (reps, 1)), np.tile(y, reps)

    def rows(got, want, tol, what):
        want, tol = want.astype(np.float32), (tol + R.U * np.abs(want)).astype(np.float32)
        for g in got.reshape(reps, base, v):
            assert (g[~keep] == 0).all() and (np.abs(g[keep] - want) <= tol).all(), (what, np.abs(g[keep] - want).max())

    kept = int(keep.sum()) * reps
    print(f"\n[past the caches] {n} x {v}", flush=True)
    g = run_logprobs_bwd(ctx, Z, yy, np.tile(dl, reps), np.tile(dh, reps), shift=1)
    rows(g, *R.token_logprobs_backward(z[keep], y[keep], dl[keep], dh[keep]), "log probabilities")
    for temperature, inplace in ((1.0, False), (2.0, True)):
        row, tol, want, g_tol = R.distillation(z[keep], y[keep], ids[keep], teacher[keep], temperature, 0.5, kept)
        loss, g = run_distill(ctx, Z, yy, np.tile(ids, (reps, 1)), np.tile(teacher, (reps, 1)), temperature, 0.5, inplace=inplace)
        near(np.float32(loss), row.mean(), tol.mean() + R.U * abs(row.mean()), "loss")
        rows(g, want, g_tol, ("distillation", temperature))


def test_more_lists_than_the_workspace_takes(ctx):
    # 16257 rows' lists of 256 entries in two parts are 64 MiB: rows on both sides of that, behind others that are left out
    v, n, k = 32800, 16300, 256
    Z = ctx.empty((n, v))
    z, y, _ = drawn(6, v, 22)
    at = 16254
    targets = np.full(n, -1, np.int32)
    targets[at:at + 6] = y
    mh.check(mh.lib().mmh_upload(ctx.handle, Z.offset(at * v), z.ctypes.data, z.nbytes))
    s = mh.token_logprobs(ctx, Z, targets, k=k)
    want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, k)
    near(s.logprobs.numpy()[at:at + 6], *want_lp, "logprobs")
    near(s.entropy.numpy()[at:at + 6], *want_h, "entropy")
    ids, top = s.top_ids.numpy(), s.top_logprobs.numpy()
    assert np.array_equal(ids[at:at + 6], want_ids)
    near(top[at:at + 6], *want_top, "top")
    assert (np.delete(ids, np.arange(at, at + 6), 0) == -1).all()
    Z.free()


def test_more_parts_than_a_join_holds(ctx):
    z, y, _ = drawn(2, 257 * 32768 + 5, 23)
    z[0, -1], z[1, 0] = 30.0, 30.0
    for k in (0, 3):
        lp, h, ids, top = run_logprobs(ctx, z, y, k, shift=7)
        want_lp, want_h, (want_ids, want_top) = R.token_logprobs(z, y, k)
        near(lp, *want_lp, "logprobs")
        near(h, *want_h, "entropy")
        assert np.array_equal(ids, want_ids)
        near(top, *want_top, "top")


@pytest.mark.parametrize("v", [2, 3, 50, 100, 200, 255, 256])
def test_a_student_that_is_its_teacher(ctx, v):
    # Every token has a slot, in another order, and the same logit but for a constant: the loss is 0, and so it is here, since
    # all sums of equal logits and of halves are exact and every logarithm is of 1. Temperatures up to 1000 do not change it.
    n = 6
    r = np.random.default_rng(v)
    ids = np.stack([r.permutation(v) for _ in range(n)]).astype(np.int32)
    for t in (1.0, 2.0, 64.0, 1000.0):
        for low in (0.0, t * HALF if t != 1000.0 else 0.0):
            z = np.full((n, v), -low, np.float32)
            z[np.arange(n), r.integers(0, v, n)] = 0.0
            teacher = np.take_along_axis(z, ids.astype(np.int64), 1)
            if low == 0.0:
                teacher += np.float32(8.0)
            loss, g = run_distill(ctx, z, None, ids, teacher, t, 1.0)
            assert loss == 0.0, (t, low, loss)
            assert np.abs(g).max() <= 8 * R.U * t / n


def test_losses_at_high_temperatures(ctx):
    # A student near its teacher: beside the exact sums above, each exponential is within (3 + 2 |d| / T) u, and a sum of 200
    # has 14 roundings on its way at most, so both sums' quotient is within 2 (3 + 2 |d| / T + 14) + 3 u, and the loss within
    # T^2 of that.
    n, v = 64, 200
    r = np.random.default_rng(31)
    z = (2 * r.standard_normal((n, v))).astype(np.float32)
    ids = np.stack([r.permutation(v) for _ in range(n)]).astype(np.int32)
    teacher = (np.take_along_axis(z, ids.astype(np.int64), 1) + 0.3 * r.standard_normal((n, v))).astype(np.float32)
    for t in (1.0, 5.0, 50.0, 200.0, 1000.0):
        row, tol, want, g_tol = R.distillation(z, None, ids, teacher, t, 1.0, n)
        loss, g = run_distill(ctx, z, None, ids, teacher, t, 1.0)
        print(f"\n[high temperature] T={t}: loss {loss}, off by {abs(loss - row.mean()) / t ** 2 / R.U:.2f} u T^2", flush=True)
        d = np.abs(z - z.max(1, keepdims=True)).max() + 1.0
        assert abs(loss - row.mean()) <= t * t * (2 * (3 + 2 * d / t + 14) + 3) * R.U + 16 * R.U * row.mean()
        near(g, want, g_tol, "dlogits")


@pytest.mark.parametrize("n,v", KERNELS)
def test_masked_targets_and_slots_keep_their_share(ctx, n, v):
    # a target of logit -inf: its log probability is -inf, its gradient dlogprob (less nothing), the others' as they are
    z, y, r = drawn(n, v, v + 1)
    z[np.arange(n), y] = -np.inf
    lp, h, ids, top = run_logprobs(ctx, z, y, 2)
    _, want_h, _ = R.token_logprobs(z, None, 2)
    assert (lp == -np.inf).all()
    near(h, *want_h, "entropy")
    dl, dh = r.standard_normal(n).astype(np.float32), r.standard_normal(n).astype(np.float32)
    g = run_logprobs_bwd(ctx, z, y, dl, dh)
    near(g, *R.token_logprobs_backward(z, y, dl, dh), "dlogits")
    assert (g[np.arange(n), y] == dl).all()
    ids, teacher = y[:, None].copy(), np.zeros((n, 1), np.float32)
    for temperature, alpha in ((1.0, 0.5), (2.0, 0.5), (2.0, 1.0)):
        loss, g = run_distill(ctx, z, y, ids, teacher, temperature, alpha)
        assert loss == np.inf
        want = -(alpha * temperature + (1 - alpha)) / n
        assert np.abs(g[np.arange(n), y] / want - 1).max() <= 8 * R.U
        with np.errstate(invalid="ignore"):
            near(g, *R.distillation(z, y, ids, teacher, temperature, alpha, n)[2:], "dlogits")


def test_many_ids_of_queued_calls_are_each_calls_own(ctx):
    # behind work that takes a while, with ids of 16 MiB that change as soon as the call is back
    a = ctx.empty((8192, 8192))
    out = ctx.empty((8192, 8192))
    n = 1 << 22
    r = np.random.default_rng(41)
    X, tables = ctx.to_device(r.standard_normal((1, 1, n, 2)).astype(np.float32)), mh.ScaledRotaryTables(ctx, 2, 1000)
    Z = ctx.to_device(r.standard_normal((n, 2)).astype(np.float32))
    cos, sin, x, z = tables.cos.numpy(), tables.sin.numpy(), X.numpy(), Z.numpy()
    at, y = r.integers(0, 1000, (1, n)).astype(np.int32), r.integers(0, 2, n).astype(np.int32)
    at0, y0 = at.copy(), y.copy()
    for _ in range(4):
        mh.gemm(ctx, "nn", a, a, out, 8192, 8192, 8192)
    q = mh.rotary(ctx, X, None, tables, positions=at)[0]
    at[:] = 0
    for _ in range(4):
        mh.gemm(ctx, "nn", a, a, out, 8192, 8192, 8192)
    s = mh.token_logprobs(ctx, Z, y)
    y[:] = 0
    assert np.array_equal(q.numpy(), R.rotate(x, cos[at0][:, None], sin[at0][:, None], "half", 2))
    d = z.astype(np.float64) - z.max(1, keepdims=True)
    want = d[np.arange(n), y0] - np.log(np.exp(d).sum(1))
    near(s.logprobs.numpy(), want, 64 * R.U * (1 + np.abs(want)), "logprobs")


@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0])
def test_losses_of_many_rows_are_not_biased(ctx, temperature):
    # Each of 4096 rows' terms (5 to 9, over T^2) rounds by half a step of 2^-20 at most, either way, as do its logarithms,
    # so their mean is within 2 x 2.6e-8 as above, and the loss rounds once more.
    n, v = 4096, 8000
    z, y, r = drawn(n, v, 24)
    d = (z.astype(np.float64) - z.max(1, keepdims=True)) / temperature
    want = temperature ** 2 * np.log(np.exp(d).sum(1)).mean()
    ids = z.argmax(1).astype(np.int32)[:, None].copy()
    loss, _ = run_distill(ctx, z, None, ids, np.zeros((n, 1), np.float32), temperature, 1.0, grad=False)
    assert abs(loss - want) <= np.spacing(np.float32(want)) / 2 + temperature ** 2 * 5.2e-8
