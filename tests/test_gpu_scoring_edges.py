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
