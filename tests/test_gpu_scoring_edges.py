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
