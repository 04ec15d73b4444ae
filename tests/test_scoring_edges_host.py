"""Scoring and distillation without a device: the oracle's gradients at the rows where a term of the loss is missing."""
import numpy as np
import pytest

import scoring_oracle as R


@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("alpha", [1.0, 0.4])
def test_oracle_gradients_of_rows_without_a_teacher(alpha, temperature):
    r = np.random.default_rng(1)
    z, y = 2 * r.standard_normal((4, 9)), np.array([0, 8, 3, 5])
    ids = r.integers(0, 9, (4, 4)).astype(np.int32)
    teacher = r.standard_normal((4, 4))
    ids[1] = -1
    teacher[2] = -np.inf
    ids[3, :2], teacher[3, 2:] = -2, -np.inf

    def loss(v):
        return R.distillation(v, y, ids, teacher, temperature, alpha, 4)[0].sum() / 4

    g = R.distillation(z, y, ids, teacher, temperature, alpha, 4)[2]
    for i in range(4):
        for j in range(9):
            s = np.zeros_like(z)
            s[i, j] = 1e-5
            assert abs((loss(z + s) - loss(z - s)) / 2e-5 - g[i, j]) < 1e-8
    if alpha == 1.0:
        assert (g[1:] == 0).all() and np.abs(g[0]).max() > 0
