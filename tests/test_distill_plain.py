"""The plain distillation gradient against differences of the plain loss (64 bits), and rows without entries."""
import numpy as np
import pytest

from tests import distill_plain


@pytest.mark.parametrize("T", [1.0, 0.75, 2.0])
def test_gradient_against_differences(T):
    rng = np.random.default_rng(3)
    V = 23
    x = rng.standard_normal((1, V)) * 2
    ids = np.array([[4, 7, -1, 7, 22, 30, 0]])                          # one token twice, two that are none
    t = rng.standard_normal((1, 7)) * 2
    t[0, 4] = -np.inf
    _, stats, _ = row = distill_plain.row_loss(x[0], ids[0], t[0], T)
    dx, _ = distill_plain.gradient(x, ids, t, T, [row[1]], None, 1.0)
    h = 1e-6
    for j in range(V):
        up, down = x[0].copy(), x[0].copy()
        up[j] += h
        down[j] -= h
        diff = (distill_plain.row_loss(up, ids[0], t[0], T)[0] - distill_plain.row_loss(down, ids[0], t[0], T)[0]) / (2 * h)
        assert abs(diff - dx[0, j]) < 1e-7 * max(1.0, T * T)            # 2nd order: h^2; rounding: 1e-16 / h


def test_rows_without_entries():
    x = np.full((2, 5), np.nan)
    ids, t = np.array([[-1, 5], [0, 1]]), np.array([[1.0, 2.0], [-np.inf, -np.inf]])
    loss, stats, _ = distill_plain.loss(x.astype(np.float32), ids, t, 1.0)
    assert not loss.any() and not stats.any()
    dx, _ = distill_plain.gradient(x.astype(np.float32), ids, t, 1.0, stats, None, 1.0)
    assert not dx.any()
