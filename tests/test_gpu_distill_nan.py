"""A NaN among a teacher's logits makes its row's loss NaN, wherever it stands and whatever else the row's entries are
(against the formulas in 64 bits, tests/distill_plain.py)."""
import numpy as np
import pytest

from tests.test_gpu_distill import _both, _logits, _teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,V,k", [(9, 40, 1), (9, 500, 2), (9, 5001, 31), (9, 5001, 256), (9, 5001, 257), (9, 9000, 1000), (700, 1200, 12)])
def test_a_nan_in_the_teacher(_sampler_session, B, V, k, bf16):
    """One CTA per row and several; entries that have a thread of their own and entries that share one."""
    rng = np.random.default_rng(k)
    x = _logits(rng, B, V, bf16)
    ids, t = _teacher(rng, B, V, k)
    t[0, 0] = np.nan
    t[1, k - 1] = np.nan
    t[2, k // 2] = np.nan
    t[3] = np.nan                                               # nothing else
    t[4, ::2] = -np.inf
    t[4, k // 2] = np.nan                                       # beside entries that are none
    t[5, k // 3], t[5, k - 1] = np.inf, np.nan
    ids[6, k // 2], t[6, k // 2] = -1, np.nan                   # no entry: no NaN
    bad = np.zeros(B, bool)
    bad[:6] = True
    with np.errstate(all="ignore"):
        loss, stats, dx = _both(_sampler_session, x, ids, t, 1.5, grads=rng.standard_normal(B).astype(np.float32))
    assert np.array_equal(np.isnan(loss), bad)
    assert np.isnan(stats[bad, 3]).all() and not np.isnan(stats[~bad]).any()
    for b in range(6):
        listed = np.zeros(V, bool)
        listed[ids[b][~np.isneginf(t[b])]] = True
        assert np.array_equal(np.isnan(dx[b]), listed)
