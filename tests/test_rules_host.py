"""The host side of a request's rules: masks as words, what LogitRules refuses before it reaches the device."""
import numpy as np
import pytest

from gorch_b200 import _lib
from gorch_b200.config import PENALTY_DTYPE
from gorch_b200.rules import LogitRules, pack_masks
from tests import rules_plain


@pytest.mark.parametrize("V", [1, 31, 32, 33, 1000])
def test_masks_as_words(V):
    a = np.random.default_rng(V).random((3, V)) < 0.5
    w = pack_masks(a)
    assert w.dtype == np.uint32 and w.shape == (3, (V + 31) // 32)
    for i in range(3):
        for v in range(V):
            assert bool((int(w[i, v // 32]) >> (v % 32)) & 1) == a[i, v]


class _NoDevice:
    def _buf(self, n):
        raise AssertionError("refused arguments must not reach the device")


@pytest.mark.parametrize("kw", [dict(penalties=[[1, 0, 0]]), dict(penalties=[[0, 0, 0]] * 2), dict(penalties=[[np.nan, 0, 0]] * 2),
                                dict(penalties=[[1.1, 0, 0]] * 2, history=[[1]]), dict(penalties=[[1.1, 0, 0]] * 2, prompt_lengths=[1]),
                                dict(history=[[1], [2]]), dict(bias=[{}]), dict(mask_rows=[0, 1]), dict(masks=np.ones((2, 5)), mask_rows=[0]),
                                dict(masks=np.ones(7, np.uint32)), dict(penalties=np.zeros(1, PENALTY_DTYPE))])
def test_bad_rules_are_refused(kw):
    with pytest.raises(ValueError):
        LogitRules(_NoDevice(), 2, **kw)


def test_the_records_layout_matches_the_header():
    assert PENALTY_DTYPE.itemsize == 16
    import ctypes
    assert ctypes.sizeof(_lib.LogitAdjust) == 13 * 8


def test_the_plain_rules():
    x = np.float32([[2.0, -2.0, 1.0, 0.5]])
    y, _ = rules_plain.adjust(x, penalties=[[2.0, 0.25, 0.5]], history=[[0, 1, 1, 2]], prompt_lengths=[1], bias=[{2: 1.0}],
                              masks=np.array([[1, 1, 1, 0]], bool))
    assert y.tolist() == [[1.0, (-4.0 - 1.0) - 0.25, (0.5 - 0.5) - 0.25 + 1.0, -np.inf]]
