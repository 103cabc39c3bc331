"""Masks of truth values belong to one vocabulary: logits of another are refused before anything reaches the device."""
import numpy as np
import pytest

from gorch_b200.config import DTYPE_F32
from gorch_b200.generate import LOOP_CACHED, DeviceGenerateState
from gorch_b200.rules import LogitRules, adjust_logits, pack_masks


class _Lib:
    def gorch_cuda_buffer_device_ptr(self, buf):
        return 256

    def gorch_cuda_buffer_free(self, buf):
        pass

    def __getattr__(self, name):
        raise AssertionError("refused arguments must not reach the device")


class _Sampler:
    _lib, _ctx = _Lib(), None

    def _buf(self, n):
        return 1

    def _upload(self, buf, arr):
        pass


@pytest.mark.parametrize("V", [1000, 1009, 1024, 1025])
def test_masks_of_another_vocabulary(V):
    s = _Sampler()
    rules = LogitRules(s, 2, masks=np.ones((2, 1010), bool))
    with pytest.raises(ValueError):
        adjust_logits(s, np.zeros((2, V), np.float32), rules)
    st = DeviceGenerateState(s, [[1], [2]], 3, 100, (), LOOP_CACHED)
    with pytest.raises(ValueError):
        st.step(256, DTYPE_F32, V, V, 256, 256, rules)
    with pytest.raises(ValueError):
        LogitRules(s, 3, masks=np.ones((3, V), bool)).check(2, V)


def test_words_and_rules_without_masks_say_nothing_of_it():
    s = _Sampler()
    LogitRules(s, 2, masks=pack_masks(np.ones((2, 1010), bool))).check(2, 1000)
    LogitRules(s, 2, bias=[{}, {}]).check(2, 5)
    LogitRules(s, 2, masks=np.ones((2, 1010), bool)).check(2, 1010)
