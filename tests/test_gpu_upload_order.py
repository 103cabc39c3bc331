"""gorch_cuda_buffer_upload: what it was given is on the device when it returns, for kernels on any stream."""
import numpy as np
import pytest

from gorch_b200 import _lib
from gorch_b200.config import DTYPE_F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [6, 65, 130, 1220])
def test_a_kernel_behind_an_upload_reads_all_of_it(_sampler_session, B):
    """Sizes at which the driver still moves the end of a pageable buffer when cudaMemcpy returns, and at which it does not. The
    kernel is a copy (no rule is on)."""
    s, V = _sampler_session, 4096
    a, out = np.zeros((B, V), np.float32), np.empty((B, V), np.float32)
    x, y = s._buf(a.nbytes), s._buf(a.nbytes)
    ptr = s._lib.gorch_cuda_buffer_device_ptr
    try:
        for _ in range(100):
            a += 1
            s._upload(x, a)
            s.adjust_logits_ptrs(ptr(x), DTYPE_F32, B, V, V, _lib.LogitAdjust(), ptr(y), V)
            s.sync()
            s._download(y, out)
            assert np.array_equal(out, a)
    finally:
        s._lib.gorch_cuda_buffer_free(x)
        s._lib.gorch_cuda_buffer_free(y)
