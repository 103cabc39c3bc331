"""One adapter of nothing but NaN among finite ones in gorch_cuda_lm_head_adapters_dev: the others' rows are right, and the call does not
take a hundred times as long."""
import numpy as np
import pytest

from gorch_b200.workloads import f32_to_bf16_bits
from tests.test_gpu_lm_head_adapters import _Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,V,K,n,R", [(64, 3000, 1024, 8, 16), (300, 2000, 256, 20, 24)])
@pytest.mark.parametrize("what", ["b", "a"])
def test_neighbours_of_an_adapter_of_nan(_sampler_session, B, V, K, n, R, what):
    import torch
    s = _sampler_session
    c = _Case(torch, B + K, B, V, K, n, R)
    getattr(c, what)[3] = f32_to_bf16_bits(np.float32([np.nan]))[0]
    c.rows[:2] = 3
    c.upload()
    got = c.run(s)                                              # (its status is looked at there)
    c.check(got)
    assert np.isnan(got[c.rows == 3]).all() and np.isfinite(got[c.rows != 3]).all()


def test_what_it_costs(_sampler_session):
    """The rows around the adapter's are worked out again, one by one: at 64 x 1,024 x 50,000 at most 40 times a call without a NaN."""
    import torch
    s = _sampler_session
    B, V, K, n, R = 64, 50000, 1024, 8, 16
    g = torch.Generator(device="cuda").manual_seed(1)

    def make(*shape):
        return (torch.randn(*shape, device="cuda", generator=g) * 0.1).to(torch.bfloat16)
    from gorch_b200 import _lib
    x, w, a, b = make(B, K), make(V, K), make(n, R, K), make(n, V, R)
    rows = torch.arange(B, device="cuda", dtype=torch.int32) % n
    rec = _lib.Adapters()
    rec.a, rec.a_pitch, rec.a_stride, rec.b, rec.b_pitch, rec.b_stride, rec.n, rec.rank = a.data_ptr(), K, R * K, b.data_ptr(), R, V * R, n, R
    ws, out = torch.empty(s.lm_head_adapters_workspace(B, K, rec), dtype=torch.uint8, device="cuda"), torch.empty(B, V, device="cuda")
    torch.cuda.synchronize()
    s.set_stream(torch.cuda.current_stream().cuda_stream)
    try:
        def us(times):
            first, last = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            took = []
            for _ in range(times):
                first.record()
                s.lm_head_adapters_ptrs(x.data_ptr(), K, w.data_ptr(), K, B, V, K, rec, rows.data_ptr(), ws.data_ptr(), ws.numel(), out.data_ptr(), V)
                last.record()
                torch.cuda.synchronize()
                took.append(first.elapsed_time(last) * 1e3)
            return sorted(took)[times // 2]
        us(3)
        clean = us(9)
        b[3] = float("nan")
        with_nan = us(9)
        assert s.lm_head_status() == 0
        nan = torch.isnan(out)
        assert nan[rows == 3].all() and not nan[rows != 3].any()
    finally:
        s.set_stream(None)
    assert with_nan <= 40 * clean, (clean, with_nan)
