"""gorch_cuda_distill_fwd_dev / _bwd_dev on training batches: one CTA per row in the forward pass, several batches of vectors per CTA in the
backward pass, out of place, in place and added up; rows taken out of the batch against the formulas in 64 bits (tests/distill_plain.py).

The bound of tests/distill_plain.py counts 128 terms that a thread adds up one after the other. Here a thread of 256 has V / 256 of a row's
logits, in two sums: V / 512 terms, each addition off by at most half a step of the sum."""
import numpy as np
import pytest

from gorch_b200 import row_ops
from gorch_b200.config import DTYPE_BF16, DTYPE_F32
from tests import distill_plain

pytestmark = pytest.mark.gpu


def _host(torch, t):
    t = t.contiguous().cpu()
    return t.view(torch.int16).numpy().view(np.uint16) if t.dtype == torch.bfloat16 else t.numpy()


# 148 SMs: eight batches of 4,096 columns a CTA (300 x 168,320 f32), four of 8,192 (the same in bf16), two (300 x 50,257 f32), eight of a row of nine (1,200 x 36,001)
@pytest.mark.parametrize("B,V,k,bf16", [(300, 168320, 100, False), (300, 168320, 300, True), (300, 50257, 1000, False), (1200, 36001, 40, False), (620, 70001, 64, True)])
def test_training_batches(_sampler_session, B, V, k, bf16):
    import torch
    s = _sampler_session
    rng = np.random.default_rng(V + B)
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(B, V, device="cuda", generator=g).mul_(2.5)
    x[:, 7] += 12.0
    x = x.to(torch.bfloat16) if bf16 else x
    ids = torch.randint(0, V, (B, k), device="cuda", generator=g, dtype=torch.int32)
    ids[:, : k // 4] = ids[:, k // 4: k // 2][:, : k // 4]      # tokens listed twice, all over the row
    ids[:, 0] = V - 1
    ids[:, 1] = V - 1
    t = torch.randn(B, k, device="cuda", generator=g).mul_(3)
    ids[5::9] = -1                                              # padding
    T, scale = 1.5, 0.37
    grads = torch.rand(B, device="cuda", generator=g) + 0.5
    loss, stats, mean = torch.zeros(B, device="cuda"), torch.zeros(B, 4, device="cuda"), torch.zeros(1, device="cuda")
    dx, onto = torch.full((B, V), 7.0, device="cuda"), torch.randn(B, V, device="cuda", generator=g)
    before = onto.clone()
    code = DTYPE_BF16 if bf16 else DTYPE_F32
    torch.cuda.synchronize()

    def bwd(dst, accumulate):
        row_ops.distill_bwd_ptrs(s, x.data_ptr(), code, B, V, V, ids.data_ptr(), t.data_ptr(), k, k, T, stats.data_ptr(), grads.data_ptr(), scale, accumulate, dst.data_ptr(), V)
    row_ops.distill_fwd_ptrs(s, x.data_ptr(), code, B, V, V, ids.data_ptr(), t.data_ptr(), k, k, T, loss.data_ptr(), stats.data_ptr(), mean.data_ptr())
    bwd(dx, False)
    bwd(onto, True)
    s.sync()
    rows = sorted({0, 1, 5, 14, B // 2, B - 2, B - 1} | set(rng.integers(0, B, 5).tolist()))
    hx, hi, ht, hs = (_host(torch, a[rows]) for a in (x, ids, t, stats))
    want, wstats, bound = distill_plain.loss(hx, hi, ht, T)
    more = max(0.0, V / 512 - 128) * distill_plain.HALF
    hl = _host(torch, loss)
    assert np.all(np.abs(hl[rows] - want) <= bound + T * T * more)
    assert np.all(np.abs(hs[:, 1] - wstats[:, 1]) <= ((4 + 3 * np.log2(V) + 128) * distill_plain.HALF + more) * wstats[:, 1])
    assert np.array_equal(hl == 0, np.isin(np.arange(B), np.arange(5, B, 9)))
    assert abs(float(mean) - hl.astype(np.float64).mean()) <= 2.0 ** -24 * abs(float(mean))
    wdx, wbound = distill_plain.gradient(hx, hi, ht, T, hs, _host(torch, grads[rows]), scale)
    # an entry's p is added to those of its token: at most two here
    assert np.all(np.abs(_host(torch, dx[rows]) - wdx) <= wbound + 2 * distill_plain.HALF * np.abs(wdx))
    summed = _host(torch, before[rows]) + wdx
    assert np.all(np.abs(_host(torch, onto[rows]) - summed) <= wbound + 2.0 ** -24 * np.abs(summed) + 2 * distill_plain.HALF * np.abs(wdx))
    assert torch.equal(onto[5::9], before[5::9]) and not bool(dx[5::9].any())
    if not bf16:
        torch.cuda.synchronize()
        bwd(x, False)                                           # where the logits lie
        s.sync()
        assert torch.equal(x, dx)
