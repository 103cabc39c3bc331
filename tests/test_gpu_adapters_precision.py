"""gorch_cuda_lm_head_adapters_dev holds what it sums in 32 bits: the adapters' inner product h to the last bit, and the logits in sums of
at most 512 products that the tensor pipe cuts off, added up with rounding."""
import numpy as np
import pytest

from gorch_b200.workloads import f32_to_bf16_bits
from tests.test_gpu_lm_head_adapters import _Case, _f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [3, 40, 130, 256, 300])
def test_the_inner_product_keeps_its_24_bits(_sampler_session, B):
    """Weights of zero and an a with one column: h = scale * (a x) is one product, rounded to f32, and a logit of rank 1 is h b. That has
    24 bits times 8, of which the tensor pipe, adding three parts, may lose a step (2^-23) each; one more for the rounding at
    the end. (Two bf16 lost up to 2^-17.)"""
    import torch
    s = _sampler_session
    c = _Case(torch, B, B, 700, 128, 5, 1, none=0.1)
    rng = np.random.default_rng(B)
    c.w[:] = 0
    c.a[:, :, 1:] = 0
    c.scales = (rng.standard_normal(c.n) * 1.2345678).astype(np.float32)
    c.scales[0] = np.float32(3.2975e38)                         # h = 3.4005e38, next to f32's largest, which the nearest bf16 would put at infinity
    c.a[0, 0, 0] = f32_to_bf16_bits(np.float32([1.0]))[0]
    c.rows[0] = 0
    c.x[c.rows == 0, 0] = f32_to_bf16_bits(np.float32([1.03125]))[0]
    c.b[0] = f32_to_bf16_bits(_f64(c.b[0]).astype(np.float32) * np.float32(2.0 ** -60))
    c.upload()
    got = c.run(s).astype(np.float64)
    for r in range(B):
        a = int(c.rows[r])
        if a < 0:
            assert not got[r].any()
            continue
        h = np.float32(_f64(c.a[a, :1, :1])[0, 0] * _f64(c.x[r, :1])[0]) * c.scales[a]      # (8 bits times 8: exact)
        assert np.isfinite(h)
        want = float(h) * _f64(c.b[a, :, 0])
        assert np.all(np.abs(got[r] - want) <= 4 * 2.0 ** -23 * np.abs(want)), r


@pytest.mark.parametrize("B,K,R", [(2, 4096, 16), (64, 4096, 16), (200, 2048, 64), (40, 8192, 8), (5, 1024, 256)])
def test_sums_do_not_lose_with_the_hidden_size(_sampler_session, B, K, R):
    """Root mean square of the error. A sum of n steps (16 products each) is cut off n times, by half a step of f32 (2^-24 of the sum
    so far) on the average, and always towards the same side; so far is sqrt(j / n) of its size after j of n, on the average 2/3. The
    sums' sizes add up in squares to the logit's, and with them their errors: n 2^-24 2/3 of it. n is 32, and the adapters' 3 for each
    16 of the rank with it, or, at a high rank, theirs and 8. Half as much again for the roundings besides: h is an f32 sum of its own,
    and up to 16 sums are added up. (One sum over all of K: K / 16 steps, six times the bound at 4,096.)"""
    import torch
    s = _sampler_session
    c = _Case(torch, K + B, B, 2000, K, 3, R, none=0.1)
    got = c.run(s).astype(np.float64)
    want, _ = c.want()
    units = 3 * ((R + 15) // 16)
    n = max(32 + 16, 8 + units)
    off = np.sqrt(np.mean((got - want) ** 2) / np.mean(want ** 2))
    assert off <= 1.5 * n * 2.0 ** -24 * 2 / 3, off


@pytest.mark.parametrize("B,K,R", [(40, 512, 112), (200, 448, 16), (300, 512, 3)])
def test_one_sum_is_the_plain_projection(_sampler_session, B, K, R):
    """Up to 512 products rows without an adapter have the bits of gorch_cuda_lm_head_logits_dev."""
    import torch
    s = _sampler_session
    c = _Case(torch, B + R, B, 3000, K, 4, R, none=0.5)
    got = c.run(s)
    plain = torch.empty(c.B, c.V, device="cuda")
    s.lm_head_logits_ptrs(c.dx.data_ptr(), c.ldx, c.dw.data_ptr(), c.ldw, c.B, c.V, c.K, plain.data_ptr(), c.V)
    s.sync()
    assert np.array_equal(got[c.rows < 0], plain.cpu().numpy()[c.rows < 0])
    c.check(got)
