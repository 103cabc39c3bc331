"""gorch_cuda_lm_head_adapters_dev where a pair of CTAs goes from one group of 256 batch rows to the next, each with runs of its own."""
import pytest

from tests.test_gpu_lm_head_adapters import _Case

pytestmark = pytest.mark.gpu


# 79 tiles of 256 columns and three groups on 74 pairs: three items or four for a pair, each of another group; 118 tiles and two groups
@pytest.mark.parametrize("B,V,K,n,R", [(520, 20000, 256, 30, 24), (512, 30000, 128, 300, 8), (700, 40000, 64, 5, 16)])
def test_items_of_several_groups(_sampler_session, B, V, K, n, R):
    import torch
    c = _Case(torch, B + n, B, V, K, n, R)
    c.check(c.run(_sampler_session))
