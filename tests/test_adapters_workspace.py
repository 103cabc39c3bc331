"""gorch_cuda_lm_head_adapters_workspace through CudaSampler, with the hidden size and without it. The call touches no device."""
import pytest

from gorch_b200 import _lib
from gorch_b200.sampling import CudaSampler, GorchCudaError


@pytest.fixture
def sampler():
    s = CudaSampler.__new__(CudaSampler)                        # no context: there need be no GPU
    s._lib, s._ctx = _lib.load(), None
    return s


def _adapters(K, n=3, rank=16, pad=0):
    ad = _lib.Adapters()
    ad.a, ad.a_pitch, ad.a_stride = 256, K + pad, rank * (K + pad)
    ad.b, ad.b_pitch, ad.b_stride = 256, rank, 1000 * rank
    ad.n, ad.rank = n, rank
    return ad


@pytest.mark.parametrize("B", [0, 1, 31, 64, 256, 300])
@pytest.mark.parametrize("K", [64, 1024, 4096])
def test_the_hidden_size_may_be_left_out(sampler, B, K):
    ad = _adapters(K)
    assert sampler.lm_head_adapters_workspace(B, ad) == sampler.lm_head_adapters_workspace(B, K, ad)


@pytest.mark.parametrize("pad", [8, 56, 64, 1000])
def test_without_it_there_is_room_for_any_that_the_rows_hold(sampler, pad):
    ad = _adapters(192, pad=pad)
    have = sampler.lm_head_adapters_workspace(40, ad)
    widest = (192 + pad) // 64 * 64
    assert have == sampler.lm_head_adapters_workspace(40, widest, ad)
    assert all(have >= sampler.lm_head_adapters_workspace(40, K, ad) for K in range(64, widest + 1, 64))


@pytest.mark.parametrize("args", [(4, None), (4, 64, None), (4, 65, _adapters(64)), (-1, _adapters(64)), (4, _adapters(56)), (4, _adapters(64, n=0)),
                                  (4, _adapters(64, rank=300))])
def test_refusals(sampler, args):
    with pytest.raises(GorchCudaError):
        sampler.lm_head_adapters_workspace(*args)


def test_two_records_are_refused(sampler):
    with pytest.raises(TypeError):
        sampler.lm_head_adapters_workspace(4, _adapters(64), _adapters(64))
