"""gorch_cuda_adjust_logits_dev where a CTA of the kernel for short histories takes many ranges of columns, of one row and of several, and where
the kernel for long ones takes ranges of full size: against the rules in 64 bits and in f32 (tests/rules_plain.py)."""
import numpy as np
import pytest

from gorch_b200.config import DTYPE_BF16, DTYPE_F32
from gorch_b200.rules import LogitRules, adjust_logits
from tests import rules_plain
from tests.test_gpu_adjust_logits import _check, _logits

pytestmark = pytest.mark.gpu


def _mixed_rules(rng, B, V, T, most_bias, masks=3):
    """Rows with and without penalties, with no, a few and more than 256 biases, with histories from nothing to T tokens."""
    pen = np.stack([rng.choice([1.0, 1.2, 0.85], B), rng.choice([0.0, 0.4], B), rng.choice([0.0, 0.3, 0.77], B)], 1).astype(np.float32)
    pen[::5] = (1.0, 0.0, 0.0)
    hist = [(rng.random(int(n)) ** 3 * V).astype(np.int64).tolist() for n in np.where(rng.random(B) < 0.2, 0, rng.integers(0, T + 1, B))]
    hist[-1] = (rng.random(T) ** 3 * V).astype(np.int64).tolist()
    prompt = [int(rng.integers(0, len(h) + 1)) for h in hist]
    counts = np.where(rng.random(B) < 0.4, 0, rng.integers(0, most_bias + 1, B))
    counts[1], counts[2 % B] = most_bias, min(256, most_bias)
    bias = [[(int(t), float(v)) for t, v in zip(rng.integers(0, V, n), rng.choice([-100.0, 0.3, 2.5], n))] for n in counts]
    return dict(penalties=pen, history=hist, prompt_lengths=prompt, bias=bias, masks=rng.random((masks, V)) < 0.4, mask_rows=rng.integers(-1, masks, B))


# ranges per CTA on 148 SMs with four CTAs each: 64 x 151,936 four of one row or two; 1,300 x 1,001 two or three rows; 97 x 40,007 two
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,V,T,most_bias", [(64, 151936, 1500, 300), (1300, 1001, 60, 400), (97, 40007, 4096, 270), (2400, 3, 5, 2)])
def test_several_ranges_for_a_cta(_sampler_session, B, V, T, most_bias, bf16, in_place):
    rng = np.random.default_rng(B + V)
    x = _logits(rng, B, V, bf16)
    rules = _mixed_rules(rng, B, V, T, most_bias)
    with LogitRules(_sampler_session, B, **rules) as r:
        _check(adjust_logits(_sampler_session, x, r, in_place), x, **rules)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_long_and_short_histories_over_many_ranges(_sampler_session, bf16, in_place):
    """Both kernels on one batch, rows of several ranges for either."""
    rng = np.random.default_rng(21)
    B, V = 80, 90001
    x = _logits(rng, B, V, bf16)
    rules = _mixed_rules(rng, B, V, 700, 300)
    for b, n in ((0, 4096), (7, 4097), (8, 9000), (50, 20000), (79, 5000)):
        rules["history"][b] = (rng.random(n) ** 2 * V).astype(int).tolist()
        rules["prompt_lengths"][b] = n // 3
        rules["penalties"][b] = (1.15, 0.2, 0.01)
    with LogitRules(_sampler_session, B, **rules) as r:
        _check(adjust_logits(_sampler_session, x, r, in_place), x, **rules)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bf16,stride", [(True, 30000), (False, 30000), (True, 40000)])
def test_dense_long_histories_on_full_ranges(_sampler_session, bf16, stride, in_place):
    """Ranges of 16,384 columns with most of their columns touched, so that every warp's list fills many times; 16- and 32-bit counts."""
    rng = np.random.default_rng(22)
    B, V = 40, 151936
    x = _logits(rng, B, V, bf16)
    rules = dict(penalties=np.tile(np.float32([1.3, 0.1, 0.02]), (B, 1)), history=[rng.integers(0, 30000, stride).tolist() for _ in range(B)],
                 prompt_lengths=rng.integers(0, stride, B).tolist())
    with LogitRules(_sampler_session, B, **rules) as r:
        _check(adjust_logits(_sampler_session, x, r, in_place), x, **rules)


@pytest.mark.parametrize("in_place,B,V", [(False, 40, 8000001), (True, 40, 16000003)])
def test_runs_beyond_the_ranges_that_are_sorted_for(_sampler_session, in_place, B, V):
    """A CTA's run of more than 64 ranges of one row: the row's tokens are sorted a second time. Three rows are compared whole; the
    others' untouched logits keep their bits."""
    import torch
    s = _sampler_session
    rng = np.random.default_rng(23)
    T = 4000
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(B, V, device="cuda", dtype=torch.bfloat16).normal_(0, 3, generator=g)
    rules = dict(penalties=np.tile(np.float32([1.3, 0.25, 0.1]), (B, 1)), history=[rng.integers(0, V, T).tolist() for _ in range(B)],
                 prompt_lengths=rng.integers(0, T, B).tolist(),
                 bias=[[(int(t), float(v)) for t, v in zip(rng.integers(0, V, n), rng.choice([-100.0, 2.5], n))] for n in rng.integers(0, 300, B)])
    rules["history"][3] = [V - 1] * T
    out = x.clone() if in_place else torch.empty_like(x)
    torch.cuda.synchronize()
    with LogitRules(s, B, **rules) as r:
        s.adjust_logits_ptrs(out.data_ptr() if in_place else x.data_ptr(), DTYPE_BF16, B, V, V, r.record, out.data_ptr(), V)
        s.sync()

    def host(t):
        return t.cpu().view(torch.int16).numpy().view(np.uint16)
    for b in (0, 3, B - 1):
        _check(host(out[b:b + 1]), host(x[b:b + 1]), **{k: v[b:b + 1] for k, v in rules.items()})
    for b in range(B):
        touched = torch.zeros(V, dtype=torch.bool, device="cuda")
        touched[torch.tensor(rules["history"][b] + [t for t, _ in rules["bias"][b]], device="cuda")] = True
        same = out[b].view(torch.int16) == x[b].view(torch.int16)
        assert bool((same | touched).all())
