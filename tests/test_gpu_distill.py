"""gorch_cuda_distill_fwd_dev / _bwd_dev against the formulas in 64 bits (tests/distill_plain.py, where the
tolerances are derived), and behind TopK and beside the cross-entropy as a training step uses them."""
import numpy as np
import pytest

from gorch_b200 import row_ops
from gorch_b200.config import DTYPE_BF16, DTYPE_F32
from gorch_b200.sampling import GorchCudaError
from gorch_b200.workloads import f32_to_bf16_bits
from tests import distill_plain

pytestmark = pytest.mark.gpu


def _logits(rng, B, V, bf16, scale=2.5):
    x = (rng.standard_normal((B, V)) * scale).astype(np.float32)
    return f32_to_bf16_bits(x) if bf16 else x


def _teacher(rng, B, V, k):
    ids = np.stack([rng.choice(V, k, replace=k > V) for _ in range(B)]).astype(np.int32)
    t = (rng.standard_normal((B, k)) * 3).astype(np.float32)
    return ids, t


def _compare(got, want, bound):
    ok = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~ok & ~np.isnan(want)], want[~ok & ~np.isnan(want)])
    assert np.all(np.abs(got[ok].astype(np.float64) - want[ok]) <= bound[ok]), np.max(np.abs(got[ok] - want[ok]) / np.maximum(bound[ok], 1e-300))


def _both(s, x, ids, t, T, grads=None, scale=0.37, onto=None):
    mean, loss, stats = row_ops.distill(s, x, ids, t, T)
    want, wstats, bound = distill_plain.loss(x, ids, t, T)
    _compare(loss, want, bound)
    fine = np.isfinite(want)
    assert np.array_equal(stats[fine][:, [0, 2]], wstats[fine][:, [0, 2]].astype(np.float32))
    V = x.shape[1]
    off = (4 + 3 * np.log2(max(V, 2)) + 128) * 2.0 ** -24
    assert np.all(np.abs(stats[fine][:, [1, 3]] - wstats[fine][:, [1, 3]]) <= off * wstats[fine][:, [1, 3]])
    if fine.all():
        assert abs(mean - loss.astype(np.float64).mean()) <= 2.0 ** -24 * abs(mean)
    dx = row_ops.distill_backward(s, x, ids, t, T, stats, grads, scale, onto)
    wdx, wbound = distill_plain.gradient(x, ids, t, T, stats, grads, scale)
    if onto is not None:
        wdx = wdx + onto
        wbound = wbound + 2.0 ** -24 * np.abs(wdx)
    _compare(dx, wdx, wbound)
    return loss, stats, dx


# V around a vector, a CTA's chunk of the backward pass (4,096 f32 or 8,192 bf16 columns) and a cluster's slices; k from one entry to
# more than a CTA keeps on chip
SHAPES = [(1, 1, 1), (2, 2, 3), (3, 7, 2), (5, 33, 33), (4, 1000, 17), (3, 4095, 64), (3, 4097, 300), (2, 8193, 5), (2, 16384, 1), (40, 5001, 20), (3, 50257, 100),
          (2, 151936, 1000), (1, 70001, 4000)]


@pytest.mark.parametrize("T", [1.0, 2.0, 0.6])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,V,k", SHAPES)
def test_loss_and_gradient(_sampler_session, B, V, k, bf16, T):
    rng = np.random.default_rng(1000 * k + V)
    x = _logits(rng, B, V, bf16)
    ids, t = _teacher(rng, B, V, k)
    _both(_sampler_session, x, ids, t, T, grads=rng.standard_normal(B).astype(np.float32))


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_without_entries_and_entries_that_are_none(_sampler_session, bf16):
    rng = np.random.default_rng(8)
    B, V, k = 7, 9001, 12
    x = _logits(rng, B, V, bf16)
    ids, t = _teacher(rng, B, V, k)
    ids[0] = -1
    ids[1, ::2] = -1
    ids[2] = V + np.arange(k)
    t[3] = -np.inf
    t[4, 1:] = -np.inf
    ids[5, 3] = 2 ** 31 - 1
    for nothing in (0, 2, 3):
        x[nothing, 100:200] = f32_to_bf16_bits(np.float32([np.nan]))[0] if bf16 else np.nan      # not read
    onto = rng.standard_normal((B, V)).astype(np.float32)
    loss, stats, dx = _both(_sampler_session, x, ids, t, 1.5)
    assert not loss[[0, 2, 3]].any() and not stats[[0, 2, 3]].any() and not dx[[0, 2, 3]].any()
    _, _, dx = _both(_sampler_session, x, ids, t, 1.5, onto=onto)
    assert np.array_equal(dx[[0, 2, 3]], onto[[0, 2, 3]])


@pytest.mark.parametrize("bf16", [False, True])
def test_values_at_the_ends(_sampler_session, bf16):
    """Infinities, NaN, the type's lowest value, rows of one value, spreads that leave f32's range of exponents."""
    rng = np.random.default_rng(9)
    B, V, k = 10, 4500, 6
    x = _logits(rng, B, V, False)
    ids, t = _teacher(rng, B, V, k)
    x[0, 17] = np.nan
    x[1, 18] = np.inf
    x[2, :] = -np.inf
    x[3, 1::2] = -np.inf
    ids[3] = np.arange(0, 2 * k, 2)                         # finite columns
    x[4, ids[4, 2]] = -np.inf                               # an entry where the student has nothing: loss +Inf
    x[5, :] = np.finfo(np.float32).min
    x[6, :] = 3.25
    x[7, 5] = 3e4
    t[8, 0] = np.inf
    t[9] = np.float32([0, -200, -300, -1e30, 0, np.finfo(np.float32).min])
    x[9, ids[9, 3]] = -np.inf                               # an entry whose p is 0 in f32 there: no term
    if bf16:
        x = f32_to_bf16_bits(x)
    with np.errstate(all="ignore"):
        loss, _, dx = _both(_sampler_session, x, ids, t, 1.0)
    assert np.isnan(loss[[0, 1, 2, 8]]).all() and loss[4] == np.inf and np.isfinite(dx[4]).all() and np.isfinite(loss[[3, 6, 7, 9]]).all()
    # f32's lowest value is (1 - 2^-24) 2^128, which rounds to the next power of two in bf16's 8 bits: -Inf, a row of nothing else
    assert np.isnan(loss[5]) if bf16 else np.isfinite(loss[5])


def test_a_token_listed_twice_counts_twice(_sampler_session):
    rng = np.random.default_rng(10)
    x = _logits(rng, 2, 600, False)
    ids = np.int32([[5, 9, 5, 5], [599, 599, 0, 0]])
    t = np.float32([[1.0, 2.0, 0.5, -1.0], [0.0, 0.0, 3.0, 1.0]])
    _both(_sampler_session, x, ids, t, 2.0)
    ids = np.full((2, 3000), 7, np.int32)                   # and more often than a CTA keeps on chip
    t = rng.standard_normal((2, 3000)).astype(np.float32)
    # 3,000 probabilities added one after the other: 3,000 half steps
    s = _sampler_session
    _, _, stats = row_ops.distill(s, x, ids, t, 1.0)
    dx = row_ops.distill_backward(s, x, ids, t, 1.0, stats)
    want, bound = distill_plain.gradient(x, ids, t, 1.0, stats, None, 1.0)
    assert np.all(np.abs(dx - want) <= bound + 3000 * 2.0 ** -24 * np.abs(dx))


@pytest.mark.parametrize("T", [1e-6, 1e-3, 1e3, 1e6])
def test_temperatures_at_the_ends(_sampler_session, T):
    rng = np.random.default_rng(11)
    x = _logits(rng, 3, 3001, False)
    ids, t = _teacher(rng, 3, 3001, 9)
    s = _sampler_session
    _, loss, stats = row_ops.distill(s, x, ids, t, T)
    want, _, bound = distill_plain.loss(x, ids, t, T)
    _compare(loss, want, bound)
    dx = row_ops.distill_backward(s, x, ids, t, T, stats)
    wdx, wbound = distill_plain.gradient(x, ids, t, T, stats, None, 1.0)
    _compare(dx, wdx, wbound)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pitch,lead,dpitch,dlead,tpitch", [(8600, 0, 8600, 0, 33), (8501, 1, 8503, 3, 40), (8512, 5, 8512, 2, 32)])
def test_strides_and_alignment(_sampler_session, bf16, pitch, lead, dpitch, dlead, tpitch):
    import torch
    s = _sampler_session
    rng = np.random.default_rng(pitch)
    B, V, k, T = 5, 8500, 32, 1.25
    flat = torch.from_numpy((rng.standard_normal(lead + B * pitch) * 2).astype(np.float32)).cuda()
    flat = flat.to(torch.bfloat16) if bf16 else flat
    x = flat.as_strided((B, V), (pitch, 1), lead)
    ids = torch.from_numpy(rng.integers(0, V, (B, tpitch)).astype(np.int32)).cuda()
    t = torch.from_numpy(rng.standard_normal((B, tpitch)).astype(np.float32)).cuda()
    loss, stats, dflat = torch.zeros(B, device="cuda"), torch.zeros(B, 4, device="cuda"), torch.full((dlead + B * dpitch,), 7.0, device="cuda")
    dx = dflat.as_strided((B, V), (dpitch, 1), dlead)
    torch.cuda.synchronize()
    code = DTYPE_BF16 if bf16 else DTYPE_F32
    row_ops.distill_fwd_ptrs(s, x.data_ptr(), code, B, V, pitch, ids.data_ptr(), t.data_ptr(), k, tpitch, T, loss.data_ptr(), stats.data_ptr())
    row_ops.distill_bwd_ptrs(s, x.data_ptr(), code, B, V, pitch, ids.data_ptr(), t.data_ptr(), k, tpitch, T, stats.data_ptr(), None, 1.0, False,
                             dx.data_ptr(), dpitch)
    s.sync()
    hx = x.contiguous().cpu()
    hx = hx.view(torch.int16).numpy().view(np.uint16) if bf16 else hx.numpy()
    hi, ht = ids[:, :k].cpu().numpy(), t[:, :k].cpu().numpy()
    want, _, bound = distill_plain.loss(hx, hi, ht, T)
    _compare(loss.cpu().numpy(), want, bound)
    wdx, wbound = distill_plain.gradient(hx, hi, ht, T, stats.cpu().numpy(), None, 1.0)
    _compare(dx.cpu().numpy(), wdx, wbound)
    rest = dflat.clone()
    rest.as_strided((B, V), (dpitch, 1), dlead).fill_(7.0)
    assert torch.all(rest == 7.0)


def test_the_gradient_in_place_of_the_logits(_sampler_session):
    import torch
    s = _sampler_session
    rng = np.random.default_rng(13)
    B, V, k = 9, 10007, 25
    hx = _logits(rng, B, V, False)
    ids, t = _teacher(rng, B, V, k)
    ids[3] = -1
    x, di, dt = torch.from_numpy(hx).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(t).cuda()
    loss, stats, out = torch.zeros(B, device="cuda"), torch.zeros(B, 4, device="cuda"), torch.empty(B, V, device="cuda")
    torch.cuda.synchronize()
    row_ops.distill_fwd_ptrs(s, x.data_ptr(), DTYPE_F32, B, V, V, di.data_ptr(), dt.data_ptr(), k, k, 2.0, loss.data_ptr(), stats.data_ptr())
    for dst in (out, x):
        row_ops.distill_bwd_ptrs(s, x.data_ptr(), DTYPE_F32, B, V, V, di.data_ptr(), dt.data_ptr(), k, k, 2.0, stats.data_ptr(), None, 0.5, False, dst.data_ptr(), V)
    s.sync()
    assert torch.equal(out, x)


def test_the_gradient_against_differences_of_the_loss(_sampler_session):
    s = _sampler_session
    rng = np.random.default_rng(14)
    V, k, T, h = 40, 5, 2.0, 0.05
    x = rng.standard_normal((1, V)).astype(np.float32)
    ids, t = _teacher(rng, 1, V, k)
    _, _, stats = row_ops.distill(s, x, ids, t, T)
    dx = row_ops.distill_backward(s, x, ids, t, T, stats)
    up, down = (np.repeat(x, V, 0) + sign * h * np.eye(V, dtype=np.float32) for sign in (1, -1))
    many = lambda y: row_ops.distill(s, y.astype(np.float32), np.repeat(ids, V, 0), np.repeat(t, V, 0), T)[1].astype(np.float64)
    diff = (many(up) - many(down)) / (2 * h)
    # third derivative of T^2 log S: below 1 / T, times h^2 / 6; each loss off by its bound over h; x + h by half a step of x
    bound = distill_plain.loss(x, ids, t, T)[2][0]
    assert np.all(np.abs(diff - dx[0]) <= h * h / 6 / T + bound / h + 4e-6)


def test_a_training_step_topk_loss_and_both_gradients(_sampler_session):
    """The teacher's logits through TopK, the loss, the gradient on top of the cross-entropy's: as a step uses them."""
    s = _sampler_session
    rng = np.random.default_rng(15)
    B, V, k, T = 12, 30011, 40, 2.0
    x, teacher = _logits(rng, B, V, True), _logits(rng, B, V, False)
    targets = rng.integers(0, V, B)
    vals, ids = s.topk(teacher, k)
    _, _, lse = row_ops.cross_entropy(s, x, targets)
    hard = row_ops.cross_entropy_backward(s, x, targets, lse, 0.3 / B)
    mean, loss, stats = row_ops.distill(s, x, ids, vals, T)
    dx = row_ops.distill_backward(s, x, ids, vals, T, stats, None, 0.7 / B, onto=hard)
    want, _, bound = distill_plain.loss(x, ids, vals, T)
    _compare(loss, want, bound)
    soft, sbound = distill_plain.gradient(x, ids, vals, T, stats, None, 0.7 / B)
    _compare(dx, hard + soft, sbound + 2.0 ** -24 * np.abs(hard + soft))
    f = distill_plain.upcast(x).astype(np.float64)
    q = np.exp(f - f.max(1, keepdims=True))
    ce = q / q.sum(1, keepdims=True)
    ce[np.arange(B), targets] -= 1
    # the cross-entropy's own: lse is f32, so its exponentials are off by half a step of lse and more (1e-6 of q)
    assert np.all(np.abs(dx - (0.3 / B * ce + soft)) <= sbound + 3e-6 * (0.3 / B * np.abs(ce) + np.abs(soft)) + 1e-9)


def test_captured_and_on_another_stream_the_same_bits(_sampler_session):
    import torch
    s = _sampler_session
    rng = np.random.default_rng(16)
    B, V, k = 33, 50257, 50
    x = torch.from_numpy(_logits(rng, B, V, False)).cuda()
    ids, t = (torch.from_numpy(a).cuda() for a in _teacher(rng, B, V, k))

    def buffers():
        return torch.zeros(B, device="cuda"), torch.zeros(B, 4, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros(B, V, device="cuda")

    def step(b):
        row_ops.distill_fwd_ptrs(s, x.data_ptr(), DTYPE_F32, B, V, V, ids.data_ptr(), t.data_ptr(), k, k, 1.5, b[0].data_ptr(), b[1].data_ptr(), b[2].data_ptr())
        row_ops.distill_bwd_ptrs(s, x.data_ptr(), DTYPE_F32, B, V, V, ids.data_ptr(), t.data_ptr(), k, k, 1.5, b[1].data_ptr(), None, 1.0 / B, False, b[3].data_ptr(), V)
    first, captured, again = buffers(), buffers(), buffers()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    step(first)
    s.sync()
    try:
        with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
            s.set_stream(torch.cuda.current_stream().cuda_stream)
            step(captured)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(first, captured))
            captured[3].zero_()
            torch.cuda.synchronize()
        s.set_stream(side.cuda_stream)
        step(again)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    finally:
        s.set_stream(None)


def test_rows_beyond_32_bit_offsets(_sampler_session):
    import torch
    s = _sampler_session
    V, pitch, dpitch = 3001, (1 << 31) + 40, (1 << 30) + 12
    x, dx = torch.zeros(pitch + V, dtype=torch.bfloat16, device="cuda"), torch.zeros(dpitch + V, device="cuda")
    row = torch.randn(V, device="cuda").bfloat16()
    x[:V], x[pitch:] = row, row
    ids, t = torch.tensor([[3, 3000]] * 2, dtype=torch.int32, device="cuda"), torch.tensor([[1.0, 2.0]] * 2, device="cuda")
    loss, stats = torch.zeros(2, device="cuda"), torch.zeros(2, 4, device="cuda")
    torch.cuda.synchronize()
    row_ops.distill_fwd_ptrs(s, x.data_ptr(), DTYPE_BF16, 2, V, pitch, ids.data_ptr(), t.data_ptr(), 2, 2, 1.0, loss.data_ptr(), stats.data_ptr())
    row_ops.distill_bwd_ptrs(s, x.data_ptr(), DTYPE_BF16, 2, V, pitch, ids.data_ptr(), t.data_ptr(), 2, 2, 1.0, stats.data_ptr(), None, 1.0, False, dx.data_ptr(), dpitch)
    s.sync()
    assert loss[0] == loss[1] != 0 and torch.equal(stats[0], stats[1]) and torch.equal(dx[:V], dx[dpitch:]) and dx[dpitch:].abs().sum() > 0


def test_refusals(_sampler_session):
    import torch
    s = _sampler_session
    B, V, k = 2, 100, 4
    x, dx = torch.zeros(B * V + 8, device="cuda"), torch.full((B * V + 8,), 5.0, device="cuda")
    ids, t, out = torch.zeros(B, k, dtype=torch.int32, device="cuda"), torch.zeros(B, k, device="cuda"), torch.full((64,), 5.0, device="cuda")
    p = dict(x=x.data_ptr(), dtype=DTYPE_F32, B=B, V=V, stride=V, ids=ids.data_ptr(), t=t.data_ptr(), k=k, ts=k, T=1.0, loss=out.data_ptr(), stats=out.data_ptr() + 64,
             mean=out.data_ptr() + 128, dx=dx.data_ptr(), dstride=V, acc=False, grads=0)
    torch.cuda.synchronize()

    def fwd(**kw):
        a = {**p, **kw}
        row_ops.distill_fwd_ptrs(s, a["x"], a["dtype"], a["B"], a["V"], a["stride"], a["ids"], a["t"], a["k"], a["ts"], a["T"], a["loss"], a["stats"], a["mean"])

    def bwd(**kw):
        a = {**p, **kw}
        row_ops.distill_bwd_ptrs(s, a["x"], a["dtype"], a["B"], a["V"], a["stride"], a["ids"], a["t"], a["k"], a["ts"], a["T"], a["stats"], a["grads"] or None, 1.0,
                                 a["acc"], a["dx"], a["dstride"])
    both = [dict(x=0), dict(dtype=3), dict(B=-1), dict(V=0), dict(stride=V - 1), dict(ids=0), dict(t=0), dict(k=0), dict(k=5), dict(k=20000, ts=20000), dict(T=0.0),
            dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(T=1e-7), dict(stats=0), dict(x=p["x"] + 2), dict(ids=p["ids"] + 2), dict(t=p["t"] + 1),
            dict(stats=p["stats"] + 2)]
    for kw in both + [dict(loss=0), dict(loss=p["loss"] + 2), dict(mean=p["mean"] + 1)]:
        with pytest.raises(GorchCudaError):
            fwd(**kw)
    for kw in both + [dict(dx=0), dict(dstride=V - 1), dict(dx=p["dx"] + 2), dict(grads=p["dx"] + 2), dict(dx=p["x"] + 4), dict(dx=p["x"], acc=True),
                      dict(dx=p["x"], dtype=DTYPE_BF16), dict(dx=p["x"], dstride=V + 1)]:
        with pytest.raises(GorchCudaError):
            bwd(**kw)
    fwd(B=0)
    bwd(B=0)
    s.sync()
    assert torch.all(dx == 5.0) and torch.all(out == 5.0)
