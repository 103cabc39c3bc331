"""gorch_cuda_adjust_logits_dev against the rules written out in 64 bits, and against the same operations in
f32 bit for bit; gorch_cuda_generate_step_adjusted_dev against a host loop over those rules.

Tolerances: each f32 operation is off by half a step of its result (tests/rules_plain.py adds them up), a
bf16 result by half a step more (2^-8 of its value). Untouched logits keep their bits."""
import numpy as np
import pytest

from gorch_b200 import _lib
from gorch_b200.config import CFG_DTYPE, DTYPE_BF16, DTYPE_F32, MODE_A, MODE_B, PENALTY_DTYPE
from gorch_b200.generate import GEN_ERROR, GEN_LIVE, GEN_MAX_NEW, LOOP_CACHED, LOOP_QWEN, LOOP_UNCACHED, DeviceGenerateState, generate_on_device
from gorch_b200.rules import LogitRules, adjust_logits, pack_masks
from gorch_b200.sampling import GorchCudaError
from gorch_b200.workloads import f32_to_bf16_bits
from tests import rules_plain

pytestmark = pytest.mark.gpu


def _check(got, x, **rules):
    want, bound = rules_plain.adjust(x, **rules)
    f32, _ = rules_plain.adjust(x, dtype=np.float32, **rules)
    bits = rules_plain.rounded(f32, x)
    fine = ~np.isnan(rules_plain.upcast(bits))
    assert np.array_equal(np.isnan(rules_plain.upcast(got)), ~fine)
    assert np.array_equal(got[fine], bits[fine])
    y = rules_plain.upcast(got).astype(np.float64)
    ok = np.isfinite(want) & np.isfinite(y)
    rel = 2.0 ** -8 if x.dtype == np.uint16 else 0.0
    assert np.all(np.abs(y[ok] - want[ok]) <= bound[ok] + rel * (np.abs(want[ok]) + bound[ok]))
    return y


def _rules(rng, B, V, T, nb, nm, density=0.3):
    pen = np.stack([rng.choice([1.0, 1.1, 1.37, 0.8], B), rng.choice([0.0, 0.5, -0.3], B), rng.choice([0.0, 0.2, 0.71], B)], 1).astype(np.float32)
    hist = [(rng.random(int(rng.integers(0, T + 1))) ** 3 * V).astype(np.int64).tolist() for _ in range(B)]
    hist[0] = (rng.random(T) ** 3 * V).astype(np.int64).tolist()
    prompt = [int(rng.integers(0, len(h) + 1)) for h in hist]
    bias = [[(int(t), float(v)) for t, v in zip(rng.integers(0, V, n), rng.choice([-100.0, 0.3, 2.5], n))]
            for n in rng.integers(0, nb + 1, B)] if nb else None
    masks = rng.random((nm, V)) < density if nm else None
    rows = rng.integers(-1, nm + 1, B) if nm else None
    return dict(penalties=pen, history=hist, prompt_lengths=prompt, bias=bias, masks=masks, mask_rows=rows)


def _logits(rng, B, V, bf16):
    x = (rng.standard_normal((B, V)) * 3).astype(np.float32)
    return f32_to_bf16_bits(x) if bf16 else x


def _run(s, x, in_place, **rules):
    with LogitRules(s, x.shape[0], **rules) as r:
        return adjust_logits(s, x, r, in_place)


# V around a chunk of the kernel (8,192 f32 or 16,384 bf16 columns) and a mask's words; odd V gives rows that start anywhere
SHAPES = [(1, 1, 3, 2, 1), (3, 2, 0, 0, 2), (5, 31, 40, 3, 2), (4, 33, 1, 0, 0), (2, 8191, 100, 20, 3), (2, 8192, 100, 20, 3), (3, 8193, 77, 9, 3),
          (2, 16385, 5000, 700, 2), (7, 50257, 300, 60, 4), (2, 151936, 2048, 5, 1)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("B,V,T,nb,nm", SHAPES)
def test_all_rules_together(_sampler_session, B, V, T, nb, nm, bf16, in_place):
    rng = np.random.default_rng(B * 1000003 + V)
    x = _logits(rng, B, V, bf16)
    rules = _rules(rng, B, V, T, nb, nm)
    _check(_run(_sampler_session, x, in_place, **rules), x, **rules)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("what", ["penalties", "bias", "masks", "nothing"])
def test_one_rule_alone(_sampler_session, what, bf16, in_place):
    rng = np.random.default_rng(5)
    B, V = 6, 20011
    x = _logits(rng, B, V, bf16)
    rules = _rules(rng, B, V, 200, 30, 3)
    keep = {"penalties": ("penalties", "history", "prompt_lengths"), "bias": ("bias",), "masks": ("masks", "mask_rows"), "nothing": ()}[what]
    rules = {k: v for k, v in rules.items() if k in keep}
    got = _run(_sampler_session, x, in_place, **rules)
    _check(got, x, **rules)
    if what == "nothing":
        assert np.array_equal(got, x)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_masks_that_leave_nothing_or_everything_and_odd_values_behind_them(_sampler_session, bf16, in_place):
    rng = np.random.default_rng(6)
    B, V = 8, 9001
    x = _logits(rng, B, V, False)
    x[:, ::7] = np.nan
    x[:, 1::7] = np.inf
    x[:, 2::7] = -np.inf
    x[:, 3::7] = np.finfo(np.float32).min
    x[:, 4::7] = -0.0
    if bf16:
        x = f32_to_bf16_bits(x)
    masks = np.stack([np.zeros(V, bool), np.ones(V, bool), np.arange(V) % 2 == 0, np.arange(V) == V - 1])
    rows = [0, 1, 2, 3, -1, 4, 0, 2]
    pen = np.tile(np.float32([1.3, 0.25, 0.5]), (B, 1))
    hist = [list(range(0, 60)) + list(range(0, 60, 2)) for _ in range(B)]
    with np.errstate(all="ignore"):
        y = _check(_run(_sampler_session, x, in_place, penalties=pen, history=hist, prompt_lengths=[10] * B, masks=masks, mask_rows=rows), x,
                   penalties=pen, history=hist, prompt_lengths=[10] * B, masks=masks, mask_rows=rows)
    assert np.all(y[[0, 6]] == -np.inf)
    assert np.all(y[3, :-1] == -np.inf)


def test_tokens_outside_the_vocabulary_are_passed_over(_sampler_session):
    rng = np.random.default_rng(7)
    x = _logits(rng, 2, 1000, False)
    hist = [[-1, 1000, 5, 2 ** 31 - 1, -2 ** 31, 5], [999, 0, 1001]]
    rules = dict(penalties=np.float32([[1.5, 0.1, 0.2]] * 2), history=hist, bias=[[(-1, 9.0), (1000, 9.0), (7, 1.0)], []])
    _check(_run(_sampler_session, x, False, **rules), x, **rules)


def test_a_token_listed_twice_takes_its_last_bias(_sampler_session):
    x = np.zeros((1, 64), np.float32)
    rules = dict(bias=[[(3, 1.0), (4, 5.0), (3, 2.0), (3, -7.0), (4, 6.0)]])
    y = _run(_sampler_session, x, False, **rules)
    assert y[0, 3] == -7.0 and y[0, 4] == 6.0
    many = [(int(t), float(i)) for i, t in enumerate(np.random.default_rng(0).integers(0, 50, 3000))]   # more than a chunk keeps on chip
    y = _run(_sampler_session, x, True, bias=[many])
    for t, v in dict(many).items():
        assert y[0, t] == v


def test_one_token_held_many_times(_sampler_session):
    x = np.full((1, 300), 2.0, np.float32)
    rules = dict(penalties=np.float32([[1.25, 0.5, 0.001]]), history=[[7] * 100000 + [8] * 3])
    y = _check(_run(_sampler_session, x, False, **rules), x, **rules)
    assert y[0, 7] == np.float32(np.float32(np.float32(1.6) - np.float32(0.001) * np.float32(100000)) - np.float32(0.5))


def _tensors(torch, rng, B, V, bf16, pitch, lead):
    """(storage, view [B, V] at row pitch `pitch`, `lead` elements into it)"""
    x = rng.standard_normal(lead + B * pitch).astype(np.float32) * 3
    flat = torch.from_numpy(x).cuda()
    flat = flat.to(torch.bfloat16) if bf16 else flat
    return flat, flat[lead:lead + (B - 1) * pitch + V].as_strided((B, V), (pitch, 1), lead)


def _host(torch, t):
    t = t.contiguous().cpu()
    return t.view(torch.int16).numpy().view(np.uint16) if t.dtype == torch.bfloat16 else t.numpy()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("pitch_in,lead_in,pitch_out,lead_out", [(9000, 0, 8600, 0), (8501, 1, 8503, 3), (8512, 5, 8512, 2), (8704, 0, 8704, 7)])
def test_strides_and_alignment(_sampler_session, bf16, pitch_in, lead_in, pitch_out, lead_out):
    """Rows that start on any element, in and out; what lies between and behind the rows stays as it was."""
    import torch
    s = _sampler_session
    rng = np.random.default_rng(pitch_in + lead_out)
    B, V = 5, 8500
    rules = _rules(rng, B, V, 300, 20, 2)
    src, x = _tensors(torch, rng, B, V, bf16, pitch_in, lead_in)
    dst, out = _tensors(torch, rng, B, V, bf16, pitch_out, lead_out)
    before_dst, before_src = dst.clone(), src.clone()
    torch.cuda.synchronize()
    with LogitRules(s, B, **rules) as r:
        code = DTYPE_BF16 if bf16 else DTYPE_F32
        s.adjust_logits_ptrs(x.data_ptr(), code, B, V, pitch_in, r.record, out.data_ptr(), pitch_out)
        s.sync()
        _check(_host(torch, out), _host(torch, x), **rules)
        assert torch.equal(src, before_src)
        got = dst.clone()
        got.as_strided((B, V), (pitch_out, 1), lead_out).copy_(before_dst.as_strided((B, V), (pitch_out, 1), lead_out))
        assert torch.equal(got, before_dst)
        s.adjust_logits_ptrs(x.data_ptr(), code, B, V, pitch_in, r.record, x.data_ptr(), pitch_in)
        s.sync()
        _check(_host(torch, x), _host(torch, before_src.as_strided((B, V), (pitch_in, 1), lead_in)), **rules)
        back = src.clone()
        back.as_strided((B, V), (pitch_in, 1), lead_in).copy_(before_src.as_strided((B, V), (pitch_in, 1), lead_in))
        assert torch.equal(back, before_src)


def test_rows_beyond_32_bit_offsets(_sampler_session):
    """A row pitch that puts the second row more than 2^32 bytes behind the first."""
    import torch
    s = _sampler_session
    V, pitch = 5000, (1 << 31) + 24
    flat = torch.zeros(pitch + V, dtype=torch.bfloat16, device="cuda")
    flat[:V] = 1.0
    flat[pitch:] = 2.0
    torch.cuda.synchronize()
    with LogitRules(s, 2, penalties=np.float32([[1.0, 0.0, 0.0], [2.0, 0.0, 0.0]]), history=[[], [4999, 0]], masks=[np.arange(V) != 3] * 2) as r:
        s.adjust_logits_ptrs(flat.data_ptr(), DTYPE_BF16, 2, V, pitch, r.record, flat.data_ptr(), pitch)
        s.sync()
    want = torch.full((V,), 2.0)
    want[0] = want[4999] = 1.0
    want[3] = -np.inf
    assert torch.equal(flat[pitch:].float().cpu(), want)
    del flat


def test_the_same_call_gives_the_same_bits_captured_and_on_another_stream(_sampler_session):
    import torch
    s = _sampler_session
    rng = np.random.default_rng(12)
    B, V = 40, 50257
    rules = _rules(rng, B, V, 900, 40, 3)
    x = torch.from_numpy(_logits(rng, B, V, False)).cuda()
    out = torch.empty_like(x)
    with LogitRules(s, B, **rules) as r:
        def call(dst):
            s.adjust_logits_ptrs(x.data_ptr(), DTYPE_F32, B, V, V, r.record, dst.data_ptr(), V)
        torch.cuda.synchronize()
        call(out)
        s.sync()
        first = out.clone()
        side, graph, captured = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.zeros_like(x)
        torch.cuda.synchronize()
        try:
            with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
                s.set_stream(torch.cuda.current_stream().cuda_stream)
                call(captured)
            for _ in range(2):
                captured.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(captured, first)
            s.set_stream(side.cuda_stream)
            again = torch.zeros_like(x)
            torch.cuda.synchronize()
            call(again)
            side.synchronize()
            assert torch.equal(again, first)
        finally:
            s.set_stream(None)


def _bad(record, field, value):
    setattr(record, field, value)
    return record


def test_refusals(_sampler_session):
    import torch
    s = _sampler_session
    B, V = 3, 100
    x = torch.zeros(B * V + 64, device="cuda")
    x0 = x.clone()
    rng = np.random.default_rng(1)
    with LogitRules(s, B, **_rules(rng, B, V, 10, 4, 2)) as r:
        def call(rec=r.record, ptr=x.data_ptr(), out=x.data_ptr(), B=B, V=V, stride=V, out_stride=V, dtype=DTYPE_F32):
            s.adjust_logits_ptrs(ptr, dtype, B, V, stride, rec, out, out_stride)

        def changed(**kw):
            rec = _lib.LogitAdjust.from_buffer_copy(r.record)
            for k, v in kw.items():
                setattr(rec, k, v)
            return rec
        for bad in (dict(rec=None), dict(ptr=0), dict(out=0), dict(dtype=7), dict(V=0), dict(stride=V - 1), dict(out_stride=V - 1), dict(B=-1),
                    dict(ptr=x.data_ptr() + 2), dict(out=x.data_ptr() + 2), dict(out=x.data_ptr() + 4), dict(out_stride=V + 1),
                    dict(out=x.data_ptr() + 4 * V),
                    dict(rec=changed(history_lengths=0)), dict(rec=changed(history=0)), dict(rec=changed(history_stride=-1)),
                    dict(rec=changed(history_stride=1 << 30)), dict(rec=changed(n_bias=-1)), dict(rec=changed(n_bias=1 << 31)),
                    dict(rec=changed(bias_ids=0)), dict(rec=changed(bias_values=0)), dict(rec=changed(mask_stride=3)), dict(rec=changed(n_masks=0)),
                    dict(rec=changed(mask_rows=0)), dict(rec=changed(n_masks=1 << 31)),
                    dict(rec=changed(history=r.record.history + 1)), dict(rec=changed(mask=r.record.mask + 2)),
                    dict(rec=changed(penalties=r.record.penalties + 2))):
            with pytest.raises(GorchCudaError) as e:
                call(**bad)
            assert e.value.code in (1, 5), bad
        call(B=0)
        s.sync()
        assert torch.equal(x, x0)


def test_rows_side_by_side_in_one_tensor_are_no_overlap(_sampler_session):
    import torch
    s = _sampler_session
    rng = np.random.default_rng(2)
    B, V = 6, 1001
    wide = torch.from_numpy(_logits(rng, B, 2 * V, False)).cuda()
    before = wide.clone()
    rules = _rules(rng, B, V, 50, 5, 2)
    torch.cuda.synchronize()
    with LogitRules(s, B, **rules) as r:
        s.adjust_logits_ptrs(wide.data_ptr(), DTYPE_F32, B, V, 2 * V, r.record, wide.data_ptr() + 4 * V, 2 * V)
        s.sync()
    assert torch.equal(wide[:, :V], before[:, :V])
    _check(wide[:, V:].contiguous().cpu().numpy(), before[:, :V].contiguous().cpu().numpy(), **rules)


# ---- in front of the sampling step, in the generate loop

CONFIGS = [(0.0, 0, 0.0, MODE_A), (0.8, 40, 0.0, MODE_A), (1.0, 0, 0.9, MODE_B), (0.7, 50, 0.95, MODE_B)]


class _Model:
    """Logits of its own for every step, the same whatever was sampled."""

    def __init__(self, torch, steps, code):
        self.steps, self.code, self.at = [torch.from_numpy(x.view(np.int16) if x.dtype == np.uint16 else x).cuda() for x in steps], code, -1

    def forward_dev(self, st):
        self.at += 1
        x = self.steps[self.at]
        return x.data_ptr(), self.code, x.shape[1], x.shape[1]

    prefill_dev = forward_dev


@pytest.mark.parametrize("loop", [LOOP_UNCACHED, LOOP_CACHED, LOOP_QWEN])
@pytest.mark.parametrize("B,V,bf16", [(9, 3000, False), (100, 5000, True), (420, 2003, False)])
def test_generation_under_rules_matches_the_host_loop(_sampler_session, oracle, loop, B, V, bf16):
    """Several steps with growing histories, grammars that change from step to step, rows that end early: ids by the oracle on
    the adjusted logits."""
    import torch
    s = _sampler_session
    rng = np.random.default_rng(B + V)
    max_new, stop = 6, 11
    steps = [_logits(rng, B, V, bf16) for _ in range(max_new)]
    prompts = [rng.integers(0, V, int(rng.integers(1, 9))).tolist() for _ in range(B)]
    cfgs = np.zeros(B, dtype=CFG_DTYPE)
    for b in range(B):
        cfgs[b] = CONFIGS[b % 4]
    u = rng.random((max_new, B))
    pen = np.stack([rng.choice([1.0, 1.4], B), rng.choice([0.0, 0.8], B), rng.choice([0.0, 0.3], B)], 1).astype(np.float32)
    bias = [{int(rng.integers(0, V)): 6.0, stop: 5.0 if b % 5 == 0 else -50.0} for b in range(B)]
    masks = [rng.random((3, V)) < 0.4 for _ in range(max_new)]
    for m in masks:
        m[:, stop] = True
    rows = rng.integers(-1, 3, B)
    per_step = [LogitRules(s, B, penalties=pen, bias=bias, masks=m, mask_rows=rows) for m in masks]
    torch.cuda.synchronize()
    s.set_stream(torch.cuda.current_stream().cuda_stream)
    try:
        got = generate_on_device(_Model(torch, steps, DTYPE_BF16 if bf16 else DTYPE_F32), prompts, cfgs, u, s, max_new, 1 << 20, [stop], loop,
                                 poll_every=2, rules=lambda i: per_step[i])
    finally:
        s.set_stream(None)
        for r in per_step:
            r.release()
    held = [list(p) for p in prompts]
    live = np.ones(B, bool)
    unsure = np.zeros(B, bool)                            # a draw within rounding of its interval's edge: the row's later tokens may differ
    for i in range(max_new):
        f32, _ = rules_plain.adjust(steps[i], pen, held, [len(p) for p in prompts], bias, masks[i], rows, dtype=np.float32)
        want = oracle.sample_batch(np.ascontiguousarray(rules_plain.rounded(f32, steps[i])), cfgs, u[i], flags=oracle.FAST_KTH, threads=oracle.hw_threads())
        for b in range(B):
            if not live[b]:
                continue
            at = len(held[b])
            mine = got["tokens"][b][at] if at < len(got["tokens"][b]) else stop
            if mine != want["ids"][b]:
                info = want["info"][b]
                assert info["cut_in_tie"] or min(abs(u[i, b] - info["edge_lo"]), abs(u[i, b] - info["edge_hi"])) <= 1e-6, (i, b)
                unsure[b], live[b] = True, False
            elif mine == stop:
                live[b] = False
            else:
                held[b].append(mine)
    assert unsure.sum() <= 1 + B // 50
    for b in range(B):
        if not unsure[b]:
            assert got["tokens"][b] == held[b] and got["n_new"][b] == len(held[b]) - len(prompts[b])


def test_a_grammar_that_allows_nothing_ends_its_row(_sampler_session):
    import torch
    s = _sampler_session
    B, V = 6, 700
    x = torch.from_numpy(_logits(np.random.default_rng(3), B, V, False)).cuda()
    cfgs = np.zeros(B, dtype=CFG_DTYPE)
    for b in range(B):
        cfgs[b] = CONFIGS[b % 4]
    masks = np.stack([np.zeros(V, bool), np.arange(V) == 5])
    st = DeviceGenerateState(s, [[1, 2]] * B, 3, 100, (), LOOP_CACHED)
    ended = DeviceGenerateState(s, [[1, 2]] * B, 0, 100, (), LOOP_CACHED)
    bufs = [s._buf(16 * B), s._buf(8 * B)]
    torch.cuda.synchronize()
    try:
        s._upload(bufs[0], cfgs)
        s._upload(bufs[1], np.full(B, 0.5))
        ptr = s._lib.gorch_cuda_buffer_device_ptr
        with LogitRules(s, B, masks=masks, mask_rows=[0, 0, 0, 1, 1, -1]) as r:
            st.step(x.data_ptr(), DTYPE_F32, V, V, ptr(bufs[0]), ptr(bufs[1]), r)
            out = st.results()
        assert out["done"].tolist()[:3] == [GEN_ERROR] * 3 and out["done"].tolist()[3:] == [GEN_LIVE] * 3
        assert out["tokens"][:3] == [[1, 2]] * 3 and out["tokens"][3:5] == [[1, 2, 5]] * 2
        # rows that have ended are left as they are, logits too
        y = x.clone()
        torch.cuda.synchronize()
        with LogitRules(s, B, masks=masks, mask_rows=[1] * 6) as r:
            st.step(x.data_ptr(), DTYPE_F32, V, V, ptr(bufs[0]), ptr(bufs[1]), r)
            s.sync()
        assert torch.equal(x[:3], y[:3]) and not torch.equal(x[5], y[5])
    finally:
        for b in bufs:
            s._lib.gorch_cuda_buffer_free(b)
        st.release()
        ended.release()


def test_generation_with_long_prompts(_sampler_session, oracle):
    """Token buffers beyond what the kernel for short histories holds, and one beyond 2^15 tokens: the rows' own tokens are the history."""
    import torch
    s = _sampler_session
    rng = np.random.default_rng(77)
    V, max_new = 9000, 3
    for longest in (6000, 40000):
        prompts = [(rng.random(n) ** 3 * V).astype(int).tolist() for n in (longest, 5, 4097, 1)]
        B = len(prompts)
        steps = [_logits(rng, B, V, False) for _ in range(max_new)]
        cfgs = np.zeros(B, dtype=CFG_DTYPE)                     # greedy: the ids follow from the adjusted logits alone
        pen = np.tile(np.float32([1.3, 0.4, 0.2]), (B, 1))
        with LogitRules(s, B, penalties=pen) as r:
            torch.cuda.synchronize()
            s.set_stream(torch.cuda.current_stream().cuda_stream)
            try:
                got = generate_on_device(_Model(torch, steps, DTYPE_F32), prompts, cfgs, np.zeros((max_new, B)), s, max_new, 1 << 20, rules=r)
            finally:
                s.set_stream(None)
        held = [list(p) for p in prompts]
        for i in range(max_new):
            y, _ = rules_plain.adjust(steps[i], pen, held, [len(p) for p in prompts], dtype=np.float32)
            for b in range(B):
                held[b].append(int(y[b].argmax()))
        assert got["tokens"] == held


def test_rules_of_another_batch_size_are_refused(_sampler_session):
    s = _sampler_session
    st = DeviceGenerateState(s, [[1], [2]], 3, 100, (), LOOP_CACHED)
    try:
        with LogitRules(s, 1, masks=np.ones((1, 64), bool)) as r:
            with pytest.raises(ValueError):
                st.step(16, DTYPE_F32, 64, 64, 16, 16, r)
            with pytest.raises(ValueError):
                adjust_logits(s, np.zeros((2, 64), np.float32), r)
    finally:
        st.release()


@pytest.mark.parametrize("T,stride", [(4096, 4096), (4097, 4097), (4500, 40000), (32767, 32767), (32768, 32768)])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_histories_around_the_kernels_limits(_sampler_session, T, stride, bf16, in_place):
    """As many tokens as the registers hold and one more, as 16-bit counts hold and one more; all rules; tokens crowded into a few
    columns, one of them in every place."""
    rng = np.random.default_rng(T)
    B, V = 3, 20000
    x = _logits(rng, B, V, bf16)
    rules = _rules(rng, B, V, 50, 400, 2)
    rules["history"] = [(rng.random(T) ** 6 * V).astype(int).tolist(), [V - 1] * T, list(range(100))]
    rules["prompt_lengths"] = [T // 3, 1, 200]
    rules["penalties"] = np.float32([[1.2, 0.3, 0.01], [0.9, 0.0, 0.001], [1.1, -0.2, 0.5]])
    s = _sampler_session
    with LogitRules(s, B, **rules) as r:
        if stride > T:                                          # room for more tokens than there are
            import torch
            wide = torch.full((B, stride), 3, dtype=torch.int32)
            for b, h in enumerate(rules["history"]):
                wide[b, : len(h)] = torch.tensor(h, dtype=torch.int32)
            wide = wide.cuda()
            torch.cuda.synchronize()
            r.record.history, r.record.history_stride = wide.data_ptr(), stride
        _check(adjust_logits(s, x, r, in_place), x, **rules)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_short_and_long_histories_in_one_large_batch(_sampler_session, bf16, in_place):
    """Room for more tokens than the kernel for short histories holds, in a batch that both kernels share: every row once."""
    rng = np.random.default_rng(4)
    B, V = 70, 5001
    x = _logits(rng, B, V, bf16)
    rules = _rules(rng, B, V, 300, 40, 3)
    for b, n in ((3, 4096), (4, 4097), (5, 6000), (40, 5000), (69, 4500)):
        rules["history"][b] = (rng.random(n) ** 3 * V).astype(int).tolist()
        rules["prompt_lengths"][b] = n // 2
    rules["penalties"][5] = (1.0, 0.0, 0.0)                     # long, and without a penalty
    _check(_run(_sampler_session, x, in_place, **rules), x, **rules)


def test_refused_steps_leave_the_logits_alone(_sampler_session):
    import torch
    s = _sampler_session
    B, V = 2, 64
    x = torch.ones(B, V, device="cuda")
    st = DeviceGenerateState(s, [[1]] * B, 3, 100, (), LOOP_CACHED)
    torch.cuda.synchronize()
    try:
        with LogitRules(s, B, masks=np.zeros((B, V), bool)) as r:
            for bad in ("mask_stride", "cfgs", "null", "record"):
                rec = _lib.LogitAdjust.from_buffer_copy(r.record)
                if bad == "mask_stride":
                    rec.mask_stride = 1
                done = st.gc.done
                if bad == "record":
                    st.gc.done = None
                with pytest.raises(GorchCudaError):
                    st.step(0 if bad == "null" else x.data_ptr(), DTYPE_F32, V, V, 0 if bad == "cfgs" else x.data_ptr(), x.data_ptr(), rec)
                st.gc.done = done
            s.sync()
            assert torch.all(x == 1)
    finally:
        st.release()
