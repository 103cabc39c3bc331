"""gorch_cuda_lm_head_adapters_dev: the LM-head projection with an adapter of its own for each row, against a float64
matmul of the same bf16 operands.

Tolerance, logit by logit: the tensor cores add K / 16 + 2 rank / 16 partial products in f32, each step off by at most a step of
the sum of all terms' magnitudes so far (2^-22 with what a step keeps of 16 products); h is an f32 sum of K products over 32 lanes
(K / 32 + 5 roundings of half a step) and loses 2^-16 on its way in two bf16."""
import numpy as np
import pytest

from gorch_b200 import _lib
from gorch_b200.config import CFG_DTYPE, DTYPE_F32, MODE_A, MODE_B
from gorch_b200.rules import LogitRules
from gorch_b200.sampling import GorchCudaError
from gorch_b200.workloads import f32_to_bf16_bits
from tests import rules_plain
from tests.parity import compare

pytestmark = pytest.mark.gpu


def _f64(bits):
    return rules_plain.upcast(bits).astype(np.float64)


def _bits(rng, *shape, scale=1.0):
    return f32_to_bf16_bits((rng.standard_normal(shape) * scale).astype(np.float32))


class _Case:
    """Operands on the device at the given pitches (elements behind a row are NaN: never read)."""

    def __init__(self, torch, seed, B, V, K, n, R, none=0.2, scales=True, pad=0):
        rng = np.random.default_rng(seed)
        self.torch, self.B, self.V, self.K, self.n, self.R = torch, B, V, K, n, R
        self.x, self.w = _bits(rng, B, K, scale=0.5), _bits(rng, V, K, scale=4 / np.sqrt(K))
        self.a, self.b = _bits(rng, n, R, K, scale=2 / np.sqrt(K)), _bits(rng, n, V, R, scale=1 / np.sqrt(R))
        self.scales = rng.choice(np.float32([0.5, 1.0, -2.0]), n) if scales else None
        self.rows = rng.integers(0, n, B).astype(np.int32)
        self.rows[rng.random(B) < none] = -1
        self.ldx, self.ldw = K + pad, K + pad
        self.a_pitch, self.b_pitch = K + pad, (R + 7) // 8 * 8 + pad
        self.a_stride, self.b_stride = R * self.a_pitch + pad, V * self.b_pitch + pad
        self.upload()

    def _placed(self, arr, pitch, stride=None):
        nan = np.uint16(0x7fc0)
        if arr.ndim == 2:
            flat = np.full((arr.shape[0], pitch), nan)
            flat[:, : arr.shape[1]] = arr
        else:
            flat = np.full((arr.shape[0], stride), nan)
            for i in range(arr.shape[0]):
                flat[i, : arr.shape[1] * pitch].reshape(arr.shape[1], pitch)[:, : arr.shape[2]] = arr[i]
        return self.torch.from_numpy(flat.view(np.int16)).cuda()

    def upload(self):
        t = self.torch
        self.dx, self.dw = self._placed(self.x, self.ldx), self._placed(self.w, self.ldw)
        self.da, self.db = self._placed(self.a, self.a_pitch, self.a_stride), self._placed(self.b, self.b_pitch, self.b_stride)
        self.ds = None if self.scales is None else t.from_numpy(self.scales).cuda()
        self.dr = t.from_numpy(self.rows).cuda()
        self.rec = _lib.Adapters()
        self.rec.a, self.rec.a_pitch, self.rec.a_stride = self.da.data_ptr(), self.a_pitch, self.a_stride
        self.rec.b, self.rec.b_pitch, self.rec.b_stride = self.db.data_ptr(), self.b_pitch, self.b_stride
        self.rec.scales, self.rec.n, self.rec.rank = None if self.ds is None else self.ds.data_ptr(), self.n, self.R
        t.cuda.synchronize()

    def space(self, s):
        ws = self.torch.empty(s.lm_head_adapters_workspace(self.B, self.K, self.rec), dtype=self.torch.uint8, device="cuda")
        return ws.fill_(0xff)                                   # NaN patterns: what is not written must not matter

    def call(self, s, ws, out, ld=None):
        s.lm_head_adapters_ptrs(self.dx.data_ptr(), self.ldx, self.dw.data_ptr(), self.ldw, self.B, self.V, self.K, self.rec, self.dr.data_ptr(),
                                ws.data_ptr(), ws.numel(), out.data_ptr(), ld or self.V)

    def run(self, s):
        out = self.torch.full((self.B, self.V), 7.0, device="cuda")
        ws = self.space(s)
        self.torch.cuda.synchronize()
        self.call(s, ws, out)
        s.sync()
        assert s.lm_head_status() == 0
        return out.cpu().numpy()

    def want(self):
        x, w = _f64(self.x), _f64(self.w)
        with np.errstate(all="ignore"):
            y, size = x @ w.T, np.abs(x) @ np.abs(w).T
            lost = np.zeros_like(y)
            for r in range(self.B):
                i = self.rows[r]
                if 0 <= i < self.n:
                    sc = 1.0 if self.scales is None else float(self.scales[i])
                    a, b = _f64(self.a[i]), _f64(self.b[i])
                    h = sc * (a @ x[r])
                    y[r] += b @ h
                    size[r] += np.abs(b) @ np.abs(h)
                    lost[r] = np.abs(b) @ (abs(sc) * (np.abs(a) @ np.abs(x[r])) * (self.K / 32 + 6) * 2.0 ** -24 + np.abs(h) * 2.0 ** -16)
            return y, lost + (self.K / 16 + 2 * (self.R / 16 + 1) + 2) * 2.0 ** -22 * size

    def check(self, got):
        y, bound = self.want()
        assert np.array_equal(np.isnan(got), np.isnan(y))
        ok = np.isfinite(y)
        assert np.array_equal(got[~ok & ~np.isnan(y)], y[~ok & ~np.isnan(y)])
        assert np.all(np.abs(got[ok] - y[ok]) <= bound[ok]), np.max(np.abs(got[ok] - y[ok]) / bound[ok])


# batch rows around an item (32, 256) and beyond a group (256); ranks below, at and above a unit (16) and a stage (64); more adapters than rows
SHAPES = [(1, 1000, 64, 1, 16), (1, 50257, 1024, 3, 8), (2, 7, 64, 2, 1), (7, 4100, 128, 3, 8), (33, 5000, 192, 33, 4), (64, 50257, 768, 8, 16), (32, 2001, 320, 5, 17),
          (130, 20000, 1024, 40, 24), (256, 4096, 128, 256, 16), (300, 8192, 256, 90, 32), (600, 1111, 64, 12, 65), (5, 3000, 128, 4, 256), (90, 300, 1024, 200, 100)]


@pytest.mark.parametrize("B,V,K,n,R", SHAPES)
def test_against_float64(_sampler_session, B, V, K, n, R):
    import torch
    c = _Case(torch, 100 * B + R, B, V, K, n, R)
    c.check(c.run(_sampler_session))


@pytest.mark.parametrize("B,V,K,n,R,pad", [(20, 900, 128, 4, 16, 8), (70, 2500, 192, 9, 20, 24)])
def test_pitches_and_scales_left_out(_sampler_session, B, V, K, n, R, pad):
    import torch
    s = _sampler_session
    c = _Case(torch, pad, B, V, K, n, R, scales=False, pad=pad)
    c.check(c.run(s))
    flat = torch.full((B, V + 13), 3.0, device="cuda")
    ws = c.space(s)
    torch.cuda.synchronize()
    c.call(s, ws, flat, V + 13)
    s.sync()
    c.check(flat[:, :V].contiguous().cpu().numpy())
    assert torch.all(flat[:, V:] == 3.0)


def test_rows_without_an_adapter_are_the_plain_projection(_sampler_session):
    """All rows, and some: bit for bit what gorch_cuda_lm_head_logits_dev writes."""
    import torch
    s = _sampler_session
    for some in (False, True):
        c = _Case(torch, 5, 40, 6000, 256, 4, 16)
        c.rows[:] = [-1, 4, 2 ** 31 - 1, -2 ** 31] * 10
        if some:
            c.rows[::5] = 2
        c.upload()
        got = c.run(s)
        plain = torch.empty(c.B, c.V, device="cuda")
        s.lm_head_logits_ptrs(c.dx.data_ptr(), c.ldx, c.dw.data_ptr(), c.ldw, c.B, c.V, c.K, plain.data_ptr(), c.V)
        s.sync()
        without = (c.rows < 0) | (c.rows >= c.n)
        assert np.array_equal(got[without], plain.cpu().numpy()[without])
        c.check(got)


def test_what_an_adapter_holds_stays_with_its_rows(_sampler_session):
    """Inf and NaN in one adapter's b, in its a, in one row of x and in w."""
    import torch
    s = _sampler_session
    c = _Case(torch, 9, 70, 3000, 128, 6, 16, none=0.3)
    inf, nan = f32_to_bf16_bits(np.float32([np.inf, np.nan]))
    c.rows[:8] = [0, 1, 2, 3, 0, -1, 5, 1]
    c.b[1, 5:40] = inf
    c.b[1, 41, 3] = nan
    c.b[2, 100] = nan
    c.a[3, 2, 7] = inf
    c.x[4, 9] = nan
    c.x[6, 10] = inf
    c.w[2500, 3] = inf
    c.upload()
    got = c.run(s)
    c.check(got)
    clean = (c.rows == 0) | (c.rows == 5) | (c.rows == 4) | (c.rows == -1)
    clean[[4, 6]] = False
    assert clean.sum() > 20 and np.isfinite(np.delete(got[clean], 2500, axis=1)).all()
    one = _Case(torch, 10, 3, 500, 64, 1, 16, none=0.0)          # rows that all use the adapter
    one.b[0, 7] = inf
    one.upload()
    one.check(one.run(s))


def test_a_projection_of_nothing_but_nan(_sampler_session):
    """Weights, then hidden states of NaN and infinities throughout: every logit is worked out again or known to be NaN, in no time
    to speak of."""
    import torch
    s = _sampler_session
    c = _Case(torch, 11, 256, 6000, 256, 8, 16)
    inf, nan = f32_to_bf16_bits(np.float32([np.inf, np.nan]))
    w = c.w.copy()
    c.w[:, -1] = nan
    c.upload()
    assert np.isnan(c.run(s)).all()
    c.w = w
    c.x[:, ::2], c.x[:, 1::2] = inf, inf | np.uint16(0x8000)
    c.upload()
    c.check(c.run(s))


def test_the_same_call_gives_the_same_bits_and_two_graphs_run_at_once(_sampler_session):
    import torch
    s = _sampler_session
    cases = [_Case(torch, 20 + i, 50, 9000, 256, 7, 24) for i in range(2)]
    first = [c.run(s) for c in cases]
    streams, graphs = [torch.cuda.Stream() for _ in cases], [torch.cuda.CUDAGraph() for _ in cases]
    outs, spaces = [torch.zeros(c.B, c.V, device="cuda") for c in cases], [c.space(s) for c in cases]
    torch.cuda.synchronize()
    try:
        for c, st, g, o, ws in zip(cases, streams, graphs, outs, spaces):
            with torch.cuda.graph(g, stream=st, capture_error_mode="thread_local"):
                s.set_stream(torch.cuda.current_stream().cuda_stream)
                c.call(s, ws, o)
                s.set_stream(None)
        for _ in range(5):
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for o, f in zip(outs, first):
                assert np.array_equal(o.cpu().numpy(), f)
    finally:
        s.set_stream(None)


def test_a_served_step_adapters_rules_and_tokens(_sampler_session, oracle):
    """Hidden states to tokens for a batch in which every request has an adapter, penalties, biases and a grammar of its own."""
    import torch
    s = _sampler_session
    c = _Case(torch, 30, 24, 20000, 256, 5, 16)
    rng = np.random.default_rng(31)
    B, V = c.B, c.V
    cfgs = np.zeros(B, dtype=CFG_DTYPE)
    for b in range(B):
        cfgs[b] = [(0.0, 0, 0.0, MODE_A), (0.8, 40, 0.0, MODE_A), (1.0, 0, 0.9, MODE_B)][b % 3]
    u = rng.random(B)
    rules = dict(penalties=np.tile(np.float32([1.2, 0.3, 0.1]), (B, 1)), history=[rng.integers(0, V, 200).tolist() for _ in range(B)],
                 prompt_lengths=[150] * B, bias=[{int(rng.integers(0, V)): 3.0} for _ in range(B)], masks=rng.random((3, V)) < 0.5,
                 mask_rows=rng.integers(-1, 3, B))
    logits, ids, flags = torch.empty(B, V, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
    ws, dc, du = c.space(s), torch.from_numpy(cfgs.view(np.uint8).reshape(B, 16).copy()).cuda(), torch.from_numpy(u).cuda()
    torch.cuda.synchronize()
    with LogitRules(s, B, **rules) as r:
        c.call(s, ws, logits)
        s.sync()
        raw = logits.cpu().numpy()
        c.call(s, ws, logits)                                   # again, and on to the tokens without a wait
        s.adjust_logits_ptrs(logits.data_ptr(), DTYPE_F32, B, V, V, r.record, logits.data_ptr(), V)
        s.sample_dev_ptrs(logits.data_ptr(), DTYPE_F32, B, V, V, dc.data_ptr(), du.data_ptr(), ids.data_ptr(), flags.data_ptr())
        s.sync()
    c.check(raw)
    want, _ = rules_plain.adjust(raw, dtype=np.float32, **rules)
    assert np.array_equal(logits.cpu().numpy(), want)
    ora = oracle.sample_batch(want, cfgs, u, flags=oracle.FAST_KTH, threads=oracle.hw_threads())
    rep = compare({"ids": ids.cpu().numpy(), "flags": flags.cpu().numpy().view(np.uint32)}, ora, u, check_probs=False, allow_tie_cut=True)
    assert rep["id_mismatch"] == rep["boundary_mismatch"]


def test_refusals(_sampler_session):
    import torch
    s = _sampler_session
    c = _Case(torch, 40, 4, 100, 64, 2, 16)
    out, ws = torch.full((4, 100), 7.0, device="cuda"), c.space(s)
    p = dict(x=c.dx.data_ptr(), ldx=64, w=c.dw.data_ptr(), ldw=64, B=4, V=100, K=64, rec=c.rec, rows=c.dr.data_ptr(), ws=ws.data_ptr(), nb=ws.numel(), out=out.data_ptr(), ld=100)

    def call(**kw):
        a = {**p, **kw}
        s.lm_head_adapters_ptrs(a["x"], a["ldx"], a["w"], a["ldw"], a["B"], a["V"], a["K"], a["rec"], a["rows"], a["ws"], a["nb"], a["out"], a["ld"])

    def rec(**kw):
        r = _lib.Adapters.from_buffer_copy(c.rec)
        for k, v in kw.items():
            setattr(r, k, v)
        return r
    for kw in (dict(x=0), dict(w=0), dict(B=-1), dict(V=0), dict(K=60), dict(ldx=63), dict(x=p["x"] + 2), dict(rec=None), dict(rows=0), dict(rows=p["rows"] + 2), dict(ws=0),
               dict(ws=p["ws"] + 16), dict(nb=p["nb"] - 1), dict(out=0), dict(out=p["out"] + 2), dict(ld=99), dict(rec=rec(a=0)), dict(rec=rec(b=0)), dict(rec=rec(n=0)),
               dict(rec=rec(rank=0)), dict(rec=rec(rank=257)), dict(rec=rec(a_pitch=63)), dict(rec=rec(a_pitch=68)), dict(rec=rec(b_pitch=8)), dict(rec=rec(b_pitch=20)),
               dict(rec=rec(a_stride=8)), dict(rec=rec(b_stride=8)), dict(rec=rec(b_stride=1604)), dict(rec=rec(a=c.rec.a + 8)), dict(rec=rec(b=c.rec.b + 2)),
               dict(rec=rec(scales=c.rec.scales + 2))):
        with pytest.raises(GorchCudaError):
            call(**kw)
    for bad in (dict(B=-1), dict(K=65), dict(rec=None), dict(rec=rec(n=-1)), dict(rec=rec(rank=300))):
        with pytest.raises(GorchCudaError):
            s.lm_head_adapters_workspace(bad.get("B", 4), bad.get("K", 64), bad.get("rec", c.rec))
    call(B=0)
    assert s.lm_head_adapters_workspace(0, 64, c.rec) == 0
    s.sync()
    assert torch.all(out == 7.0)
