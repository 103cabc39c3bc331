"""A draw that runs past the last kept token is token V - 1 (model/generate.go:239). In gorch_cuda_generate_step_adjusted_dev, where the
row's mask does not allow that token but others, the row goes on with its largest logit."""
import ctypes as C

import numpy as np
import pytest

from gorch_b200.config import CFG_DTYPE, DTYPE_BF16, DTYPE_F32, FLAG_FALLBACK, MODE_A, MODE_B
from gorch_b200.generate import GEN_ERROR, GEN_LIVE, GEN_STOP, LOOP_CACHED, DeviceGenerateState
from gorch_b200.rules import LogitRules
from gorch_b200.workloads import f32_to_bf16_bits
from tests import rules_plain

pytestmark = pytest.mark.gpu

CONFIGS = [(0.8, 0, 0.0, MODE_A), (0.8, 40, 0.0, MODE_A), (1.0, 0, 0.9, MODE_B), (0.7, 50, 0.95, MODE_B), (1.3, 300, 0.0, MODE_A)]


def _step(s, torch, x, cfgs, u, masks, rows, stops=(), with_flags=True):
    """One step over logits x: (results, ids, flags, logits after it)."""
    B, V = x.shape
    dev = torch.from_numpy(x.view(np.int16) if x.dtype == np.uint16 else x.copy()).cuda()
    st = DeviceGenerateState(s, [[1, 2]] * B, 5, 100, stops, LOOP_CACHED)
    bufs = [s._buf(16 * B), s._buf(8 * B)]
    torch.cuda.synchronize()
    try:
        s._upload(bufs[0], cfgs)
        s._upload(bufs[1], u)
        pc, pu = (s._lib.gorch_cuda_buffer_device_ptr(b) for b in bufs)
        code = DTYPE_BF16 if x.dtype == np.uint16 else DTYPE_F32
        with LogitRules(s, B, masks=masks, mask_rows=rows) as r:
            if with_flags:
                st.step(dev.data_ptr(), code, V, V, pc, pu, r)
            else:
                err = C.c_void_p()
                assert s._lib.gorch_cuda_generate_step_adjusted_dev(s._ctx, dev.data_ptr(), code, B, V, V, C.byref(r.record), pc, pu, st.ids_ptr,
                                                                    None, C.byref(st.gc), C.byref(err)) == 0
            live = st.live()
            out = st.results()
            after = dev.cpu().numpy()
            return out, st._get("ids", B), st._get("flags", B).view(np.uint32), after.view(np.uint16) if x.dtype == np.uint16 else after, live
    finally:
        for b in bufs:
            s._lib.gorch_cuda_buffer_free(b)
        st.release()


@pytest.mark.parametrize("with_flags", [True, False])
@pytest.mark.parametrize("B,V,bf16", [(5, 3001, False), (5, 3001, True), (300, 2003, False), (300, 2003, True), (40, 50257, False)])
def test_rows_that_fall_through_go_on_with_an_allowed_token(_sampler_session, B, V, bf16, with_flags):
    """Uniforms of 1 and the largest one below 1: whether a row falls through depends on how its sums round (1 times the total may lie
    below the walk's own last sum, which adds in another order), and its flag says so."""
    import torch
    s = _sampler_session
    rng = np.random.default_rng(B + V)
    x = (rng.standard_normal((B, V)) * 2).astype(np.float32)
    x[:, V - 1] = 20.0                                          # what the mask takes away is what would have been drawn anyway
    x = f32_to_bf16_bits(x) if bf16 else x
    masks = rng.random((4, V)) < 0.3
    masks[:, V - 1] = False
    masks[3, V - 1] = True
    rows = np.arange(B) % 5                                     # 4: none
    cfgs = np.zeros(B, dtype=CFG_DTYPE)
    for b in range(B):
        cfgs[b] = CONFIGS[b % 7 % 5]
    u = np.where(rng.random(B) < 0.5, 1.0, np.nextafter(1.0, 0.0))
    out, ids, flags, after, live = _step(s, torch, x, cfgs, u, masks, rows, with_flags=with_flags)
    assert live == B and (out["done"] == GEN_LIVE).all()
    y = rules_plain.upcast(after)
    fell = 0
    for b in range(B):
        token = out["tokens"][b][-1]
        assert len(out["tokens"][b]) == 3 and ids[b] == token == out["next_input"][b]
        assert rows[b] == 4 or masks[rows[b], token]
        if with_flags and flags[b] & FLAG_FALLBACK:
            assert token == (V - 1 if rows[b] >= 3 else int(y[b].argmax()))
            fell += rows[b] < 3
    assert fell or not with_flags


@pytest.mark.parametrize("bf16", [False, True])
def test_what_cannot_be_sampled_still_ends_its_row(_sampler_session, bf16):
    import torch
    s = _sampler_session
    B, V = 8, 700
    x = np.random.default_rng(3).standard_normal((B, V)).astype(np.float32)
    x[1, 10] = np.nan
    x[2, 10] = np.inf
    x[3, 11] = np.nan                                           # masked away: the row goes on
    x[6, :] = -np.inf
    x[7, 20] = x[7, 21] = 9.0                                   # equal largest ones: the lower index
    x = f32_to_bf16_bits(x) if bf16 else x
    masks = np.stack([np.zeros(V, bool), np.arange(V) % 2 == 0, np.isin(np.arange(V), [20, 21, 33])])
    rows = [0, 1, 1, 1, 2, 1, 1, 2]
    cfgs = np.zeros(B, dtype=CFG_DTYPE)
    cfgs[:] = CONFIGS[0]
    cfgs[5] = (1.0, 0, 1e-9, MODE_A)                            # mode A's top_p removes every token
    past = np.full(B, 1.5)                                      # past every sum, which stands for rounding that cannot be had at will
    out, ids, _, after, live = _step(s, torch, x, cfgs, past, masks, rows)
    y = rules_plain.upcast(after)
    assert out["done"].tolist() == [GEN_ERROR] * 3 + [GEN_LIVE] * 3 + [GEN_ERROR, GEN_LIVE] and live == 4
    assert [t[2:] for t in out["tokens"]] == [[], [], [], [int(y[3].argmax())], [int(y[4].argmax())], [int(y[5].argmax())], [], [20]]
    stop = int(y[4].argmax())
    out, *_ = _step(s, torch, x, cfgs, past, masks, rows, stops=[stop])
    assert out["done"][4] == GEN_STOP and out["tokens"][4] == [1, 2]
