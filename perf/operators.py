"""What stands between the LM head and a token, or a loss, as cases that can be prepared, run and timed.

Four operators on rows of logits: the rules of a request on its logits (penalties for tokens that it
already holds, biases, a grammar's mask), distillation from a teacher's top logits (the loss, and its
gradient), and the LM-head projection with a low-rank adapter of its own for each request. `run` makes
the framework's calls where `own` is true, and computes the same from elementary PyTorch operations in
32 bits where it is false.

Vocabularies are GPT-2's (50,257), Qwen's (151,936) and the 168,320 columns of the cross-entropy
workload; drawn cases take any size from 1,000 columns up to those. Logits are seeded normals with
peaked columns, made on the GPU.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

GPT2_VOCAB = 50257
QWEN_VOCAB = 151936
CE_VOCAB = 168320
MIN_VOCAB = 1000
MAX_ROWS = 512
MAX_CE_BYTES = 1500 * CE_VOCAB * 4               # logits of one distillation call
MAX_WEIGHTS = QWEN_VOCAB * 2048                  # elements of an LM head
MAX_LM_MACS = 256 * QWEN_VOCAB * 1024            # multiply-adds of one projection
MAX_ADAPTER_WEIGHTS = 32 * QWEN_VOCAB * 32       # elements of all adapters' output sides
TORCH_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODES = {"f32": 0, "bf16": 1}


def listed() -> list:
    return [
        # One user's chat on GPT-2: the penalties over a short history, a call where latency counts.
        {"name": "adjust_1", "kind": "adjust", "rows": 1, "vocab": GPT2_VOCAB, "dtype": "f32", "history": 300, "penalties": True, "bias": 0,
         "masks": 0, "allowed": 0.0, "in_place": False},
        # A serving batch in which every request has settings of its own: penalties, a logit_bias map, and a grammar for half the rows.
        {"name": "adjust_64", "kind": "adjust", "rows": 64, "vocab": QWEN_VOCAB, "dtype": "f32", "history": 2048, "penalties": True, "bias": 64,
         "masks": 16, "allowed": 0.3, "in_place": False},
        # A large batch of bf16 rows.
        {"name": "adjust_512", "kind": "adjust", "rows": 512, "vocab": QWEN_VOCAB, "dtype": "bf16", "history": 1000, "penalties": True, "bias": 16,
         "masks": 64, "allowed": 0.3, "in_place": False},
        # Long documents in the context: the history is as long as a fifth of the row.
        {"name": "adjust_long_16", "kind": "adjust", "rows": 16, "vocab": QWEN_VOCAB, "dtype": "bf16", "history": 32768, "penalties": True, "bias": 0,
         "masks": 0, "allowed": 0.0, "in_place": False},
        # Structured output: a grammar state that allows few tokens, on the logits where they lie.
        {"name": "grammar_256", "kind": "adjust", "rows": 256, "vocab": QWEN_VOCAB, "dtype": "f32", "history": 0, "penalties": False, "bias": 0,
         "masks": 40, "allowed": 0.002, "in_place": True},
        # The loss of a short evaluation batch against a teacher's 20 best tokens.
        {"name": "distill_loss_24", "kind": "distill_fwd", "rows": 24, "vocab": GPT2_VOCAB, "dtype": "f32", "k": 20, "temperature": 1.0},
        # The loss of a training batch on the cross-entropy workload's shape, a softened teacher.
        {"name": "distill_loss_1500", "kind": "distill_fwd", "rows": 1500, "vocab": CE_VOCAB, "dtype": "f32", "k": 100, "temperature": 2.0},
        # The gradient of a small batch of bf16 logits.
        {"name": "distill_grad_32", "kind": "distill_bwd", "rows": 32, "vocab": QWEN_VOCAB, "dtype": "bf16", "k": 64, "temperature": 1.0},
        # The gradient of the training batch.
        {"name": "distill_grad_1500", "kind": "distill_bwd", "rows": 1500, "vocab": CE_VOCAB, "dtype": "f32", "k": 100, "temperature": 2.0},
        # One request with an adapter: the weights' read decides.
        {"name": "adapters_1", "kind": "adapters", "rows": 1, "vocab": QWEN_VOCAB, "hidden": 1024, "adapters": 1, "rank": 16, "without": 0.0},
        # A serving batch over eight adapters, some requests without one.
        {"name": "adapters_64", "kind": "adapters", "rows": 64, "vocab": QWEN_VOCAB, "hidden": 1024, "adapters": 8, "rank": 16, "without": 0.2},
        # A large batch over many adapters of a higher rank.
        {"name": "adapters_256", "kind": "adapters", "rows": 256, "vocab": QWEN_VOCAB, "hidden": 1024, "adapters": 32, "rank": 32, "without": 0.1},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["adjust", "adjust", "distill_fwd", "distill_bwd", "adapters"])
    dtype = rng.choice(["f32", "bf16"])
    es = 4 if dtype == "f32" else 2
    if kind == "adjust":
        vocab = _log_int(rng, MIN_VOCAB, QWEN_VOCAB)
        rows = _log_int(rng, 1, min(MAX_ROWS, MAX_ROWS * QWEN_VOCAB * 2 // (vocab * es)))
        if rng.random() < 0.2:
            return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "history": 0, "penalties": False, "bias": 0,
                    "masks": _log_int(rng, 1, 64), "allowed": rng.choice([0.0005, 0.01, 0.5]), "in_place": True}
        history = _log_int(rng, 1, min(32768, 512 * 2000 // rows))
        return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "history": history, "penalties": rng.random() < 0.9,
                "bias": rng.choice([0, 0, _log_int(rng, 1, 300)]), "masks": rng.choice([0, _log_int(rng, 1, 64)]),
                "allowed": rng.choice([0.002, 0.3, 0.9]), "in_place": False}
    if kind in ("distill_fwd", "distill_bwd"):
        vocab = _log_int(rng, MIN_VOCAB, CE_VOCAB)
        rows = _log_int(rng, 8, min(2048, MAX_CE_BYTES // (vocab * 4)))
        return {"kind": kind, "rows": rows, "vocab": vocab, "dtype": dtype, "k": _log_int(rng, 1, 500), "temperature": rng.choice([1.0, 1.5, 2.0, 4.0])}
    vocab = _log_int(rng, MIN_VOCAB, QWEN_VOCAB)
    hidden = 64 * _log_int(rng, 8, min(64, MAX_WEIGHTS // (vocab * 64)))
    rows = _log_int(rng, 1, min(256, MAX_LM_MACS // (vocab * hidden)))
    rank = rng.choice([4, 8, 16, 24, 32, 64])
    adapters = _log_int(rng, 1, max(1, min(rows, 64, MAX_ADAPTER_WEIGHTS // (vocab * rank))))
    return {"kind": kind, "rows": rows, "vocab": vocab, "hidden": hidden, "adapters": adapters, "rank": rank, "without": rng.choice([0.0, 0.1, 0.5])}


# ---- what a user's program has in hand

_handle = None


def _sampler():
    """The one handle that a program keeps, on PyTorch's stream: its inputs come from there."""
    global _handle
    if _handle is None:
        from gorch_b200 import sampling
        _handle = sampling.CudaSampler(torch.cuda.current_device())
        _handle.set_stream(torch.cuda.current_stream().cuda_stream)
    return _handle


def _logits(rows: int, vocab: int, dtype: str, gen) -> torch.Tensor:
    x = torch.randn(rows, vocab, device="cuda", generator=gen).mul_(2.0)
    cols = torch.randint(0, vocab, (rows, 16), device="cuda", generator=gen)
    x.scatter_add_(1, cols, torch.full((rows, 16), 8.0, device="cuda"))
    return x.to(TORCH_DTYPES[dtype])


def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    kind, B, V = case["kind"], case["rows"], case["vocab"]
    st = {}
    if kind == "adjust":
        st["x"] = _logits(B, V, case["dtype"], gen)
        T = case["history"]
        if case["penalties"]:
            pen = np.zeros((B, 4), dtype=np.float32)               # repetition, presence, frequency, unused
            pen[:, 0] = rng.choice([1.0, 1.05, 1.1, 1.3, 0.9], B)
            pen[:, 1] = rng.choice([0.0, 0.5, 1.0, -0.3], B)
            pen[:, 2] = rng.choice([0.0, 0.2, 0.7], B)
            lengths = rng.integers(T // 2, T + 1, B)
            lengths[0] = T
            # token ids of text: few tokens make up most of it
            u = torch.rand(B, T, device="cuda", generator=gen)
            st["history"] = (u.pow(4) * V).to(torch.int32).clamp_(max=V - 1)
            st["lengths"] = torch.from_numpy(lengths.astype(np.int32)).cuda()
            st["prompt_lengths"] = torch.from_numpy((lengths * rng.random(B)).astype(np.int32)).cuda()
            st["penalties"] = torch.from_numpy(pen).cuda()
        if case["bias"]:
            n = min(case["bias"], V)
            counts = rng.integers(0, n + 1, B)
            counts[0] = n
            st["bias_offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()
            st["bias_ids"] = torch.from_numpy(np.concatenate([rng.choice(V, c, replace=False) for c in counts]).astype(np.int32)).cuda()
            st["bias_values"] = torch.from_numpy(rng.choice([-100.0, -3.5, 0.25, 2.0, 5.0], int(counts.sum())).astype(np.float32)).cuda()
        if case["masks"]:
            bits = torch.rand(case["masks"], (V + 31) // 32, 32, device="cuda", generator=gen) < case["allowed"]
            weights = torch.tensor([1 << i for i in range(32)], device="cuda", dtype=torch.int64)
            words = (bits.to(torch.int64) * weights).sum(2)
            st["mask"] = torch.where(words < 1 << 31, words, words - (1 << 32)).to(torch.int32).contiguous()
            which = rng.integers(0, case["masks"], B)
            if not case["in_place"]:
                which[rng.random(B) < 0.5] = -1                    # a row without a grammar
            st["mask_rows"] = torch.from_numpy(which.astype(np.int32)).cuda()
    elif kind in ("distill_fwd", "distill_bwd"):
        x = _logits(B, V, case["dtype"], gen)
        k = min(case["k"], V)
        teacher = x.float().mul_(0.8).add_(torch.randn(B, V, device="cuda", generator=gen))
        values, ids = teacher.topk(k, dim=1)
        del teacher
        ids = ids.to(torch.int32)
        pad = torch.from_numpy(rng.random(B) < 0.05).cuda()        # positions of padding have no teacher
        pad[0] = False
        ids[pad] = -1
        st.update(x=x, teacher_ids=ids.contiguous(), teacher=values.contiguous())
        if kind == "distill_bwd":
            st["row_grads"] = torch.rand(B, device="cuda", generator=gen) + 0.5
            xs, ts = x.float() / case["temperature"], values / case["temperature"]
            stats = torch.empty(B, 4, device="cuda")               # as the forward pass leaves them
            stats[:, 0] = x.amax(1).float()
            stats[:, 1] = (xs - xs.amax(1, keepdim=True)).exp_().sum(1)
            stats[:, 2] = values.amax(1)
            stats[:, 3] = (ts - ts.amax(1, keepdim=True)).exp_().sum(1)
            stats[pad] = 0.0
            st["row_stats"] = stats
    else:
        K, n, R = case["hidden"], case["adapters"], case["rank"]
        pitch = (R + 7) // 8 * 8                                   # an adapter's rows start on 16 bytes
        st["x"] = (torch.randn(B, K, device="cuda", generator=gen) * 0.5).to(torch.bfloat16)
        st["w"] = (torch.randn(V, K, device="cuda", generator=gen) * (4.0 / math.sqrt(K))).to(torch.bfloat16)
        st["a"] = (torch.randn(n, R, K, device="cuda", generator=gen) * (2.0 / math.sqrt(K))).to(torch.bfloat16)
        st["b"] = (torch.randn(n, V, pitch, device="cuda", generator=gen) * (0.5 / math.sqrt(R))).to(torch.bfloat16)
        st["scales"] = torch.from_numpy(rng.choice([0.5, 1.0, 2.0], n).astype(np.float32)).cuda()
        which = rng.integers(0, n, B)
        which[rng.random(B) < case["without"]] = -1
        st["row_adapter"] = torch.from_numpy(which.astype(np.int32)).cuda()
    return st


def prepare(case: dict, seed: int) -> dict:
    st = _inputs(case, seed)
    st["case"] = case
    kind, B, V = case["kind"], case["rows"], case["vocab"]
    if kind == "adjust":
        st["out"] = st["x"] if case["in_place"] else torch.empty_like(st["x"])
    elif kind == "distill_fwd":
        st.update(loss=torch.empty(B, device="cuda"), row_stats=torch.empty(B, 4, device="cuda"), mean=torch.empty(1, device="cuda"))
    elif kind == "distill_bwd":
        st["dx"] = torch.empty(B, V, device="cuda")
    else:
        st["out"] = torch.empty(B, V, device="cuda")
    if not own:
        return st
    from gorch_b200 import _lib
    st["s"] = s = _sampler()
    if kind == "adjust":
        adj = _lib.LogitAdjust()
        if case["penalties"]:
            adj.penalties, adj.history, adj.history_stride = st["penalties"].data_ptr(), st["history"].data_ptr(), st["history"].shape[1]
            adj.history_lengths, adj.prompt_lengths = st["lengths"].data_ptr(), st["prompt_lengths"].data_ptr()
        if case["bias"]:
            adj.bias_offsets, adj.bias_ids, adj.bias_values = st["bias_offsets"].data_ptr(), st["bias_ids"].data_ptr(), st["bias_values"].data_ptr()
            adj.n_bias = st["bias_ids"].numel()
        if case["masks"]:
            adj.mask, adj.mask_stride, adj.n_masks, adj.mask_rows = st["mask"].data_ptr(), st["mask"].shape[1], case["masks"], st["mask_rows"].data_ptr()
        st["adjust"] = adj
    elif kind == "adapters":
        ad = _lib.Adapters()
        ad.a, ad.a_pitch, ad.a_stride = st["a"].data_ptr(), st["a"].stride(1), st["a"].stride(0)
        ad.b, ad.b_pitch, ad.b_stride = st["b"].data_ptr(), st["b"].stride(1), st["b"].stride(0)
        ad.scales, ad.n, ad.rank = st["scales"].data_ptr(), case["adapters"], case["rank"]
        st["adapters"] = ad
        st["workspace"] = torch.empty(s.lm_head_adapters_workspace(B, ad), device="cuda", dtype=torch.uint8)
    return st


# ---- one pass

def _run_own(st: dict):
    from gorch_b200 import row_ops
    case, s = st["case"], st["s"]
    kind, B, V = case["kind"], case["rows"], case["vocab"]
    if kind == "adapters":
        K = case["hidden"]
        s.lm_head_adapters_ptrs(st["x"].data_ptr(), K, st["w"].data_ptr(), K, B, V, K, st["adapters"], st["row_adapter"].data_ptr(),
                                st["workspace"].data_ptr(), st["workspace"].numel(), st["out"].data_ptr(), V)
        return st["out"]
    x, code = st["x"].data_ptr(), CODES[case["dtype"]]
    if kind == "adjust":
        s.adjust_logits_ptrs(x, code, B, V, V, st["adjust"], st["out"].data_ptr(), V)
        return st["out"]
    ids, teacher, k, T = st["teacher_ids"].data_ptr(), st["teacher"].data_ptr(), st["teacher"].shape[1], case["temperature"]
    if kind == "distill_fwd":
        row_ops.distill_fwd_ptrs(s, x, code, B, V, V, ids, teacher, k, k, T, st["loss"].data_ptr(), st["row_stats"].data_ptr(), st["mean"].data_ptr())
        return [st["loss"], st["row_stats"], st["mean"]]
    row_ops.distill_bwd_ptrs(s, x, code, B, V, V, ids, teacher, k, k, T, st["row_stats"].data_ptr(), st["row_grads"].data_ptr(), 1.0 / B, False,
                             st["dx"].data_ptr(), V)
    return st["dx"]


def _allowed(st: dict, V: int) -> torch.Tensor:
    """[rows, V] truth values; every token of a row without a mask."""
    bits = (st["mask"].unsqueeze(2) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    bits = bits.reshape(bits.shape[0], -1)[:, :V].bool()
    rows = st["mask_rows"].long()
    return bits[rows.clamp(min=0)] | (rows < 0).unsqueeze(1)


def _run_plain(st: dict):
    case = st["case"]
    kind, B, V = case["kind"], case["rows"], case["vocab"]
    if kind == "adjust":
        if case["in_place"]:
            return st["x"].masked_fill_(~_allowed(st, V), -math.inf)
        y = st["x"].float()
        if case["penalties"]:
            at = torch.arange(st["history"].shape[1], device="cuda")
            held = at < st["lengths"].unsqueeze(1)
            new = held & (at >= st["prompt_lengths"].unsqueeze(1))
            ids = st["history"].long()
            seen = torch.zeros(B, V, device="cuda", dtype=torch.int32).scatter_add_(1, ids, held.int())
            count = torch.zeros(B, V, device="cuda", dtype=torch.int32).scatter_add_(1, ids, new.int())
            rep, pres, freq = (st["penalties"][:, i:i + 1] for i in range(3))
            y = torch.where(seen > 0, torch.where(y > 0, y / rep, y * rep), y)
            y = y - freq * count.float()
            y = torch.where(count > 0, y - pres, y)
        if case["bias"]:
            per_row = torch.diff(st["bias_offsets"]).long()
            row = torch.repeat_interleave(torch.arange(B, device="cuda"), per_row, output_size=st["bias_ids"].numel())
            y.view(-1).index_add_(0, row * V + st["bias_ids"].long(), st["bias_values"])
        if case["masks"]:
            y = y.masked_fill(~_allowed(st, V), -math.inf)
        return y.to(st["x"].dtype)
    if kind == "adapters":
        x = st["x"].float()
        y = x @ st["w"].float().t()
        R = case["rank"]
        for a in range(case["adapters"]):
            mine = (st["row_adapter"] == a).unsqueeze(1)
            h = (x @ st["a"][a].float().t()) * st["scales"][a]
            y += torch.where(mine, h, torch.zeros_like(h)) @ st["b"][a, :, :R].float().t()
        return y
    T = case["temperature"]
    ids, t = st["teacher_ids"].long(), st["teacher"]
    there = ids >= 0
    at = ids.clamp(min=0)
    x = st["x"].float()
    t = torch.where(there, t, torch.full_like(t, -math.inf))
    some = there.any(1)
    if kind == "distill_fwd":
        m, tm = x.amax(1, keepdim=True), t.amax(1, keepdim=True)
        s = ((x - m) / T).exp().sum(1, keepdim=True)
        d = torch.where(there, (t - tm) / T, torch.full_like(t, -math.inf))
        e = d.exp()
        ts = e.sum(1, keepdim=True)
        p = e / ts
        logp = d - ts.log()
        logq = (x.gather(1, at) - m) / T - s.log()
        loss = T * T * torch.where(p > 0, p * (logp - logq), torch.zeros_like(p)).sum(1)
        loss = torch.where(some, loss, torch.zeros_like(loss))
        stats = torch.cat([m, s, tm, ts], 1).masked_fill(~some.unsqueeze(1), 0.0)
        return [loss, stats, loss.sum().reshape(1) / B]
    m, s, tm, ts = (st["row_stats"][:, i:i + 1] for i in range(4))
    q = ((x - m) / T).exp_().div_(s)
    p = torch.where(there, ((t - tm) / T).exp() / ts, torch.zeros_like(t))
    q.scatter_add_(1, at, -p)
    return q.mul_((st["row_grads"] * T / B).unsqueeze(1)).masked_fill_(~some.unsqueeze(1), 0.0)


def run(st: dict):
    return _run_own(st) if own else _run_plain(st)


# ---- the same from the definitions, in 64 bits

def exact(case: dict, seed: int):
    st = _inputs(case, seed)
    kind, B, V = case["kind"], case["rows"], case["vocab"]
    x = st["x"].double()
    if kind == "adjust":
        if case["penalties"]:
            pen = st["penalties"].double().tolist()
            lengths, prompts = st["lengths"].tolist(), st["prompt_lengths"].tolist()
            for b in range(B):
                toks = st["history"][b, : lengths[b]].long()
                prompt, made = torch.bincount(toks[: prompts[b]], minlength=V), torch.bincount(toks[prompts[b]:], minlength=V)
                rep, pres, freq = pen[b][:3]
                hit = (prompt + made).nonzero().squeeze(1)
                z = x[b, hit]
                c = made[hit].double()
                z = torch.where(z > 0, z / rep, z * rep) - freq * c - pres * (c > 0).double()
                x[b, hit] = z
        if case["bias"]:
            off = st["bias_offsets"].tolist()
            for b in range(B):
                x[b, st["bias_ids"][off[b]:off[b + 1]].long()] += st["bias_values"][off[b]:off[b + 1]].double()
        if case["masks"]:
            words = st["mask"].cpu().numpy().view(np.uint8)
            bits = torch.from_numpy(np.unpackbits(words, axis=1, bitorder="little")[:, :V]).cuda()
            for b, r in enumerate(st["mask_rows"].tolist()):
                if r >= 0:
                    x[b, bits[r] == 0] = -math.inf
        return x
    if kind == "adapters":
        y = x @ st["w"].double().t()
        for b, a in enumerate(st["row_adapter"].tolist()):
            if a >= 0:
                h = st["a"][a].double() @ x[b]
                y[b] += st["scales"][a].double() * (st["b"][a, :, : case["rank"]].double() @ h)
        return y
    T = case["temperature"]
    out_loss, out_stats = torch.zeros(B, dtype=torch.float64, device="cuda"), torch.zeros(B, 4, dtype=torch.float64, device="cuda")
    for b in range(B):
        ids = st["teacher_ids"][b]
        keep = ids >= 0
        if kind == "distill_fwd":
            if bool(keep[0]):
                m = x[b].max()
                s = ((x[b] - m) / T).exp().sum()
                out_stats[b, 0], out_stats[b, 1] = m, s
                t = st["teacher"][b].double()
                logp = torch.log_softmax(t / T, 0)
                logq = x[b, ids.long()] / T - (m / T + s.log())
                out_loss[b] = T * T * (logp.exp() * (logp - logq)).sum()
                out_stats[b, 2] = t.max()
                out_stats[b, 3] = ((t - t.max()) / T).exp().sum()
        else:
            if not bool(keep[0]):
                x[b] = 0.0
                continue
            stats = st["row_stats"][b].double()
            q = ((x[b] - stats[0]) / T).exp() / stats[1]
            q[ids.long()] -= ((st["teacher"][b].double() - stats[2]) / T).exp() / stats[3]
            x[b] = q * (st["row_grads"][b].double() * T / B)
    return x if kind == "distill_bwd" else [out_loss, out_stats, out_loss.mean().reshape(1)]


def work(case: dict) -> dict:
    """Each input read once, each output written once; in place, only the logits that change are touched, and the mask that says so."""
    kind, B, V = case["kind"], case["rows"], case["vocab"]
    es = 2 if case.get("dtype") == "bf16" else 4
    if kind == "adjust":
        words = min(case["masks"], B) * ((V + 31) // 32) * 4
        if case["in_place"]:
            return {"bytes": int(B * V * es * (1.0 - case["allowed"])) + words + 4 * B, "flops": 0}
        hist = B * (case["history"] * 3 + 24) if case["penalties"] else 0      # lengths lie between half the history and all of it
        return {"bytes": 2 * B * V * es + hist + B * case["bias"] * 4 + words, "flops": 0}
    taught = int(0.95 * B)                                         # the other rows' logits need not be read
    if kind == "distill_fwd":
        return {"bytes": taught * V * es + B * (8 * min(case["k"], V) + 20), "flops": 4 * taught * V}
    if kind == "distill_bwd":
        return {"bytes": taught * V * es + B * (V * 4 + 8 * min(case["k"], V) + 20), "flops": 4 * taught * V}
    K, n, R = case["hidden"], min(case["adapters"], B), case["rank"]
    with_one = B * (1.0 - case["without"])
    return {"bytes": (V + B) * K * 2 + n * R * (K + V) * 2 + B * V * 4, "flops": int(2 * B * V * K + 2 * with_one * R * (K + V))}
