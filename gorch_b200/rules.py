"""The rules of a request on its logits, in front of the sampling step: penalties for tokens that it
already holds, a bias map, the mask of a grammar (gorch_cuda_adjust_logits_dev; the reference samples
from the bare logits, model/generate.go:75-79).

`LogitRules` uploads them once and keeps the record that `CudaSampler.adjust_logits_ptrs`,
`DeviceGenerateState.step` and `generate_on_device` take. Callers whose arrays lie on the device already
fill `_lib.LogitAdjust` themselves.
"""
from __future__ import annotations

import numpy as np

from . import _lib
from .config import PENALTY_DTYPE
from .sampling import CudaSampler


def pack_masks(allowed) -> np.ndarray:
    """[n, V] truth values -> [n, (V + 31) // 32] uint32: bit v % 32 of word v // 32 says that token v is allowed."""
    a = np.ascontiguousarray(allowed, dtype=bool)
    n, V = a.shape
    padded = np.zeros((n, (V + 31) // 32 * 32), dtype=bool)
    padded[:, :V] = a
    return np.packbits(padded, axis=1, bitorder="little").view("<u4")


class LogitRules:
    """Device copies of B rows' rules.

    penalties    PENALTY_DTYPE [B], or [B, 3] floats (repetition, presence, frequency)
    history      B lists of token ids, prompt first (a generation takes its own tokens instead)
    prompt_lengths  how many of them are prompt (none when left out)
    bias         B mappings token -> bias, or lists of (token, bias)
    masks        [n, V] truth values, or uint32 words as pack_masks makes them
    mask_rows    the mask of each row, outside 0 .. n - 1: none; without it row b has mask b
    """

    def __init__(self, sampler: CudaSampler, B: int, penalties=None, history=None, prompt_lengths=None, bias=None, masks=None,
                 mask_rows=None):
        parts, rec = [], _lib.LogitAdjust()
        self.V = None                                                 # the vocabulary, where the masks say it

        def add(field, arr):
            parts.append((field, arr))

        if penalties is not None:
            pen = np.asarray(penalties)
            if pen.dtype != PENALTY_DTYPE:
                cols = np.asarray(penalties, dtype=np.float32)
                if cols.shape != (B, 3):
                    raise ValueError("penalties must be PENALTY_DTYPE [B] or floats [B, 3]")
                pen = np.zeros(B, dtype=PENALTY_DTYPE)
                pen["repetition"], pen["presence"], pen["frequency"] = cols.T
            if pen.shape != (B,):
                raise ValueError("penalties must have one entry per row")
            if np.any(~(pen["repetition"] > 0)):
                raise ValueError("a repetition penalty must be above 0 (1 is none)")
            add("penalties", pen)
            rows = [[] for _ in range(B)] if history is None else [list(map(int, h)) for h in history]
            if len(rows) != B:
                raise ValueError("history must have one list per row")
            width = max(max((len(h) for h in rows), default=0), 1)
            held = np.full((B, width), -1, dtype=np.int32)
            for b, h in enumerate(rows):
                held[b, : len(h)] = h
            add("history", held)
            add("history_lengths", np.array([len(h) for h in rows], dtype=np.int32))
            rec.history_stride = width
            if prompt_lengths is not None:
                pl = np.ascontiguousarray(prompt_lengths, dtype=np.int32)
                if pl.shape != (B,):
                    raise ValueError("prompt_lengths must have one entry per row")
                add("prompt_lengths", pl)
        elif history is not None or prompt_lengths is not None:
            raise ValueError("a history serves the penalties: give them too")
        if bias is not None:
            rows = [list(m.items()) if hasattr(m, "items") else list(m) for m in bias]
            if len(rows) != B:
                raise ValueError("bias must have one map per row")
            add("bias_offsets", np.concatenate([[0], np.cumsum([len(r) for r in rows])]).astype(np.int32))
            flat = [e for r in rows for e in r]
            add("bias_ids", np.array([t for t, _ in flat], dtype=np.int32))
            add("bias_values", np.array([x for _, x in flat], dtype=np.float32))
            rec.n_bias = len(flat)
        if masks is not None:
            words = np.asarray(masks)
            if words.dtype == np.uint32:
                words = np.ascontiguousarray(words)
            else:
                words = pack_masks(words)
                self.V = np.shape(masks)[1]
            if words.ndim != 2:
                raise ValueError("masks must be [n, V] truth values or [n, words] uint32")
            add("mask", words)
            rec.n_masks, rec.mask_stride = words.shape
            if mask_rows is not None:
                mr = np.ascontiguousarray(mask_rows, dtype=np.int32)
                if mr.shape != (B,):
                    raise ValueError("mask_rows must have one entry per row")
                add("mask_rows", mr)
        elif mask_rows is not None:
            raise ValueError("mask_rows without masks")
        at, places = 0, []
        for field, arr in parts:
            places.append((field, arr, at))
            at += max((arr.nbytes + 255) & ~255, 256)
        self.s, self.B, self.record = sampler, B, rec
        packed = np.zeros(max(at, 256), dtype=np.uint8)
        for _, arr, o in places:
            packed[o:o + arr.nbytes] = np.ascontiguousarray(arr).view(np.uint8).reshape(-1)
        self._buf = sampler._buf(packed.nbytes)
        sampler._upload(self._buf, packed)
        base = sampler._lib.gorch_cuda_buffer_device_ptr(self._buf)
        for field, _, o in places:
            setattr(rec, field, base + o)

    def check(self, B: int, V: int) -> None:
        """Refuses logits [B, V] that these rules are not for. (Masks of truth values for fewer tokens than V would go unnoticed, as
        their words have room for up to 31 more, and forbid those tokens.)"""
        if B != self.B:
            raise ValueError("the rules are of another batch size")
        if self.V not in (None, V):
            raise ValueError(f"the masks are for {self.V} tokens, the logits have {V}")

    def release(self) -> None:
        if self._buf:
            self.s._lib.gorch_cuda_buffer_free(self._buf)
        self._buf = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.release()


def adjust_logits(s: CudaSampler, logits, rules: LogitRules, in_place: bool = False) -> np.ndarray:
    """logits [B,V] float32, or uint16 bf16 bit patterns -> the same with the rows' rules applied (through the in-place form
    of the device call where in_place is set; the host array is not changed)."""
    from .row_ops import _Bufs
    from .sampling import _logits_arg
    a, dtype = _logits_arg(logits)
    B, V = a.shape
    rules.check(B, V)
    out = np.empty_like(a)
    bufs = _Bufs(s)
    try:
        b_x = bufs.new(a)
        b_o = b_x if in_place else bufs.new(a.nbytes)
        s.adjust_logits_ptrs(bufs.ptr(b_x), dtype, B, V, V, rules.record, bufs.ptr(b_o), V)
        s.sync()
        if out.nbytes:
            s._download(b_o, out)
    finally:
        bufs.free()
    return out
