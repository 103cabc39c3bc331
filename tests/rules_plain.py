"""The rules of gorch_cuda_adjust_logits_dev written out one logit at a time, on numpy arrays."""
import numpy as np

from gorch_b200.workloads import f32_to_bf16_bits


def upcast(x):
    """f32, or bf16 bit patterns (uint16), as f32."""
    return (x.astype(np.uint32) << 16).view(np.float32) if x.dtype == np.uint16 else x


def tokens_of(history, prompt, V):
    """(held, count) over V columns for one row's tokens."""
    held, count = np.zeros(V, bool), np.zeros(V, np.int64)
    for i, t in enumerate(history):
        if 0 <= t < V:
            held[t] = True
            count[t] += i >= prompt
    return held, count


def adjust(x, penalties=None, history=None, prompt_lengths=None, bias=None, masks=None, mask_rows=None, dtype=np.float64):
    """[B,V] in `dtype` (64 bits: the definition; float32: the device's own order of operations, unrounded), and the bound
    on the device's f32 rounding errors for each logit."""
    B, V = x.shape
    y = upcast(x).astype(dtype)
    bound = np.zeros((B, V))
    half = 2.0 ** -24
    with np.errstate(all="ignore"):
        for b in range(B):
            if penalties is not None:
                rep, pres, freq = (dtype(v) for v in penalties[b])
                if (rep, pres, freq) != (1, 0, 0):
                    held, count = tokens_of(history[b], 0 if prompt_lengths is None else prompt_lengths[b], V)
                    z = y[b]
                    z = np.where(held, np.where(z > 0, z / rep, z * rep), z)
                    fc = freq * count.astype(dtype)
                    # x / rep, freq * c and the two differences, each off by half a step of its result
                    bound[b] += held * half * (3 * np.abs(z) + 3 * np.abs(fc) + abs(pres)).astype(np.float64)
                    y[b] = np.where(count > 0, (z - fc) - pres, z)
            if bias is not None:
                last = dict(bias[b].items() if hasattr(bias[b], "items") else bias[b])
                for t, v in last.items():
                    if 0 <= t < V:
                        y[b, t] = y[b, t] + dtype(np.float32(v))
                        bound[b, t] += half * abs(float(y[b, t]))
            if masks is not None:
                m = b if mask_rows is None else mask_rows[b]
                if 0 <= m < len(masks):
                    y[b, ~np.asarray(masks[m], bool)] = -np.inf
    return y, bound * 1.001


def rounded(y32, like):
    """f32 results in the type of the logits."""
    return f32_to_bf16_bits(y32) if like.dtype == np.uint16 else y32
