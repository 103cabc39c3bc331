"""The distillation loss and its gradient written out in 64 bits on numpy arrays, with bounds on what f32 terms may be off by."""
import numpy as np

from tests.rules_plain import upcast

HALF = 2.0 ** -24                                          # half a step of f32, relative


def entries(ids, t, V):
    """The entries of one row that count."""
    ids, t = np.asarray(ids), np.asarray(t, np.float64)
    keep = (ids >= 0) & (ids < V) & ~(t == -np.inf)
    return ids[keep], t[keep]


def softmax(x):
    with np.errstate(all="ignore"):
        e = np.exp(x - x.max()) if x.size else x
        return e / e.sum()


def row_loss(x, ids, t, T):
    """(loss, (M, S, tM, tS), bound on the loss's error) of one row."""
    V = x.size
    i, t = entries(ids, t, V)
    if i.size == 0:
        return 0.0, (0.0, 0.0, 0.0, 0.0), 0.0
    with np.errstate(all="ignore"):
        M, tM = np.nanmax(np.append(x, -np.inf)), np.nanmax(np.append(t, -np.inf))
        S, tS = np.exp((x - M) / T).sum(), np.exp((t - tM) / T).sum()
        if not M > -np.inf:
            S = np.nan
        p = np.exp((t - tM) / T) / tS
        logq = (x[i] - M) / T - np.log(S)
        logp = (t - tM) / T - np.log(tS)
        terms = np.where(p == 0, 0.0, p * (logp - logq))                 # (a NaN p, of a teacher logit of +Inf, stays a NaN)
        loss = T * T * terms.sum()
        # S: its terms 2^t are off by 2^-22 (the special function unit) and 3 half steps of |t| ln 2, |t| at most log2 V on the
        # sum's average; a thread adds up to 128 of them one after the other. p: by 4 half steps and the same of its exponent.
        s_off = (4 + 3 * np.log2(max(V, 2)) + 128) * HALF
        p_off = 8 * HALF * np.sum(p * np.abs(np.where(p == 0, 0.0, logp - logq)) * (1 + np.abs(t - tM) / T)) if np.isfinite(loss) else 0.0
        return loss, (M, S, tM, tS), T * T * (s_off + p_off + 4 * HALF) + 2 * HALF * abs(loss)


def loss(x, ids, t, T):
    x, T = upcast(x).astype(np.float64), float(np.float32(T))      # the entry point takes a float: 0.6 is 0.6 (1 + 4e-8) there, 1e-6 of exp(-28)
    rows = [row_loss(x[b], ids[b], t[b], T) for b in range(len(x))]
    return np.array([r[0] for r in rows]), np.array([r[1] for r in rows]), np.array([r[2] for r in rows])


def gradient(x, ids, t, T, stats, grads, scale):
    """(dx, bound) from the stats that the backward pass is given."""
    x, T = upcast(x).astype(np.float64), float(np.float32(T))
    B, V = x.shape
    dx, bound = np.zeros((B, V)), np.zeros((B, V))
    with np.errstate(all="ignore"):
        for b in range(B):
            M, S, tM, tS = np.asarray(stats[b], np.float64)
            if tS == 0:
                continue
            g = float(scale) * (1.0 if grads is None else float(grads[b])) * T
            d = (x[b] - M) / T
            q = np.exp(d) / S
            # the exponential: 3e-7; its argument's difference half a step, and two products
            off = q * (3e-7 + HALF * (np.where(np.isfinite(d), np.abs(d), 0.0) + 4))
            i, tt = entries(ids[b], t[b], V)
            p = np.exp((tt - tM) / T) / tS
            np.subtract.at(q, i, p)
            np.add.at(off, i, p * HALF * (8 + 2 * np.abs(tt - tM) / T))
            dx[b] = g * q
            bound[b] = abs(g) * (off + 4 * HALF * np.abs(q)) + 1e-37
    return dx, bound
