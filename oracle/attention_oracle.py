"""Plain 64-bit forms of the attention operators and of their gradients, with bounds on what fp32 arithmetic and the
operand type's roundings may add (test infrastructure; numpy on the CPU).

A rounding to a type of relative step 2 u is off by at most u times the value.  Every `*_bound` below adds up, element
by element, the roundings that the operator's documentation allows: operands and results are rounded once, fp32 sums
lose at most `terms * 2^-24` of the sum of their terms' magnitudes, and 16-bit operands have the probabilities (and the
scores' gradients) rounded to 16 bits in front of the second product.
"""
import numpy as np

F32 = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def allowed_keys(N, Tk, lengths=None, mask=None):
    ok = np.ones((N, Tk), bool)
    if lengths is not None:
        ok &= np.arange(Tk)[None] < np.asarray(lengths)[:, None]
    if mask is not None:
        ok &= np.asarray(mask, bool)
    return ok


def _by_head(x, group=1):
    """[N, T, H, D] -> [N, H * group, T, D]"""
    return np.repeat(np.moveaxis(x, 2, 1), group, axis=1)


def attention(q, k, v, g=None, ok=None, scale=None, dtype="f32"):
    """Returns {name: (value, bound)} for out and, given the output's gradient g, dq, dk, dv; all in float64."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    N, Tq, Hq, D = q.shape
    Tk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    u = HALF_STEP[dtype]
    if ok is None:
        ok = np.ones((N, Tk), bool)
    keep = ok[:, :, None, None]
    k, v = np.where(keep, k, 0.0), np.where(keep, v, 0.0)
    Q, K, V = _by_head(q), _by_head(k, G), _by_head(v, G)
    S = Q @ np.swapaxes(K, 2, 3) * scale
    okb = ok[:, None, None, :]
    S = np.where(okb, S, -np.inf)
    top = np.max(S, axis=3, keepdims=True, initial=-np.inf)
    top = np.where(np.isinf(top), 0.0, top)
    E = np.exp(S - top)
    L = E.sum(axis=3, keepdims=True)
    some = L > 0
    P = np.where(some, E / np.where(some, L, 1.0), 0.0)
    O = P @ V

    # relative error of a probability: its score's (D products and sums, the scaling; twice, its own and the
    # normaliser's), exp2's argument and result, the sum of the probabilities
    mag = (np.abs(Q) @ np.swapaxes(np.abs(K), 2, 3)) * scale
    worst = mag.max(axis=3, keepdims=True, initial=0.0)
    rel = F32 * (2 * (D + 8) * worst + 16 + Tk)
    # exp2 gives zero for what is below fp32's smallest normal number: a probability, its sum being at least 1, may be off
    # by that much however small it is
    flush = 2.0 ** -126
    # fp16: half a step of its smallest numbers, 2^-25, of probabilities that are multiplied by 2^7 at least (2^12 in the
    # gradients' pass)
    tiny = flush + 2.0 ** -32 if dtype == "f16" else flush
    tiny_back = flush + 2.0 ** -37 if dtype == "f16" else flush
    rnd = 0.0 if dtype == "f32" else u
    A = P @ np.abs(V)
    o_err = (rnd + rel + Tk * F32) * A + tiny * np.abs(V).sum(axis=2, keepdims=True)
    back = lambda x: np.moveaxis(x, 1, 2)
    res = {"out": (back(O), back(o_err + u * np.abs(O) + 1e-37))}
    if g is None:
        return res
    Gr = _by_head(np.asarray(g, np.float64))
    dP = Gr @ np.swapaxes(V, 2, 3)
    delta = (P * dP).sum(axis=3, keepdims=True)
    dS = P * (dP - delta)
    shared = lambda x: back(x.reshape(N, Hk, G, Tk, D).sum(axis=2))
    # delta is sum dO O with the rounded result; dO V^T is D products and sums
    delta_err = (np.abs(Gr) * (o_err + u * np.abs(O) + D * F32 * np.abs(O))).sum(axis=3, keepdims=True)
    dp_err = D * F32 * (np.abs(Gr) @ np.swapaxes(np.abs(V), 2, 3))
    ds_mag = P * (np.abs(dP) + np.abs(delta))
    ds_err = rnd * np.abs(dS) + P * (delta_err + dp_err) + (rel + 4 * F32) * ds_mag + flush * (np.abs(dP) + np.abs(delta))
    # fp16: scores' gradients are scaled so that a row's or column's largest is far from fp16's smallest
    least = 2.0 ** -30 if dtype == "f16" else 0.0
    rows_err = ds_err + least * np.abs(dS).max(axis=3, keepdims=True, initial=0.0)
    cols_err = ds_err + least * np.abs(dS).max(axis=2, keepdims=True, initial=0.0)
    dQ = dS @ K * scale
    q_err = (rows_err + Tk * F32 * np.abs(dS)) @ np.abs(K) * scale
    dK = np.swapaxes(dS, 2, 3) @ Q * scale
    k_err = np.swapaxes(cols_err + G * Tq * F32 * np.abs(dS), 2, 3) @ np.abs(Q) * scale
    dV = np.swapaxes(P, 2, 3) @ Gr
    p_err = P * (rnd + rel + G * Tq * F32) + tiny_back
    v_err = np.swapaxes(p_err * np.ones_like(P), 2, 3) @ np.abs(Gr)
    res["dq"] = (back(dQ), back(q_err + u * np.abs(dQ) + 1e-37))
    for name, d, e in (("dk", dK, k_err), ("dv", dV, v_err)):
        d, e = shared(d), shared(e) + 1e-37
        res[name] = (np.where(keep, d, 0.0), np.where(keep, e + u * np.abs(d), 0.0))
    if dtype == "f16":   # a result itself may be one of fp16's smallest numbers
        res = {n: (x, b + 2.0 ** -25 * (b > 0)) for n, (x, b) in res.items()}
    return res


def pairs(n, interleaved):
    i = np.arange(n)
    return (2 * i, 2 * i + 1) if interleaved else (i, n + i)


def _turn(y, co, si, n, interleaved):
    a, b = pairs(n, interleaved)
    y = y.copy()
    ya, yb = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = ya * co - yb * si, yb * co + ya * si
    return y


def norm_rotate(x, w=None, freqs=None, pos=None, eps=1e-6, interleaved=False, g=None, dtype="f32", sums=0):
    """Returns {name: (value, bound)} for y and, given y's gradient g, dx and dw.  `sums`: the most terms that one fp32
    chain of the weight gradient's sum may have."""
    x = np.asarray(x, np.float64)
    N, T, H, D = x.shape
    u = HALF_STEP[dtype]
    w = np.ones(D) if w is None else np.asarray(w, np.float64)
    n = 0 if freqs is None else len(freqs)
    pos = np.arange(T) if pos is None else np.asarray(pos)
    angle = np.broadcast_to(pos, (N, T))[..., None, None].astype(np.float64) * (np.zeros(0) if n == 0 else np.asarray(freqs, np.float64))
    co, si = np.cos(angle), np.sin(angle)
    r = 1.0 / np.sqrt((x * x).mean(axis=3, keepdims=True) + eps)
    base = x * r * w
    y = _turn(base, co, si, n, interleaved)
    # r: 8 squares per lane and 5 steps of the butterfly, halved by the root, the root itself, two products; the angle:
    # its fraction's rounding (2 pi 2^-25 absolute) and the functions' own; the rotation's product and sum
    spread = lambda z: np.abs(_turn(np.abs(z), np.ones_like(co), -np.ones_like(si), n, interleaved)) + np.abs(
        _turn(np.abs(z), np.ones_like(co), np.ones_like(si), n, interleaved)) + np.abs(z)
    res = {"y": (y, u * np.abs(y) + 24 * F32 * spread(base) + 1e-37)}
    if g is not None:
        g = np.asarray(g, np.float64)
        t = _turn(g, co, -si, n, interleaved)
        m = (w * t * x).mean(axis=3, keepdims=True)
        dx = r * (w * t) - x * r ** 3 * m
        sg = spread(g)
        mag = r * np.abs(w) * sg + np.abs(x) * r ** 3 * (np.abs(w) * sg * np.abs(x)).mean(axis=3, keepdims=True)
        res["dx"] = (dx, u * np.abs(dx) + 48 * F32 * mag + 1e-37)
        dw = (t * x * r).sum(axis=(0, 1, 2))
        res["dw"] = (dw, (32 + sums) * F32 * (sg * np.abs(x) * r).sum(axis=(0, 1, 2)) + F32 * np.abs(dw) + 1e-37)
    if dtype == "f16":
        res = {k: (v, b + (2.0 ** -25 if k != "dw" else 0.0)) for k, (v, b) in res.items()}
    return res
