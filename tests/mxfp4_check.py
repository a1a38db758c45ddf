"""MXFP4 and the grouped route from their definitions, in numpy: what the
kernels of k_mxfp4.cu, k_linear_mxfp4.cu and k_route_grouped.cu are held to.
Values and sums in binary64; the route's scores in binary32 with each
exponential and each softmax sum rounded once from binary64, as the
operator's definition says, because whole numbers come out of comparing them."""

import numpy as np

from tests import model_check as MC

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# Half the gap between neighbours: a value on one of these lies between two
# grid values, and the one with mantissa bit 0 (an even code) takes it.
MIDDLE = (GRID[1:] + GRID[:-1]) / 2


def narrow(t, x):
    """x in the element type t as the kernels read it: f32, or 16-bit words."""
    x = np.ascontiguousarray(x, np.float32)
    return x if t == "f32" else np.asarray(MC.narrow(t, x)).reshape(x.shape)


def widen_type(t, x):
    return x if t == "f32" else np.asarray(MC.widen(t, x)).reshape(x.shape)


def quantise(x):
    """(codes [.., k / 2] u8, scales [.., k / 32] u8) of f32 x [.., k]."""
    x = np.asarray(x, np.float32)
    b = x.reshape(x.shape[:-1] + (-1, 32)).astype(np.float64)
    amax = np.abs(b).max(-1)
    ok = np.isfinite(b).all(-1)
    _, ex = np.frexp(np.where(ok, amax, 1.0))  # amax = f 2^ex, f in [1/2, 1)
    s = np.where(ok & (amax > 0), np.clip(ex - 1 - 2 + 127, 0, 254), 0)
    t = np.where(ok[..., None], np.abs(b), 0.0) * np.exp2(127.0 - s)[..., None]
    up = np.searchsorted(MIDDLE, t, "left")  # ties to the lower neighbour ...
    tie = np.isin(t, MIDDLE) & (up % 2 == 1)  # ... but an odd code gives way to the even one above
    code = (up + tie).astype(np.uint8) | (np.where(ok[..., None], np.signbit(b), False).astype(np.uint8) << 3)
    code = code.reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), np.where(ok, s, 255).astype(np.uint8)


def widen(codes, scales):
    """The binary64 values of codes [.., k / 2] and scales [.., k / 32]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1,))
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return v * np.repeat(s, 32, -1)


def linear_bound(w, x, t):
    """How far y = w x may be, elementwise, for w [n, kk] and x [m, kk] in
    binary64, y of type t. An input is held as parts relative to the largest
    of a run of at most 512: within 2^-22 of itself, or 2^-38 of that
    largest. At most 64 sums in a row keep 23 bits each of at most the sum of
    magnitudes, the runs' sums 24 bits each; then y's own rounding."""
    aw, ax = np.abs(w), np.abs(x)
    total = ax @ aw.T
    kk = x.shape[-1]
    run = np.zeros_like(total)
    for i in range(0, kk, 512):
        run += ax[:, i:i + 512].max(-1, keepdims=True) * aw[:, i:i + 512].sum(-1)[None]
    far = total * ((64 + kk / 512) * 2.0 ** -23 + 2.0 ** -22) + run * 2.0 ** -38
    y = np.abs(x @ w.T)
    return far + {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -10}[t] * (y + far) + {"f16": 2.0 ** -24}.get(t, 2.0 ** -140)


def route_grouped(x, k, groups=1, top_groups=1, group_by=1, sigmoid=False, renorm=False, factor=1.0, bias=None):
    """(ids, weights in binary64, scores) of f32 logits x [m, n]."""
    x = np.asarray(x, np.float32)
    m, n = x.shape
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if sigmoid:
            s = np.float32(1) / (np.float32(1) + np.exp(-x.astype(np.float64)).astype(np.float32))
        else:
            top = np.fmax.reduce(x, -1)[:, None]
            e = np.exp((x - top).astype(np.float64)).astype(np.float32)
            e = np.where((top == -np.inf) & ~np.isnan(x), np.float32(0), e)
            total = e.astype(np.float64).sum(-1, keepdims=True)
            s = e / np.where(total == 0, 1, total).astype(np.float32)
        c = s if bias is None else s + np.asarray(bias, np.float32)
    low = lambda v: -np.inf if np.isnan(v) else float(v)  # noqa: E731
    per = n // groups
    ids = np.zeros((m, k), np.uint32)
    ws = np.zeros((m, k))
    for r in range(m):
        among = range(n)
        if top_groups < groups:
            worth = []
            for g in range(groups):
                v = sorted(c[r, g * per:(g + 1) * per], key=lambda z: (np.isnan(z), -low(z)))
                worth.append(np.float32(v[0] + v[1]) if group_by == 2 and per > 1 else v[0])
            kept = sorted(range(groups), key=lambda g: (np.isnan(worth[g]), -low(worth[g]), g))[:top_groups]
            among = [i for g in sorted(kept) for i in range(g * per, (g + 1) * per)]
        ids[r] = sorted(among, key=lambda i: (np.isnan(c[r, i]), -low(c[r, i]), i))[:k]
        v = s[r, ids[r]].astype(np.float64)
        if renorm:
            v = np.zeros(k) if v.sum() == 0 else v / v.sum()
        ws[r] = v * factor
    return ids, ws, s
