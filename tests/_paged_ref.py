"""The paged cache's operators in 64 bits on the CPU (numpy), from their
definitions, and the error bounds that the tests hold the kernels to."""

import math

import numpy as np
import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# half the smallest positive number of a type: what a rounding near zero may be off by
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def f64(t):
    return t.detach().to("cpu").double().numpy()


def rotate(x, pos, table, rot, interleaved):
    """x (B,H,L,D) float64, pos (B,L) int, table (N,2,rot/2) fp32 -> float64."""
    x = np.array(x, dtype=np.float64)
    t = table.astype(np.float64)
    inside = (pos >= 0) & (pos < t.shape[0])
    cs = t[np.where(inside, pos, 0)]  # (B,L,2,rot/2)
    cs = np.where(inside[..., None, None], cs, np.nan)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    y = x.copy()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def e4m3_value(codes):
    codes = codes.astype(np.int64)
    e, m, sign = (codes >> 3) & 15, codes & 7, np.where(codes >> 7, -1.0, 1.0)
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    return np.where((codes & 127) == 127, np.nan, sign * v)


_LEVELS = e4m3_value(np.arange(127))  # the magnitudes, ascending


def e4m3_encode(rows):
    """rows (..., D) float64 (fp32 numbers) -> codes, e + 127: nearest level
    by distance, the even code of two equally near."""
    finite = np.isfinite(rows)
    amax = np.where(finite, np.abs(rows), 0.0).max(-1)
    e = np.zeros(amax.shape, dtype=np.int64)
    for i, a in np.ndenumerate(amax):
        if a > 0:
            k = math.frexp(a / 448.0)[1] - 1
            while 448.0 * 2.0 ** k < a:
                k += 1
            while 448.0 * 2.0 ** (k - 1) >= a:
                k -= 1
            e[i] = max(k, -126)
    u = np.where(finite, rows, 0.0) * 2.0 ** (-e[..., None].astype(np.float64))
    mag = np.abs(u)
    hi = np.clip(np.searchsorted(_LEVELS, mag), 1, 126)
    lo = hi - 1
    dl, dh = mag - _LEVELS[lo], _LEVELS[hi] - mag
    code = np.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.signbit(u), code | 128, code)
    return np.where(finite, code, 127).astype(np.uint8), (e + 127).astype(np.uint8)


def int4_encode(rows):
    """rows (..., D) float64 -> codes (..., D) 0..15, scale fp32, min fp32."""
    lo, hi = rows.min(-1), rows.max(-1)
    s = ((hi - lo) / 15.0).astype(np.float32)
    d = rows - lo[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s[..., None] > 0, d / s[..., None].astype(np.float64), 0.0)
    return np.clip(np.rint(q), 0, 15).astype(np.uint8), s, lo.astype(np.float32)


def page_values(layer):
    """Every row of a layer's pages (n_pages,H,page,D) in float64: keys,
    values, and what a value's error in attention is relative to, its
    magnitude.  For INT4 that is |scale * code| + |min|: the kernel sums
    w scale code and w min apart, the first with weights w scale rounded to 16
    bits, so its error is 2^-16 of sum w |scale code|, and more than that of
    sum w |v| where scale * code and min cancel."""
    if layer.k_exp is None:
        v = f64(layer.v)
        return f64(layer.k), v, np.abs(v)

    def scale(t):
        b = t.cpu().numpy().astype(np.int64)
        return np.where(b > 0, 2.0 ** (b - 127.0), 0.0)[..., None]

    k = e4m3_value(layer.k.cpu().numpy()) * scale(layer.k_exp)
    if layer.fmt == "fp8":
        v = e4m3_value(layer.v.cpu().numpy()) * scale(layer.v_scale)
        return k, v, np.abs(v)
    c = layer.v.cpu().numpy()
    c = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1).astype(np.float64)
    sz = f64(layer.v_scale)
    return k, c * sz[..., :1] + sz[..., 1:], np.abs(c * sz[..., :1]) + np.abs(sz[..., 1:])


def sequence(values, table, b, n, page, n_pages):
    """Tokens [0, n) of sequence b: rows (H, n, D), and which take part."""
    ids = table[b, np.arange(n) // page] if n else np.zeros(0, dtype=np.int64)
    ok = (ids >= 0) & (ids < n_pages)
    return [v[np.where(ok, ids, 0), :, np.arange(n) % page].transpose(1, 0, 2) for v in values], ok


def attend(q, values, table, lens, page, n_pages, scale):
    """-> out, lse and the error scale sum_t w_t |v_t| (see page_values) with the largest error of
    a score, both per head (see bound)."""
    B, Hq, D = q.shape
    H = values[0].shape[1]
    G = Hq // H
    out, lse = np.zeros((B, Hq, D)), np.full((B, Hq), -np.inf)
    spread, ds = np.zeros((B, Hq, D)), np.zeros((B, Hq))
    for b in range(B):
        n = int(min(max(lens[b], 0), table.shape[1] * page))
        (k, v, mag), ok = sequence(values, table, b, n, page, n_pages)
        k, v, mag = k[:, ok], v[:, ok], mag[:, ok]
        if k.shape[1] == 0:
            continue
        for h in range(Hq):
            s = k[h // G] @ q[b, h] * scale
            m = s.max()
            w = np.exp(s - m)
            lse[b, h] = m + math.log(w.sum())
            w /= w.sum()
            out[b, h] = w @ v[h // G]
            spread[b, h] = w @ mag[h // G]
            # fp32 accumulation of D exact products, and the scale's and
            # log2 e's rounding
            ds[b, h] = (D + 4) * 2.0 ** -24 * (np.abs(k[h // G]) @ np.abs(q[b, h]) * abs(scale)).max()
    return out, lse, spread, ds


def attend_bound(out, spread, ds, lens, dtype):
    """What the kernel's result may be off by: its own rounding; each weight's
    relative error, from its score (exp magnifies it by 1 + ds; twice, once in
    the sum), from exp2 (2^-22) and from its rounding (as a sum of two bf16
    numbers 2^-16, of two fp16 ones less); the value of an INT4 row in fp32 (scale times code plus minimum,
    folded into the weights: as a weight's error); fp32 sums over n tokens in
    pieces of 32 and then waves and workgroups (n / 32 + 64 roundings)."""
    w = 2.0 ** -16
    n = max(int(max(lens)), 1)
    rel = 2 * ds[..., None] * 1.01 + w + 2.0 ** -21 + (n / 32 + 64) * 2.0 ** -24
    return UNIT[dtype] * np.abs(out) + TINY[dtype] + rel * spread
