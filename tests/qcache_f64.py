"""Caches in 4 or 8 bits: their definitions in 64 bits (numpy) and the error
bounds of what reads them.

Rows are computed in 64 bits and rounded once: half a step of fp32 (u = 2^-24),
and 2^-48 of the pair's size for the arithmetic before.  Codes and parameters
follow from the fp32 rows exactly.

Attention.  A score is sum over groups of step * (q . c) + mid * (sum of q): with
A = sum |q| (step |c| + |mid|), q keeps 22 bits (2^-21 with truncated remainders)
and its sums add at most 17u of A.  The scale, the shift, a cap, a bias and the
exponential add what cache_ops_f64.attention states.  A weight times a step keeps 22
bits, or 2^-32 of the largest step its row sees (halves down to 2^-25 in fp16,
steps brought to 2^8 and more, sums of weights of 1/2 and more); numerator and denominator
each carry (N/16 + 32)u of their sums.
"""
import numpy as np

U = 2.0 ** -24


def order(what, hd, bits):
    """The element at each place of a row's codes (pocr_hip.h, pocr_qcache)."""
    out = []
    for m in range(hd // 8):
        if what == "k" and bits == 4:
            u, c = m // (hd // 32), m % (hd // 32)
            out += [32 * c + 8 * u + e for e in (0, 2, 4, 6, 1, 3, 5, 7)]
        elif what == "k":
            c, u = 2 * (m // 8) + m % 2, m // 2 % 4
            out += [32 * c + 8 * u + e for e in range(8)]
        elif hd == 128:
            out += [4 * m + e for e in range(4)] + [64 + 4 * m + e for e in range(4)]
        else:
            out += [8 * m + e for e in range(8)]
    return np.array(out)


def quantise(x, bits):
    """fp32 rows [..., hd] → codes (from 0 on) [..., hd], params [..., hd / 32] fp16."""
    half = 1 << (bits - 1)
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    bad = ~np.isfinite(g).all(-1)
    g = np.clip(np.where(np.isfinite(g), g, 0), -65504, 65504).astype(np.float64)
    lo, hi = g.min(-1), g.max(-1)
    mid = (((half - 1) * lo + half * hi) * (1.0 / (2 * half - 1))).astype(np.float32).astype(np.float16)
    need = np.maximum((hi - mid.astype(np.float64)) * (1.0 / (half - 1)), (mid.astype(np.float64) - lo) / half)
    step = need.astype(np.float32).astype(np.float16)
    step = np.where(step.astype(np.float64) < need, np.nextafter(step, np.float16(np.inf)), step).astype(np.float16)
    with np.errstate(divide="ignore"):
        inv = np.where(step > 0, 1.0 / step.astype(np.float64), 0.0)
    c = np.clip(np.rint((g - mid.astype(np.float64)[..., None]) * inv[..., None]), -half, half - 1).astype(np.int64) + half
    c[bad] = 0
    step[bad] = mid[bad] = np.float16(np.nan)
    return c.reshape(x.shape), np.concatenate([step, mid], -1)


def values(codes, params, bits, parts=False):
    """Rows of codes (from 0 on) and parameters, in 64 bits; parts: step * code and mid."""
    step, mid = np.split(params.astype(np.float64), 2, -1)
    c = (codes - (1 << (bits - 1))).reshape(*codes.shape[:-1], codes.shape[-1] // 64, 64).astype(np.float64)
    a, b = c * step[..., None], np.broadcast_to(mid[..., None], c.shape)
    a, b = a.reshape(codes.shape), b.reshape(codes.shape)
    return (a, b) if parts else a + b


def pack(codes, what, bits):
    c = codes[..., order(what, codes.shape[-1], bits)].astype(np.uint8)
    return c if bits == 8 else c[..., 0::2] | c[..., 1::2] << 4


def unpack(raw, what, hd, bits):
    c = raw if bits == 8 else np.stack([raw & 15, raw >> 4], -1).reshape(*raw.shape[:-1], hd)
    return c[..., np.argsort(order(what, hd, bits))].astype(np.int64)


def axes_of(half, axes, sections, interleaved):
    if not interleaved:
        return np.repeat(np.arange(axes), sections[:axes])
    out = np.zeros(half, np.int64)
    for a in range(1, axes):
        out[a::axes][:sections[a]] = a
    return out


def rotate(x, norm, eps, angle, adjacent):
    """One head's rows [n][hd], angles [n][pairs] or None → 64 bits, and the sizes of each element's pair."""
    y = x.astype(np.float64)
    if norm is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * norm.astype(np.float64)
    size = np.abs(y)
    if angle is not None:
        half = angle.shape[-1]
        a = np.arange(half) * 2 if adjacent else np.arange(half)
        b = a + 1 if adjacent else a + half
        ya, yb, c, s = y[..., a], y[..., b], np.cos(angle), np.sin(angle)
        y, size = y.copy(), size.copy()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
        size[..., a] = size[..., b] = np.abs(ya) + np.abs(yb)
    return y, size


def attention(q, k, v, seen, scale, cap=0.0, slope=None, dist=None):
    """One KV head: q [R][hd] fp32; k, v: (step * code, mid) pairs of [L][hd]; slope [R], dist [R][L]
    → out, lse and the bounds of their errors."""
    q = np.asarray(q, np.float64)
    used = seen.any(0)
    (ka, kb), (va, vb) = ((np.where(used[:, None], x, 0.0) for x in pair) for pair in (k, v))
    s = q @ (ka + kb).T * scale
    size = np.abs(ka) + np.abs(kb)
    err = np.abs(q) @ size.T * scale * (17 * U + 2.0 ** -21) + np.abs(s) * 4 * U
    err += scale * 2.0 ** -32 * np.abs(q).max(1)[:, None] * size.sum(1)
    if cap:
        s = cap * np.tanh(s / cap)
        err = err + np.abs(s) * 8 * U
    if slope is not None:
        s = s - slope[:, None] * dist
        err = err + slope[:, None] * np.abs(dist) * 2 * U + np.abs(s) * U
    s = np.where(seen, s, -np.inf)
    m = s.max(1, keepdims=True) if s.shape[1] else np.full((s.shape[0], 1), -np.inf)
    m0 = np.where(np.isfinite(m), m, 0.0)
    e = np.exp(s - m0)
    total = e.sum(1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    with np.errstate(divide="ignore"):
        lse = np.where(total[:, 0] == 0, -np.inf, m0[:, 0] + np.log(total[:, 0]))
    steps = (seen.sum(1) / 16 + 32) * U
    d = np.where(seen, err + np.abs(np.where(seen, s, 0.0) - m0) * 2 * U + 2 * U, 0.0)
    rows = (p * d).sum(1) + steps
    lse_err = rows + np.abs(np.where(np.isfinite(lse), lse, 0.0)) * 2 * U + 2 * U
    size = np.abs(va) + np.abs(vb)
    out_err = (p * (d + rows[:, None])) @ size + (p @ size) * (2.0 ** -21 + steps[:, None] + 2 * U) + 1e-38
    out_err += (np.where(seen, size.max(1), 0.0).max(1, initial=0.0) * seen.sum(1))[:, None] * 2.0 ** -32
    return p @ (va + vb), lse, out_err, lse_err
