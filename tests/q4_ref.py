"""The 4-bit cache's format and softmax attention in 64 bits, in plain numpy: what
tests/test_q4_cache.py and tests/test_packed.py compare the library with."""
from __future__ import annotations

import numpy as np

Q4_MAX = 65280.0


def quantise(x: np.ndarray):
    """(codes [rows, blocks, 32], s, z [rows, blocks] float16) of float32 rows. The
    arithmetic of s and of the quotient is 32-bit by definition."""
    x = np.where(np.isnan(x), np.float32(0), x).astype(np.float32)
    b = np.clip(x, np.float32(-Q4_MAX), np.float32(Q4_MAX)).reshape(x.shape[0], -1, 32)
    lo, hi = b.min(-1), b.max(-1)
    s, z = ((hi - lo) * (np.float32(1) / np.float32(15))).astype(np.float16), lo.astype(np.float16)
    sf, zf = s.astype(np.float32)[..., None], z.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(sf > 0, np.rint((b - zf) / sf), 0)
    return np.clip(c, 0, 15).astype(np.uint8), s, z


def values(q) -> np.ndarray:
    """What the codes stand for, float64 (one rounding to float16)."""
    c, s, z = q
    v = c.astype(np.float64) * s.astype(np.float64)[..., None] + z.astype(np.float64)[..., None]
    return v.astype(np.float16).astype(np.float64).reshape(c.shape[0], -1)


def raw(q) -> np.ndarray:
    """The interchange rows: per block s, z, then elements i and i + 16 in byte i."""
    c, s, z = q
    sz = np.stack([s, z], -1).view(np.uint8).reshape(*s.shape, 4)
    return np.concatenate([sz, c[..., :16] | (c[..., 16:] << 4)], -1).reshape(c.shape[0], -1)


def span(causal: bool, window: int, pos: int, n_seq: int):
    if causal:
        return (max(0, pos + 1 - window) if window > 0 else 0), min(pos, n_seq - 1)
    if window > 0:
        return max(0, pos - window // 2), min(n_seq - 1, pos + window // 2)
    return 0, n_seq - 1


def attend(q, k, v, *, pos0, n_seq, window, causal, n_head, n_kv, head_dim, scale):
    """(out, bound, mean |V|) of q [n_tok, n_head * head_dim] over the keys of positions 0 ..
    n_seq - 1, float64. bound: how far an output computed with fp32 sums and
    operands of 22 significant bits may be off. A score's products sum to at most
    A = scale max_k sum |q k|; their sum has the operands' roundings (2^-23 each)
    and a rounding of 2^-24 per partial sum, of which the matrix cores make two
    per 32 products: (head_dim / 16 + 8) 2^-24 A covers both. A weight moves by
    that and by its exponential's and its own split's few 2^-24 (2^-21 in all), an
    output by twice its weights' relative error times the largest |V|."""
    n_tok, g = q.shape[0], n_head // n_kv
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, bound, spread = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    for t in range(n_tok):
        first, last = span(causal, window, pos0 + t, n_seq)
        if last < first:
            continue
        for h in range(n_head):
            at, kv = slice(h * head_dim, (h + 1) * head_dim), slice(h // g * head_dim, (h // g + 1) * head_dim)
            kk, vv = k[first:last + 1, kv], v[first:last + 1, kv]
            with np.errstate(invalid="ignore", over="ignore"):
                s = kk @ q[t, at] * scale
                w = np.exp(s - s.max())
                out[t, at] = w @ vv / w.sum()
                spread[t, at] = w @ np.abs(vv) / w.sum()
                a = (np.abs(kk) @ np.abs(q[t, at])).max() * abs(scale)
                bound[t, at] = 2 * np.abs(vv).max() * (a * (head_dim / 16 + 8) * 2.0**-24 + 2.0**-21)
    return out, bound, spread
