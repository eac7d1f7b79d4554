"""8-bit paged KV oracle (numpy, 64 bits).  TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).

The reference's pool is 16-bit (core/pool.py:20-71); this restates the 8-bit format of
``unifiedkv_b200/kv_quant.py`` from its definition: a row is e4m3 codes and one
power-of-two scale, value = code * 2^(byte - 127).
"""
from __future__ import annotations

import numpy as np

_ALL = np.arange(256)
_FIELD, _FRAC = (_ALL >> 3) & 15, _ALL & 7
#: value of each e4m3 code (0x7f and 0xff are NaN)
E4M3 = np.where(_FIELD == 0, _FRAC * 2.0 ** -9, (8 + _FRAC) * 2.0 ** (_FIELD - 10.0))
E4M3 = np.where(_ALL >= 128, -E4M3, E4M3)
E4M3[[0x7F, 0xFF]] = np.nan


def quantise(x):
    """rows [..., d] -> (codes uint8 [..., d], scale bytes uint8 [...])."""
    x = np.asarray(x, np.float64)
    amax = np.abs(x).max(-1)
    finite = np.isfinite(amax)
    e = np.full(amax.shape, -127)
    for k in range(-127, 120):  # the smallest e in [-127, 119] with amax <= 448 * 2^e, else 119
        e = np.where((e == k) & (amax > 448.0 * 2.0 ** k) & (k < 119), k + 1, e)
    y = np.clip(np.where(finite[..., None], x, 0.0) / 2.0 ** e[..., None], -448.0, 448.0)
    _, octave = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
    step = 2.0 ** (octave - 4.0)
    v = np.rint(np.abs(y) / step) * step  # rint: halves to even
    _, octave = np.frexp(np.maximum(v, 2.0 ** -6))
    sub = v < 2.0 ** -6
    codes = np.where(sub, v * 512, (octave + 6) * 8 + v * 2.0 ** (4.0 - octave) - 8).astype(np.int64)
    codes = np.where(np.signbit(y), codes | 128, codes)
    codes = np.where(finite[..., None], codes, 0x7F)
    return codes.astype(np.uint8), np.where(finite, e + 127, 255).astype(np.uint8)


def dequantise(codes, scales):
    """codes uint8 [..., d], scale bytes [...] -> values."""
    return E4M3[codes] * 2.0 ** (scales.astype(np.float64) - 127)[..., None]


def request_rows(codes, scales, table_row, n):
    """Values [n, h_kv, d] of a request's first n tokens; NaN rows where its table has no page of the pool."""
    out = np.full((n,) + codes.shape[2:], np.nan)
    there = np.zeros(n, bool)
    for j in range(-(-n // 16)):
        page = int(table_row[j]) if j < len(table_row) else -1
        if not 0 <= page < codes.shape[0]:
            continue
        m = min(16, n - 16 * j)
        out[16 * j:16 * j + m] = dequantise(codes[page, :m], scales[page].T[:m])
        there[16 * j:16 * j + m] = True
    return out, there


def attention(q, k, v, there, n_new, scale, causal=True):
    """q [n_new, h_q, d]; k, v [n, h_kv, d]; there [n].  -> out, lse, and per output the weighted mean of |v|
    and the largest sum |q_i k_i| scale of the row: what error bounds are made of."""
    n_q, h_q, d = q.shape
    n, h_kv = k.shape[:2]
    rep = h_q // h_kv
    out, mean_abs = np.zeros((n_q, h_q, d)), np.zeros((n_q, h_q, d))
    lse, size = np.full((n_q, h_q), -np.inf), np.zeros((n_q, h_q))
    for i in range(n_q):
        see = there & (np.arange(n) <= (n - n_new + i if causal else n - 1))
        if not see.any():
            continue
        for h in range(h_q):
            kk, vv = k[see, h // rep], v[see, h // rep]
            s = kk @ q[i, h] * scale
            m = s.max()
            p = np.exp(s - m)
            l = p.sum()
            out[i, h] = p @ vv / l
            mean_abs[i, h] = p @ np.abs(vv) / l
            lse[i, h] = m + np.log(l)
            size[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * scale
    return out, lse, mean_abs, size
