"""The 8-bit page pool from its definition, in numpy (64 bits unless a value is f32 by
definition): quantiser, pool layout, kernel (1)'s norm and rotation, attention."""
from __future__ import annotations

import numpy as np

D, PAGE, TILE = 128, 16, 4224
INT8, E4M3 = 0, 1
F32, F16, BF16 = 0, 1, 30
TINY = np.float32(2.0 ** -126)


def e4m3_values() -> np.ndarray:
    """The 256 values of an e4m3 byte (S.1111.111 is NaN, no infinities)."""
    b = np.arange(256)
    e, f = (b >> 3) & 15, b & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8.0 + f) * 2.0 ** (e - 10.0))
    v[(e == 15) & (f == 7)] = np.nan
    return np.where(b >> 7, -v, v)


E4M3_VALUES = e4m3_values()
_POS = E4M3_VALUES[:127]           # 0 .. 448, ascending


def _e4m3_bytes(y: np.ndarray) -> np.ndarray:
    """|y| <= 448 rounded to e4m3, ties to the even byte."""
    a = np.abs(y)
    hi = np.clip(np.searchsorted(_POS, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    b = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    b = np.where(a == _POS[hi], hi, b)
    return (b + np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def quantise(x: np.ndarray, fmt: int):
    """(bytes uint8, scales f32) of x [..., 128] (f32 values)."""
    x = np.asarray(x, np.float64)
    amax = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    amax = np.where(bad, 0.0, amax)
    if fmt == INT8:
        d = np.maximum((amax / 127).astype(np.float32), TINY)
        q = np.rint(x / d.astype(np.float64)[..., None]).astype(np.int8).view(np.uint8)
    else:
        m, e = np.frexp(amax)
        k = np.maximum(np.where(m > 0.875, e - 8, e - 9), -126)
        d = np.ldexp(1.0, np.where(amax > 0, k, -126)).astype(np.float32)
        q = _e4m3_bytes(x / d.astype(np.float64)[..., None])
        q = np.where(bad[..., None], 0, q).astype(np.uint8)
    return q, np.where(bad, np.float32(np.nan), d).astype(np.float32)


def values(raw: np.ndarray, fmt: int) -> np.ndarray:
    return raw.view(np.int8).astype(np.float64) if fmt == INT8 else E4M3_VALUES[raw]


def parts(pool: np.ndarray):
    """Views of a pool [..., 4224] uint8: bytes [..., K|V, 16, 128], scales [..., K|V, 16] f32."""
    raw = pool[..., : 2 * PAGE * D].reshape(*pool.shape[:-1], 2, PAGE, D)
    assert np.shares_memory(raw, pool)
    return raw, pool[..., 2 * PAGE * D:].view(np.float32).reshape(*pool.shape[:-1], 2, PAGE)


def write(pool, bt, slot, pos, k, v, fmt):
    """k, v [M][layers][kv heads][128] into pool [layers][pages][kv heads][4224], in place."""
    for m in range(len(slot)):
        if pos[m] < 0:
            continue
        tile = pool[:, bt[slot[m], pos[m] // PAGE]]                       # [layers][heads][4224], a view
        t = pos[m] % PAGE
        for part, x in ((0, k), (1, v)):
            q, d = quantise(x[m], fmt)
            at = (part * PAGE + t) * D
            tile[:, :, at:at + D] = q
            at = 2 * PAGE * D + (part * PAGE + t) * 4
            tile[:, :, at:at + 4] = np.ascontiguousarray(d)[..., None].view(np.uint8).reshape(*d.shape, 4)


def read(pool, bt_row, t0, t1, fmt):
    """K, V [layers][kv heads][t1 - t0][128] in 64 bits of one sequence's tokens."""
    raw, scales = parts(pool)
    t = np.arange(t0, t1)
    page = bt_row[t // PAGE]
    out = []
    for part in (0, 1):
        x = values(raw[:, page, :, part, t % PAGE], fmt)                  # [tokens][layers][heads][128]
        d = scales[:, page, :, part, t % PAGE].astype(np.float64)
        out.append(np.moveaxis(x * d[..., None], 0, 2))
    return out


def norm_rotate(x, w, rot, eps=np.float32(1e-5)):
    """Kernel (1) on head vectors x [M][heads][128] f32: the sum of squares in double, all
    else single f32 operations in the kernel's order. rot [M][64][2]."""
    ss = (x * x).astype(np.float64).sum(-1)
    mean = (ss / D).astype(np.float32)
    scale = np.float32(1.0) / np.sqrt(mean + np.float32(eps))
    y = (x * scale[..., None]) * w
    a, b = y[..., :64], y[..., 64:]
    c, s = rot[:, None, :, 0], rot[:, None, :, 1]
    return np.concatenate([a * c - b * s, a * s + b * c], -1).astype(np.float32)


def norm_rotate_exact(x, w, rot, eps=np.float32(1e-5)):
    """norm_rotate in 64 bits (x, w, rot and eps are f32 values)."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(eps)) * w.astype(np.float64)
    a, b = y[..., :64], y[..., 64:]
    c, s = rot[:, None, :, 0].astype(np.float64), rot[:, None, :, 1].astype(np.float64)
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def attention(q, k, v):
    """q [Hq][128], k and v [Hkv][n][128]: softmax(q k) v in 64 bits, [Hq][128]."""
    q = np.asarray(q, np.float64)
    g = len(q) // len(k)
    out = np.zeros((len(q), D))
    for h in range(len(q)):
        s = k[h // g] @ q[h]
        p = np.exp(s - s.max())
        out[h] = (p / p.sum()) @ v[h // g]
    return out
