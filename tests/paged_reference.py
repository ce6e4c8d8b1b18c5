"""The paged cache operators in 64 bits, from their definitions (include/neko_cuda.h), one value after the other as
far as numpy allows. Pages are float64 arrays [pages][kv heads][page][hd] of values (codes times nothing)."""
import math

import numpy as np

SCALE_MIN_EXP = -100


def e4m3_table():
    """The 256 codes' values: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7F and 0xFF are NaN."""
    out = np.zeros(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = math.nan if c & 0x7F == 0x7F else -v if c & 0x80 else v
    return out


E4M3 = e4m3_table()


def e4m3_round(x):
    """To the nearest code's value, ties to even mantissa, beyond 448 (infinities too) to +-448; NaN stays."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), 448.0)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    return np.where(np.isnan(x), np.nan, np.copysign(np.minimum(np.rint(a / step) * step, 448.0), x))


def block_scale(x):
    """The smallest power of two, at least 2^-100, that brings the finite magnitudes to 448 or less."""
    a = np.abs(x[np.isfinite(x)])
    most = a.max() if a.size else 0.0
    e = SCALE_MIN_EXP
    while most > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def turn(x, pos, cs, interleaved, gain, eps):
    """x [heads][hd] of one token."""
    x = np.array(x, np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gain, np.float64)
    if cs is not None:
        half = cs.shape[1]
        y = x.copy()
        for j in range(half):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
            c, s = float(cs[pos, j, 0]), float(cs[pos, j, 1])
            y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
        x = y
    return x


def append(k, v, k_pages, v_pages, table, start, q_start, k_scale=None, v_scale=None, q=None, cs=None,
           interleaved=False, q_gain=None, k_gain=None, eps=1e-6):
    """In place on the pages (values of codes for an 8-bit cache) and scales; returns the turned q."""
    pages, n_kv, ps, hd = k_pages.shape
    out = None if q is None else np.zeros(q.shape)
    for s in range(len(start)):
        a, b = q_start[s], q_start[s + 1]
        if start[s] < 0:
            continue
        fresh = {"k": [], "v": []}
        for i in range(a, b):
            pos = start[s] + i - a
            inside = cs is None or pos < cs.shape[0]
            if q is not None:
                out[i] = turn(q[i], pos, cs if inside else None, interleaved, q_gain, eps)
            if inside:
                fresh["k"].append(turn(k[i], pos, cs, interleaved, k_gain, eps))
                fresh["v"].append(np.array(v[i], np.float64))
        count = len(fresh["k"])
        at = 0
        while at < count:
            pos = start[s] + at
            n = min(count - at, ps - pos % ps)
            slot, o = pos // ps, pos % ps
            p = table[s][slot] if slot < table.shape[1] else -1
            if 0 <= p < pages:
                for name, pool, scale in (("k", k_pages, k_scale), ("v", v_pages, v_scale)):
                    for h in range(n_kv):
                        new = np.stack([x[h] for x in fresh[name][at:at + n]])
                        if scale is None:
                            pool[p, h, o:o + n] = new
                            continue
                        sc = block_scale(new)
                        if o:
                            sc = max(sc, scale[p, h])
                            pool[p, h, :o] = e4m3_round(pool[p, h, :o] * (scale[p, h] / sc))
                        scale[p, h] = sc
                        pool[p, h, o:o + n] = e4m3_round(new / sc)
            at += n
    return out


def attention(q, k_pages, v_pages, table, kv_len, q_start, scale, softcap=0.0, window=0, slopes=None, prefix=None):
    """Pages of values (an 8-bit cache's codes times their scales). Unseen keys and values are never touched."""
    pages, n_kv, ps, hd = k_pages.shape
    heads = q.shape[1]
    out = np.zeros(q.shape)
    for s in range(len(kv_len)):
        a, b = q_start[s], q_start[s + 1]
        pre = prefix[s] if prefix is not None else 0
        for i in range(a, b):
            pos = kv_len[s] - (b - a) + i - a
            keys = []
            for j in range(max(kv_len[s], 0)):
                if (j <= pos and (not window or pos - j < window)) or j < pre:
                    p = table[s][j // ps] if j // ps < table.shape[1] else -1
                    if 0 <= p < pages:
                        keys.append((j, p, j % ps))
            if not keys:
                continue
            js, ps_, os_ = (np.array(x) for x in zip(*keys))
            for h in range(heads):
                kk, vv = k_pages[ps_, h // (heads // n_kv), os_], v_pages[ps_, h // (heads // n_kv), os_]
                z = kk @ q[i, h] * scale
                if softcap:
                    z = softcap * np.tanh(z / softcap)
                if slopes is not None:
                    z = z + float(slopes[h]) * (js - pos)
                w = np.exp(z - z.max())
                out[i, h] = w @ vv / w.sum()
    return out
