"""Trees of drafted tokens, sampling and moving tokens, from their definitions (include/neko_cuda.h), in 64 bits or whole numbers,
one after the other as far as numpy allows."""
import numpy as np

from tests import paged_reference as ref


def lines(parent):
    """For each node of a tree, the nodes from itself up to its root."""
    out = []
    for i, p in enumerate(parent):
        out.append([i] + (out[p] if 0 <= p < i else []))
    return out


def masks(parents, words):
    """parents: a list for each sequence. Masks uint64 [nodes][words] and depths."""
    m, d = [], []
    for parent in parents:
        for line in lines(parent):
            bits = sum(1 << j for j in line)
            m.append([bits >> 64 * w & (1 << 64) - 1 for w in range(words)])
            d.append(len(line) - 1)
    return np.array(m, np.uint64).reshape(-1, words), np.array(d, np.int32)


def accept(chosen, draft, parent):
    """Of one sequence: the nodes walked through and the token chosen at the last."""
    if not len(parent):
        return [], -1
    walk = [0]
    while True:
        nxt = [i for i in range(walk[-1] + 1, len(parent)) if parent[i] == walk[-1] and draft[i] == chosen[walk[-1]]]
        if not nxt:
            return walk, chosen[walk[-1]]
        walk.append(nxt[0])


def sees(mask, depth, q_start, kv_len, n_keys, window=0):
    """Which keys a sequence's nodes see [n][n_keys], and their distance pos_q - pos_k."""
    a, b = q_start
    n, base = b - a, kv_len - (b - a)
    j = np.arange(n_keys)
    bit = np.zeros((n, n_keys), bool)
    where = j.copy()
    for t in range(n):
        if 0 <= base + t < n_keys:
            bit[:, base + t] = [int(mask[a + i, t >> 6]) >> (t & 63) & 1 for i in range(n)]
            where[base + t] = base + depth[a + t]
    gap = (base + depth[a:b])[:, None] - where[None]
    see = ((j < base)[None] | bit) & (j < kv_len)[None]
    return (see & (gap < window) if window else see), gap


def compact(pool, scale, table, start, path, count):
    """In place on pool [planes][pages][heads][page][hd] (values of codes for an 8-bit cache) and scale."""
    planes, pages, heads, ps, hd = pool.shape
    old, old_scale = pool.copy(), None if scale is None else scale.copy()
    at = lambda s, pos: table[s][pos // ps] if 0 <= pos // ps < table.shape[1] and 0 <= table[s][pos // ps] < pages else -1  # noqa: E731
    for s, n in enumerate(count):
        if start[s] < 0:
            continue
        into = {}
        for k in range(n):
            p, src = at(s, start[s] + k), start[s] + int(path[s][k])
            if p >= 0 and at(s, src) >= 0:
                into.setdefault((start[s] + k) // ps, []).append((k, src))
        for slot, moves in into.items():
            p = table[s][slot]
            stay = start[s] % ps if slot == start[s] // ps else 0
            if scale is not None:
                new = np.max([old_scale[:, at(s, src)] for _, src in moves] + ([old_scale[:, p]] if stay else []), axis=0)  # [planes][heads]
                scale[:, p] = new
                pool[:, p, :, :stay] = ref.e4m3_round(old[:, p, :, :stay] * (old_scale[:, p] / new)[..., None, None])
            for k, src in moves:
                v = old[:, at(s, src), :, src % ps]
                pool[:, p, :, (start[s] + k) % ps] = v if scale is None else ref.e4m3_round(v * (old_scale[:, at(s, src)] / new)[..., None])


def sample(x, u, temperature, top_k, top_p, min_p, held=True):
    """One row of float logits. held: weights as the operator holds them, whole numbers of 2^-44 of the largest; else in extended
    precision as they are. Returns the token and its probability."""
    x = np.asarray(x, np.float64)
    ids = np.flatnonzero(x > -np.inf)
    if not len(ids):
        return -1, 0.0
    best = x[ids].max()
    if not temperature > 0:
        return int(ids[x[ids] == best][0]), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x[ids] == best, 1.0, np.exp(-(best - x[ids]) / np.float64(np.float32(temperature))))
    plain = w.copy()
    down = np.argsort(-x[ids], kind="stable")
    one = 1 << 44 if held else 1
    w = np.rint(w * 2.0 ** 44).astype(np.int64) if held else w.astype(np.longdouble)
    if top_k > 0:
        down = down[:top_k]
    p = np.float64(np.float32(top_p))
    if p < 1:
        mass = np.cumsum(w[down])
        total = mass[-1]
        down = down[:max(1, int(np.searchsorted(mass.astype(np.float64) if held else mass, p * (float(total) if held else total))) + 1)]
    down = np.sort(down[plain[down] >= min(np.float64(np.float32(min_p)), 1.0)])
    mass = np.cumsum(w[down])
    at = int(np.searchsorted(mass, np.floor(u * float(mass[-1])) if held else np.longdouble(u) * mass[-1], side="right"))
    at = down[min(at, len(down) - 1)]
    return int(ids[at]), float(plain[at] * one / float(mass[-1]))
