"""Operators behind drafted tokens and sampling against their definitions (drafts_reference.py): trees over the paged cache, rows'
sampling, masks and walks, moving tokens and pages, and all of them together.

Whole numbers are equal. Attention: the bound of test_gpu_cache_edges (scores 2^-20 of their reach, weights 2^-18 or f16's 2^-11,
the output's rounding). Probabilities: sums and exponentials in 64 bits, weights to 2^-45 of the largest, one rounding to f32: 2^-23."""
import math

import numpy as np
import pytest

from tests import drafts_reference as want_of
from tests import paged_reference as ref
from tests.test_gpu_cache_edges import bound, ints, quantize
from tests.test_gpu_paged import Cache, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


# ------------------------------------------------------------------------------------------------ trees over the cache
def some_trees(rng, new):
    """Parents of each sequence's nodes: chains with branches, some more roots."""
    out = []
    for n in new:
        out.append([-1 if i == 0 or rng.random() < 0.05 else i - 1 if rng.random() < 0.5 else int(rng.integers(0, i)) for i in range(n)])
    return out


def exact(torch, cache, q, lens, new, mask, depth, scale, softcap, window, slopes):
    """The definition in 64 bits; mass and reach as in test_gpu_cache_edges, and what the weights' f16 cannot hold: a weight times its
    value's scale is off by up to 2^-32 of the row's largest such product (at most the largest scale seen), in units of the
    value's scale, so a sum of codes c_j by up to 2^-32 max scale sum |c_j| (f16 pages: scales of 1)."""
    pages, n_kv, ps, hd = cache.k.shape
    k, v = (torch.from_numpy(x).cuda() for x in cache.values())
    code = torch.from_numpy(cache.values(scaled=False)[1]).cuda()
    table = cache.table
    out, mass, lost = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(3))
    reach = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    G, at = q.shape[1] // n_kv, starts(new)
    for s, (L, n) in enumerate(zip(lens, new)):
        L_ = min(L, table.shape[1] * ps)
        if not n or L_ <= 0:
            continue
        see, gap = want_of.sees(mask, depth, (at[s], at[s + 1]), L, L_, window)
        t = table[s, :-(-L_ // ps)]
        see &= np.repeat((t >= 0) & (t < pages), ps)[None, :L_]
        see, gap = torch.from_numpy(see).cuda(), torch.from_numpy(gap).cuda().double()
        pick = torch.from_numpy(np.clip(t, 0, pages - 1)).long().cuda()
        rows = slice(at[s], at[s + 1])
        for h in range(q.shape[1]):
            kk, vv, cc = (torch.where(see.any(0)[:, None], x[pick, h // G].reshape(-1, hd)[:L_], 0.0) for x in (k, v, code))
            sc = cache.vs[pick, h // G].double().repeat_interleave(ps)[:L_] if cache.e4m3 else torch.ones(L_, device="cuda", dtype=torch.float64)
            most = torch.where(see, sc, 0).amax(1)
            lost[rows, h] = 2.0 ** -32 * most[:, None] * (see.double() @ cc.abs())
            qq = q[rows, h].double()
            z = qq @ kk.T * scale
            reach[rows, h] = torch.where(see, qq.abs() @ kk.abs().T * abs(scale), 0).amax(1)
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            if slopes is not None:
                z = z - slopes[h].double() * gap
            p = torch.softmax(torch.where(see, z, -torch.inf), 1).nan_to_num(0.0)
            out[rows, h], mass[rows, h] = p @ vv, p @ vv.abs()
    return out, mass, reach, lost


def tree_call(torch, cache, lens, new, heads, dtype, seed, mask=None, depth=None, softcap=0.0, window=0, alibi=False, max_new=None,
              strided=False):
    """One call on random queries, every value within its bound."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(seed)
    hd, T = cache.k.shape[3], int(sum(new))
    words = (max(max(new), 1) + 63) // 64
    if mask is None:
        mask, depth = want_of.masks(some_trees(rng, new), words)
    wide = torch.from_numpy(rng.standard_normal((T, heads + 3, hd + 8)).astype(np.float32)).to(getattr(torch, dtype)).cuda()
    q = wide[:, 1:1 + heads, 4:4 + hd] if strided else wide[:, :heads, :hd].contiguous()
    out = torch.full((T + 2, heads + 1, hd + 4), 7.0, dtype=q.dtype, device="cuda")
    slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if alibi else None
    got = ops.paged_tree_attention(q, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, *lens),
                                   torch.from_numpy(mask.view(np.int64)).cuda(), torch.from_numpy(depth).cuda(), k_scale=cache.ks,
                                   v_scale=cache.vs, q_start=ints(torch, *starts(new).tolist()), max_new=max_new or max(new),
                                   softcap=softcap, window=window, slopes=slopes, out=out[:T, :heads, :hd])
    ops.status()
    assert (out[T:] == 7).all() and (out[:, heads:] == 7).all() and (out[:, :, hd:] == 7).all()
    want, mass, reach, lost = exact(torch, cache, q, lens, new, mask, depth, hd ** -0.5, softcap, window, slopes)
    off = (got.double() - want).abs()
    far = ~(off <= bound(dtype, want, mass, reach, softcap) + lost)
    assert not far.any(), f"{int(far.sum())} of {far.numel()}, worst {off[far].max().item():.3g}, first {far.nonzero()[0].tolist()}"
    return got, want


SHAPES = [([1], [1]), ([1], [700]), ([12], [789]), ([3, 8, 5, 1], [40, 300, 5, 17]), ([0, 4, 0, 2], [9, 4, 0, 1000]),
          ([63, 21, 64], [63, 500, 330]), ([65, 130, 7], [65, 700, 2050]), ([200], [5000])]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,ps", [(128, 16, 8, 16), (64, 9, 3, 32), (32, 4, 4, 16), (128, 8, 1, 128)])
@pytest.mark.parametrize("new,lens", SHAPES)
def test_trees(torch, new, lens, hd, heads, n_kv, ps, e4m3, dtype):
    rng = np.random.default_rng(1)
    cache = Cache(torch, rng, lens, n_kv, ps, hd, e4m3)
    cache.fill(rng, lens)
    tree_call(torch, cache, lens, new, heads, dtype, 2)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,lens", [([5, 9], [60, 300]), ([40, 70], [90, 1200]), ([130], [130])])
@pytest.mark.parametrize("opts", [dict(softcap=30.0), dict(window=1), dict(window=3), dict(window=100), dict(alibi=True),
                                  dict(alibi=True, window=40, softcap=20.0), dict(window=1 << 30, alibi=True)])
def test_tree_masks_and_biases(torch, opts, new, lens, e4m3, dtype):
    """Windows and biases go by depth, of keys too."""
    rng = np.random.default_rng(3)
    for hd in (64, 128):
        cache = Cache(torch, rng, lens, 2, 16, hd, e4m3)
        cache.fill(rng, lens)
        tree_call(torch, cache, lens, new, 8, dtype, 4, strided=True, **opts)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("new,lens", [([7, 6], [7, 50]), ([90, 70], [90, 300])])
def test_masks_that_are_no_trees(torch, new, lens, dtype):
    """Any bits: nodes that see later ones, rows that see none of them and, without keys before the tree, nothing at all; bits past
    the nodes that there are say nothing."""
    rng = np.random.default_rng(5)
    cache = Cache(torch, rng, lens, 2, 16, 128, False)
    cache.fill(rng, lens)
    T, words = sum(new), (max(new) + 63) // 64 + 1
    mask = rng.integers(0, 1 << 63, (T, words), dtype=np.uint64) | rng.integers(0, 2, (T, words), dtype=np.uint64) << np.uint64(63)
    mask[2], mask[new[0] + 3], mask[4] = 0, 0, np.uint64((1 << 64) - 1)
    got, want = tree_call(torch, cache, lens, new, 8, dtype, 6, mask=mask, depth=np.zeros(T, np.int32))
    assert (got[2] == 0).all() and (got[new[0] + 3] != 0).any()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,lens", [([6], [40]), ([80], [400])])
def test_nodes_that_are_not_seen_have_no_effect(torch, new, lens, dtype, e4m3):
    """Keys and values that are not numbers at nodes that a row does not see; those that see them get NaN. Pages that are not
    resident, in the tree as before it."""
    rng = np.random.default_rng(7)
    n, L = new[0], lens[0]
    cache = Cache(torch, rng, lens, 2, 16, 128, e4m3)
    cache.fill(rng, lens)
    parents = [[-1, 0, 0, 1, 2] + [int(rng.integers(0, 3)) for _ in range(n - 5)]]
    mask, depth = want_of.masks(parents, (n + 63) // 64)
    nan = 0x7F if e4m3 else float("nan")
    p = int(cache.table[0, (L - n + 2) // 16])
    cache.v[p, 1, (L - n + 2) % 16, 9] = nan
    cache.k[p, 0, (L - n + 2) % 16, 5] = nan
    sees_it = torch.from_numpy(mask[:, 0] >> np.uint64(2) & np.uint64(1)).cuda().bool()
    from nekochat_b200 import ops
    q = torch.randn((n, 4, 128), device="cuda", dtype=getattr(torch, dtype))
    got = ops.paged_tree_attention(q, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, L),
                                   torch.from_numpy(mask.view(np.int64)).cuda(), torch.from_numpy(depth).cuda(), k_scale=cache.ks,
                                   v_scale=cache.vs, q_start=ints(torch, 0, n), max_new=n)
    assert torch.equal(got[:, :2].isnan().all(-1).all(-1), sees_it) and torch.equal(got[:, 2:, 9].isnan().all(-1), sees_it)
    assert torch.isfinite(got[~sees_it]).all() and torch.isfinite(got[:, 2:, 10:]).all()
    cache.v[p, 1, (L - n + 2) % 16, 9] = 0
    cache.k[p, 0, (L - n + 2) % 16, 5] = 0
    cache.table[0, (L - n // 2) // 16] = -1
    cache.table[0, 0] = 10 ** 6
    tree_call(torch, cache, lens, new, 4, dtype, 8, mask=mask, depth=depth)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n,ctx", [(6, 50), (40, 300)])
def test_a_node_sees_what_its_line_alone_would(torch, n, ctx, e4m3):
    """Append with depths, then tree attention: each node's row is the last row of its line appended and attended as plain tokens
    (8-bit pages: scales go by all tokens of a page, so codes of 4 bits are off by a step)."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(9)
    hd, heads, n_kv = 128, 8, 2
    parent = some_trees(rng, [n])[0]
    parent[:1] = [-1]
    q, k, v = (torch.from_numpy(rng.standard_normal((ctx + n, h, hd)).astype(np.float32)).cuda() for h in (heads, n_kv, n_kv))
    cs, gain = ops.rope_table(600, hd, 1e4), torch.rand(hd, device="cuda") + 0.5
    put = dict(cs=cs, q_gain=gain, k_gain=gain)

    def cached(rows, L):
        c = Cache(torch, np.random.default_rng(1), [L], n_kv, 16, hd, e4m3)
        t = torch.from_numpy(c.table).cuda()
        sc = dict(k_scale=c.ks, v_scale=c.vs)
        ops.paged_append(k[:ctx], v[:ctx], c.k, c.v, t, ints(torch, 0), q=q[:ctx], q_start=ints(torch, 0, ctx), max_new=ctx, **put, **sc)
        return c, t, sc

    mask, depth = ops.tree_masks(ints(torch, *parent), ints(torch, 0, n), n)
    c, t, sc = cached(range(n), ctx + n)
    nodes = dict(q_start=ints(torch, 0, n), max_new=n, **sc)
    turned = ops.paged_append(k[ctx:], v[ctx:], c.k, c.v, t, ints(torch, ctx), q=q[ctx:], depth=depth, **put, **nodes)
    got = ops.paged_tree_attention(turned, c.k, c.v, t, ints(torch, ctx + n), mask, depth, **nodes)
    for i in range(0, n, max(1, n // 12)):
        line = [ctx + j for j in reversed(want_of.lines(parent)[i])]
        m = len(line)
        c, t, sc = cached(line, ctx + m)
        args = dict(q_start=ints(torch, 0, m), max_new=m, **sc)
        rows = ops.paged_append(k[line], v[line], c.k, c.v, t, ints(torch, ctx), q=q[line], **put, **args)
        want = ops.paged_attention(rows, c.k, c.v, t, ints(torch, ctx + m), **args)[-1]
        # f16 pages: the same numbers in another order of sums, 2^-18 of the largest value twice; 8-bit: 2^-4 of what they hold
        tol = 6.0 * (2.0 ** -3 if e4m3 else 2.0 ** -17)
        assert (got[i] - want).abs().max() <= tol, i
        if not e4m3:
            assert (turned[i] - rows[-1]).abs().max() <= 2e-6 * rows[-1].abs().max()
    ops.status()


# ------------------------------------------------------------------------------------------------ masks and walks
@pytest.mark.parametrize("new,spare", [([1], 0), ([12], 0), ([0, 5, 0, 64, 65, 1], 3), ([200, 3, 129], 0), ([4096], 1), ([17] * 300, 0)])
def test_masks_and_walks(torch, new, spare):
    from nekochat_b200 import ops
    rng = np.random.default_rng(10)
    parents = some_trees(rng, new) if new != [4096] else [list(range(-1, 4095))]
    flat = [p for x in parents for p in x] + [0] * spare
    for i in range(len(flat)):
        if flat[i] < 0 and i % 3 == 0:
            flat[i] = 9999  # no earlier node: a root too
    at, n = starts(new).tolist(), max(new)
    mask, depth = ops.tree_masks(ints(torch, *flat), ints(torch, *at), n)
    m, d = want_of.masks(parents, (n + 63) // 64)
    T = at[-1]
    assert np.array_equal(mask[:T].cpu().numpy().view(np.uint64), m) and np.array_equal(depth[:T].cpu().numpy(), d)
    assert not mask[T:].any() and not depth[T:].any()
    draft = rng.integers(0, 3, len(flat))
    chosen = rng.integers(0, 3, len(flat))
    path, count, token = (x.cpu().numpy() for x in ops.tree_accept(ints(torch, *chosen), ints(torch, *draft), ints(torch, *flat), ints(torch, *at), n))
    for s, parent in enumerate(parents):
        walk, t = want_of.accept(chosen[at[s]:at[s + 1]], draft[at[s]:at[s + 1]], flat[at[s]:at[s + 1]])
        assert count[s] == len(walk) and token[s] == t and path[s].tolist() == walk + [0] * (n - len(walk))
    ops.status()


def test_trees_left_out_are_reported(torch):
    """More nodes than max_new, and rows that are not there: the sequence is left out, the others are not."""
    from nekochat_b200 import NekoError, ops
    parent = ints(torch, -1, 0, 1, -1, 0)
    path, count, token = ops.tree_accept(ints(torch, 5, 6, 7, 8, 9), ints(torch, 0, 5, 6, 0, 8), parent, ints(torch, 0, 3, 5), 2)
    assert count[1] == 2 and token[1] == 9
    with pytest.raises(NekoError, match="max_new"):
        ops.status()
    mask, depth = ops.tree_masks(parent, ints(torch, 0, 2, 9), 4)
    assert depth.tolist() == [0, 1, 0, 0, 0]
    with pytest.raises(NekoError, match="max_new"):
        ops.status()
    pool = torch.zeros((2, 4, 2, 16, 32), dtype=torch.float16, device="cuda")
    pool.copy_(torch.randn(pool.shape))
    before = pool.clone()
    ops.paged_compact(pool, ints(torch, 0, 1)[None], ints(torch, 3), ints(torch, 1, 2)[None], ints(torch, 3))
    with pytest.raises(NekoError, match="max_new"):
        ops.status()
    assert torch.equal(pool, before)
    ops.status()


# ------------------------------------------------------------------------------------------------ moving tokens and pages
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,n_kv,ps", [(128, 8, 16), (64, 3, 64), (32, 5, 32), (128, 1, 128)])
def test_compact(torch, hd, n_kv, ps, e4m3):
    """Paths within a page and over several, into shared sequences' last pages, tokens that stay, sequences of no tokens, inactive
    ones and pages that are not resident; scales of all sizes. Nothing else changes."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(11)
    planes, width = 3, 2 * -(-300 // ps) + 2
    paths = [[0], [0, 1, 2], [1], [0, 2, 5, 6], list(range(1, 40)), sorted(rng.choice(200, 70, replace=False)), [], [0, 3], [0, 1, 2, 90, 91],
             list(range(150, 290)), [0, 1 << 30, 2 ** 31 - 1]]
    start = [0, ps - 1, 5, ps - 2, 3 * ps - 7, ps, 4, -1, 2 * ps - 3, 0, 7]
    count = [len(p) for p in paths]
    path = np.zeros((len(paths), max(count)), np.int32)
    for i, p in enumerate(paths):
        path[i, :len(p)] = p
    held = [min(width, (max(s, 0) + min(max(p + [0]), 400)) // ps + 1) for s, p in zip(start, paths)]
    pages = sum(held) + 2
    order = rng.permutation(pages)
    table = np.full((len(paths), width), -1, np.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    table[8, (start[8] + 91) // ps] = -5  # its last tokens come from nowhere, or go nowhere
    shape = (planes, pages, n_kv, ps, hd)
    scale = None
    if e4m3:
        pool = torch.from_numpy(rng.integers(0, 256, shape).astype(np.uint8)).cuda()
        scale = torch.from_numpy((2.0 ** rng.integers(-9, 3, shape[:3])).astype(np.float32)).cuda()
        want, ws = ref.E4M3[pool.cpu().numpy()], scale.cpu().numpy().astype(np.float64)
    else:
        pool = torch.randn(shape, device="cuda").half()
        want, ws = pool.cpu().numpy().astype(np.float64), None
    before = want.copy()
    want_of.compact(want, ws, table, start, path, count)
    wide = torch.from_numpy(np.concatenate([path, path + 7], 1)).cuda()[:, :path.shape[1]]  # any row stride
    ops.paged_compact(pool.view(torch.float8_e4m3fn) if e4m3 else pool, torch.from_numpy(table).cuda(), ints(torch, *start), wide, ints(torch, *count), scale=scale)
    ops.status()
    got = ref.E4M3[pool.cpu().numpy()] if e4m3 else pool.cpu().numpy().astype(np.float64)
    # what lies at and past start + count is not the sequence's any more
    free = np.zeros((pages, ps), bool)
    for i in range(len(paths)):
        for pos in range(max(start[i], 0) + count[i], width * ps):
            p = table[i, pos // ps]
            if 0 <= p < pages and start[i] >= 0:
                free[p, pos % ps] = True
    keep = np.broadcast_to(~free[None, :, None, :, None], shape)
    assert np.array_equal(got[keep], want[keep], equal_nan=True)
    assert (want[keep] != before[keep]).any()
    if e4m3:
        assert np.array_equal(scale.cpu().numpy().astype(np.float64), ws)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,n_kv,ps,n", [(128, 8, 16, 3), (64, 3, 64, 40), (32, 1, 16, 1), (128, 12, 128, 7)])
def test_copy(torch, hd, n_kv, ps, n, e4m3):
    """Pages and their scales, from one page to several, pairs with an entry out of range skipped; pools with gaps between pages
    and planes, which stay as they are."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(12)
    pages = 3 * n + 4
    order = rng.permutation(pages)
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    src[-1] = src[0]
    pairs = [(s, d) for s, d in zip(src, dst)] + [(-1, int(order[-1])), (int(order[0]), pages), (pages + 7, int(order[-2])), (int(order[-3]),) * 2]
    wide = torch.randint(0, 256, (2, 4, pages + 1, n_kv, ps, hd * (1 if e4m3 else 2)), dtype=torch.uint8, device="cuda")
    pool = wide.view(torch.float8_e4m3fn if e4m3 else torch.float16)[:, 1:, :pages]
    assert pool.shape[1] == 3
    pool = pool[1]  # planes a constant step apart
    sc_wide = torch.rand((2, 4, pages + 1, n_kv + 2), device="cuda")
    scale = sc_wide[:, 1:, :pages, 1:1 + n_kv][1] if e4m3 else None
    want, want_s = wide.clone(), sc_wide.clone()
    for s, d in pairs:
        if 0 <= s < pages and 0 <= d < pages:
            want[1, 1:, d] = wide[1, 1:, s]
            if e4m3:
                want_s[1, 1:, d, 1:1 + n_kv] = sc_wide[1, 1:, s, 1:1 + n_kv]
    ops.paged_copy(pool, ints(torch, *(s for s, _ in pairs)), ints(torch, *(d for _, d in pairs)), scale=scale)
    assert torch.equal(wide, want) and torch.equal(sc_wide, want_s)


def test_moves_past_32_bits(torch):
    """Planes and pages more than 2^32 elements apart."""
    from nekochat_b200 import ops
    pool = torch.empty((2, 5, 1, 128, 128), dtype=torch.float16, device="cuda")
    step = (1 << 32) + 8 * 128 * 128
    big = torch.empty(step + 5 * (1 << 20), dtype=torch.float16, device="cuda")
    pool = big.as_strided((2, 5, 1, 128, 128), (step, 1 << 20, 128 * 128, 128, 1))
    pool.copy_(torch.randn(pool.shape, device="cuda"))
    want = pool.clone()
    ops.paged_copy(pool, ints(torch, 4), ints(torch, 1))
    want[:, 1] = want[:, 4]
    ops.paged_compact(pool, ints(torch, 3, 2)[None], ints(torch, 5), ints(torch, 0, 130)[None], ints(torch, 2))
    want[:, 3, :, 6] = want[:, 2, :, 7]
    assert torch.equal(pool, want)


# ------------------------------------------------------------------------------------------------ sampling
def rows_of(rng, kind, rows, V):
    x = rng.standard_normal((rows, V)) * 2
    if kind == "peaked":
        x[np.arange(rows)[:, None], rng.integers(0, V, (rows, 12))] += 12 * rng.random((rows, 12))
    elif kind == "flat":
        x[:] = 1.5
    elif kind == "wide":
        x *= 20
    elif kind == "ties":
        x = np.round(x)
    elif kind == "few":
        x[rng.random((rows, V)) < 0.99] = -np.inf
        x[0] = -np.inf
    elif kind == "odd":
        x[rng.random((rows, V)) < 0.2] = np.nan
        x[rng.random((rows, V)) < 0.2] = -np.inf
        x[rows // 2:, rng.integers(0, V, 3)] = np.inf
        x[-1] = np.nan
    elif kind == "zeros":
        x = np.where(rng.random((rows, V)) < 0.5, 0.0, -0.0)
        x[:, :V // 2] -= 1
    return x.astype(np.float32)


PARAMS = [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.95, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (1.3, 200, 1.0, 0.02), (0.6, 1, 0.5, 0.0),
          (1.0, 3000, 0.97, 0.0), (1.0, 5000, 1.0, 0.0), (5.0, 0, 0.99, 0.0), (0.05, 0, 0.9, 0.0), (1e-3, 50, 0.9, 0.1), (100.0, 700, 0.4, 0.0),
          (0.9, 0, 0.0, 0.0), (0.9, 0, 1.0, 1.0), (0.9, 0, 0.3, 2.0), (0.0, 40, 0.9, 0.0), (1.0, -3, 2.0, -1.0), (1e30, 0, 0.5, 0.0)]


def sampled(torch, x, dtype, params, u, stride=0):
    """ops.sample_rows on rows x of one type and stride, against the definition."""
    from nekochat_b200 import ops
    rows, V = x.shape
    wide = torch.full((rows, V + stride), 9.0, dtype=getattr(torch, dtype), device="cuda")
    wide[:, :V] = torch.from_numpy(x).cuda()
    before = wide.clone()
    logits = wide[:, :V]
    token, prob = ops.sample_rows(logits, torch.from_numpy(u).cuda(), *params)
    assert torch.equal(wide.view(torch.uint8), before.view(torch.uint8))
    x = logits.float().cpu().numpy()
    of = lambda p, r: p[r].item() if torch.is_tensor(p) else p  # noqa: E731
    for r in range(rows):
        t, p = want_of.sample(x[r], u[r], *(of(y, r) for y in params))
        assert int(token[r]) == t, (r, params, u[r])
        assert abs(float(prob[r]) - p) <= 2.0 ** -23 * p, (r, params)
    return token


@pytest.mark.parametrize("V", [1, 2, 5, 31, 1000, 4097, 50257, 151936])
@pytest.mark.parametrize("kind", ["normal", "peaked", "flat", "wide", "ties", "few", "odd", "zeros"])
def test_samples(torch, kind, V):
    """Every set of parameters on every kind of row, from the ends of u's range too."""
    rng = np.random.default_rng(V)
    rows = 6
    x = rows_of(rng, kind, rows, V)
    for i, params in enumerate(PARAMS if V < 100000 else PARAMS[:10]):
        u = rng.random(rows)
        u[:3] = [0.0, 0.5, 1 - 2.0 ** -20]
        sampled(torch, x, ["float32", "bfloat16", "float16"][i % 3], params, u, stride=i % 4)


def test_samples_of_the_largest_vocabulary(torch):
    rng = np.random.default_rng(13)
    for kind in ("normal", "flat"):
        x = rows_of(rng, kind, 2, 262144)
        for params in ((1.0, 0, 0.9, 0.0), (1.0, 20000, 1.0, 0.0), (1.0, 0, 1.0, 0.0)):
            for dtype in ("float32", "bfloat16"):
                sampled(torch, x, dtype, params, rng.random(2))


def test_samples_with_parameters_of_each_row(torch):
    rng = np.random.default_rng(14)
    rows = 120
    for V in (300, 50257):
        x = rows_of(rng, "peaked", rows, V)
        pick = lambda a, t: torch.tensor(rng.choice(a, rows), dtype=t, device="cuda")  # noqa: E731
        params = (pick([0.0, 0.5, 0.8, 1.0, 1.5], torch.float32), pick([0, 1, 7, 40, 500, 2000], torch.int32),
                  pick([0.2, 0.8, 0.95, 1.0], torch.float32), pick([0.0, 0.03, 0.2], torch.float32))
        a = sampled(torch, x, "float32", params, rng.random(rows))
        assert len(set(a.tolist())) > 10


def test_samples_are_as_likely_as_they_should_be(torch):
    """2^16 numbers spread evenly over [0, 1): each token is taken as often as its weight says, to within one of its two ends."""
    from nekochat_b200 import ops
    x = torch.tensor([[0.3, -1.0, 2.0, 0.5, float("-inf"), 1.0, 0.25]], device="cuda").expand(1 << 16, 7)
    u = (torch.arange(1 << 16, device="cuda", dtype=torch.float64) + 0.5) / (1 << 16)
    token, prob = ops.sample_rows(x, u, 0.7)
    p = torch.softmax(x[0].double() / np.float64(np.float32(0.7)), 0)
    n = torch.bincount(token.long(), minlength=7)
    assert ((n / 65536 - p).abs() <= 2 / 65536).all() and (token[1:] >= token[:-1]).all()
    assert ((prob - p[token.long()]).abs() <= 1e-7).all()
    greedy, one = ops.sample_rows(x[:3], None, 0.0)
    assert greedy.tolist() == [2, 2, 2] and (one == 1).all()


# ------------------------------------------------------------------------------------------------ together
def test_a_step_in_a_graph_and_on_another_stream(torch):
    """Masks, append, attention, sampling, the walk and the compaction captured once and replayed on other inputs: the bits of the
    calls themselves, made on another stream at the same time."""
    from nekochat_b200 import ops
    lens, new, heads = [300, 40, 700], [12, 3, 40], 8
    base, T = [x - n for x, n in zip(lens, new)], sum(new)
    rng = np.random.default_rng(15)
    g = torch.Generator("cuda").manual_seed(16)

    def filled():
        c = Cache(torch, np.random.default_rng(17), lens, 2, 16, 128, True)
        g.manual_seed(18)
        quantize(torch, c, *(torch.randn(c.k.shape, device="cuda", generator=g) for _ in range(2)))
        return c

    torch.manual_seed(19)
    q, k, v = (torch.randn((T, h, 128), device="cuda") for h in (heads, 2, 2))
    parent, draft = ints(torch, *sum(some_trees(rng, new), [])), torch.randint(0, 2, (T,), device="cuda", dtype=torch.int32)
    head, u = torch.randn((heads * 128, 1000), device="cuda"), torch.rand(T, device="cuda", dtype=torch.float64)
    at, held, qs, cs = ints(torch, *base), ints(torch, *lens), ints(torch, *starts(new).tolist()), ops.rope_table(800, 128, 1e4)
    likely = torch.tensor([20.0] * 2 + [0.0] * 998, device="cuda")  # the tokens that the drafts are

    def step(c):
        table, sc = torch.from_numpy(c.table).cuda() if not hasattr(c, "t") else c.t, dict(k_scale=c.ks, v_scale=c.vs, q_start=qs, max_new=max(new))
        c.t = table
        mask, depth = ops.tree_masks(parent, qs, max(new))
        turned = ops.paged_append(k, v, c.k, c.v, table, at, q=q, cs=cs, depth=depth, **sc)
        o = ops.paged_tree_attention(turned, c.k, c.v, table, held, mask, depth, window=500, **sc)
        token, prob = ops.sample_rows(torch.tanh(o.view(T, -1) @ head) + likely, u, 0.8, 40, 0.95, 0.01)
        path, count, last = ops.tree_accept(token, draft, parent, qs, max(new))
        for pool, s in ((c.k, c.ks), (c.v, c.vs)):
            ops.paged_compact(pool.view(torch.float8_e4m3fn), table, at, path, count, scale=s)
        return o, token, prob, path, count, last

    one, two = filled(), filled()
    step(one), step(two)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(one)
    other, walked = torch.cuda.Stream(), 0
    for _ in range(3):
        for x in (q, k, v):
            x.normal_()
        u.uniform_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            want = step(two)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(one.k, two.k) and torch.equal(one.v, two.v) and torch.equal(one.ks, two.ks)
        walked += int(want[4].sum())
    assert walked > 9  # more than the roots
    ops.status()


@pytest.fixture(scope="module")
def model():
    from nekochat_b200 import paged, workload
    m = paged.build("qwen3-tiny", kind="f16", page=16, pages=60, max_len=256, perturb=True, max_seqs=12)
    m.prompts = [workload.prompt(m.s, n, seed=i + 5).tolist() for i, n in enumerate((40, 1, 37))]
    m.prompts.append(m.prompts[0][:9] * 5)
    return m


@pytest.mark.parametrize("how", [dict(), dict(temperature=0.8, top_k=40, top_p=0.95, seed=3), dict(temperature=0.3, min_p=0.1)])
def test_drafts_do_not_change_the_answers(model, how):
    """Greedy and sampled: the tokens that one at a time gives, in fewer steps; pages come back."""
    plain = model.generate(model.prompts, 40, **how)
    for draft in (1, 7, 70):
        steps = []
        verify = model.verify
        model.verify = lambda *a: steps.append(1) or verify(*a)
        try:
            got = model.generate(model.prompts, 40, draft=draft, **how)
        finally:
            del model.verify
        assert got == plain and len(model.cache.free) == 60 and not model.cache.held
        assert 0 < len(steps) < 40
    stop = plain[0][20]
    assert model.generate(model.prompts, 40, stop_ids={stop}, draft=7, **how) == model.generate(model.prompts, 40, stop_ids={stop}, **how)


def test_answers_of_a_forked_prompt(model):
    """Copies share the prompt's pages: the answers are those of prompts of their own with the same numbers, and differ."""
    how = dict(temperature=1.0, seed=4)
    got = model.generate(model.prompts[:2], 12, copies=3, **how)
    assert got == model.generate([p for p in model.prompts[:2] for _ in range(3)], 12, **how) and got[0] != got[1]
    assert got == model.generate(model.prompts[:2], 12, copies=3, draft=5, **how)
    assert len(model.cache.free) == 60 and not model.cache.held and not any(model.cache.holders)


def test_forks_cuts_and_packing(model, torch):
    """Sequences that share pages give the logits of their own tokens whatever the others do, before and after pages move."""
    c, p = model.cache, model.prompts[0]
    alone = lambda tokens: (lambda s: (model.forward([(s, tokens)])[0].clone(), c.close(s))[0])(c.open())  # noqa: E731
    want = [alone(p + x) for x in ([7], [8, 9], [10], [11])]
    a, filler = c.open(), c.open()
    model.forward([(filler, p * 2)])
    model.forward([(a, p)])
    b, d = c.fork(a, 2)
    assert c.held[a][:2] == c.held[b][:2] and len({c.held[x][2] for x in (a, b, d)}) == 3
    got = list(model.forward([(a, [7]), (b, [8, 9])]))
    c.close(filler)
    free = len(c.free)
    assert c.pack() == 60 - free and sorted({x for s in (a, b, d) for x in c.held[s]}) == list(range(60 - free))
    got.append(model.forward([(d, [10])])[0].clone())
    c.cut(b, len(p) - 20), c.cut(a, len(p))
    got.append(model.forward([(b, p[-20:] + [11])])[0].clone())
    for x, y in zip(got, want):
        assert (x - y).abs().max() <= 2e-2
    for s in (a, b, d):
        c.close(s)
    assert len(c.free) == 60


def test_command_samples_and_drafts():
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-m", "nekochat_b200.paged", "--max-new", "4", "--temperature", "0.8", "--top-k", "40", "--draft", "6", "--copies", "2"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "tokens/s" in r.stdout and r.stdout.count("prompt tokens") == 6, r.stderr


# ------------------------------------------------------------------------------------------------ rows and sequences that are left out
def test_rows_of_no_sequence_are_zeros(torch):
    """Before the first sequence, behind the last and of a sequence that is left out, in memory that held other things; as many as
    several CTAs clear."""
    from nekochat_b200 import NekoError, ops
    for starts, tokens, n, bad in (([2, 5, 5, 9], 12, 70, ()), ([0, 1], 3000, 900, ()), ([7, 7], 40, 64, ()), ([0, 3, 9, 12], 12, 4, (3, 9))):
        parent = torch.arange(-1, tokens - 1, dtype=torch.int32, device="cuda")
        parent[[s for s in starts[:-1] if s < tokens]] = -1
        for a, b in zip(starts, starts[1:]):
            parent[a:b] = torch.arange(-1, b - a - 1, dtype=torch.int32)
        words = -(-n // 64)
        for shape in ((tokens, words * 2), (tokens,)):  # the allocator hands these out again
            torch.full(shape, -1, dtype=torch.int32, device="cuda")
        mask, depth = ops.tree_masks(parent, ints(torch, *starts), n)
        want_mask, want_depth = np.zeros((tokens, words), np.uint64), np.zeros(tokens, np.int32)
        for a, b in zip(starts, starts[1:]):
            if (a, b) == bad:
                continue
            for i in range(b - a):  # lines
                want_depth[a + i] = i
                for j in range(i + 1):
                    want_mask[a + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
        assert np.array_equal(mask.cpu().numpy().view(np.uint64), want_mask) and np.array_equal(depth.cpu().numpy(), want_depth)
        if bad:
            with pytest.raises(NekoError, match="max_new"):
                ops.status()
        ops.status()
    mask, depth = ops.tree_masks(parent, ints(torch, 0), 5)
    assert not mask.any() and not depth.any() and mask.shape == (12, 1)


def test_a_sequence_left_out_walks_nowhere(torch):
    from nekochat_b200 import NekoError, ops
    parent, draft = ints(torch, -1, 0, 1, 2, -1, 0), ints(torch, 1, 2, 3, 4, 5, 6)
    torch.full((2, 3), 7, dtype=torch.int32, device="cuda")
    path, count, token = ops.tree_accept(ints(torch, 2, 3, 4, 5, 6, 8), draft, parent, ints(torch, 0, 4, 6), 3)
    assert path.tolist() == [[0, 0, 0], [0, 1, 0]] and count.tolist() == [0, 2] and token.tolist() == [-1, 8]
    with pytest.raises(NekoError, match="max_new"):
        ops.status()


@pytest.mark.parametrize("n_seq", [2, 128, 129, 300])
def test_trees_of_many_sequences(torch, n_seq):
    """Sequences in any order of their lengths, alike and empty ones, up to and past the number that is ordered by them."""
    from nekochat_b200 import ops
    H, KV, hd, ps, new = 8, 2, 64, 32, 9  # 36 rows of a KV head: the kernel for many rows
    rng = np.random.default_rng(n_seq)
    ctx = rng.choice([0, 1, 31, 150, 150, 300], n_seq)
    sizes = np.where(rng.random(n_seq) < 0.1, 0, rng.integers(1, new + 1, n_seq))
    kv_len, at = ctx + sizes, np.concatenate([[0], np.cumsum(sizes)])
    width = -(-int(kv_len.max()) // ps)
    table = rng.permutation(n_seq * width).reshape(n_seq, width).astype(np.int32)
    k, v = (torch.randn((n_seq * width, KV, ps, hd), device="cuda").half() for _ in range(2))
    parent = np.concatenate([[-1] + [int(rng.integers(0, i)) for i in range(1, m)] if m else [] for m in sizes]).astype(np.int32)
    q = torch.randn((len(parent), H, hd), device="cuda")
    mask, depth = ops.tree_masks(ints(torch, *parent), ints(torch, *at), new)
    whole = ops.paged_tree_attention(q, k, v, torch.from_numpy(table).cuda(), ints(torch, *kv_len), mask, depth, q_start=ints(torch, *at), max_new=new)
    ops.status()
    for s in range(n_seq):  # each by the definition
        a, b = int(at[s]), int(at[s + 1])
        if a == b:
            continue
        n = int(kv_len[s])
        kk, vv = (x[torch.from_numpy(table[s]).long().cuda()].transpose(0, 1).reshape(KV, -1, hd)[:, :n].double() for x in (k, v))
        z = torch.einsum("tghd,gjd->ghtj", q[a:b].double().view(b - a, KV, H // KV, hd), kk) / hd ** 0.5
        seen = torch.ones((b - a, n), dtype=torch.bool, device="cuda")
        bits = mask[a:b, 0, None] >> torch.arange(b - a, device="cuda") & 1
        seen[:, n - (b - a):] = bits.bool()
        w = torch.softmax(z.masked_fill(~seen, -float("inf")), -1)
        want = torch.einsum("ghtj,gjd->tghd", w, vv).reshape(b - a, H, hd)
        # |values| < 6. Queries and weights enter as two f16 (22 bits); scores, of 64 products of sizes up to 16 and divided by 8, are
        # off by less than 64 * 16 / 8 * 2^-21 = 2^-14 even if all errors agree, a softmax by as much times |value|
        assert (whole[a:b].double() - want).abs().max() < 6 * 2.0 ** -14, s


def test_numbers_of_a_call_out_of_range(torch):
    """A temperature that is no number is greedy; numbers beyond f32 and 32 bits count as the ends of the range."""
    from nekochat_b200 import ops
    x = torch.randn((4, 500), device="cuda")
    u = torch.rand(4, dtype=torch.float64, device="cuda")
    greedy = x.argmax(1).int()
    assert torch.equal(ops.sample_rows(x, u, math.nan)[0], greedy)
    t = torch.tensor([math.nan, -1.0, 0.0, -math.inf], device="cuda")
    assert torch.equal(ops.sample_rows(x, u, t)[0], greedy)
    flat = (u * 500).floor().int()
    for hot in (1e300, math.inf, 1e36):
        assert torch.equal(ops.sample_rows(x, u, hot)[0], flat)
    for k in (2 ** 40, -2 ** 40, 0):
        assert torch.equal(ops.sample_rows(x, u, 0.9, k, 1e300, -1e300)[0], ops.sample_rows(x, u, 0.9)[0])
    assert torch.equal(ops.sample_rows(x, u, 0.9, 0, -1e300)[0], greedy) and torch.equal(ops.sample_rows(x, u, 0.9, 0, 1.0, 1e300)[0], greedy)


@pytest.mark.parametrize("e4m3", [False, True])
def test_two_streams_at_once(torch, e4m3):
    """Calls that run beside each other, each on inputs of its own, give what they give alone."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(3)
    sets = []
    for n_seq, new in ((5, 40), (40, 3)):
        ps, KV, hd, ctx = 64, 4, 128, 1500
        width = -(-(ctx + new) // ps)
        k, v = (torch.randn((n_seq * width, KV, ps, hd), device="cuda").half() for _ in range(2))
        scales = {}
        if e4m3:
            k, v = (x.to(torch.float8_e4m3fn) for x in (k, v))
            scales = dict(k_scale=torch.ones((n_seq * width, KV), device="cuda"), v_scale=torch.ones((n_seq * width, KV), device="cuda"))
        table = torch.randperm(n_seq * width, device="cuda").int().view(n_seq, width)
        at = torch.arange(n_seq + 1, device="cuda").int() * new
        parent = ints(torch, *[int(rng.integers(0, i)) if i else -1 for _ in range(n_seq) for i in range(new)])
        q, x = torch.randn((n_seq * new, 8, hd), device="cuda"), torch.randn((n_seq * new, 20000), device="cuda")
        u = torch.rand(n_seq * new, dtype=torch.float64, device="cuda")
        kv_len = torch.full((n_seq,), ctx + new, dtype=torch.int32, device="cuda")

        def call(q=q, k=k, v=v, table=table, kv_len=kv_len, parent=parent, at=at, new=new, scales=scales, x=x, u=u):
            mask, depth = ops.tree_masks(parent, at, new)
            out = ops.paged_tree_attention(q, k, v, table, kv_len, mask, depth, q_start=at, max_new=new, **scales)
            token, prob = ops.sample_rows(x, u, 0.9, 0, 0.9)
            return (out, token, prob, *ops.tree_accept(token, token, parent, at, new))
        sets.append(call)
    alone = [call() for call in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(10):
        for i, (stream, call) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(stream):
                got[i].append(call())
    torch.cuda.synchronize()
    for want, runs in zip(alone, got):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, want))
    ops.status()
