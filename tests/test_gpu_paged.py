"""The paged key/value cache operators (neko_op_paged_append, neko_op_paged_attention) against their definitions in 64
bits (paged_reference.py).

Tolerances, from the arithmetic. Attention: scores carry 22 bits of q and exact keys, so an error of a few 2^-22 of
sum |q||k| scale (about 10 at these sizes), the weights a few 2^-22 more, and a softcap of 50 tanh's 2^-22: together
4e-5 of the largest value seen. 16-bit queries are exact and add their weights' rounding to f16 (2^-12 relative each,
2^-11 taken) and the output's (2^-12 for f16, 2^-9 for bf16, of at most the largest value). Append: q in f32 carries the
norm's and the rotation's few roundings, 2e-6 of the row's largest value; a stored f16 half a unit (2^-11 relative)
more, a stored e4m3 half a unit of 3 mantissa bits (2^-4) of its value, or 2^-10 of its scale when subnormal."""
import numpy as np
import pytest

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
ROUND = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


class Cache:
    """A pool of pages with some that nobody holds, in no order, every unused place poisoned with NaN."""

    def __init__(self, torch, rng, lens, n_kv, ps, hd, e4m3, spare=3, together=False, width=None):
        self.torch, self.ps, self.e4m3 = torch, ps, e4m3
        need = [-(-max(x, 0) // ps) for x in lens]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        width = width or max(max(need), 1)
        self.table = np.full((len(lens), width), -1, np.int32)
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = order[at:at + m][:width]
            at += m
        shape = (pages, 2, n_kv, ps, hd) if together else (2, pages, n_kv, ps, hd)
        if e4m3:
            pool = torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda")
            sc = torch.full(shape[:3], float("nan"), device="cuda")
        else:
            pool = torch.full(shape, float("nan"), dtype=torch.float16, device="cuda")
            sc = None
        pick = (lambda t, i: t[:, i]) if together else (lambda t, i: t[i])
        self.k, self.v = pick(pool, 0), pick(pool, 1)
        self.ks, self.vs = (pick(sc, 0), pick(sc, 1)) if e4m3 else (None, None)

    def fill(self, rng, lens, scale=1.0, exps=3):
        """Random keys and values at the places that sequences hold."""
        t = self.torch
        for pool, sc in ((self.k, self.ks), (self.v, self.vs)):
            x = rng.standard_normal(pool.shape) * scale
            mine = np.zeros(pool.shape[:1] + pool.shape[2:3], bool)
            for s, n in enumerate(lens):
                for i, p in enumerate(self.table[s]):
                    if p >= 0:
                        mine[p, :max(0, min(self.ps, n - i * self.ps))] = True
            m = t.from_numpy(mine).cuda()[:, None, :, None]
            if self.e4m3:
                codes = np.abs(rng.standard_normal(pool.shape) * 30).clip(0, 120).astype(np.uint8)
                codes |= (rng.integers(0, 2, pool.shape) << 7).astype(np.uint8)
                pool.copy_(t.where(m, t.from_numpy(codes).cuda(), pool))
                used = t.from_numpy(mine.any(1)).cuda()[:, None]
                e = t.from_numpy((2.0 ** rng.integers(-4, -4 + exps, sc.shape)).astype(np.float32)).cuda()
                sc.copy_(t.where(used, e, sc))
            else:
                pool.copy_(t.where(m, t.from_numpy(x.astype(np.float16)).cuda(), pool))

    def values(self, scaled=True):
        out = []
        for pool, sc in ((self.k, self.ks), (self.v, self.vs)):
            if self.e4m3:
                x = ref.E4M3[pool.cpu().numpy()]
                out.append(x * sc.cpu().numpy().astype(np.float64)[:, :, None, None] if scaled else x)
            else:
                out.append(pool.cpu().numpy().astype(np.float64))
        return out


def starts(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def attend(torch, cache, lens, new, heads, dtype, seed, softcap=0.0, window=0, alibi=False, prefix=None, scale=None,
           strided=False, q_start=True, q_scale=1.0, bad_v=None, stream=None):
    from nekochat_b200 import ops
    rng = np.random.default_rng(seed)
    dt = getattr(torch, dtype)
    hd = cache.k.shape[3]
    T = int(sum(new))
    qs = starts(new)
    wide = torch.from_numpy((rng.standard_normal((T, heads + 3, hd + 8)) * q_scale).astype(np.float32)).to(dt).cuda()
    q = wide[:, 1:1 + heads, 4:4 + hd] if strided else wide[:, :heads, :hd].contiguous()
    out = torch.full((T, heads + 1, hd + 4), 7.0, dtype=dt, device="cuda") if strided else None
    slopes = (2.0 ** (-8.0 * np.arange(1, heads + 1) / heads)).astype(np.float32) if alibi else None
    ints = lambda x: None if x is None else torch.tensor(list(x), dtype=torch.int32, device="cuda")  # noqa: E731
    args = dict(k_scale=cache.ks, v_scale=cache.vs, q_start=ints(qs) if q_start else None, max_new=max(max(new), 1),
                softcap=softcap, window=window, slopes=None if slopes is None else torch.from_numpy(slopes).cuda(),
                prefix=ints(prefix), scale=scale, out=None if out is None else out[:, :heads, :hd])
    table = torch.from_numpy(cache.table).cuda()
    got = ops.paged_attention(q, cache.k, cache.v, table, ints(lens), **args)
    torch.cuda.synchronize()
    if strided:
        assert (out[:, heads] == 7.0).all() and (out[:, :, hd:] == 7.0).all()
    kv, vv = cache.values()
    want = ref.attention(q.float().cpu().numpy().astype(np.float64), kv, vv, cache.table, list(lens), qs,
                         hd ** -0.5 if scale is None else scale, softcap, window, slopes, prefix)
    got = got.float().cpu().numpy().astype(np.float64)
    seen = np.abs(vv[np.isfinite(vv)])
    vmax = seen.max() if seen.size else 1.0
    tol = (4e-5 + (0 if dtype == "float32" else 2.0 ** -11) + ROUND[dtype]) * vmax
    assert np.array_equal(np.isfinite(got), np.isfinite(want)), "finite elsewhere than the definition"
    f = np.isfinite(want)
    err = np.abs(got[f] - want[f])
    assert err.size == 0 or err.max() <= tol, f"{err.max()} > {tol}"
    return got, want


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,ps", [(128, 16, 8, 16), (128, 32, 8, 64), (64, 12, 12, 32), (32, 4, 4, 16),
                                              (128, 8, 1, 128), (64, 9, 3, 16), (128, 24, 2, 32)])
def test_single_tokens(torch, hd, heads, n_kv, ps, e4m3, dtype):
    """Decode steps: lengths from one token on, around the groups of 16, pages and the warps' rounds."""
    rng = np.random.default_rng(hd + heads + ps + e4m3)
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 130, 257]
    cache = Cache(torch, rng, lens, n_kv, ps, hd, e4m3)
    cache.fill(rng, lens)
    attend(torch, cache, lens, [1] * len(lens), heads, dtype, 1, q_start=False)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,ps", [(128, 16, 8, 16), (64, 12, 12, 64), (32, 6, 2, 32), (128, 8, 1, 128)])
def test_ragged_rows(torch, hd, heads, n_kv, ps, e4m3, dtype):
    """Several new tokens per sequence, some sequences without any, some all new, one empty."""
    rng = np.random.default_rng(hd + heads + ps + 7 * e4m3)
    new = [3, 0, 17, 1, 40, 5, 0, 2]
    lens = [3, 20, 50, 1, 40, 133, 0, 66]
    cache = Cache(torch, rng, lens, n_kv, ps, hd, e4m3)
    cache.fill(rng, lens)
    attend(torch, cache, lens, new, heads, dtype, 2)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("opts", [dict(softcap=30.0), dict(softcap=0.5), dict(window=1), dict(window=20),
                                  dict(window=33, softcap=50.0, alibi=True), dict(alibi=True), dict(pre=True),
                                  dict(pre=True, window=18), dict(scale=0.5), dict(strided=True),
                                  dict(q_scale=1e-6, scale=1e5), dict(q_scale=3e3, scale=1e-4)])
def test_masks_and_biases(torch, opts, e4m3, dtype):
    opts = dict(opts)
    rng = np.random.default_rng(len(opts) + e4m3)
    new = [1, 4, 30, 9, 2]
    lens = [100, 4, 75, 41, 90]
    if opts.pop("pre", False):
        opts["prefix"] = [40, 4, 60, 0, 200]
    if dtype == "float16" and "q_scale" in opts:
        opts["q_scale"] = min(opts["q_scale"], 1e3)
    cache = Cache(torch, rng, lens, 4, 16, 128, e4m3)
    cache.fill(rng, lens)
    attend(torch, cache, lens, new, 8, dtype, 3, **opts)


@pytest.mark.parametrize("e4m3", [False, True])
def test_pages_that_are_not_resident(torch, e4m3):
    """Entries of -1 and out of range inside a sequence, a table narrower than the length, rows that see nothing."""
    rng = np.random.default_rng(11)
    lens, new = [100, 100, 40, 64], [1, 5, 3, 2]
    cache = Cache(torch, rng, lens, 2, 16, 64, e4m3)
    cache.fill(rng, lens)
    cache.table[0, 1:3] = -1
    cache.table[1, 6] = 1 << 20
    cache.table[2, :] = -1
    got, want = attend(torch, cache, lens, new, 4, "float32", 4)
    assert (want[6:9] == 0).all() and (got[6:9] == 0).all()
    attend(torch, cache, lens, new, 4, "float32", 4, window=3)
    cache.table = np.ascontiguousarray(cache.table[:, :3])
    attend(torch, cache, lens, new, 4, "float32", 4)


def test_rows_without_keys(torch):
    """No tokens at all, inactive sequences, more new tokens than the cache is said to hold (negative positions)."""
    rng = np.random.default_rng(12)
    lens, new = [0, -5, 3, 10], [1, 2, 6, 1]
    cache = Cache(torch, rng, lens, 2, 16, 128, False)
    cache.fill(rng, lens)
    got, _ = attend(torch, cache, lens, new, 4, "float32", 5)
    assert (got[:6] == 0).all()
    attend(torch, cache, lens, new, 4, "float32", 5, prefix=[5, 5, 2, 20])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_that_are_not_seen_have_no_effect(torch, dtype, e4m3):
    """NaN in keys and values of later tokens reaches the rows that see them and no other; NaN and infinities in
    masked places change nothing."""
    rng = np.random.default_rng(13)
    lens, new = [50, 70, 20], [20, 1, 20]
    cache = Cache(torch, rng, lens, 2, 16, 64, e4m3)
    cache.fill(rng, lens)
    nan = 0x7F if e4m3 else float("nan")
    cache.v[int(cache.table[0, 45 // 16]), :, 45 % 16, 3:40] = nan
    cache.k[int(cache.table[0, 48 // 16]), 1, 48 % 16, 5] = nan
    cache.v[int(cache.table[2, 0]), 0, 10, :] = nan
    got, want = attend(torch, cache, lens, new, 4, dtype, 6)
    assert np.isfinite(want[:15]).all() and np.isnan(want[15:20, :, 3:40]).all() and np.isnan(want[18:20, 2:]).all()
    if not e4m3:
        cache.v[int(cache.table[1, 0]), :, 2, :] = float("-inf")
    else:
        cache.v[int(cache.table[1, 0]), :, 2, :] = nan
    attend(torch, cache, lens, new, 4, dtype, 6, window=10)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
def test_blocks_of_very_different_scales(torch, e4m3, dtype):
    """Keys and values whose blocks' magnitudes differ by 2^12, and a softmax that prefers the small ones."""
    rng = np.random.default_rng(14)
    lens = [200, 77]
    cache = Cache(torch, rng, lens, 2, 16, 128, e4m3)
    cache.fill(rng, lens, exps=1)
    if e4m3:
        cache.vs.copy_(torch.from_numpy((2.0 ** rng.integers(-8, 5, tuple(cache.vs.shape))).astype(np.float32)).cuda())
    attend(torch, cache, lens, [1, 1], 4, dtype, 7)


def test_pages_between_each_other_and_other_streams(torch):
    """K and V pages of one pool, scales likewise; a call on a stream of its own."""
    rng = np.random.default_rng(15)
    lens, new = [90, 33, 17], [1, 6, 17]
    for e4m3 in (False, True):
        cache = Cache(torch, rng, lens, 2, 32, 128, e4m3, together=True)
        cache.fill(rng, lens)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            attend(torch, cache, lens, new, 4, "float32", 8)


def test_offsets_past_32_bits(torch):
    """Pages whose byte offsets pass 2^32 and element offsets 2^31."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(16)
    ps, hd, stride = 16, 64, 3 << 30
    pool = torch.empty(2 * stride + 2 * ps * hd + 64, dtype=torch.uint8, device="cuda")
    k = pool.as_strided((3, 1, ps, hd), (stride, ps * hd, hd, 1))
    v = pool.as_strided((3, 1, ps, hd), (stride, ps * hd, hd, 1), ps * hd)
    sc = torch.full((3, 1), 0.125, device="cuda")
    x = torch.from_numpy(rng.standard_normal((40, 1, hd)).astype(np.float32)).cuda()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    one = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.paged_append(x, -x, k, v, table, one(0), k_scale=sc, v_scale=sc.clone(), q_start=one(0, 40), max_new=40)
    got = ops.paged_attention(x, k, v, table, one(40), k_scale=sc, v_scale=sc, q_start=one(0, 40), max_new=40)
    kv = ref.E4M3[k.cpu().numpy()] * sc.cpu().numpy()[:, :, None, None]
    vv = ref.E4M3[v.cpu().numpy()] * sc.cpu().numpy()[:, :, None, None]
    want = ref.attention(x.cpu().numpy().astype(np.float64), kv, vv, table.cpu().numpy(), [40], [0, 40], hd ** -0.5)
    assert np.abs(got.cpu().numpy() - want).max() <= 4e-5 * np.abs(vv).max()
    back = kv[[2, 0, 1]].reshape(48, hd)[:40]
    assert np.abs(back - x[:, 0].cpu().numpy()).max() <= 2.0 ** -4 * np.abs(back).max()


# ------------------------------------------------------------------ append
def fresh_rows(torch, rng, T, heads, n_kv, hd, dt, spread=1.0):
    x = rng.standard_normal((T, heads + 2 * n_kv, hd)) * np.exp(spread * rng.standard_normal((T, 1, 1)))
    qkv = torch.from_numpy(x.astype(np.float32)).to(dt).cuda()
    return qkv[:, :heads], qkv[:, heads:heads + n_kv], qkv[:, heads + n_kv:]


def append(torch, cache, start, new, heads, dtype, rng, rot=0, interleaved=False, norm=False, cs_rows=600, spread=1.0,
           q_start=True, in_place=False):
    from nekochat_b200 import ops
    n_kv, hd = cache.k.shape[1], cache.k.shape[3]
    qs = starts(new)
    q, k, v = fresh_rows(torch, rng, int(sum(new)), heads, n_kv, hd, getattr(torch, dtype), spread)
    cs = ops.rope_table(cs_rows, rot, 1e4, device="cuda") if rot else None
    gains = [torch.from_numpy((1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)).cuda() for _ in range(2)] if norm else [None] * 2
    ints = lambda x: torch.tensor(list(x), dtype=torch.int32, device="cuda")  # noqa: E731
    f64 = lambda t: None if t is None else t.float().cpu().numpy().astype(np.float64)  # noqa: E731
    before = cache.values(scaled=False)
    scales = [f64(cache.ks), f64(cache.vs)]
    host = [f64(t) for t in (q, k, v)]
    got_q = ops.paged_append(k, v, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(start),
                             k_scale=cache.ks, v_scale=cache.vs, q_start=ints(qs) if q_start else None,
                             max_new=max(max(new), 1), q=q, cs=cs, interleaved=interleaved, q_gain=gains[0],
                             k_gain=gains[1], q_out=q if in_place else None)
    torch.cuda.synchronize()
    assert not in_place or got_q is q
    want_q = ref.append(host[1], host[2], *before, cache.table, list(start), qs, scales[0], scales[1], host[0],
                        None if cs is None else cs.cpu().numpy(), interleaved, f64(gains[0]), f64(gains[1]))
    top = np.abs(want_q).max(-1, keepdims=True)
    err = np.abs(f64(got_q) - want_q)
    assert (err <= 2e-6 * top + ROUND[dtype] * np.abs(want_q)).all(), err.max()
    after = cache.values(scaled=False)
    for got, want, gs, ws in zip(after, before, [f64(cache.ks), f64(cache.vs)], scales):
        assert np.array_equal(np.isnan(got), np.isnan(want))
        if cache.e4m3:
            # a maximum within rounding of 448 * 2^e may take either scale
            near = ~np.isnan(ws)
            same = np.where(near, gs == ws, True)
            assert (np.isnan(gs) == np.isnan(ws)).all() and same.mean() > 0.9
            assert (np.where(near & ~same, np.abs(np.log2(gs / ws)), 1) == 1).all()
            g, w = got * gs[:, :, None, None], want * ws[:, :, None, None]
            # equal codes, or neighbours where the value was at a tie within rounding
            assert (np.abs(g - w)[~np.isnan(w)] <= (2.0 ** -3 * np.abs(w) + 2.0 ** -9 * ws[:, :, None, None])[~np.isnan(w)]).all()
            flat = same[:, :, None, None] & ~np.isnan(want)
            assert (got != want)[flat].mean() < 1e-3
        else:
            f = ~np.isnan(want)
            rows = np.where(f, np.abs(want), 0).max(-1, keepdims=True)
            assert (np.abs(got - want)[f] <= (2.0 ** -11 * np.abs(want) + 2e-6 * rows + 2.0 ** -24)[f]).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,rot,interleaved,norm", [(128, 128, False, True), (128, 64, True, False),
                                                     (128, 0, False, True), (64, 48, False, False),
                                                     (64, 64, True, True), (32, 32, False, True), (32, 8, True, False)])
def test_append(torch, hd, rot, interleaved, norm, e4m3, dtype):
    """Ragged new tokens at every alignment to the pages, some sequences without any."""
    rng = np.random.default_rng(hd + rot + e4m3)
    for ps in (16, 64):
        start, new = [0, 15, 16, 5, 130, 33, 0], [1, 1, 40, 0, 3, 90, 64]
        lens = [a + b for a, b in zip(start, new)]
        cache = Cache(torch, rng, lens, 3, ps, hd, e4m3)
        cache.fill(rng, start)
        append(torch, cache, start, new, 6, dtype, rng, rot, interleaved, norm)


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("e4m3", [False, True])
def test_append_single_tokens(torch, ps, e4m3):
    """One token after the other; growing magnitudes move a block's scale under the codes it holds."""
    rng = np.random.default_rng(ps + e4m3)
    lens = [ps * 2 + 5, 3]
    cache = Cache(torch, rng, lens, 2, ps, 64, e4m3)
    for i in range(0, lens[0]):
        append(torch, cache, [i, min(i, 2)], [1, 1], 4, "float32", rng, 64, norm=bool(i % 2), spread=2.0,
               q_start=bool(i % 3), in_place=not i % 2)


@pytest.mark.parametrize("e4m3", [False, True])
def test_append_refuses_places_and_keeps_the_rest(torch, e4m3):
    """Inactive sequences, pages that are not resident, tables that end: nothing else changes."""
    rng = np.random.default_rng(21)
    start, new = [10, -1, 40, 30, 0], [3, 2, 30, 4, 17]
    lens = [a + b for a, b in zip(start, new)]
    cache = Cache(torch, rng, lens, 2, 16, 64, e4m3)
    cache.fill(rng, start)
    cache.table[2, 3] = -1
    cache.table[3, 1] = 10 ** 6
    append(torch, cache, start, new, 4, "float32", rng, 64)
    cache.table = np.ascontiguousarray(cache.table[:, :2])
    append(torch, cache, start, new, 4, "float32", rng, 32, interleaved=True)


def test_append_special_values(torch):
    """Zeros, subnormals, infinities and NaN in an 8-bit block: the scale comes from the finite ones."""
    from nekochat_b200 import ops
    k = torch.zeros((16, 4, 32), device="cuda")
    k[:, 1] = 1e-42
    k[:, 2] = 3.0
    k[3, 2, 5], k[4, 2, 6], k[5, 2, 7] = float("inf"), float("-inf"), float("nan")
    k[:, 3] = 448.0 * 2 ** 20
    pages = torch.zeros((1, 4, 16, 32), dtype=torch.float8_e4m3fn, device="cuda")
    sc = torch.ones((1, 4), device="cuda")
    sv = torch.ones((1, 4), device="cuda")
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    ops.paged_append(k, k, pages, pages.clone(), i(0)[None], i(0), k_scale=sc, v_scale=sv, q_start=i(0, 16), max_new=16)
    assert sc.tolist() == [[2.0 ** -100, 2.0 ** -100, 2.0 ** -7, 2.0 ** 20]] and sv.tolist() == sc.tolist()
    got = pages.float()[0]
    assert (got[0] == 0).all() and (got[3] == 448).all()
    assert got[2, 3, 5] == 448 and got[2, 4, 6] == -448 and got[2, 5, 7].isnan() and got[2, 0, 0] == 384


def test_a_step_equals_a_prompt(torch):
    """Tokens appended one by one leave the same f16 cache as all at once, and attention the same result."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(31)
    T, heads, n_kv, hd = 45, 4, 2, 128
    q, k, v = fresh_rows(torch, rng, T, heads, n_kv, hd, torch.float32)
    cs = ops.rope_table(64, 128, 1e6)
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    a, b = (Cache(torch, np.random.default_rng(1), [T], n_kv, 16, hd, False) for _ in range(2))
    table = torch.from_numpy(a.table).cuda()
    qa = ops.paged_append(k, v, a.k, a.v, table, i(0), q_start=i(0, T), max_new=T, q=q, cs=cs)
    all_at_once = ops.paged_attention(qa, a.k, a.v, table, i(T), q_start=i(0, T), max_new=T)
    for s in range(T):
        qb = ops.paged_append(k[s:s + 1], v[s:s + 1], b.k, b.v, table, i(s), q=q[s:s + 1], cs=cs)
        one = ops.paged_attention(qb, b.k, b.v, table, i(s + 1))
        assert torch.equal(qb, qa[s:s + 1])
        assert (one - all_at_once[s:s + 1]).abs().max() <= 8e-5 * v.abs().max()
    assert torch.equal(a.k.nan_to_num(9), b.k.nan_to_num(9)) and torch.equal(a.v.nan_to_num(9), b.v.nan_to_num(9))


def test_results_repeat(torch):
    """The same call twice: the same bits."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(41)
    lens = [700, 3000, 65]
    cache = Cache(torch, rng, lens, 2, 64, 128, True)
    cache.fill(rng, lens)
    q = torch.randn((3, 8, 128), device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    table = torch.from_numpy(cache.table).cuda()
    outs = [ops.paged_attention(q, cache.k, cache.v, table, n, k_scale=cache.ks, v_scale=cache.vs) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("hd,heads,n_kv,ps", [(128, 16, 8, 16), (64, 12, 12, 64), (128, 8, 1, 128), (64, 6, 2, 32)])
def test_prompts(torch, hd, heads, n_kv, ps, e4m3, dtype):
    """Row tiles of 128 packed rows and their ragged ends, key tiles of 128 and theirs, earlier turns."""
    rng = np.random.default_rng(hd + heads + ps + 3 * e4m3)
    new = [130, 1, 64, 257, 0]
    lens = [130, 77, 300, 400, 30]
    cache = Cache(torch, rng, lens, n_kv, ps, hd, e4m3)
    cache.fill(rng, lens)
    attend(torch, cache, lens, new, heads, dtype, 52)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("opts", [dict(softcap=30.0), dict(window=1), dict(window=100),
                                  dict(window=140, softcap=50.0, alibi=True), dict(alibi=True), dict(pre=True),
                                  dict(pre=True, window=18), dict(scale=0.5), dict(scale=-0.1), dict(strided=True),
                                  dict(gone=True), dict(odd=True), dict(odd=True, window=30)])
def test_prompt_masks_and_biases(torch, opts, e4m3, dtype):
    """Masks on whole tiles and inside them, pages that are not resident, NaN that only some rows see."""
    opts = dict(opts)
    rng = np.random.default_rng(len(opts) + e4m3)
    new, lens = [200, 40, 150], [330, 600, 150]
    if opts.pop("pre", False):
        opts["prefix"] = [290, 40, 150]
    cache = Cache(torch, rng, lens, 2, 16, 128, e4m3)
    cache.fill(rng, lens)
    if opts.pop("gone", False):
        cache.table[0, 2:5] = -1
        cache.table[0, 8:16] = 1 << 20
        cache.table[2, :] = -1
    if opts.pop("odd", False):
        nan = 0x7F if e4m3 else float("nan")
        for s, j in ((0, 250), (0, 140), (1, 570), (2, 0)):
            cache.v[int(cache.table[s, j // 16]), s % 2, j % 16, 3:70] = nan
        cache.k[int(cache.table[2, 6]), 1, 7, 5] = nan
    attend(torch, cache, lens, new, 4, dtype, 53, **opts)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prompt_of_blocks_of_very_different_scales(torch, dtype):
    rng = np.random.default_rng(54)
    lens = [500, 260]
    cache = Cache(torch, rng, lens, 2, 16, 128, True)
    cache.fill(rng, lens, exps=1)
    cache.vs.copy_(torch.from_numpy((2.0 ** rng.integers(-8, 5, tuple(cache.vs.shape))).astype(np.float32)).cuda())
    attend(torch, cache, lens, [60, 200], 4, dtype, 55)
    cache.vs.copy_(torch.from_numpy(rng.uniform(0.01, 0.3, tuple(cache.vs.shape)).astype(np.float32)).cuda())
    cache.ks.copy_(torch.from_numpy((rng.integers(0, 5, tuple(cache.ks.shape)) * 0.03).astype(np.float32)).cuda())
    attend(torch, cache, lens, [60, 200], 4, dtype, 55)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,ctx,heads,n_kv", [(300, 2900, 4, 2), (40, 5000, 8, 2), (1024, 1024, 16, 8)])
def test_long_prompts_keep_f32_precision(torch, new, ctx, heads, n_kv, e4m3):
    """Thousands of keys a row: the relative error (2-norm) of f32 results stays that of f32 sums. Half a unit of 2^-24 at
    each of the 64 steps between two sums of the tensor core's accumulator and 22 bits of queries and weights: 3e-6."""
    rng = np.random.default_rng(ctx)
    cache = Cache(torch, rng, [new + ctx], n_kv, 64, 128, e4m3)
    from nekochat_b200 import ops
    cache.fill(rng, [new + ctx])
    q = torch.randn((new, heads, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(7))
    i = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.paged_attention(q, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), i(new + ctx), k_scale=cache.ks,
                              v_scale=cache.vs, q_start=i(0, new), max_new=new).double()
    kv, vv = (torch.from_numpy(x).cuda()[torch.from_numpy(cache.table[0]).long().cuda()].transpose(0, 1).reshape(n_kv, -1, 128)[:, :new + ctx]
              for x in cache.values())
    see = torch.arange(new + ctx, device="cuda")[None] <= ctx + torch.arange(new, device="cuda")[:, None]
    for h in range(heads):
        z = torch.where(see, q[:, h].double() @ kv[h * n_kv // heads].T * 128 ** -0.5, -torch.inf)
        want = torch.softmax(z, -1) @ vv[h * n_kv // heads]
        assert (got[:, h] - want).norm() <= 3e-6 * want.norm()


@pytest.mark.parametrize("n,L,heads,n_kv,hd", [(48, 9000, 16, 8, 128), (1, 30000, 8, 2, 128), (60, 5000, 12, 12, 64)])
def test_long_steps_keep_f32_precision(torch, n, L, heads, n_kv, hd):
    """Single tokens over long contexts: 22-bit products and sums rounded to nearest, an error of 1.5e-6 (2-norm) at most."""
    from nekochat_b200 import ops
    g = torch.Generator("cuda").manual_seed(9)
    P = -(-L // 64)
    k, v = (torch.randn((n * P, n_kv, 64, hd), device="cuda", generator=g, dtype=torch.float16) for _ in range(2))
    q = torch.randn((n, heads, hd), device="cuda", generator=g)
    table = torch.randperm(n * P, device="cuda", generator=g).int().view(n, P)
    got = ops.paged_attention(q, k, v, table, torch.full((n,), L, dtype=torch.int32, device="cuda")).double()
    for s in (0, n // 2, n - 1):
        kk, vv = (x[table[s].long()].double().transpose(0, 1).reshape(n_kv, -1, hd)[:, :L] for x in (k, v))
        for h in range(heads):
            want = torch.softmax(kk[h * n_kv // heads] @ q[s, h].double() * hd ** -0.5, -1) @ vv[h * n_kv // heads]
            assert (got[s, h] - want).norm() <= 1.5e-6 * want.norm()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
def test_prompts_whose_keys_are_split(torch, dtype, e4m3):
    """Few row tiles on thousands of keys: the keys of a row tile go to several CTAs, which join."""
    rng = np.random.default_rng(61)
    cache = Cache(torch, rng, [1900], 2, 32, 128, e4m3)
    cache.fill(rng, [1900])
    if e4m3:
        cache.vs.copy_(torch.from_numpy((2.0 ** rng.integers(-8, 5, tuple(cache.vs.shape))).astype(np.float32)).cuda())
    attend(torch, cache, [1900], [150], 8, dtype, 62)
    attend(torch, cache, [1900], [150], 8, dtype, 62, window=700, softcap=20.0, prefix=[100])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
def test_a_few_tokens_of_many_short_contexts(torch, dtype, e4m3):
    """More row tiles than SMs on a page or two each, of ragged lengths."""
    rng = np.random.default_rng(63)
    new = [int(x) for x in rng.integers(0, 10, 112)]
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 60, 112))]
    cache = Cache(torch, rng, lens, 4, 64, 128, e4m3)
    cache.fill(rng, lens)
    attend(torch, cache, lens, new, 12, dtype, 64, softcap=30.0, alibi=True)
