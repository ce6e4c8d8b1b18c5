"""The paged operators where arguments, values and lengths are at their ends: what is left out is reported, what is not seen
has no effect, and memory outside is not touched. Definitions in 64 bits: paged_reference.py."""
import numpy as np
import pytest

from tests import paged_reference as ref
from tests.test_gpu_paged import Cache, append, attend, fresh_rows, starts  # noqa: F401

pytestmark = pytest.mark.gpu
ROUND = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def ints(torch, *a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def native():
    from nekochat_b200 import model, workload
    s = workload.shape("qwen3-tiny")
    m = model.Model(s, 1, context=64, max_seqs=1, max_rows=16).load(workload.weights(s, 0, True))
    yield m
    m.close()


@pytest.mark.parametrize("rows", [3, 40])
def test_rows_left_out_are_reported_to_who_asks(torch, native, rows):
    """A sequence with more rows than max_new, and positions past the rotation table: the operators' own status says so,
    once, and a model's steps do not fail for it."""
    from nekochat_b200 import NekoError, ops, workload
    ops.status()
    rng = np.random.default_rng(rows)
    cache = Cache(torch, rng, [rows], 2, 16, 64, False)
    table = torch.from_numpy(cache.table).cuda()
    q, k, v = fresh_rows(torch, rng, rows, 4, 2, 64, torch.float32)
    held = dict(q_start=ints(torch, 0, rows))
    calls = [lambda: ops.paged_append(k, v, cache.k, cache.v, table, ints(torch, 0), max_new=rows - 1, **held),
             lambda: ops.paged_append(k, v, cache.k, cache.v, table, ints(torch, 0), max_new=rows, q=q,
                                      cs=ops.rope_table(rows - 1, 64, 1e4), **held),
             lambda: ops.paged_attention(q, cache.k, cache.v, table, ints(torch, rows), max_new=rows - 1, **held),
             lambda: ops.paged_attention(q[:-1], cache.k, cache.v, table, ints(torch, rows), max_new=rows, **held)]
    for call in calls:
        call()
        native.forward(workload.prompt(workload.shape("qwen3-tiny"), 3), 0)
        with pytest.raises(NekoError, match="max_new"):
            ops.status()
        ops.status()


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("at", [2 ** 31 - 2, 2 ** 31 - 40, 2 ** 30, 2 ** 30 + 1])
def test_starts_past_every_table(torch, at, e4m3, n):
    """Positions that do not fit 31 bits: nothing is read from before the rotation table, nothing is stored, the queries are
    what they are without a rotation, and the status says so."""
    from nekochat_b200 import NekoError, ops
    rng = np.random.default_rng(122)
    cache = Cache(torch, rng, [9, 50], 2, 16, 64, e4m3)
    cache.fill(rng, [9, 50])
    q, k, v = fresh_rows(torch, rng, n, 4, 2, 64, torch.float32)
    gain = torch.rand(64, device="cuda") + 0.5
    args = dict(k_scale=cache.ks, v_scale=cache.vs, q_start=ints(torch, 0, n, n), max_new=n, q=q, q_gain=gain, k_gain=gain)
    table, start = torch.from_numpy(cache.table).cuda(), ints(torch, at, 50)
    before = [x.clone() for x in (cache.k, cache.v) + ((cache.ks, cache.vs) if e4m3 else ())]
    plain = ops.paged_append(k, v, cache.k, cache.v, table, start, **args)
    ops.status()
    turned = ops.paged_append(k, v, cache.k, cache.v, table, start, cs=ops.rope_table(600, 64, 1e4), **args)
    with pytest.raises(NekoError, match="positions past the rotation table"):
        ops.status()
    want = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * gain
    for got in (plain, turned):
        assert ((got - want).abs() <= 2e-6 * want.abs().amax(-1, keepdim=True)).all()
    for x, y in zip(before, (cache.k, cache.v, cache.ks, cache.vs)):
        assert torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8))


def exact(torch, cache, q, lens, new, scale, softcap=0.0, window=0, slopes=None, prefix=None):
    """The definition in 64 bits, and for each row and head what its rounding errors are measured by: mass = sum_j p_j |v_j| per value
    and reach = max_j sum_d |q_d k_jd| scale."""
    pages, n_kv, ps, hd = cache.k.shape
    if cache.e4m3:
        code = torch.from_numpy(ref.E4M3).cuda()
        k, v = (code[x.view(torch.uint8).long()] * s[:, :, None, None].double() for x, s in ((cache.k, cache.ks), (cache.v, cache.vs)))
    else:
        k, v = cache.k.double(), cache.v.double()
    table = torch.from_numpy(cache.table).cuda().long()
    out, mass = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    reach = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    G = q.shape[1] // n_kv
    at = 0
    for s, (L, n) in enumerate(zip(lens, new)):
        rows, at = slice(at, at + n), at + n
        L_ = min(L, table.shape[1] * ps)
        if n == 0 or L_ <= 0:
            continue
        t = table[s, :-(-L_ // ps)]
        held = ((t >= 0) & (t < pages)).repeat_interleave(ps)[:L_]
        j, pos = torch.arange(L_, device="cuda")[None], (L - n + torch.arange(n, device="cuda"))[:, None]
        see = (j <= pos) & ((pos - j < window) if window else True)
        if prefix is not None:
            see = see | (j < prefix[s])
        see = see & held[None]
        for h in range(q.shape[1]):
            kk, vv = (x[t.clamp(0, pages - 1), h // G].reshape(-1, hd)[:L_] for x in (k, v))
            kk, vv = (torch.where(see.any(0)[:, None], x, 0.0) for x in (kk, vv))
            qq = q[rows, h].double()
            z = qq @ kk.T * scale
            reach[rows, h] = torch.where(see, qq.abs() @ kk.abs().T * abs(scale), 0).amax(1)
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            if slopes is not None:
                z = z + slopes[h].double() * (j - pos)
            z = torch.where(see, z, -torch.inf)
            p = torch.softmax(z, 1).nan_to_num(0.0)
            out[rows, h], mass[rows, h] = p @ vv, p @ vv.abs()
    return out, mass, reach


def bound(dtype, want, mass, reach, softcap=0.0):
    """What a row's arithmetic may be off by. Scores: 22 bits of q, sums of hd / 16 steps, together 2^-20 of reach; a cap 2^-21 of
    itself; exponentials, hi + lo weights and the sums 2^-18 of mass (16-bit rows: weights to f16, 2^-11). The output's rounding
    2^-11 (f16) or 2^-8 (bf16) of itself, f16 subnormals 2^-25."""
    rel = 2.0 ** -20 * reach[..., None] + 2.0 ** -21 * softcap + (2.0 ** -18 if dtype == "float32" else 2.0 ** -11 + 2.0 ** -16)
    return rel * mass + ROUND[dtype] * want.abs() + (2.0 ** -25 if dtype == "float16" else 0.0)


def held_to(torch, cache, lens, new, heads, dtype, seed, q_scale=1.0, q=None, softcap=0.0, window=0, alibi=False, prefix=None, max_new=None,
            scale=None):
    """One call, every value within bound()."""
    from nekochat_b200 import ops
    g = torch.Generator("cuda").manual_seed(seed)
    hd = cache.k.shape[3]
    if q is None:
        q = torch.randn((int(sum(new)), heads, hd), device="cuda", generator=g) * q_scale
    q = q.to(getattr(torch, dtype))
    slopes = (2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads)) if alibi else None
    got = ops.paged_attention(q, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, *lens), k_scale=cache.ks,
                              v_scale=cache.vs, q_start=ints(torch, *starts(new).tolist()), max_new=max_new or max(new), softcap=softcap,
                              window=window, slopes=slopes, prefix=None if prefix is None else ints(torch, *prefix), scale=scale)
    ops.status()
    want, mass, reach = exact(torch, cache, q, lens, new, hd ** -0.5 if scale is None else scale, softcap, window, slopes, prefix)
    off = (got.double() - want).abs()
    far = ~(off <= bound(dtype, want, mass, reach, softcap))
    assert not far.any(), f"{int(far.sum())} of {far.numel()} values, the worst off by {off[far].max().item():.3g} at {far.nonzero()[0].tolist()}"
    return got, want


def quantize(torch, cache, k, v):
    """Normal values into the cache's pages ([pages][n_kv][ps][hd] f32): f16, or codes with the append's scales."""
    if not cache.e4m3:
        cache.k.copy_(k), cache.v.copy_(v)
        return
    for x, pool, sc in ((k, cache.k, cache.ks), (v, cache.v, cache.vs)):
        e = torch.ceil(torch.log2(x.abs().amax((2, 3)).double() / 448)).clamp(min=-100)
        sc.copy_(torch.exp2(e).float())
        pool.copy_((x / sc[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8))


@pytest.mark.parametrize("hd", [32, 128])
@pytest.mark.parametrize("max_new", [1000, 1 << 24, 2 ** 31 - 1])
def test_a_loose_limit_of_new_tokens(torch, hd, max_new):
    """max_new far above what any sequence has: the same results."""
    rng = np.random.default_rng(116)
    new, lens = [40, 1, 7], [60, 200, 7]
    cache = Cache(torch, rng, lens, 2, 16, hd, False)
    cache.fill(rng, lens)
    held_to(torch, cache, lens, new, 8, "float32", 117, max_new=max_new)


@pytest.mark.parametrize("max_new", [1 << 24, 2 ** 31 - 1])
def test_a_loose_limit_of_appended_tokens(torch, max_new):
    """max_new far above what any sequence has: the pages and queries of a tight one, to the last bit."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(123)
    new, at = [40, 1, 7], [20, 199, 0]
    q, k, v = fresh_rows(torch, rng, sum(new), 4, 2, 64, torch.float32)
    cs, outs = ops.rope_table(300, 64, 1e4), []
    for limit in (40, max_new):
        cache = Cache(torch, np.random.default_rng(1), [a + n for a, n in zip(at, new)], 2, 16, 64, False)
        outs.append((ops.paged_append(k, v, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, *at),
                                      q_start=ints(torch, *starts(new).tolist()), max_new=limit, q=q, cs=cs), cache.k.nan_to_num(9), cache.v.nan_to_num(9)))
        ops.status()
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("max_new", [1, 9])
def test_one_row_with_any_stride(torch, max_new):
    """The token stride of a single row: 2^24 and more, as a dimension of one may have it."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(124)
    outs = []
    q, k, v = fresh_rows(torch, rng, 1, 4, 2, 64, torch.float32)
    far = lambda x: x.as_strided(x.shape, (1 << 33, x.stride(1), 1))  # noqa: E731
    for f in (lambda x: x, far):
        cache = Cache(torch, np.random.default_rng(1), [30], 2, 16, 64, False)
        outs.append((ops.paged_append(f(k), f(v), cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, 29), q_start=ints(torch, 0, 1),
                                      max_new=max_new, q=f(q), q_out=f(torch.empty_like(q))).clone(), cache.k.nan_to_num(9), cache.v.nan_to_num(9)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("softcap,q_scale", [(30.0, 1.0), (0.5, 1.0), (2.0, 50.0)])
@pytest.mark.parametrize("new,lens", [([3, 1, 2], [60, 70, 20]), ([200, 40, 150], [330, 600, 150])])
def test_scores_that_are_not_numbers_stay_so_under_a_cap(torch, new, lens, softcap, q_scale, e4m3, dtype):
    """tanh(NaN) is NaN: rows that see such a key give NaN, whatever the other scores are, and no other row does."""
    rng = np.random.default_rng(81)
    cache = Cache(torch, rng, lens, 2, 16, 128, e4m3)
    cache.fill(rng, lens)
    nan = 0x7F if e4m3 else float("nan")
    for s, j in ((0, lens[0] - 2), (2, lens[2] - 1)):
        cache.k[int(cache.table[s, j // 16]), s // 2, j % 16, 5] = nan
    got, want = attend(torch, cache, lens, new, 4, dtype, 82, softcap=softcap, q_scale=q_scale)
    assert np.isnan(want).any() and np.isfinite(want).any()


@pytest.mark.parametrize("n", [1, 9, 200])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_a_query_that_is_not_a_number(torch, n, softcap):
    """Its row and head are NaN, with and without a cap; the rows beside it are not."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(83)
    cache = Cache(torch, rng, [300], 2, 16, 128, False)
    cache.fill(rng, [300])
    q = torch.randn((n, 4, 128), device="cuda")
    q[n // 2, 1, 77] = float("nan")
    got = ops.paged_attention(q, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, 300),
                              q_start=ints(torch, 0, n), max_new=n, softcap=softcap)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[n // 2, 1] = True
    assert torch.equal(got.isnan(), bad)


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_that_do_not_turn_stay_apart(torch, dtype, interleaved, e4m3, n):
    """Infinities and NaN in the part of a head that a rotation leaves alone change no other value, in the steps' kernel and
    the prompts', and those in a pair reach that pair alone. f32 arithmetic, one rounding: 2e-6 of the row's largest finite
    value and half a unit of the type; 8-bit codes are as the definition's but for ties within that (none at these values)."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(84)
    hd, rot, start = 64, 32, 5
    cache = Cache(torch, rng, [start + n], 2, 16, hd, e4m3)
    cache.fill(rng, [start])
    q, k, v = fresh_rows(torch, rng, n, 4, 2, hd, getattr(torch, dtype))
    for x in (q, k, v):
        x[1, 0, 40], x[1, 1, 50], x[2, 0, 63] = float("nan"), float("inf"), float("-inf")
        x[2, 1, 3] = float("inf")
        x[0, 1, 33] = float("inf")
    cs = ops.rope_table(100, rot, 1e4)
    f64 = lambda t: t.float().cpu().numpy().astype(np.float64)  # noqa: E731
    before, scales = cache.values(scaled=False), [f64(cache.ks), f64(cache.vs)] if e4m3 else [None, None]
    got = ops.paged_append(k, v, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, start), k_scale=cache.ks,
                           v_scale=cache.vs, q_start=ints(torch, 0, n), max_new=n, q=q, cs=cs, interleaved=interleaved)
    want = ref.append(f64(k), f64(v), *before, cache.table, [start], [0, n], *scales, f64(q), cs.cpu().numpy(), interleaved)

    def same(g, w, near):
        assert np.array_equal(np.isnan(g), np.isnan(w))
        assert np.array_equal(np.where(np.isinf(g), g, 0), np.where(np.isinf(w), w, 0))
        f = np.isfinite(w)
        top = np.where(f, np.abs(w), 0).max(-1, keepdims=True)
        assert (np.abs(g[f] - w[f]) <= (2e-6 * top + near * np.where(f, np.abs(w), 0))[f]).all()

    same(f64(got), want, 0 if dtype == "float32" else 2.0 ** -8)
    for g, w in zip(cache.values(scaled=False), before):
        same(g, w, 2.0 ** -3 if e4m3 else 2.0 ** -11)


@pytest.mark.parametrize("new,lens", [([6, 1], [3, 40]), ([100, 1], [60, 300])])
def test_a_window_that_leaves_nothing_out(torch, new, lens):
    """The largest window there is gives what no window gives, also where positions are negative."""
    rng = np.random.default_rng(110)
    cache = Cache(torch, rng, lens, 2, 16, 128, False)
    cache.fill(rng, lens)
    a, _ = held_to(torch, cache, lens, new, 4, "float32", 111)
    b, _ = held_to(torch, cache, lens, new, 4, "float32", 111, window=2 ** 31 - 1)
    assert (a - b).abs().max() <= 1e-5 * a.abs().max()


def free(torch):
    torch.cuda.synchronize()
    return torch.cuda.mem_get_info()[0]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n,ctx", [(2500, 0), (1200, 3000)])
def test_prompts_on_heads_of_32(torch, n, ctx, e4m3):
    rng = np.random.default_rng(112)
    cache = Cache(torch, rng, [n + ctx, 77], 2, 64, 32, e4m3)
    g = torch.Generator("cuda").manual_seed(113)
    quantize(torch, cache, *(torch.randn(cache.k.shape, device="cuda", generator=g) for _ in range(2)))
    for dtype in ("float32", "bfloat16"):
        held_to(torch, cache, [n + ctx, 77], [n, 77], 6, dtype, 114)


@pytest.mark.parametrize("n,dtype", [(8192, "float32"), (66000, "float32"), (140000, "bfloat16")])
def test_long_prompts_on_heads_of_32_take_little_scratch_memory(torch, n, dtype):
    """More row tiles than a grid's second dimension counts, with at most 256 MiB of scratch memory; some rows against the
    definition (a window keeps the time short)."""
    from nekochat_b200 import ops
    heads, ps, window = 8, 128, 500
    g = torch.Generator("cuda").manual_seed(115)
    pages = -(-n // ps)
    k, v = (torch.randn((pages, 1, ps, 32), device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn((n, heads, 32), device="cuda", generator=g).to(getattr(torch, dtype))
    table = torch.randperm(pages, device="cuda", generator=g).int()[None]
    out = torch.empty_like(q)
    before = free(torch)
    ops.paged_attention(q, k, v, table, ints(torch, n), q_start=ints(torch, 0, n), max_new=n, window=window, out=out)
    ops.status()
    assert before - free(torch) <= 256 << 20
    kk, vv = (x[table[0].long(), 0].reshape(-1, 32)[:n].double() for x in (k, v))
    for i in (0, 1, 499, 500, n // 3, n - 1):
        lo = max(0, i - window + 1)
        z = kk[lo:i + 1] @ q[i].double().T * 32 ** -0.5
        p = torch.softmax(z, 0)
        want, mass = (p.T @ x[lo:i + 1] for x in (vv, vv.abs()))
        reach = (kk[lo:i + 1].abs() @ q[i].double().abs().T * 32 ** -0.5).amax(0)
        assert ((out[i].double() - want).abs() <= bound(dtype, want, mass, reach)).all()


FORMS = {  # new tokens, length, query heads, KV heads, head dim
    "step": (1, 300, 4, 2, 128), "step, many keys": (1, 6000, 8, 2, 64), "verify": (7, 300, 8, 2, 128), "head dim 32": (30, 200, 4, 2, 32),
    "rows of a few tiles": (200, 300, 4, 2, 128),
    "prompt on keys": (60, 2500, 8, 2, 64), "prompt": (700, 800, 4, 2, 128), "prompt, heads of 64": (900, 1000, 4, 2, 64),
}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("form", FORMS)
def test_small_blocks_keep_their_bits_beside_large_ones(torch, form, dtype):
    """Blocks of values 2^-30 the size of their neighbours', which the softmax prefers by 2^-90: the result is theirs, in
    all its bits."""
    new, L, heads, n_kv, hd = FORMS[form]
    rng = np.random.default_rng(94)
    cache = Cache(torch, rng, [L], n_kv, 16, hd, True)
    g = torch.Generator("cuda").manual_seed(95)
    k, v = (torch.randn(cache.k.shape, device="cuda", generator=g) for _ in range(2))
    k[..., 0] = 0
    order = torch.from_numpy(cache.table[0]).cuda().long()
    k[order[1::2], :, :, 0] = -31.25  # times 2 of q: 62.5 less
    v[order[0::2]] *= 2.0 ** -30
    quantize(torch, cache, k, v)
    q = torch.randn((new, heads, hd), device="cuda", generator=g) * 0.1
    q[..., 0] = 2.0
    held_to(torch, cache, [L], [new], heads, dtype, 96, q=q, scale=1.0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,L,window", [(200, 330, 24), (9, 60, 5), (300, 300, 0), (700, 900, 24), (700, 700, 0)])
def test_blocks_that_a_row_does_not_see_take_none_of_its_bits(torch, new, L, window, dtype):
    """Values 2^40 larger in every fourth block: rows whose window or place leaves those out are exact in their own size."""
    rng = np.random.default_rng(97)
    cache = Cache(torch, rng, [L], 2, 16, 128, True)
    g = torch.Generator("cuda").manual_seed(98)
    k, v = (torch.randn(cache.k.shape, device="cuda", generator=g) for _ in range(2))
    v[torch.from_numpy(cache.table[0]).cuda().long()[3::4]] *= 2.0 ** 40
    quantize(torch, cache, k, v)
    held_to(torch, cache, [L], [new], 4, dtype, 99, window=window)


@pytest.mark.parametrize("new,L", [(1, 200), (100, 200), (700, 800)])
def test_values_at_the_ends_of_the_scales(torch, new, L):
    """All values about 2^-95, about 2^100, and blocks of zeros (scale 2^-100) beside others: relative to their own size."""
    rng = np.random.default_rng(100)
    for size in (2.0 ** -95, 2.0 ** 100, 0.0):
        cache = Cache(torch, rng, [L], 2, 16, 128, True)
        g = torch.Generator("cuda").manual_seed(101)
        k, v = (torch.randn(cache.k.shape, device="cuda", generator=g) for _ in range(2))
        if size:
            v *= size
        else:
            v[torch.from_numpy(cache.table[0]).cuda().long()[::2]] = 0
        quantize(torch, cache, k, v)
        held_to(torch, cache, [L], [new], 4, "float32", 102)


SHAPES = {  # what takes the call: new tokens, lengths, query heads, KV heads, head dim, page
    "one token, short": ([1] * 4, [1, 17, 500, 777], 16, 8, 128, 16),
    "one token, long": ([1] * 9, [9000, 1, 5000, 33, 700, 8191, 64, 4097, 128], 16, 2, 128, 64),
    "one token, wide heads": ([1] * 40, [300 + 41 * i for i in range(40)], 12, 12, 64, 32),
    "verify": ([5, 3, 9, 1], [2000, 3, 4100, 900], 8, 4, 128, 64),
    "head dim 32": ([7, 130, 1], [300, 130, 900], 8, 2, 32, 16),
    "chunk": ([64], [576], 16, 8, 128, 16),
    "prompts": ([300, 41, 257, 1], [300, 900, 800, 650], 12, 4, 128, 64),
    "prompts, narrow heads": ([200, 129], [1500, 129], 6, 2, 64, 128),
    "a prompt among steps": ([500] + [1] * 12, [900] + [50 + 97 * i for i in range(12)], 8, 2, 128, 64),
}


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("opts", [dict(), dict(softcap=20.0, window=150, alibi=True), dict(window=70, prefix=True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_value_within_its_own_bound(torch, shape, opts, e4m3, dtype):
    """Normal keys and values, 8-bit ones quantized as the append does: a wrong head, key range, window's edge or scale moves an
    output by its own size, and the bounds are 2 to 3 orders below that."""
    new, lens, heads, n_kv, hd, ps = SHAPES[shape]
    opts = dict(opts)
    if opts.pop("prefix", False):
        opts["prefix"] = [max(0, x // 2 - 5) for x in lens]
    rng = np.random.default_rng(91)
    cache = Cache(torch, rng, lens, n_kv, ps, hd, e4m3)
    g = torch.Generator("cuda").manual_seed(92)
    k, v = (torch.randn(cache.k.shape, device="cuda", generator=g) * torch.exp(0.5 * torch.randn((cache.k.shape[0], n_kv, ps, 1), device="cuda", generator=g))
            for _ in range(2))
    quantize(torch, cache, k, v)
    held_to(torch, cache, lens, new, heads, dtype, 93, **opts)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new,L,page_gone", [(700, 128, False), (700, 100, False), (100, 60, False), (7, 3, False), (150, 150, True), (1, 40, True)])
def test_rows_that_see_nothing_beside_rows_that_do(torch, new, L, page_gone, e4m3, dtype):
    """Zeros, not NaN, whatever the values' scale: positions before the first token, and pages that are gone."""
    rng = np.random.default_rng(107)
    cache = Cache(torch, rng, [L], 2, 16, 128, e4m3)
    g = torch.Generator("cuda").manual_seed(108)
    k, v = (torch.randn(cache.k.shape, device="cuda", generator=g) for _ in range(2))
    quantize(torch, cache, k, v if not e4m3 else v * 2.0 ** 17)
    if page_gone:
        cache.table[0, :3] = -1
    got, want = held_to(torch, cache, [L], [new], 4, dtype, 109)
    none = (want == 0).all(-1)
    assert none.any() and (got[none] == 0).all()


@pytest.mark.parametrize("new,heads,n_kv", [(1, 2, 1), (40, 2, 2)])
def test_many_small_weights_count(torch, new, heads, n_kv):
    """40,000 keys whose weights are 2^-29 of one key's: together 7.5e-5 of the result, which is within 2.5e-5 of the
    definition's."""
    L = 40000
    rng = np.random.default_rng(103)
    cache = Cache(torch, rng, [L], n_kv, 64, 128, False)
    k, v = torch.zeros(cache.k.shape, device="cuda"), torch.ones(cache.k.shape, device="cuda")
    k[int(cache.table[0, 0]), :, 0, 0] = 1.0
    quantize(torch, cache, k, v)
    q = torch.zeros((new, heads, 128), device="cuda")
    q[..., 0] = 29 * np.log(2.0)
    held_to(torch, cache, [L], [new], heads, "float32", 104, q=q, scale=1.0)


@pytest.mark.parametrize("dtype,L,hd,near", [("float32", 16384, 128, 1.5e-6), ("float32", 1100, 64, 1.5e-6), ("float16", 262144, 64, 0.0)])
def test_a_first_key_that_takes_all_weight(torch, dtype, L, hd, near):
    """The result is that key's value however many keys of no weight follow: for f32 within the two roundings of a weight's
    f16 halves, of the sum and of the quotient (together 1.5e-6), for f16, which that error does not reach, exactly."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(105)
    n = 64
    cache = Cache(torch, rng, [L], 1, 128, hd, False)
    g = torch.Generator("cuda").manual_seed(106)
    k, v = torch.zeros(cache.k.shape, device="cuda"), torch.randn(cache.k.shape, device="cuda", generator=g)
    first = int(cache.table[0, 0])
    k[first, :, 0, 0] = 8.0
    quantize(torch, cache, k, v)
    q = torch.zeros((n, 2, hd), device="cuda", dtype=getattr(torch, dtype))
    q[..., 0] = 16.0  # the others' weights are e^-128 of the first's
    got = ops.paged_attention(q, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, L), q_start=ints(torch, 0, n), max_new=n, scale=1.0)
    want = cache.v[first, 0, 0].double().expand(n, 2, hd)
    assert ((got.double() - want).abs() <= near * want.abs()).all(), ((got.double() - want) / want).abs().max()


def test_f32_precision_of_more_prompts_than_run_at_once(torch):
    """8,800 row tiles of 16,384 keys (one sequence's pages, shared): sums kept outside the tensor cores for those that run, at
    most 64 MiB in all, and the error of every row as small as for few (2-norm, 3e-6)."""
    from nekochat_b200 import ops
    n_seq, n, L, n_kv, ps = 1100, 32, 16384, 8, 128
    g = torch.Generator("cuda").manual_seed(125)
    k, v = (torch.randn((L // ps, n_kv, ps, 128), device="cuda", generator=g).half() for _ in range(2))
    q = torch.randn((n_seq * n, n_kv, 128), device="cuda", generator=g)
    table = torch.randperm(L // ps, device="cuda", generator=g).int().repeat(n_seq, 1)
    out = torch.empty_like(q)
    before = free(torch)
    ops.paged_attention(q, k, v, table, torch.full((n_seq,), L, dtype=torch.int32, device="cuda"),
                        q_start=torch.arange(0, n_seq * n + 1, n, dtype=torch.int32, device="cuda"), max_new=n, out=out)
    ops.status()
    assert before - free(torch) <= 64 << 20
    see = torch.arange(L, device="cuda")[None] <= (L - n + torch.arange(n, device="cuda"))[:, None]
    for h in (0, 5):
        kk, vv = (x[table[0].long(), h].reshape(L, 128).double() for x in (k, v))
        for s in (0, 1, 147, 148, 600, n_seq - 1):
            rows = slice(s * n, s * n + n)
            want = torch.softmax(torch.where(see, q[rows, h].double() @ kk.T * 128 ** -0.5, -torch.inf), -1) @ vv
            assert (out[rows, h] - want).norm() <= 3e-6 * want.norm()


@pytest.mark.parametrize("new,lens", [([1] * 3, [700, 3000, 65]), ([300, 5], [2000, 900])])
def test_calls_in_a_graph(torch, new, lens):
    """Append and attention captured once and replayed on other inputs: the bits of the calls themselves."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(118)
    cache, other = (Cache(torch, np.random.default_rng(119), lens, 2, 64, 128, True, width=80) for _ in range(2))
    g = torch.Generator("cuda").manual_seed(120)
    for c in (cache, other):
        g.manual_seed(121)
        quantize(torch, c, *(torch.randn(c.k.shape, device="cuda", generator=g) for _ in range(2)))
    T = sum(new)
    q, k, v = fresh_rows(torch, rng, T, 8, 2, 128, torch.float32)
    cs = ops.rope_table(4000, 128, 1e6)
    at, n, qs, table = ints(torch, *[a - b for a, b in zip(lens, new)]), ints(torch, *lens), ints(torch, *starts(new).tolist()), torch.from_numpy(cache.table).cuda()

    def both(c):
        turned = ops.paged_append(k, v, c.k, c.v, table, at, k_scale=c.ks, v_scale=c.vs, q_start=qs, max_new=max(new), q=q, cs=cs)
        return ops.paged_attention(turned, c.k, c.v, table, n, k_scale=c.ks, v_scale=c.vs, q_start=qs, max_new=max(new))

    both(other)
    for x, y in ((other.k, cache.k), (other.v, cache.v), (other.ks, cache.ks), (other.vs, cache.vs)):
        x.copy_(y)  # scales and codes go by what a page has held
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = both(cache)
    for turn in range(3):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        graph.replay()
        want = both(other)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(cache.k, other.k) and torch.equal(cache.vs, other.vs)
    ops.status()


@pytest.mark.parametrize("new,L", [(1, 50), (700, 800)])
@pytest.mark.parametrize("size,scale", [(2.0 ** 125, 2.0 ** -125), (2.0 ** -135, 2.0 ** 125)])
def test_queries_at_the_ends_of_f32(torch, size, scale, new, L):
    """Rows whose largest magnitude is above 2^127 or subnormal, brought back by the scale."""
    rng = np.random.default_rng(126)
    cache = Cache(torch, rng, [L], 2, 16, 128, False)
    g = torch.Generator("cuda").manual_seed(127)
    k, v = (torch.randn(cache.k.shape, device="cuda", generator=g) for _ in range(2))
    quantize(torch, cache, k * 0.05, v)
    q = torch.randn((new, 4, 128), device="cuda", generator=g).clamp(-7, 7)
    q[..., 3] = 7.5
    held_to(torch, cache, [L], [new], 4, "float32", 128, q=(q.double() * size).float(), scale=scale)


def test_scratch_memory_is_given_back_when_asked(torch):
    """f16 copies of a long 8-bit cache's pages (491 MB) stay with the library until trim; calls after it work as before."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(129)
    lens, new = [120000], [300]
    cache = Cache(torch, rng, lens, 8, 128, 128, True)
    g = torch.Generator("cuda").manual_seed(130)
    cache.k.copy_(torch.randint(0, 100, cache.k.shape, device="cuda", generator=g, dtype=torch.uint8))
    cache.v.copy_(cache.k)
    cache.ks.fill_(0.01), cache.vs.fill_(0.01)
    q = torch.randn((300, 16, 128), device="cuda", generator=g)
    call = lambda: ops.paged_attention(q, cache.k, cache.v, torch.from_numpy(cache.table).cuda(), ints(torch, *lens), k_scale=cache.ks,  # noqa: E731
                                       v_scale=cache.vs, q_start=ints(torch, 0, 300), max_new=300, out=out)
    out = torch.empty_like(q)
    ops.trim()
    call()
    held, first = free(torch), out.clone()
    ops.trim()
    assert free(torch) - held >= 450 << 20
    call()
    torch.cuda.synchronize()
    assert torch.equal(out, first)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("form", FORMS)
def test_large_values_of_small_weight_count(torch, form, dtype):
    """Blocks of values 2^45 the size of their neighbours', whose keys' weights are 2^-43 of theirs: both make up the result."""
    new, L, heads, n_kv, hd = FORMS[form]
    rng = np.random.default_rng(131)
    cache = Cache(torch, rng, [L], n_kv, 16, hd, True)
    g = torch.Generator("cuda").manual_seed(132)
    k, v = (torch.randn(cache.k.shape, device="cuda", generator=g) for _ in range(2))
    k[..., 0] = 0
    order = torch.from_numpy(cache.table[0]).cuda().long()
    k[order[1::2], :, :, 0] = -15.0  # times 2 of q: 30 less
    v[order[1::2]] *= 2.0 ** 45
    quantize(torch, cache, k, v)
    q = torch.randn((new, heads, hd), device="cuda", generator=g) * 0.1
    q[..., 0] = 2.0
    held_to(torch, cache, [L], [new], heads, dtype, 133, q=q, scale=1.0)


def test_a_prompt_on_a_gpu_that_the_cache_fills(torch):
    """Where there is no room for f16 copies of an 8-bit cache's pages (491 MB here), the call does without."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(134)
    lens, new = [120000], [300]
    cache = Cache(torch, rng, lens, 8, 128, 128, True)
    g = torch.Generator("cuda").manual_seed(135)
    cache.k.copy_(torch.randint(0, 100, cache.k.shape, device="cuda", generator=g, dtype=torch.uint8))
    cache.v.copy_(cache.k)
    cache.ks.fill_(0.01), cache.vs.fill_(0.01)
    q = torch.randn((300, 16, 128), device="cuda", generator=g)
    table, out = torch.from_numpy(cache.table).cuda(), torch.empty_like(q)

    def call(n, L):
        ops.paged_attention(q[:n], cache.k, cache.v, table[:, :-(-L // 128)], ints(torch, L), k_scale=cache.ks, v_scale=cache.vs,
                            q_start=ints(torch, 0, n), max_new=n, out=out[:n])

    call(60, 4000)  # one row tile: the kernel without copies is loaded
    call(300, lens[0])
    want = out.clone()
    torch.cuda.synchronize()
    ops.trim()
    torch.cuda.empty_cache()
    full = torch.empty(torch.cuda.mem_get_info()[0] - (300 << 20), dtype=torch.uint8, device="cuda")
    out.zero_()
    call(300, lens[0])
    torch.cuda.synchronize()
    del full
    torch.cuda.empty_cache()
    assert (out - want).abs().max() <= 2e-6 * want.abs().max()
