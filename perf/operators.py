"""Cases of the paged key/value cache operators: appending a step's or a prompt's keys and values (with the query /
key norm and the position rotation on the way) and attention over the cached pages.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes what a serving program
holds before the call, ``run()`` is one call (the library's operator where ``own`` is true, elementary torch operations
in 32 bits otherwise), ``exact()`` the same from the definition in 64 bits and ``work()`` its bytes and operations.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0
SCALE_MIN_EXP = -100

BASE = dict(dtype="f32", cache="f16", n_seq=1, new_lo=1, new_hi=1, ctx_lo=512, ctx_hi=512, heads=16, kv_heads=8,
            hd=128, page=16, norm=False, rot=0, interleaved=False, softcap=0.0, window=0, alibi=False, prefix=0)


def case(name, op, **kw):
    return dict(BASE, name=name, op=op, **kw)


def listed():
    return [
        # One chat, one new token: the smallest call of a decode step. Qwen3-0.6B heads, f16 cache.
        case("append 1x1 f16", "append", ctx_lo=777, ctx_hi=777, norm=True, rot=128),
        # 64 chats, one new token each, at ragged positions inside their 64-token blocks, 8-bit cache.
        case("append 64x1 e4m3", "append", cache="e4m3", n_seq=64, ctx_lo=100, ctx_hi=1000, page=64, norm=True,
             rot=128),
        # Prompts of several chats in one call (ragged), 16-bit activations, 8-bit cache, Qwen3-4B heads.
        case("append prompts e4m3", "append", dtype="bf16", cache="e4m3", n_seq=12, new_lo=333, new_hi=1777, ctx_lo=0,
             ctx_hi=100, heads=32, page=64, norm=True, rot=128),
        # One long prompt on 64-wide heads, no norm, part of each head rotated in interleaved pairs, f16 cache.
        case("append prompt partial", "append", new_lo=4001, new_hi=4001, ctx_lo=0, ctx_hi=0, heads=12, kv_heads=12,
             hd=64, page=32, rot=48, interleaved=True),
        # One chat, one new token after a 512-token prompt and a reply: the latency case of a decode step.
        case("decode 1x777 f16", "attention", ctx_lo=776, ctx_hi=776),
        # One chat deep into a long context on an 8-bit cache (40,000 of Qwen3's 40,960 positions).
        case("decode 1x40000 e4m3", "attention", cache="e4m3", ctx_lo=39999, ctx_hi=39999, heads=32, page=64),
        # A batched decode step, 64 chats of about the benchmark's length, 8-bit cache.
        case("decode 64x700 e4m3", "attention", cache="e4m3", n_seq=64, ctx_lo=300, ctx_hi=1100, page=64),
        # The largest batched step: 128 ragged contexts up to 8192 tokens, 16-bit activations.
        case("decode 128x8192 e4m3", "attention", dtype="bf16", cache="e4m3", n_seq=128, ctx_lo=900, ctx_hi=8191,
             heads=32, page=64),
        # Windowed, capped scores with a distance bias, one KV head per query head, 64-wide heads, f16 cache.
        case("decode 48 window cap alibi", "attention", dtype="f16", n_seq=48, ctx_lo=50, ctx_hi=5000, heads=12,
             kv_heads=12, hd=64, page=32, softcap=30.0, window=1024, alibi=True),
        # The engine's prompt chunk: 64 tokens against 512 that the cache already holds.
        case("chunk 64 on 512 f16", "attention", new_lo=64, new_hi=64, ctx_lo=512, ctx_hi=512),
        # A long prompt in one call, 16-bit activations: bound by the tensor cores.
        case("prompt 8192 bf16", "attention", dtype="bf16", new_lo=8192, new_hi=8192, ctx_lo=0, ctx_hi=0, page=64),
        # Ragged prompts with earlier turns in an 8-bit cache, a bidirectional prefix and capped scores.
        case("prompts on turns e4m3", "attention", cache="e4m3", n_seq=5, new_lo=129, new_hi=1501, ctx_lo=0,
             ctx_hi=2999, heads=32, page=64, softcap=50.0, prefix=200),
    ]


def spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    plain = max(plain_cells(c) for c in listed())
    while True:
        c = dict(BASE)
        c["op"] = rng.choice(["append", "attention", "attention"])
        c["dtype"] = rng.choice(["f32", "f32", "bf16", "f16"])
        c["cache"] = rng.choice(["f16", "e4m3"])
        c["page"] = rng.choice([16, 32, 64, 128])
        c["hd"] = rng.choice([64, 128, 128])
        c["kv_heads"] = rng.choice([1, 2, 4, 8, 8, 12])
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 2, 3, 4, 8])
        c["n_seq"] = spread(rng, 1, 150)
        kind = rng.choice(["step", "verify", "prompt"])
        top = {"step": 1, "verify": 9, "prompt": 4096}[kind]
        c["new_hi"] = 1 if top == 1 else spread(rng, 2 if kind == "verify" else 17, top)
        c["new_lo"] = rng.choice([c["new_hi"], max(1, c["new_hi"] // 3)])
        c["ctx_hi"] = spread(rng, 1, 20000) - 1
        c["ctx_lo"] = rng.choice([c["ctx_hi"], c["ctx_hi"] // 8])
        if c["op"] == "append":
            c["ctx_hi"] = min(c["ctx_hi"], 2000)
            c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])
            c["norm"] = rng.random() < 0.5
            c["rot"] = rng.choice([0, c["hd"], c["hd"], c["hd"] // 2, 3 * c["hd"] // 4])
            c["interleaved"] = rng.random() < 0.4
        else:
            c["softcap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
            c["window"] = rng.choice([0, 0, spread(rng, 16, 4096)])
            c["alibi"] = rng.random() < 0.25
            c["prefix"] = rng.choice([0, 0, 0, spread(rng, 1, 500)])
        w = work(c)
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and plain_cells(c) <= plain:
            return c


# ------------------------------------------------------------------------------------------------ sizes of a case
def spans(c):
    """[(tokens held before, new tokens)] of each sequence: spread evenly over the case's ranges, the same for every
    seed, the first sequence at the upper ends."""
    out = []
    for i in range(c["n_seq"]):
        f, g = (1.0 - i * 0.6180339887498949) % 1.0 or 1.0, (1.0 - i * 0.7548776662466927) % 1.0 or 1.0
        out.append((c["ctx_lo"] + round(f * (c["ctx_hi"] - c["ctx_lo"])),
                    c["new_lo"] + round(g * (c["new_hi"] - c["new_lo"]))))
    return out


def seen(c, ctx, new):
    """(keys that some query of the sequence sees, pairs of a query and a key it sees)."""
    win, pre, total = c["window"], min(c["prefix"], ctx + new), ctx + new
    first = max(0, ctx - win + 1) if win else 0
    keys = total - first + min(first, pre)
    if not win and not pre:
        return keys, new * ctx + new * (new + 1) // 2
    pairs = 0
    for p in range(ctx, total):
        lo = max(0, p - win + 1) if win else 0
        pairs += p + 1 - lo + min(lo, pre) + max(0, pre - p - 1)
    return keys, pairs


def work(c):
    """Queries, new keys and values read once, outputs written once, the keys and values that are seen read once."""
    H, KV, hd, a, b = c["heads"], c["kv_heads"], c["hd"], BYTES[c["dtype"]], BYTES[c["cache"]]
    tokens = sum(n for _, n in spans(c))
    if c["op"] == "append":
        return {"bytes": tokens * (2 * H * hd * a + 2 * KV * hd * (a + b) + 4 * c["rot"]),
                "flops": tokens * (H + KV) * ((4 * hd if c["norm"] else 0) + 3 * c["rot"])}
    keys = pairs = 0
    for ctx, n in spans(c):
        k, p = seen(c, ctx, n)
        keys, pairs = keys + k, pairs + p
    return {"bytes": 2 * tokens * H * hd * a + 2 * keys * KV * hd * b, "flops": 4 * pairs * H * hd}


def plain_cells(c):
    """Numbers that the plain form holds at its widest (padded scores, gathered keys)."""
    sp = spans(c)
    longest, rows = max(x + n for x, n in sp), max(n for _, n in sp)
    if c["op"] == "append":
        return sum(x + n for x, n in sp) * c["kv_heads"] * c["hd"]
    return c["n_seq"] * (longest + c["page"]) * max(rows * c["heads"], 2 * c["kv_heads"] * c["hd"])


# ------------------------------------------------------------------------------------------------ inputs
def quantized(x):
    """[pages][heads][page][hd] f32 as 8-bit codes and their power-of-two scales [pages][heads]."""
    m, e = torch.frexp(x.abs().amax(dim=(2, 3)) / E4M3_MAX)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=SCALE_MIN_EXP)
    scale = torch.ldexp(torch.ones_like(m), e)
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    H, KV, hd, ps, dt = c["heads"], c["kv_heads"], c["hd"], c["page"], DTYPES[c["dtype"]]
    sp = spans(c)
    n = len(sp)
    held = [-(-(x + t) // ps) for x, t in sp]
    pages = sum(held) + 1 + sum(held) // 16  # a pool with a few pages that nobody holds
    # keys have a few strong channels, values and keys a size that differs from token to token
    chan = torch.exp(0.5 * torch.randn((KV, 1, hd), generator=g, device=dev))

    def rows(count, strong):
        x = torch.randn((count, KV, ps, hd), generator=g, device=dev)
        x *= torch.exp(0.3 * torch.randn((count, KV, ps, 1), generator=g, device=dev))
        return x * chan if strong else x

    store = torch.float16 if c["cache"] == "f16" else torch.float8_e4m3fn
    s = {"case": c, "k_scale": None, "v_scale": None}
    for name, strong in (("k", True), ("v", False)):
        pool = torch.empty((pages, KV, ps, hd), dtype=store, device=dev)
        scale = torch.empty((pages, KV), device=dev) if c["cache"] == "e4m3" else None
        step = max(1, (1 << 26) // (KV * ps * hd))
        for b in range(0, pages, step):
            x = rows(min(step, pages - b), strong)
            if scale is None:
                pool[b:b + step] = x.half()
            else:
                codes, scale[b:b + step] = quantized(x)
                pool[b:b + step].view(torch.uint8).copy_(codes.view(torch.uint8))
        s[name + "_pages"] = pool
        if scale is not None:
            s[name + "_scale"] = scale
    # pages in the order that a pool hands them out after a while: none
    order = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((n, max(held)), -1, dtype=torch.int32)
    at = 0
    where = []
    for h in held:
        where.append((at, h))
        at += h
    order_host = order.cpu()
    for i, (b, h) in enumerate(where):
        table[i, :h] = order_host[b:b + h]
    s["table"] = table.to(dev)
    starts = [0]
    for _, t in sp:
        starts.append(starts[-1] + t)
    T = starts[-1]
    s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    s["start"] = torch.tensor([x for x, _ in sp], dtype=torch.int32, device=dev)
    s["kv_len"] = torch.tensor([x + t for x, t in sp], dtype=torch.int32, device=dev)
    s["max_new"] = max(t for _, t in sp)
    if c["op"] == "append":
        # the fused projection's output: q, k and v are column ranges of its rows
        qkv = torch.randn((T, (H + 2 * KV) * hd), generator=g, device=dev)
        qkv *= torch.exp(0.3 * torch.randn((T, 1), generator=g, device=dev))
        s["qkv"] = qkv.to(dt)
        s["gain_q"] = s["gain_k"] = s["cs"] = None
        if c["norm"]:
            s["gain_q"] = 1 + 0.1 * torch.randn(hd, generator=g, device=dev)
            s["gain_k"] = 1 + 0.1 * torch.randn(hd, generator=g, device=dev)
        if c["rot"]:
            half = c["rot"] // 2
            freq = 1e6 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
            ang = torch.arange(max(x + t for x, t in sp), device=dev, dtype=torch.float64)[:, None] * freq
            s["cs"] = torch.stack([ang.cos(), ang.sin()], -1).float()
    else:
        s["q"] = torch.randn((T, H, hd), generator=g, device=dev).to(dt)
        s["slopes"] = None
        if c["alibi"]:
            s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device=dev, dtype=torch.float32) / H)
        s["prefix"] = s["kv_len"].clamp(max=c["prefix"]) if c["prefix"] else None
    return s


def parts(s):
    """The q, k and v columns of the fused projection."""
    c = s["case"]
    H, KV, hd = c["heads"], c["kv_heads"], c["hd"]
    q, k, v = s["qkv"].split([H * hd, KV * hd, KV * hd], dim=1)
    return q.unflatten(1, (H, hd)), k.unflatten(1, (KV, hd)), v.unflatten(1, (KV, hd))


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    if c["op"] == "append":
        q, k, v = parts(s)
        if own:
            from nekochat_b200 import ops
            q = ops.paged_append(k, v, s["k_pages"], s["v_pages"], s["table"], s["start"], k_scale=s["k_scale"],
                                 v_scale=s["v_scale"], q_start=s["q_start"], max_new=s["max_new"], q=q, cs=s["cs"],
                                 interleaved=c["interleaved"], q_gain=s["gain_q"], k_gain=s["gain_k"])
        else:
            q = plain_append(s, q, k, v)
        return [q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]
    if own:
        from nekochat_b200 import ops
        return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], k_scale=s["k_scale"],
                                   v_scale=s["v_scale"], q_start=s["q_start"], max_new=s["max_new"],
                                   softcap=c["softcap"], window=c["window"], slopes=s["slopes"], prefix=s["prefix"])
    return plain_attention(s)


def rotated(x, gain, cs, pos, c, eps=1e-6):
    """Root-mean-square norm of each head (with `gain`), then the rotation of its first `rot` values."""
    x = x.float()
    if gain is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * gain
    if cs is None:
        return x
    r = c["rot"]
    cos, sin = cs[pos, :, 0][:, None], cs[pos, :, 1][:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., r:]], -1)


def plain_append(s, q, k, v):
    c = s["case"]
    ps = c["page"]
    T = q.shape[0]
    at = torch.arange(T, device=q.device)
    seq = torch.searchsorted(s["q_start"][1:].contiguous(), at.int(), right=True)
    pos = s["start"][seq] + at - s["q_start"][seq]
    page, off = s["table"][seq, pos // ps].long(), pos % ps
    out = rotated(q, s["gain_q"], s["cs"], pos, c).to(q.dtype)
    for x, name in ((rotated(k, s["gain_k"], s["cs"], pos, c), "k"), (v.float(), "v")):
        pool = s[name + "_pages"]
        if c["cache"] == "f16":
            pool[page, :, off] = x.half()
            continue
        # the scale of each (block, head) that gets tokens: the smallest power of two that holds them, and no smaller
        # than the scale of the tokens that the block held before
        scale = s[name + "_scale"]
        most = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
        m, e = torch.frexp(most / E4M3_MAX)
        e = torch.where(m == 0.5, e - 1, e).clamp(min=SCALE_MIN_EXP)
        fresh = torch.ldexp(torch.ones_like(m), e)
        first = s["table"].gather(1, (s["start"] // ps)[:, None].long())[:, 0].long()  # each sequence's first block
        before = s["start"] % ps
        old = scale[first]
        kept = torch.where(before[:, None] > 0, torch.maximum(old, fresh[first]), fresh[first])
        codes = pool[first].float() * (old / kept)[:, :, None, None]
        mine = torch.arange(ps, device=q.device)[None, None, :, None] < before[:, None, None, None]
        codes = torch.where(mine, codes, pool[first].float()).to(torch.float8_e4m3fn)
        scale[page] = fresh[page]
        scale[first] = kept
        raw = pool.view(torch.uint8)
        raw[first] = codes.view(torch.uint8)
        raw[page, :, off] = (x / scale[page][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return out


def plain_attention(s):
    c = s["case"]
    H, KV, hd, ps = c["heads"], c["kv_heads"], c["hd"], c["page"]
    n, width = s["table"].shape
    L, R = width * ps, s["max_new"]
    held = s["table"].long().clamp(min=0)

    def gathered(name):
        x = s[name + "_pages"][held].float()  # [n][width][KV][ps][hd]
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][held][..., None, None]
        return x.transpose(1, 2).reshape(n, KV, L, hd)

    i = torch.arange(R, device=s["q"].device)
    new = s["q_start"][1:] - s["q_start"][:-1]
    rows = (s["q_start"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    pos = (s["kv_len"] - new)[:, None] + i
    q = s["q"][rows].float().reshape(n, R, KV, H // KV, hd).permute(0, 2, 3, 1, 4).reshape(n, KV, H // KV * R, hd)
    sc = (q @ gathered("k").transpose(2, 3)).mul_(hd ** -0.5).view(n, KV, H // KV, R, L)
    if c["softcap"]:
        sc = sc.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    j = torch.arange(L, device=q.device)
    if s["slopes"] is not None:
        sc = sc + s["slopes"].view(1, KV, H // KV, 1, 1) * (j - pos[:, :, None])[:, None, None].float()
    see = j <= pos[:, :, None]
    if c["window"]:
        see &= pos[:, :, None] - j < c["window"]
    if s["prefix"] is not None:
        see |= j < s["prefix"][:, None, None]
    see &= (j < s["kv_len"][:, None, None]) & (i < new[:, None])[:, :, None]
    see = see[:, None, None]
    sc = sc.masked_fill_(~see, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = (sc - torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1, total)).view(n, KV, H // KV * R, L)
    out = (p @ gathered("v")).view(n, KV, H // KV, R, hd).permute(0, 3, 1, 2, 4).reshape(n, R, H, hd)
    return out[i < new[:, None]].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    return exact_append(s) if c["op"] == "append" else exact_attention(s)


def e4m3_nearest(x):
    """The nearest value with 4 significant bits, no finer than 2^-9, ties to even, no larger than 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact_append(s):
    c = s["case"]
    KV, hd, ps, r = c["kv_heads"], c["hd"], c["page"], c["rot"]
    q, k, v = (x.double() for x in parts(s))
    begin, start, table = s["q_start"].tolist(), s["start"].tolist(), s["table"].tolist()

    def turn(x, gain, first):
        if gain is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain.double()
        if r:
            z = torch.view_as_complex(s["cs"][first:first + x.shape[0]].double().contiguous())[:, None]
            y = x[..., :r]
            pair = y.unflatten(-1, (r // 2, 2)) if c["interleaved"] else y.unflatten(-1, (2, r // 2)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
            y = y if c["interleaved"] else y.transpose(-1, -2)
            x = torch.cat([y.flatten(-2), x[..., r:]], -1)
        return x

    out_q = torch.empty_like(q)
    pools = {m: s[m + "_pages"].double() for m in "kv"}
    scales = {m: s[m + "_scale"].double() if c["cache"] == "e4m3" else None for m in "kv"}
    for i, (x, y) in enumerate(zip(begin, begin[1:])):
        out_q[x:y] = turn(q[x:y], s["gain_q"], start[i])
        for m, new in (("k", turn(k[x:y], s["gain_k"], start[i])), ("v", v[x:y])):
            a, end = start[i], start[i] + y - x
            while a < end:
                b, p, o = min(end, (a // ps + 1) * ps), table[i][a // ps], a % ps
                block = new[a - start[i]:b - start[i]].transpose(0, 1)  # [KV][tokens][hd]
                if scales[m] is not None:
                    most = block.abs().amax((1, 2)) / E4M3_MAX
                    most = most.clamp(min=2.0 ** SCALE_MIN_EXP)
                    sc = torch.ldexp(torch.ones_like(most), torch.round(torch.log2(most)))
                    sc = torch.where(sc < most, 2 * sc, torch.where(sc / 2 >= most, sc / 2, sc))
                    if o:
                        sc = torch.maximum(sc, scales[m][p])
                        pools[m][p, :, :o] = e4m3_nearest(pools[m][p, :, :o] * (scales[m][p] / sc)[:, None, None])
                    scales[m][p] = sc
                    block = e4m3_nearest(block / sc[:, None, None])
                pools[m][p, :, o:o + b - a] = block
                a = b
    return [out_q, pools["k"], pools["v"], scales["k"], scales["v"]]


def exact_attention(s):
    c = s["case"]
    H, KV, hd, G = c["heads"], c["kv_heads"], c["hd"], c["heads"] // c["kv_heads"]
    begin, lens, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"]
    prefix = s["prefix"].tolist() if s["prefix"] is not None else [0] * len(lens)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, L in enumerate(lens):
        a, b = begin[i], begin[i + 1]
        pages = table[i, :-(-L // c["page"])].long()
        j = torch.arange(L, device=out.device)[None]
        t = torch.arange(L - (b - a), L, device=out.device)[:, None]
        see = (j <= t) & ((t - j < c["window"]) if c["window"] else True) | (j < prefix[i])
        for h in range(KV):
            k, v = (s[m + "_pages"][pages, h].double() for m in "kv")
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][pages, h][:, None, None].double(), v * s["v_scale"][pages, h][:, None, None].double()
            k, v = k.reshape(-1, hd)[:L], v.reshape(-1, hd)[:L]
            for g in range(h * G, h * G + G):
                z = s["q"][a:b, g].double() @ k.T / math.sqrt(hd)
                if c["softcap"]:
                    z = c["softcap"] * torch.tanh(z / c["softcap"])
                if s["slopes"] is not None:
                    z = z - s["slopes"][g].double() * (t - j)
                out[a:b, g] = torch.softmax(torch.where(see, z, -math.inf), -1) @ v
    return out
