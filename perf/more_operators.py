"""Cases of the operators behind drafted tokens and sampling on the paged key/value cache: attention of a tree of drafted
tokens over the cache, choosing a token from each row of logits, walking the tree along the chosen tokens, bringing the
accepted tokens' keys and values together, and copying pages.

``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``prepare()`` makes what a serving program
holds before the call, ``run()`` is one call (the library's operators where ``own`` is true, elementary torch operations
otherwise), ``exact()`` the same from the definition in 64 bits and ``work()`` its bytes and operations.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
E4M3_MAX = 448.0

TREE = dict(op="tree", dtype="f32", cache="f16", n_seq=1, new_lo=1, new_hi=1, ctx_lo=512, ctx_hi=512, heads=16, kv_heads=8,
            hd=128, page=64, softcap=0.0, window=0, alibi=False)
SAMPLE = dict(op="sample", dtype="f32", rows=1, vocab=151936, temperature=0.8, top_k=40, top_p=0.95, min_p=0.0, mixed=False)
ACCEPT = dict(op="accept", n_seq=1, new_lo=1, new_hi=1)
COMPACT = dict(op="compact", cache="f16", planes=56, n_seq=1, new_lo=8, new_hi=8, ctx_lo=512, ctx_hi=512, kv_heads=8, hd=128,
               page=64)
COPY = dict(op="copy", cache="f16", planes=56, pages=64, moved=4, kv_heads=8, hd=128, page=64)


def case(name, base, **kw):
    return dict(base, name=name, **kw)


def listed():
    return [
        # One chat, a small tree of drafts behind its newest token: the smallest call of a drafted step. Qwen3-0.6B heads.
        case("tree 1x12 on 777 f16", TREE, new_lo=12, new_hi=12, ctx_lo=777, ctx_hi=777, page=16),
        # 64 chats of about the benchmark's length with up to eight tokens each, 8-bit cache.
        case("tree 64x8 on 700 e4m3", TREE, cache="e4m3", n_seq=64, new_lo=3, new_hi=8, ctx_lo=300, ctx_hi=1100),
        # Wide trees over long ragged contexts, 16-bit activations, capped scores, Qwen3-4B heads: the largest.
        case("tree 16x63 on 8192 f16", TREE, dtype="bf16", n_seq=16, new_lo=21, new_hi=63, ctx_lo=900, ctx_hi=8191,
             heads=32, softcap=50.0),
        # One reply's next token with the engine's default parameters, Qwen3's vocabulary.
        case("sample 1x151936", SAMPLE),
        # A batch whose chats each bring their own parameters, some greedy; 16-bit logits, GPT-2's vocabulary (odd rows).
        case("sample 64x50257 mixed", SAMPLE, dtype="bf16", rows=64, vocab=50257, mixed=True),
        # Every node of 64 chats' trees, the nucleus of the whole vocabulary: the largest.
        case("sample 320x151936 nucleus", SAMPLE, rows=320, temperature=1.0, top_k=0, top_p=0.9),
        # The masks of one chat's tree and the walk along its chosen tokens.
        case("accept 1x12", ACCEPT, new_lo=12, new_hi=12),
        # The same for 128 chats with wide trees.
        case("accept 128x64", ACCEPT, n_seq=128, new_lo=17, new_hi=64),
        # One chat's accepted tokens brought together in all of Qwen3-0.6B's layers.
        case("compact 1x5 f16", COMPACT, new_lo=5, new_hi=5, ctx_lo=777, ctx_hi=777, page=16),
        # The same for 64 chats on an 8-bit cache, Qwen3-4B's layers.
        case("compact 64x16 e4m3", COMPACT, cache="e4m3", planes=72, n_seq=64, new_lo=2, new_hi=16, ctx_lo=300, ctx_hi=1100),
        # A reply forked into four: their partly filled last pages.
        case("copy 3 pages f16", COPY, moved=3),
        # Pages of ended chats' neighbours moved down, 8-bit cache.
        case("copy 301 pages e4m3", COPY, cache="e4m3", planes=72, pages=640, moved=301),
    ]


def spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["tree", "tree", "tree", "sample", "sample", "sample", "accept", "compact", "copy"])
        most = [max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")]
        kv, hd, page = rng.choice([1, 2, 4, 8, 8, 12]), rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
        cache = rng.choice(["f16", "e4m3"])
        if op == "tree":
            c = dict(TREE, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), cache=cache, page=page, hd=hd, kv_heads=kv,
                     heads=kv * rng.choice([1, 2, 2, 3, 4, 8]), n_seq=spread(rng, 1, 150), new_hi=spread(rng, 1, 200),
                     ctx_hi=spread(rng, 1, 20000) - 1, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                     window=rng.choice([0, 0, spread(rng, 2, 4096)]), alibi=rng.random() < 0.25)
            c["new_lo"] = rng.choice([c["new_hi"], max(1, c["new_hi"] // 3)])
            c["ctx_lo"] = rng.choice([c["ctx_hi"], c["ctx_hi"] // 8])
        elif op == "sample":
            c = dict(SAMPLE, dtype=rng.choice(["f32", "f32", "bf16", "f16"]), rows=spread(rng, 1, 400),
                     vocab=rng.choice([50257, 151936, spread(rng, 50, 250000)]), mixed=rng.random() < 0.3,
                     temperature=round(rng.uniform(0.3, 1.5), 3), top_k=rng.choice([0, 0, spread(rng, 1, 5000)]),
                     top_p=rng.choice([1.0, round(rng.uniform(0.4, 0.99), 3)]),
                     min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.01, 0.3), 3)]))
        elif op == "accept":
            c = dict(ACCEPT, n_seq=spread(rng, 1, 200), new_hi=spread(rng, 1, 200))
            c["new_lo"] = rng.choice([c["new_hi"], max(1, c["new_hi"] // 3)])
        elif op == "compact":
            c = dict(COMPACT, cache=cache, planes=2 * spread(rng, 1, 40), n_seq=spread(rng, 1, 100), new_hi=spread(rng, 1, 64),
                     ctx_hi=spread(rng, 1, 2000) - 1, kv_heads=kv, hd=hd, page=page)
            c["new_lo"] = rng.choice([c["new_hi"], max(1, c["new_hi"] // 3)])
            c["ctx_lo"] = rng.choice([c["ctx_hi"], c["ctx_hi"] // 8])
        else:
            c = dict(COPY, cache=cache, planes=2 * spread(rng, 1, 40), moved=spread(rng, 1, 400), kv_heads=kv, hd=hd, page=page)
            c["pages"] = 2 * c["moved"] + rng.randrange(50)
        w = work(c)
        if w["bytes"] > most[0] or w["flops"] > max(most[1], w["bytes"]):
            continue
        if op == "tree" and plain_cells(c) > max(plain_cells(x) for x in listed() if x["op"] == "tree"):
            continue
        if op in ("compact", "copy") and pool_bytes(c) > 4 << 30:
            continue
        return c


# ------------------------------------------------------------------------------------------------ sizes of a case
def spans(c):
    """[(tokens held before, new tokens)] of each sequence: spread evenly over the case's ranges, the same for every
    seed, the first sequence at the upper ends."""
    out = []
    for i in range(c["n_seq"]):
        f, g = (1.0 - i * 0.6180339887498949) % 1.0 or 1.0, (1.0 - i * 0.7548776662466927) % 1.0 or 1.0
        lo, hi = c.get("ctx_lo", 0), c.get("ctx_hi", 0)
        out.append((lo + round(f * (hi - lo)), c["new_lo"] + round(g * (c["new_hi"] - c["new_lo"]))))
    return out


def work(c):
    """What comes in read once, what goes out written once, the keys and values that are seen read once."""
    op = c["op"]
    if op == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * BYTES[c["dtype"]] + 16 * c["rows"], "flops": 2 * n}
    if op == "copy":
        return {"bytes": 2 * c["planes"] * c["moved"] * page_bytes(c), "flops": 0}
    sp = spans(c)
    tokens = sum(n for _, n in sp)
    if op == "accept":
        return {"bytes": tokens * (12 + 8 * words_of(c) + 4), "flops": tokens}
    if op == "compact":
        return {"bytes": 2 * c["planes"] * tokens * c["kv_heads"] * c["hd"] * BYTES[c["cache"]], "flops": 0}
    H, KV, hd, a, b = c["heads"], c["kv_heads"], c["hd"], BYTES[c["dtype"]], BYTES[c["cache"]]
    keys = pairs = 0
    for ctx, n in sp:
        seen = min(ctx, c["window"] - 1) if c["window"] else ctx
        keys += seen + n
        pairs += n * seen + n * min(n, 4)
    return {"bytes": 2 * tokens * H * hd * a + 2 * keys * KV * hd * b, "flops": 4 * pairs * H * hd}


def words_of(c):
    return (c["new_hi"] + 63) // 64


def page_bytes(c):
    return c["kv_heads"] * (c["page"] * c["hd"] * BYTES[c["cache"]] + (4 if c["cache"] == "e4m3" else 0))


def pool_bytes(c):
    pages = c["pages"] if c["op"] == "copy" else sum(-(-(x + 2 * t + 3) // c["page"]) for x, t in spans(c)) + 4
    return c["planes"] * pages * page_bytes(c)


def plain_cells(c):
    """Numbers that the plain form holds at its widest (padded scores, gathered keys)."""
    sp = spans(c)
    longest, rows = max(x + n for x, n in sp), max(n for _, n in sp)
    return c["n_seq"] * (longest + c["page"]) * max(rows * c["heads"], 2 * c["kv_heads"] * c["hd"])


# ------------------------------------------------------------------------------------------------ inputs
def quantized(x):
    """[..., page, hd] f32 as 8-bit codes and their power-of-two scales [...]."""
    m, e = torch.frexp(x.abs().amax(dim=(-2, -1)) / E4M3_MAX)
    scale = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e).clamp(min=-100))
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def pool_of(c, planes, pages, g):
    """Pages [planes][pages][heads][page][hd] with values whose size differs from token to token, and their scales."""
    KV, ps, hd, dev = c["kv_heads"], c["page"], c["hd"], g.device
    store = torch.float16 if c["cache"] == "f16" else torch.float8_e4m3fn
    pool = torch.empty((planes * pages, KV, ps, hd), dtype=store, device=dev)
    scale = torch.empty((planes * pages, KV), device=dev) if c["cache"] == "e4m3" else None
    step = max(1, (1 << 27) // (KV * ps * hd))
    for b in range(0, planes * pages, step):
        n = min(step, planes * pages - b)
        x = torch.randn((n, KV, ps, hd), generator=g, device=dev)
        x *= torch.exp(0.7 * torch.randn((n, KV, ps, 1), generator=g, device=dev))
        if scale is None:
            pool[b:b + n] = x.half()
        else:
            codes, scale[b:b + n] = quantized(x)
            pool[b:b + n].view(torch.uint8).copy_(codes.view(torch.uint8))
    return pool.view(planes, pages, KV, ps, hd), None if scale is None else scale.view(planes, pages, KV)


def tables(held, pages, g):
    """A page table whose sequences hold `held` pages each, in the order that a pool hands them out after a while: none."""
    order = torch.randperm(pages, generator=g, device=g.device).int().cpu()
    table = torch.full((len(held), max(held)), -1, dtype=torch.int32)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    return table.to(g.device)


def trees(sp, rng):
    """parent of every node, counted from its sequence's first: node 0 is the newest token, the rest are drafts behind it,
    often along a chain, sometimes beside it."""
    out = []
    for _, n in sp:
        parent = [-1]
        for i in range(1, n):
            parent.append(i - 1 if rng.random() < 0.45 else int(rng.integers(max(0, i - 12), i)))
        out += parent
    return np.array(out, np.int32)


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": c}
    op = c["op"]
    put = lambda x, t: torch.tensor(np.asarray(x), dtype=t, device=dev)  # noqa: E731
    if op == "sample":
        R, V = c["rows"], c["vocab"]
        x = torch.randn((R, V), generator=g, device=dev) * torch.exp(0.4 * torch.randn((R, 1), generator=g, device=dev)) * 2
        # a few dozen likely tokens in each row, and rows where a grammar leaves few tokens
        hot = torch.randint(0, V, (R, 24), generator=g, device=dev)
        x.scatter_add_(1, hot, 9 * torch.rand((R, 24), generator=g, device=dev))
        few = torch.rand((R, 1), generator=g, device=dev) < 0.1
        x.masked_fill_(few & (torch.rand((R, V), generator=g, device=dev) < 0.97), -math.inf)
        s["logits"] = x.to(DTYPES[c["dtype"]])
        s["u"] = torch.rand(R, generator=g, device=dev, dtype=torch.float64)
        if c["mixed"]:
            pick = lambda a, t: put(rng.choice(a, R), t)  # noqa: E731
            s["temperature"] = pick([0.0, 0.6, 0.7, 0.8, 1.0, 1.3], torch.float32)
            s["top_k"] = pick([0, 1, 20, 40, 40, 50, 200, 1000], torch.int32)
            s["top_p"] = pick([0.5, 0.8, 0.9, 0.95, 0.95, 1.0], torch.float32)
            s["min_p"] = pick([0.0, 0.0, 0.02, 0.05, 0.1], torch.float32)
        else:
            s.update({k: c[k] for k in ("temperature", "top_k", "top_p", "min_p")})
        return s
    if op == "copy":
        s["pool"], s["scale"] = pool_of(c, c["planes"], c["pages"], g)
        order = torch.randperm(c["pages"], generator=g, device=dev).int()
        s["src"], s["dst"] = order[:c["moved"]].clone(), order[c["moved"]:2 * c["moved"]].clone()
        return s
    sp = spans(c)
    n = len(sp)
    starts = np.concatenate([[0], np.cumsum([t for _, t in sp])])
    s["q_start"] = put(starts, torch.int32)
    s["max_new"] = max(t for _, t in sp)
    if op == "accept":
        s["parent_host"] = trees(sp, rng)
        s["parent"] = put(s["parent_host"], torch.int32)
        draft = rng.integers(0, 151936, starts[-1])
        # most nodes' chosen token is one of the drafts behind it
        chosen = rng.integers(0, 151936, starts[-1])
        for a, b in zip(starts, starts[1:]):
            for i in range(a + 1, b):
                if rng.random() < 0.6:
                    chosen[a + s["parent_host"][i]] = draft[i]
        s["draft"], s["chosen"] = put(draft, torch.int32), put(chosen, torch.int32)
        return s
    if op == "compact":
        # accepted tokens of a tree of about twice as many nodes
        held = [-(-(x + 2 * t + 3) // c["page"]) for x, t in sp]
        pages = sum(held) + 4
        s["pool"], s["scale"] = pool_of(c, c["planes"], pages, g)
        s["table"] = tables(held, pages, g)
        path = np.zeros((n, s["max_new"]), np.int32)
        for i, (_, t) in enumerate(sp):
            path[i, :t] = np.concatenate([[0], 1 + np.sort(rng.choice(2 * t + 2, t - 1, replace=False))])
        s["path"], s["count"] = put(path, torch.int32), put([t for _, t in sp], torch.int32)
        s["start"] = put([x for x, _ in sp], torch.int32)
        return s
    held = [-(-(x + t) // c["page"]) for x, t in sp]
    pages = sum(held) + 1 + sum(held) // 16
    pool, scale = pool_of(c, 2, pages, g)
    s["k_pages"], s["v_pages"] = pool[0], pool[1]
    s["k_scale"], s["v_scale"] = (None, None) if scale is None else (scale[0], scale[1])
    s["table"] = tables(held, pages, g)
    s["kv_len"] = put([x + t for x, t in sp], torch.int32)
    s["q"] = torch.randn((int(starts[-1]), c["heads"], c["hd"]), generator=g, device=dev).to(DTYPES[c["dtype"]])
    s["slopes"] = None
    if c["alibi"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, c["heads"] + 1, device=dev, dtype=torch.float32) / c["heads"])
    # the tree's masks and depths, as a step makes them once for all its layers
    s["mask"], s["depth"] = plain_masks(put(trees(sp, rng), torch.int32), s["q_start"], s["max_new"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from nekochat_b200 import ops
        if op == "tree":
            return ops.paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], s["mask"], s["depth"],
                                            k_scale=s["k_scale"], v_scale=s["v_scale"], q_start=s["q_start"],
                                            max_new=s["max_new"], softcap=c["softcap"], window=c["window"], slopes=s["slopes"])
        if op == "sample":
            return ops.sample_rows(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        if op == "accept":
            mask, depth = ops.tree_masks(s["parent"], s["q_start"], s["max_new"])
            path, count, token = ops.tree_accept(s["chosen"], s["draft"], s["parent"], s["q_start"], s["max_new"])
            return [mask, depth, path, count, token]
        if op == "compact":
            ops.paged_compact(s["pool"], s["table"], s["start"], s["path"], s["count"], scale=s["scale"])
        else:
            ops.paged_copy(s["pool"], s["src"], s["dst"], scale=s["scale"])
        return [s["pool"], s["scale"]]
    if op == "tree":
        return plain_tree(s)
    if op == "sample":
        return plain_sample(s)
    if op == "accept":
        mask, depth = plain_masks(s["parent"], s["q_start"], s["max_new"])
        return [mask, depth, *plain_accept(s)]
    if op == "compact":
        plain_compact(s)
    else:
        src, dst = s["src"].long(), s["dst"].long()
        raw = s["pool"].view(torch.int32)
        raw[:, dst] = raw[:, src]
        if s["scale"] is not None:
            s["scale"][:, dst] = s["scale"][:, src]
    return [s["pool"], s["scale"]]


def plain_masks(parent, q_start, max_new):
    """Bit j of node i's words: node j is i itself or an ancestor of it; and how many ancestors i has."""
    T = parent.shape[0]
    at = torch.arange(T, device=parent.device)
    first = q_start.long()[torch.searchsorted(q_start[1:].contiguous(), at.int(), right=True)]
    words = (max_new + 63) // 64
    mask = torch.zeros((T, words), dtype=torch.int64, device=parent.device)
    depth = torch.zeros(T, dtype=torch.int32, device=parent.device)
    node, live = at - first, torch.ones(T, dtype=torch.bool, device=parent.device)
    for _ in range(max_new):
        bit = torch.where(live, torch.ones_like(node) << (node & 63), 0)
        mask.scatter_add_(1, (node >> 6)[:, None], bit[:, None])
        node = torch.where(live, parent.long()[first + node], node)
        live = live & (node >= 0)
        node = node.clamp(min=0)
        depth += live.int()
    return mask, depth


def plain_tree(s):
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
    j = torch.arange(L, device=s["q"].device)
    new = s["q_start"][1:] - s["q_start"][:-1]
    base = s["kv_len"] - new
    rows = (s["q_start"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    pos = base[:, None] + s["depth"][rows]                        # [n][R]
    node = j - base[:, None]                                      # [n][L]: of a key, negative: cached before
    inside = (node >= 0) & (node < new[:, None])
    key = (s["q_start"][:-1, None] + node).clamp(0, s["q"].shape[0] - 1).long()
    key_pos = torch.where(inside, base[:, None] + s["depth"][key], j)
    shift = node.clamp(0, R - 1)
    bits = s["mask"][rows].gather(2, (shift >> 6)[:, None].expand(n, R, L).long())
    see = torch.where(inside[:, None], (bits >> (shift & 63)[:, None].long()) & 1 == 1, (node < 0)[:, None])
    gap = pos[:, :, None] - key_pos[:, None]                      # [n][R][L]
    if c["window"]:
        see = see & (gap < c["window"])
    see = (see & (i < new[:, None])[:, :, None])[:, None, None]
    q = s["q"][rows].float().reshape(n, R, KV, H // KV, hd).permute(0, 2, 3, 1, 4).reshape(n, KV, H // KV * R, hd)
    sc = (q @ gathered("k").transpose(2, 3)).mul_(hd ** -0.5).view(n, KV, H // KV, R, L)
    if c["softcap"]:
        sc = sc.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if s["slopes"] is not None:
        sc = sc - s["slopes"].view(1, KV, H // KV, 1, 1) * gap[:, None, None].float()
    sc = sc.masked_fill_(~see, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = (sc - torch.where(top == -math.inf, 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1, total)).view(n, KV, H // KV * R, L)
    out = (p @ gathered("v")).view(n, KV, H // KV, R, hd).permute(0, 3, 1, 2, 4).reshape(n, R, H, hd)
    return out[i < new[:, None]].to(s["q"].dtype)


def plain_sample(s):
    """In 64 bits: the sums run over a whole vocabulary, and which token a number falls on hangs on their last places."""
    x = s["logits"].double()
    R, V = x.shape
    t, k, p, m = ((s[n] if torch.is_tensor(s[n]) else torch.full((R,), float(s[n]), device=x.device)).double()[:, None]
                  for n in ("temperature", "top_k", "top_p", "min_p"))
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(V, device=x.device)
    w = torch.exp((v - v[:, :1]) / torch.where(t > 0, t, 1))
    w = torch.where(v == -math.inf, 0, w)
    w = torch.where((rank < k) | (k <= 0), w, 0)
    before = torch.cumsum(w, 1) - w
    keep = (before < p * w.sum(1, keepdim=True)) | (p >= 1) | (rank == 0)
    keep &= (w >= m) & ((t > 0) | (rank == 0))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0))
    upto = torch.cumsum(w, 1)
    total = upto[:, -1:]
    token = (upto <= s["u"][:, None] * total).sum(1)
    last = V - 1 - (w > 0).flip(1).int().argmax(1)
    token = torch.minimum(token, last)
    prob = w.gather(1, token[:, None])[:, 0] / torch.where(total[:, 0] > 0, total[:, 0], 1)
    return torch.where(total[:, 0] > 0, token, -1).int(), prob.float()


def plain_accept(s):
    begin, new = s["q_start"][:-1].long(), s["q_start"][1:] - s["q_start"][:-1]
    n, R, dev = begin.shape[0], s["max_new"], begin.device
    i = torch.arange(R, device=dev)
    rows = (begin[:, None] + i).clamp(max=s["parent"].shape[0] - 1)
    parent, draft = s["parent"][rows], s["draft"][rows]
    real = (i < new[:, None]) & (i > 0)
    path = torch.zeros((n, R), dtype=torch.int32, device=dev)
    count = torch.ones(n, dtype=torch.int32, device=dev)
    at, live = torch.zeros(n, dtype=torch.long, device=dev), torch.ones(n, dtype=torch.bool, device=dev)
    for step in range(1, R):
        want = s["chosen"][begin + at]
        hit = real & (parent == at[:, None]) & (draft == want[:, None])
        live = live & hit.any(1)
        at = torch.where(live, hit.int().argmax(1), at)
        path[:, step] = torch.where(live, at, 0).int()
        count += live.int()
    return path, count, s["chosen"][begin + at]


def plain_compact(s):
    c = s["case"]
    ps = c["page"]
    n, R = s["path"].shape
    pool, table = s["pool"], s["table"].long()
    i = torch.arange(R, device=pool.device)
    on = i < s["count"][:, None]
    to = s["start"][:, None] + i
    fro = s["start"][:, None] + s["path"]
    page = lambda x: table.gather(1, (x // ps).clamp(max=table.shape[1] - 1).long())[on]  # noqa: E731
    tp, to_off, fp, fro_off = page(to), (to % ps)[on], page(fro), (fro % ps)[on]
    raw = pool.view(torch.uint8) if s["scale"] is not None else pool
    moved = raw[:, fp, :, fro_off]                                # [tokens][planes][heads][hd]
    if s["scale"] is None:
        raw[:, tp, :, to_off] = moved
        return
    scale = s["scale"]
    old = scale.clone()
    fresh = torch.zeros_like(scale).index_reduce_(1, tp, old[:, fp], "amax")
    first = table.gather(1, (s["start"] // ps)[:, None].long())[:, 0]  # each sequence's first page
    before = s["start"] % ps
    kept = torch.where((before > 0)[None, :, None], torch.maximum(old[:, first], fresh[:, first]), fresh[:, first])
    fresh[:, first] = kept
    scale[:, tp] = fresh[:, tp]
    codes = pool[:, first].float() * (old[:, first] / kept)[..., None, None]
    mine = torch.arange(ps, device=pool.device)[None, None, None, :, None] < before[None, :, None, None, None]
    raw[:, first] = torch.where(mine, codes.to(torch.float8_e4m3fn).view(torch.uint8), raw[:, first])
    ratio = (old[:, fp] / fresh[:, tp]).transpose(0, 1)           # [tokens][planes][heads]
    value = moved.view(torch.float8_e4m3fn).float() * ratio[..., None]
    raw[:, tp, :, to_off] = value.to(torch.float8_e4m3fn).view(torch.uint8)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    return {"tree": exact_tree, "sample": exact_sample, "accept": exact_accept, "compact": exact_compact, "copy": exact_copy}[c["op"]](s)


def exact_tree(s):
    c = s["case"]
    H, KV, hd, G = c["heads"], c["kv_heads"], c["hd"], c["heads"] // c["kv_heads"]
    begin, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    mask, depth = s["mask"].cpu().numpy(), s["depth"].cpu().numpy()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for x, L in enumerate(lens):
        a, b = begin[x], begin[x + 1]
        n, base = b - a, L - (b - a)
        see = np.ones((n, L), bool)
        see[:, base:] = [[mask[a + i, j >> 6] >> (j & 63) & 1 for j in range(n)] for i in range(n)]
        where = np.concatenate([np.arange(base), base + depth[a:b]])
        gap = (base + depth[a:b])[:, None] - where[None]
        if c["window"]:
            see &= gap < c["window"]
        see, gap = torch.tensor(see, device=out.device), torch.tensor(gap, device=out.device).double()
        pages = s["table"][x, :-(-L // c["page"])].long()
        for h in range(KV):
            k, v = (s[m + "_pages"][pages, h].double() for m in "kv")
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][pages, h][:, None, None].double(), v * s["v_scale"][pages, h][:, None, None].double()
            k, v = k.reshape(-1, hd)[:L], v.reshape(-1, hd)[:L]
            for y in range(h * G, h * G + G):
                z = s["q"][a:b, y].double() @ k.T / math.sqrt(hd)
                if c["softcap"]:
                    z = c["softcap"] * torch.tanh(z / c["softcap"])
                if s["slopes"] is not None:
                    z = z - s["slopes"][y].double() * gap
                z = torch.where(see, z, -math.inf)
                w = torch.exp(z - z.max(1, keepdim=True).values)
                out[a:b, y] = (w @ v) / w.sum(1, keepdim=True)
    return out


def exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    u = s["u"].cpu().numpy()
    R = len(u)
    of = lambda n, t: (s[n].cpu().numpy() if torch.is_tensor(s[n]) else np.full(R, s[n])).astype(t).astype(np.longdouble)  # noqa: E731
    t, k, p, m = of("temperature", "f4"), of("top_k", "i4"), of("top_p", "f4"), of("min_p", "f4")
    out, probs = [], []
    for r in range(R):
        ids = np.flatnonzero(x[r] > -np.inf)
        if not len(ids):
            out.append(-1)
            probs.append(0.0)
            continue
        best = x[r].max()
        if t[r] <= 0:
            out.append(int(np.flatnonzero(x[r] == best)[0]))
            probs.append(1.0)
            continue
        # from the likeliest down, equal ones by index; weights of the likeliest's
        w = np.exp(((x[r][ids] - best) / np.float64(t[r])).astype(np.float64)).astype(np.longdouble)
        down = np.argsort(-x[r][ids], kind="stable") if k[r] > 0 or p[r] < 1 else np.arange(len(ids))
        if k[r] > 0:
            down = down[:int(k[r])]
        mass = np.cumsum(w[down])
        held = len(down)
        if p[r] < 1:
            held = min(held, int(np.searchsorted(mass, p[r] * mass[-1])) + 1)
        down = down[:held]
        down = np.sort(down[w[down] >= m[r]])
        mass = np.cumsum(w[down])
        at = int(np.searchsorted(mass, np.longdouble(u[r]) * mass[-1], side="right"))
        at = min(at, len(down) - 1)
        out.append(int(ids[down[at]]))
        probs.append(float(w[down[at]] / mass[-1]))
    return torch.tensor(out, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)


def exact_accept(s):
    begin, parent = s["q_start"].tolist(), s["parent_host"]
    draft, chosen = s["draft"].tolist(), s["chosen"].tolist()
    words, R = (s["max_new"] + 63) // 64, s["max_new"]
    mask, depth = [], []
    path, count, token = np.zeros((len(begin) - 1, R), np.int32), [], []
    for x, (a, b) in enumerate(zip(begin, begin[1:])):
        bits, deep = [], []
        for i in range(b - a):
            up = int(parent[a + i])
            bits.append((bits[up] if up >= 0 else 0) | 1 << i)
            deep.append(deep[up] + 1 if up >= 0 else 0)
        mask += [[z - (1 << 64) if z >> 63 else z for z in ((v >> (64 * w)) & (1 << 64) - 1 for w in range(words))] for v in bits]
        depth += deep
        walk = [0]
        while True:
            nxt = [i for i in range(1, b - a) if parent[a + i] == walk[-1] and draft[a + i] == chosen[a + walk[-1]]]
            if not nxt:
                break
            walk.append(nxt[0])
        path[x, :len(walk)] = walk
        count.append(len(walk))
        token.append(chosen[a + walk[-1]])
    i32 = torch.int32
    return [torch.tensor(mask, dtype=torch.int64), torch.tensor(depth, dtype=i32), torch.tensor(path), torch.tensor(count, dtype=i32),
            torch.tensor(token, dtype=i32)]


def e4m3_nearest(x):
    """The nearest value with 4 significant bits, no finer than 2^-9, ties to even, no larger than 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact_compact(s):
    c = s["case"]
    ps = c["page"]
    table, start, path, count = (s[n].tolist() for n in ("table", "start", "path", "count"))
    out = s["pool"].clone()
    wide = s["scale"] is not None
    scales = s["scale"].clone().double() if wide else None
    for x, n in enumerate(count):
        new = {}
        for k in range(n):
            src, dst = start[x] + path[x][k], start[x] + k
            new.setdefault(table[x][dst // ps], []).append((dst % ps, table[x][src // ps], src % ps))
        for page, moves in new.items():
            if not wide:
                for to, p, o in moves:
                    out[:, page, :, to] = s["pool"][:, p, :, o]
                continue
            stay = start[x] % ps if page == table[x][start[x] // ps] else 0
            moves = [(o, page, o) for o in range(stay)] + moves
            tops = torch.stack([s["scale"][:, p] for _, p, _ in moves]).double().amax(0)
            scales[:, page] = tops
            for to, p, o in moves:
                v = s["pool"][:, p, :, o].double() * (s["scale"][:, p].double() / tops)[..., None]
                out[:, page, :, to] = e4m3_nearest(v).to(torch.float8_e4m3fn)
    return [out, scales]


def exact_copy(s):
    pool, scale = s["pool"].clone(), None if s["scale"] is None else s["scale"].clone()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        pool[:, b] = s["pool"][:, a]
        if scale is not None:
            scale[:, b] = s["scale"][:, a]
    return [pool, scale]
