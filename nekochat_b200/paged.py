"""Qwen3 decoding on a paged key/value cache, from the single operators of :mod:`nekochat_b200.ops`.

The native runner (:mod:`nekochat_b200.model`) gives every sequence a slot of `context` positions in f16. Here sequences
take pages from one pool as they grow (f16, or 8 bits with a scale for each page and KV head), prompts of several
sequences run in one ragged call, and the rotation table may be scaled for longer contexts.

``python -m nekochat_b200.paged --shape qwen3-tiny --cache e4m3`` generates from random prompts and random weights.
"""
import argparse
import time

import numpy as np

from . import ACCUMULATE, NekoError, ops, workload

MAX_ROWS = 4096  # activation rows of one forward


class PagedCache:
    """Pools of `pages` pages of `page` tokens for every layer, and which sequence holds which page."""

    def __init__(self, layers, n_kv, hd, pages, page=64, kind="f16", max_seqs=64, max_len=4096, device="cuda"):
        import torch
        if kind not in ("f16", "e4m3"):
            raise NekoError(f"PagedCache: kind is f16 or e4m3, got {kind!r}")
        dt = torch.float16 if kind == "f16" else torch.float8_e4m3fn
        self.pool = torch.empty((layers, 2, pages, n_kv, page, hd), dtype=dt, device=device)
        self.scale = torch.empty((layers, 2, pages, n_kv), device=device) if kind == "e4m3" else None
        self.page, self.pages, self.max_len = page, pages, max_len
        self.free = list(range(pages - 1, -1, -1))
        self.held = {}                   # sequence -> its pages
        self.length = {}                 # sequence -> tokens it holds
        self.ids = list(range(max_seqs - 1, -1, -1))
        self.width = -(-max_len // page)

    def layer(self, l):
        """k_pages, v_pages and their scales (None for f16) of one layer."""
        s = self.scale
        return self.pool[l, 0], self.pool[l, 1], None if s is None else s[l, 0], None if s is None else s[l, 1]

    def open(self):
        """A new, empty sequence."""
        if not self.ids:
            raise NekoError("PagedCache: every sequence is in use")
        s = self.ids.pop()
        self.held[s], self.length[s] = [], 0
        return s

    def close(self, s):
        """Gives a sequence's pages back."""
        self.free.extend(reversed(self.held.pop(s)))
        del self.length[s]
        self.ids.append(s)

    def grow(self, news):
        """Makes room for news [(sequence, tokens)] or, where the pool has not enough pages, changes nothing."""
        want = []
        for s, n in news:
            if self.length[s] + n > self.max_len:
                raise NekoError(f"PagedCache: sequence {s} would hold more than {self.max_len} tokens")
            want.append(-(-(self.length[s] + n) // self.page) - len(self.held[s]))
        if sum(want) > len(self.free):
            raise NekoError(f"PagedCache: {sum(want)} pages wanted, {len(self.free)} free")
        for (s, _), w in zip(news, want):
            self.held[s].extend(self.free.pop() for _ in range(w))

    def rows(self, seqs):
        """The page table of some sequences as int32 [len(seqs)][width of the longest]."""
        width = max(max(len(self.held[s]) for s in seqs), 1)
        t = np.full((len(seqs), width), -1, np.int32)
        for i, s in enumerate(seqs):
            t[i, :len(self.held[s])] = self.held[s]
        return t


class PagedDecoder:
    """A Qwen3 model (workload.shape) with packed weights on the current device and a PagedCache."""

    def __init__(self, shape, fmt, cache, scaling="none", factor=1.0, original=0):
        if shape["arch"] != "qwen3":
            raise NekoError("PagedDecoder: Qwen3 shapes")
        self.s, self.fmt, self.cache = dict(shape), fmt, cache
        self.cs = ops.rope_table(cache.max_len, shape["head_dim"], shape["rope_theta"], scaling, factor, original)
        self.w = {}

    def load(self, tensors):
        """tensors: (name, float32 array) as workload.weights gives them; q|k|v and gate|up are concatenated like the
        engine's loader does (qwen3_model.cpp:195-209)."""
        import torch
        raw = {n: torch.from_numpy(np.ascontiguousarray(a)).cuda() for n, a in tensors}
        for l in range(self.s["layers"]):
            p = f"layers.{l}."
            q = lambda *names: ops.quantize(self.fmt, torch.cat([raw[p + n + ".weight"] for n in names]))  # noqa: E731
            self.w[l] = dict(qkv=q("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"), o=q("self_attn.o_proj"),
                             gu=q("mlp.gate_proj", "mlp.up_proj"), down=q("mlp.down_proj"),
                             ln1=raw[p + "input_layernorm.weight"], ln2=raw[p + "post_attention_layernorm.weight"],
                             qn=raw[p + "self_attn.q_norm.weight"], kn=raw[p + "self_attn.k_norm.weight"])
        self.embed = ops.quantize(self.fmt, raw["embed_tokens.weight"])  # also the tied LM head
        self.norm = raw["norm.weight"]
        return self

    def forward(self, batch):
        """batch: [(sequence, its new tokens)], ragged. Appends them and returns the logits of each sequence's last
        token, float32 [len(batch)][vocab] on the device."""
        import torch
        s, c = self.s, self.cache
        H, KV, hd, C, F = s["heads"], s["kv_heads"], s["head_dim"], s["embd"], s["ff"]
        seqs, news = [x for x, _ in batch], [len(t) for _, t in batch]
        T = sum(news)
        if not batch or min(news) <= 0 or T > MAX_ROWS or len(set(seqs)) != len(seqs):
            raise NekoError(f"forward: 1 to {MAX_ROWS} tokens, some for each of different sequences")
        tokens = np.concatenate([np.asarray(t, np.int64) for _, t in batch])
        if tokens.min() < 0 or tokens.max() >= s["vocab"]:  # the embedding is gathered by them on the device
            raise NekoError(f"forward: a token is not in the vocabulary of {s['vocab']}")
        c.grow(list(zip(seqs, news)))
        begin = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        start = np.array([c.length[x] for x in seqs], np.int32)
        table = c.rows(seqs)
        n = len(seqs)
        # one copy for all the integers
        ints = np.concatenate([tokens.astype(np.int32), begin, start, start + np.asarray(news, np.int32),
                               table.ravel()])
        d = torch.from_numpy(ints).cuda()
        tokens, q_start, at, held, table_d = d.split([T, n + 1, n, n, table.size])
        table_d = table_d.view(table.shape)
        last = (q_start[1:] - 1).long()
        step = dict(q_start=q_start, max_new=max(news))
        eps = s["eps"]
        x = ops.dequantize(self.fmt, self.embed[tokens.long()], C)
        for l in range(s["layers"]):
            w = self.w[l]
            k_pages, v_pages, k_scale, v_scale = c.layer(l)
            pages = dict(k_scale=k_scale, v_scale=v_scale, **step)
            qkv = ops.matmul(self.fmt, ops.norm(x, w["ln1"], eps=eps), w["qkv"], C)
            q, k, v = (y.unflatten(1, (-1, hd)) for y in qkv.split([H * hd, KV * hd, KV * hd], 1))
            q = ops.paged_append(k, v, k_pages, v_pages, table_d, at, q=q, q_out=q, cs=self.cs, q_gain=w["qn"],
                                 k_gain=w["kn"], eps=eps, **pages)
            o = ops.paged_attention(q, k_pages, v_pages, table_d, held, out=None, **pages)
            ops.matmul(self.fmt, o.view(T, H * hd), w["o"], H * hd, y=x, flags=ACCUMULATE)
            g = ops.matmul_fused(self.fmt, ops.norm(x, w["ln2"], eps=eps), w["gu"], C, F, swiglu=True)
            ops.matmul(self.fmt, g, w["down"], F, y=x, flags=ACCUMULATE)
        for sq, m in zip(seqs, news):
            c.length[sq] += m
        return ops.matmul(self.fmt, ops.norm(x[last], self.norm, eps=eps), self.embed, C)

    def generate(self, prompts, max_new, stop_ids=()):
        """Greedy tokens after each prompt (lists of ids), stopped at a stop id or max_new tokens. Prompts may be longer than
        one forward takes: they go through in pieces."""
        if not all(len(p) for p in prompts):
            raise NekoError("generate: an empty prompt")
        out = [[] for _ in prompts]
        if max_new <= 0:
            return out
        seqs = []
        try:
            for _ in prompts:
                seqs.append(self.cache.open())
            feed = [list(p) for p in prompts]  # what each sequence has still to take in
            live = list(range(len(prompts)))
            while live:
                room, batch = MAX_ROWS, []
                for i in live[:MAX_ROWS]:
                    batch.append((i, feed[i][:room]))
                    room -= len(batch[-1][1])
                    if not room:
                        break
                nxt = ops.argmax(self.forward([(seqs[i], t) for i, t in batch])).cpu().numpy()
                ops.status()
                done = set()
                for (i, taken), t in zip(batch, nxt):
                    feed[i] = feed[i][len(taken):]
                    if feed[i]:
                        continue
                    if int(t) in stop_ids:
                        done.add(i)
                        continue
                    out[i].append(int(t))
                    feed[i] = [int(t)]
                    if len(out[i]) == max_new:
                        done.add(i)
                live = [i for i in live if i not in done]
        finally:
            for sq in seqs:
                self.cache.close(sq)
        return out


def build(shape_name, fmt=1, kind="f16", pages=256, page=64, max_len=4096, seed=0, perturb=False, max_seqs=64,
          **rope):
    s = workload.shape(shape_name)
    cache = PagedCache(s["layers"], s["kv_heads"], s["head_dim"], pages, page, kind, max_seqs, max_len)
    return PagedDecoder(s, fmt, cache, **rope).load(workload.weights(s, seed, perturb))


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--shape", default="qwen3-tiny", choices=[k for k, v in workload.SHAPES.items() if v["arch"] == "qwen3"])
    ap.add_argument("--cache", default="e4m3", choices=["f16", "e4m3"])
    ap.add_argument("--prompts", type=int, nargs="+", default=[5, 90, 33], help="prompt lengths")
    ap.add_argument("--max-new", type=int, default=32)
    args = ap.parse_args()
    import torch
    m = build(args.shape, kind=args.cache)
    prompts = [workload.prompt(m.s, n, seed=i + 1).tolist() for i, n in enumerate(args.prompts)]
    m.generate(prompts, 2)
    torch.cuda.synchronize()
    t = time.perf_counter()
    out = m.generate(prompts, args.max_new)
    t = time.perf_counter() - t
    for p, o in zip(prompts, out):
        print(f"{len(p)} prompt tokens -> {o}")
    print(f"{sum(map(len, out)) / t:.0f} tokens/s ({args.shape}, {args.cache} cache)")


if __name__ == "__main__":
    main()
