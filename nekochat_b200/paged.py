"""Qwen3 decoding on a paged key/value cache, from the single operators of :mod:`nekochat_b200.ops`.

The native runner (:mod:`nekochat_b200.model`) gives every sequence a slot of `context` positions in f16. Here sequences
take pages from one pool as they grow (f16, or 8 bits with a scale for each page and KV head), prompts of several
sequences run in one ragged call, and the rotation table may be scaled for longer contexts. Sequences may be forked (they
share their full pages), tokens sampled, and several guessed tokens checked in one step: trees of drafts behind each newest
token, found in what the sequence holds already.

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
        self.holders = [0] * pages       # sequences that hold each page
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
        """Gives a sequence's pages back; those that others hold stay theirs."""
        self._drop(self.held.pop(s))
        del self.length[s]
        self.ids.append(s)

    def _drop(self, pages):
        for p in reversed(pages):
            self.holders[p] -= 1
            if not self.holders[p]:
                self.free.append(p)

    def _take(self):
        p = self.free.pop()
        self.holders[p] = 1
        return p

    def fork(self, s, copies=1):
        """New sequences that hold what s holds: its full pages are shared, the partly filled last one is copied (on the
        current stream). Where there is no room for all of them, nothing changes."""
        full, part = divmod(self.length[s], self.page)
        if copies > len(self.ids) or (part and copies > len(self.free)):
            raise NekoError(f"PagedCache: no room for {copies} forks ({len(self.ids)} sequences and {len(self.free)} pages free)")
        made, moves = [], []
        for _ in range(copies):
            f = self.open()
            self.held[f], self.length[f] = self.held[s][:full], self.length[s]
            for p in self.held[f]:
                self.holders[p] += 1
            if part:
                self.held[f].append(self._take())
                moves.append((self.held[s][full], self.held[f][full]))
            made.append(f)
        self._copy(moves)
        return made

    def cut(self, s, length):
        """Forgets a sequence's tokens past `length` and gives the pages behind them back. Its last page is its own again
        where it was shared (a copy), so that tokens can be appended."""
        if not 0 <= length <= self.length[s]:
            raise NekoError(f"PagedCache: sequence {s} holds {self.length[s]} tokens, not {length}")
        keep, last = -(-length // self.page), length // self.page
        copy = length % self.page and self.holders[self.held[s][last]] > 1
        if copy and not self.free and not any(self.holders[p] == 1 for p in self.held[s][keep:]):
            raise NekoError("PagedCache: no page free for a copy of a shared one")
        self._drop(self.held[s][keep:])
        del self.held[s][keep:]
        self.length[s] = length
        if copy:
            old, new = self.held[s][last], self._take()
            self.holders[old] -= 1
            self.held[s][last] = new
            self._copy([(old, new)])

    def pack(self):
        """Moves pages so that those in use are the pool's first (on the current stream). Returns how many they are."""
        used = sum(1 for h in self.holders if h)
        moves = list(zip([p for p in range(used, self.pages) if self.holders[p]], [p for p in range(used) if not self.holders[p]]))
        self._copy(moves)
        to = dict(moves)
        for s in self.held:
            self.held[s] = [to.get(p, p) for p in self.held[s]]
        for old, new in moves:
            self.holders[new], self.holders[old] = self.holders[old], 0
        self.free = [p for p in range(self.pages - 1, -1, -1) if not self.holders[p]]
        return used

    def _copy(self, moves):
        """Page src becomes page dst in every layer, for moves [(src, dst)]."""
        if moves:
            import torch
            d = torch.tensor(moves, dtype=torch.int32).T.contiguous().to(self.pool.device)
            ops.paged_copy(self.pool, d[0], d[1], scale=self.scale)

    def grow(self, news):
        """Makes room for news [(sequence, tokens)] or, where the pool has not enough pages, changes nothing."""
        want = []
        for s, n in news:
            if self.length[s] + n > self.max_len:
                raise NekoError(f"PagedCache: sequence {s} would hold more than {self.max_len} tokens")
            want.append(max(-(-(self.length[s] + n) // self.page) - len(self.held[s]), 0))
        if sum(want) > len(self.free):
            raise NekoError(f"PagedCache: {sum(want)} pages wanted, {len(self.free)} free")
        for (s, _), w in zip(news, want):
            self.held[s].extend(self._take() for _ in range(w))

    def fits(self, news):
        """Whether grow(news) finds its pages."""
        return sum(max(-(-(self.length[s] + n) // self.page) - len(self.held[s]), 0) for s, n in news) <= len(self.free)

    def shed(self, s):
        """Gives back the pages behind a sequence's tokens."""
        keep = -(-self.length[s] // self.page)
        self._drop(self.held[s][keep:])
        del self.held[s][keep:]

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

    def _batch(self, batch):
        """Checks a batch [(sequence, its new tokens, ..)] and makes room for it. Returns sequences, counts, tokens and where the
        sequences' rows begin."""
        seqs, news = [x[0] for x in batch], [len(x[1]) for x in batch]
        if not batch or min(news) <= 0 or sum(news) > MAX_ROWS or len(set(seqs)) != len(seqs):
            raise NekoError(f"forward: 1 to {MAX_ROWS} tokens, some for each of different sequences")
        tokens = np.concatenate([np.asarray(x[1], np.int64) for x in batch])
        if tokens.min() < 0 or tokens.max() >= self.s["vocab"]:  # the embedding is gathered by them on the device
            raise NekoError(f"forward: a token is not in the vocabulary of {self.s['vocab']}")
        self.cache.grow(list(zip(seqs, news)))
        return seqs, news, tokens.astype(np.int32), np.concatenate([[0], np.cumsum(news)]).astype(np.int32)

    def _layers(self, tokens, table, at, held, mask=None, depth=None, **step):
        """The hidden states behind the last layer for rows of tokens (device), appended to the cache on the way."""
        s, c = self.s, self.cache
        H, KV, hd, C, F = s["heads"], s["kv_heads"], s["head_dim"], s["embd"], s["ff"]
        T, eps = tokens.shape[0], s["eps"]
        x = ops.dequantize(self.fmt, self.embed[tokens.long()], C)
        for l in range(s["layers"]):
            w = self.w[l]
            k_pages, v_pages, k_scale, v_scale = c.layer(l)
            pages = dict(k_scale=k_scale, v_scale=v_scale, **step)
            qkv = ops.matmul(self.fmt, ops.norm(x, w["ln1"], eps=eps), w["qkv"], C)
            q, k, v = (y.unflatten(1, (-1, hd)) for y in qkv.split([H * hd, KV * hd, KV * hd], 1))
            q = ops.paged_append(k, v, k_pages, v_pages, table, at, q=q, q_out=q, cs=self.cs, q_gain=w["qn"],
                                 k_gain=w["kn"], eps=eps, depth=depth, **pages)
            if mask is None:
                o = ops.paged_attention(q, k_pages, v_pages, table, held, out=None, **pages)
            else:
                o = ops.paged_tree_attention(q, k_pages, v_pages, table, held, mask, depth, **pages)
            ops.matmul(self.fmt, o.view(T, H * hd), w["o"], H * hd, y=x, flags=ACCUMULATE)
            g = ops.matmul_fused(self.fmt, ops.norm(x, w["ln2"], eps=eps), w["gu"], C, F, swiglu=True)
            ops.matmul(self.fmt, g, w["down"], F, y=x, flags=ACCUMULATE)
        return x

    def _head(self, x):
        return ops.matmul(self.fmt, ops.norm(x, self.norm, eps=self.s["eps"]), self.embed, self.s["embd"])

    def forward(self, batch):
        """batch: [(sequence, its new tokens)], ragged. Appends them and returns the logits of each sequence's last
        token, float32 [len(batch)][vocab] on the device."""
        import torch
        c = self.cache
        seqs, news, tokens, begin = self._batch(batch)
        T, n = len(tokens), len(seqs)
        start = np.array([c.length[x] for x in seqs], np.int32)
        table = c.rows(seqs)
        # one copy for all the integers
        ints = np.concatenate([tokens, begin, start, start + np.asarray(news, np.int32), table.ravel()])
        d = torch.from_numpy(ints).cuda()
        tokens, q_start, at, held, table_d = d.split([T, n + 1, n, n, table.size])
        x = self._layers(tokens, table_d.view(table.shape), at, held, q_start=q_start, max_new=max(news))
        last = (q_start[1:] - 1).long()
        for sq, m in zip(seqs, news):
            c.length[sq] += m
        return self._head(x[last])

    def verify(self, batch, choose):
        """batch: [(sequence, tokens, parents)]: behind each sequence's newest token (tokens[0], parents[0] = -1) a tree of drafted
        ones, parents[i] < i. All of them go through the model in one step; choose(logits [nodes][vocab]) gives the token that
        the model takes at each node (int32, device). The cache keeps the nodes that those tokens walk through. Returns, for
        each sequence, the tokens gained: the drafts walked through and the one chosen at the last of them."""
        import torch
        c = self.cache
        if any(len(t) != len(p) for _, t, p in batch):
            raise NekoError("verify: a parent for each token")
        seqs, news, tokens, begin = self._batch(batch)
        T, n = len(tokens), len(seqs)
        parents = np.concatenate([np.asarray(p, np.int32) for _, _, p in batch])
        start = np.array([c.length[x] for x in seqs], np.int32)
        table = c.rows(seqs)
        ints = np.concatenate([tokens, parents, begin, start, start + np.asarray(news, np.int32), table.ravel()])
        d = torch.from_numpy(ints).cuda()
        tokens_d, parent, q_start, at, held, table_d = d.split([T, T, n + 1, n, n, table.size])
        table_d, step = table_d.view(table.shape), dict(q_start=q_start, max_new=max(news))
        mask, depth = ops.tree_masks(parent, **step)
        x = self._layers(tokens_d, table_d, at, held, mask, depth, **step)
        path, count, token = ops.tree_accept(choose(self._head(x)), tokens_d, parent, **step)
        ops.paged_compact(c.pool, table_d, at, path, count, scale=c.scale)
        out = torch.cat([path.view(-1), count, token]).cpu().numpy()
        path, count, token = np.split(out, [path.numel(), path.numel() + n])
        path, gained = path.reshape(n, -1), []
        for i, sq in enumerate(seqs):
            c.length[sq] += int(count[i])
            c.shed(sq)
            gained.append([int(tokens[begin[i] + k]) for k in path[i, 1:count[i]]] + [int(token[i])])
        return gained

    def generate(self, prompts, max_new, stop_ids=(), temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, seed=0, copies=1, draft=0):
        """Tokens after each prompt (lists of ids), stopped at a stop id or max_new tokens: greedy at temperature 0, else sampled
        (ops.sample_rows) from numbers that seed, the answer's place and the token's decide. copies answers a prompt, one after
        the other in the result; the prompt goes through the model once. draft > 0: up to that many tokens are guessed
        each step from what the answer and its prompt hold (Drafts) and checked at once, which changes how fast the answers come and not
        what they are, but for rounding (with 8-bit pages a guess with large keys or values raises its page's scale, which stays when the
        guess does not come true). Prompts may be longer than one forward takes: they go through in pieces."""
        import torch
        if not all(len(p) for p in prompts):
            raise NekoError("generate: an empty prompt")
        if copies < 1 or draft < 0:
            raise NekoError("generate: copies is 1 or more, draft not negative")
        n = len(prompts) * copies
        out = [[] for _ in range(n)]
        if max_new <= 0:
            return out
        u = [np.random.default_rng([seed, i]).random(max_new) for i in range(n)] if temperature > 0 else None

        def choose(logits, rows):
            """The tokens taken at rows [(answer, tokens before)] of logits."""
            if u is None:
                return ops.argmax(logits)
            d = torch.from_numpy(np.array([u[i][min(k, max_new - 1)] for i, k in rows])).cuda()
            return ops.sample_rows(logits, d, temperature, top_k, top_p, min_p)[0]

        seqs, guess = {}, {}
        try:
            for i in range(0, n, copies):
                seqs[i] = self.cache.open()
            feed = {i: list(prompts[i // copies]) for i in seqs}  # what each sequence has still to take in
            live = sorted(feed)
            while live:
                if draft and all(out[i] for i in live):
                    batch, rows, room = [], [], MAX_ROWS
                    for i in live:
                        nodes = min(draft + 1, max_new - len(out[i]), self.cache.max_len - self.cache.length[seqs[i]], room - (len(live) - len(batch) - 1))
                        if i not in guess:
                            guess[i] = Drafts(list(prompts[i // copies]) + out[i])
                        tokens, parents = guess[i].tree(max(nodes, 1))
                        batch.append((seqs[i], tokens, parents))
                        room -= len(tokens)
                        if not room:
                            break
                    if not self.cache.fits([(sq, len(tokens)) for sq, tokens, _ in batch]):  # no pages for guesses
                        batch = [(sq, tokens[:1], [-1]) for sq, tokens, _ in batch]
                    for i, (_, _, parents) in zip(live, batch):
                        deep = []
                        for p in parents:
                            deep.append(0 if p < 0 else deep[p] + 1)
                        rows += [(i, len(out[i]) + x) for x in deep]
                    got = list(zip(live, self.verify(batch, lambda logits: choose(logits, rows))))
                else:
                    room, batch = MAX_ROWS, []
                    for i in live[:MAX_ROWS]:
                        batch.append((i, feed[i][:room]))
                        room -= len(batch[-1][1])
                        if not room:
                            break
                    logits = self.forward([(seqs[i], t) for i, t in batch])
                    heads, got = [], []  # rows of logits and the answers that take a token from each
                    for x, (i, taken) in enumerate(batch):
                        feed[i] = feed[i][len(taken):]
                        if feed[i]:
                            continue
                        heads.append((x, i))
                        if not out[i] and i % copies == 0 and i + copies - 1 not in seqs:  # the prompt is through: its other answers
                            for f, sq in enumerate(self.cache.fork(seqs[i], copies - 1)):
                                seqs[i + 1 + f], feed[i + 1 + f] = sq, []
                                heads.append((x, i + 1 + f))
                    if heads:
                        pick = logits if [x for x, _ in heads] == list(range(len(batch))) else logits[[x for x, _ in heads]]
                        nxt = choose(pick, [(i, len(out[i])) for _, i in heads]).cpu().numpy()
                        got = [(i, [int(t)]) for (_, i), t in zip(heads, nxt)]
                ops.status()
                live, done = sorted(set(live) | {i for i, _ in got}), set()
                for i, tokens in got:
                    for t in tokens:
                        if t in stop_ids or t < 0:
                            done.add(i)
                            break
                        out[i].append(t)
                        if i in guess:
                            guess[i].add(t)
                        if len(out[i]) == max_new:
                            done.add(i)
                            break
                    feed[i] = out[i][-1:]
                live = [i for i in live if i not in done]
        finally:
            for sq in seqs.values():
                self.cache.close(sq)
        return out


class Drafts:
    """Guesses at what follows a sequence of tokens: what followed the latest `looks` earlier places at which the same `gram`
    tokens ended, or where there are none the same one."""

    def __init__(self, tokens, gram=2, looks=4):
        if gram < 1 or looks < 1:
            raise NekoError("Drafts: gram and looks are 1 or more")
        self.gram, self.looks, self.tokens, self.ends = gram, looks, [], {}
        for t in tokens:
            self.add(t)

    def add(self, token):
        last = len(self.tokens) - 1  # what ends there is an earlier place from now on
        for g in range(1, min(self.gram, last + 1) + 1):
            self.ends.setdefault(tuple(self.tokens[last - g + 1:]), []).append(last)
        self.tokens.append(token)

    def tree(self, nodes):
        """Up to `nodes` tokens and their parents: the newest, and behind it the guesses, shared beginnings once."""
        if not self.tokens:
            return [], []
        tree, parents, follow = self.tokens[-1:], [-1], {}
        for g in range(min(self.gram, len(self.tokens)), 0, -1):
            ends = self.ends.get(tuple(self.tokens[-g:]), ())[-self.looks:]
            for e in reversed(ends):
                at = 0
                for t in self.tokens[e + 1:e + nodes]:
                    if (at, t) not in follow:
                        if len(tree) >= nodes:
                            return tree, parents
                        follow[at, t] = len(tree)
                        tree.append(t)
                        parents.append(at)
                    at = follow[at, t]
            if ends:
                break
        return tree, parents


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
    ap.add_argument("--temperature", type=float, default=0.0, help="0: greedy")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--copies", type=int, default=1, help="answers to each prompt")
    ap.add_argument("--draft", type=int, default=0, help="tokens guessed and checked in each step")
    args = ap.parse_args()
    import torch
    m = build(args.shape, kind=args.cache)
    prompts = [workload.prompt(m.s, n, seed=i + 1).tolist() for i, n in enumerate(args.prompts)]
    how = dict(temperature=args.temperature, top_k=args.top_k, top_p=args.top_p, min_p=args.min_p, seed=args.seed, copies=args.copies,
               draft=args.draft)
    m.generate(prompts, 2, **how)
    torch.cuda.synchronize()
    t = time.perf_counter()
    out = m.generate(prompts, args.max_new, **how)
    t = time.perf_counter() - t
    for i, o in enumerate(out):
        print(f"{args.prompts[i // args.copies]} prompt tokens -> {o}")
    print(f"{sum(map(len, out)) / t:.0f} tokens/s ({args.shape}, {args.cache} cache)")


if __name__ == "__main__":
    main()
