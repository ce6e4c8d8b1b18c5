"""Drafted tokens, sampling and moving pages without a GPU: the argument structs, every refusal of the C entries (which come before
any CUDA call), page sharing, and how generate feeds drafts."""
import ctypes as C
import math
import os
import struct
import subprocess
import types

import numpy as np
import pytest

import nekochat_b200 as nb
from nekochat_b200 import ops, paged, workload
from tests import drafts_reference as want_of
from tests.test_paged_host import ATTEND, GOOD

PLANES = ["pages", "scale", "table", "plane_stride", "page_stride", "scale_plane", "scale_stride", "table_stride", "type", "planes", "n_seq",
          "max_pages", "num_pages", "n_kv", "page_size", "head_dim"]
POOL = dict(pages=4096, scale=64, table=64, plane_stride=9 * 8 * 16 * 128, page_stride=8 * 16 * 128, scale_plane=72, scale_stride=8,
            table_stride=4, type=3, planes=2, n_seq=2, max_pages=4, num_pages=9, n_kv=8, page_size=16, head_dim=128)
SAMPLE = ["logits", "u", "temperatures", "top_ps", "min_ps", "top_ks", "token", "prob", "row_stride", "type", "rows", "vocab", "top_k",
          "temperature", "top_p", "min_p", "reserved"]
ROWS = dict(logits=64, u=64, temperatures=0, top_ps=0, min_ps=0, top_ks=0, token=64, prob=0, row_stride=100, type=0, rows=2, vocab=100, top_k=0,
            temperature=1.0, top_p=1.0, min_p=0.0, reserved=0)


def test_structs_match_the_header(tmp_path):
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "neko_cuda.h"\n'
                   'int main(void){printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(neko_tree), sizeof(neko_paged_planes), sizeof(neko_sample_rows_args),'
                   "offsetof(neko_paged_planes, head_dim), offsetof(neko_paged_planes, scale_stride), offsetof(neko_sample_rows_args, top_k),"
                   "offsetof(neko_sample_rows_args, min_p));return 0;}\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", inc, str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got[:3] == [ops._TREE.size, ops._PLANES.size, ops._SAMPLE.size]
    a = ops._PLANES.pack(*(POOL[f] for f in PLANES))
    assert np.frombuffer(a, np.int32)[got[3] // 4] == 128 and np.frombuffer(a, np.int64)[got[4] // 8] == 8
    b = ops._SAMPLE.pack(*(dict(ROWS, top_k=77, min_p=0.5)[f] for f in SAMPLE))
    assert np.frombuffer(b, np.int32)[got[5] // 4] == 77 and np.frombuffer(b, np.float32)[got[6] // 4] == 0.5


def planes(name, *args, **over):
    d = dict(POOL, **over)
    return getattr(nb.lib(), name)(ops._PLANES.pack(*(d[f] for f in PLANES)), *args, None)


@pytest.mark.parametrize("over", [dict(pages=0), dict(scale=0), dict(type=0), dict(type=2), dict(planes=-1), dict(planes=70000), dict(n_seq=-1),
                                  dict(max_pages=-1), dict(num_pages=0), dict(n_kv=0), dict(page_size=8), dict(head_dim=96),
                                  dict(page_stride=8 * 16 * 128 - 16), dict(page_stride=8 * 16 * 128 + 8), dict(plane_stride=64),
                                  dict(plane_stride=9 * 8 * 16 * 128 + 4), dict(pages=4104), dict(scale_stride=7), dict(scale_plane=7)])
def test_refused_pools(over):
    none = dict(pages=4096) if over == dict(pages=0) else {}
    assert planes("neko_op_paged_copy", None, None, 0, **none) == 0
    assert planes("neko_op_paged_compact", None, None, 0, None, 0) == 0
    assert planes("neko_op_paged_copy", None, None, 0, **over) == -1 and b"paged_copy" in nb.lib().neko_last_error()
    assert planes("neko_op_paged_compact", None, None, 0, None, 0, **over) == -1 and b"paged_compact" in nb.lib().neko_last_error()


def test_refused_moves():
    assert planes("neko_op_paged_copy", 64, 64, -1) == -1 and planes("neko_op_paged_copy", None, 64, 1) == -1
    assert planes("neko_op_paged_copy", 64, None, 1) == -1
    assert planes("neko_op_paged_compact", 64, 64, 2, 64, 3) == -1  # rows of path overlap
    assert planes("neko_op_paged_compact", 64, 64, 2, 64, -1) == -1
    for hole in range(3):
        args = [64, 64, 64]
        args[hole] = None
        assert planes("neko_op_paged_compact", args[0], args[1], 2, args[2], 2) == -1
    assert planes("neko_op_paged_compact", 64, 64, 2, 64, 2, table=0) == -1
    assert planes("neko_op_paged_compact", 64, 64, 2, 64, 2, table_stride=3) == -1
    assert planes("neko_op_paged_compact", 64, 64, 2, 64, 2, max_pages=1 << 27, table_stride=1 << 27) == -1
    assert nb.lib().neko_op_paged_copy(None, 64, 64, 1, None) == -1 and nb.lib().neko_op_paged_compact(None, 64, 64, 1, 64, 1, None) == -1


@pytest.mark.parametrize("over,code", [(dict(logits=0), -1), (dict(token=0), -1), (dict(u=0), -1), (dict(u=0, temperature=0.0, temperatures=64), -1),
                                       (dict(type=3), -1), (dict(rows=-1), -1), (dict(vocab=0), -1), (dict(logits=66), -1),
                                       (dict(vocab=262145), -6), (dict(rows=(1 << 24) + 1), -6)])
def test_refused_samples(over, code):
    d = dict(ROWS, **over)
    assert nb.lib().neko_op_sample_rows(ops._SAMPLE.pack(*(d[f] for f in SAMPLE)), None) == code
    assert b"sample_rows" in nb.lib().neko_last_error()
    assert nb.lib().neko_op_sample_rows(ops._SAMPLE.pack(*(dict(ROWS, rows=0)[f] for f in SAMPLE)), None) == 0
    assert nb.lib().neko_op_sample_rows(None, None) == -1


def test_refused_trees():
    l = nb.lib()
    attend = lambda tree, **over: l.neko_op_paged_tree_attention(ops._ATTEND.pack(*(dict(GOOD, **over)[f] for f in ATTEND)), tree, None)  # noqa: E731
    tree = lambda **o: ops._TREE.pack(*(dict(dict(mask=64, depth=64, words=1, reserved=0), **o)[f] for f in ("mask", "depth", "words", "reserved")))  # noqa: E731
    assert attend(tree()) == 0 and attend(None) == -1 and b"paged_tree_attention" in l.neko_last_error()
    assert attend(tree(), page_size=8) == -1 and b"paged_tree_attention" in l.neko_last_error()
    for t, over in ((tree(mask=0), {}), (tree(mask=68), {}), (tree(), dict(max_new=65)), (tree(depth=0), dict(window=4)), (tree(depth=0), dict(slopes=64)),
                    (tree(), dict(prefix=64))):
        assert attend(t, **dict(dict(tokens=100, max_new=64), **over)) == -1
    ok = [64, 64, 2, 10, 5, 64, 1, 64]
    for i, bad, code in ((0, None, -1), (1, None, -1), (2, -1, -1), (3, -1, -1), (4, -1, -1), (6, 0, -1), (5, 68, -1)):
        args = list(ok)
        args[i] = bad
        assert l.neko_op_tree_masks(*args, None) == code, i
    assert l.neko_op_tree_masks(64, 64, 1, 5000, 5000, 64, 100, 64, None) == -6
    assert l.neko_op_tree_masks(None, None, 0, 10, 5, 64, 1, 64, None) == 0 and l.neko_op_tree_masks(64, 64, 2, 10, 5, None, 0, None, None) == 0
    ok = [64, 64, 64, 64, 2, 10, 5, 64, 64, 64]
    for i, bad in ((0, None), (1, None), (2, None), (3, None), (4, -1), (5, -1), (6, -1), (7, None), (8, None), (9, None)):
        args = list(ok)
        args[i] = bad
        assert l.neko_op_tree_accept(*args, None) == -1, i
    assert l.neko_op_tree_accept(64, 64, 64, 64, 2, 9000, 5000, 64, 64, 64, None) == -6
    assert l.neko_op_tree_accept(None, None, None, None, 0, 0, 5, None, None, None, None) == 0


def test_tensors_that_are_not_on_the_device_are_refused():
    import torch
    i = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.tree_masks(i, i, 2), lambda: ops.tree_accept(i, i, i, i, 2), lambda: ops.sample_rows(torch.zeros(2, 5), None, 0.0),
                 lambda: ops.paged_copy(torch.zeros(4, 1, 16, 32, dtype=torch.float16), i, i),
                 lambda: ops.paged_compact(torch.zeros(4, 1, 16, 32, dtype=torch.float16), i[None], i, i[None], i)):
        with pytest.raises(nb.NekoError):
            call()


def cache_of(monkeypatch, **kw):
    moves = []
    c = paged.PagedCache(1, 2, 32, **dict(dict(pages=10, page=16, max_seqs=5, max_len=128, device="cpu"), **kw))
    monkeypatch.setattr(c, "_copy", moves.append)
    return c, moves


def test_forks_share_full_pages(monkeypatch):
    c, moves = cache_of(monkeypatch)
    a = c.open()
    c.grow([(a, 40)])
    c.length[a] = 40
    b, d = c.fork(a, 2)
    assert c.held[b][:2] == c.held[a][:2] == c.held[d][:2] and len(c.free) == 5 and c.length[b] == 40
    assert moves.pop() == [(c.held[a][2], c.held[b][2]), (c.held[a][2], c.held[d][2])]
    c.close(a)
    assert len(c.free) == 6  # its own last page alone
    with pytest.raises(nb.NekoError, match="no room"):
        c.fork(b, 9)
    assert len(c.free) == 6 and len(c.ids) == 3
    c.cut(b, 32)
    e, = c.fork(b)
    assert moves.pop() == [] and c.held[e] == c.held[b] and len(c.free) == 7
    shared = c.held[e][1]
    c.cut(e, 20)  # within a page that others hold: a copy of its own
    assert moves.pop() == [(shared, c.held[e][1])] and c.held[e][1] != shared and c.held[b][1] == shared
    with pytest.raises(nb.NekoError):
        c.cut(e, 21)
    for s in (b, d, e):
        c.close(s)
    assert sorted(c.free) == list(range(10)) and not any(c.holders) and len(c.ids) == 5


def test_a_cut_of_a_shared_page_needs_room(monkeypatch):
    c, moves = cache_of(monkeypatch, pages=2)
    a = c.open()
    c.grow([(a, 32)])
    c.length[a] = 32
    b, = c.fork(a)
    with pytest.raises(nb.NekoError, match="no page free"):
        c.cut(b, 20)
    assert c.length[b] == 32 and c.held[b] == c.held[a]
    c.cut(b, 16)
    assert c.held[b] == c.held[a][:1]


def test_packing_moves_pages_down(monkeypatch):
    c, moves = cache_of(monkeypatch)
    s = [c.open() for _ in range(3)]
    for x in s:
        c.grow([(x, 40)])
        c.length[x] = 48
    f, = c.fork(s[2])
    c.close(s[0])
    held = {x: list(c.held[x]) for x in (s[1], s[2], f)}
    assert c.pack() == 6
    to = dict(moves.pop())
    assert all(c.held[x] == [to.get(p, p) for p in held[x]] for x in held) and c.held[f] == c.held[s[2]]
    assert {p for x in held for p in c.held[x]} == set(range(6)) and sorted(c.free) == [6, 7, 8, 9] and c.free[-1] == 6
    assert [c.holders[p] for p in range(10)].count(2) == 3 and c.pack() == 6 and moves.pop() == []


def test_guesses_follow_earlier_places():
    d = paged.Drafts([1, 2, 3, 4, 1, 2, 5, 6, 1, 2])
    assert d.tree(6) == ([2, 5, 6, 1, 2, 3], [-1, 0, 1, 2, 3, 0])
    assert d.tree(1) == ([2], [-1])
    d.add(3)
    assert d.tree(4) == ([3, 4, 1, 2], [-1, 0, 1, 2])
    assert paged.Drafts([7]).tree(5) == ([7], [-1]) and paged.Drafts([7, 8]).tree(5) == ([8], [-1])
    assert paged.Drafts([5, 5, 5, 5]).tree(4) == ([5, 5], [-1, 0]) or paged.Drafts([5, 5, 5, 5]).tree(4)[1][:2] == [-1, 0]


class Fake:
    """Stands in for the device: the token after a sequence is a number that its last two tokens decide, modulo a few, so that guesses
    come true often."""

    def __init__(self, monkeypatch, m):
        self.m, self.seen, self.steps, self.nodes = m, {}, 0, 0
        monkeypatch.setattr(paged, "ops", types.SimpleNamespace(argmax=lambda x: x, status=lambda: None, paged_copy=lambda *a, **k: None))
        monkeypatch.setattr(m, "forward", self.forward, raising=False)
        monkeypatch.setattr(m, "verify", self.verify, raising=False)

    def after(self, tokens):
        return (3 * tokens[-1] + (tokens[-2] if len(tokens) > 1 else 0) + 1) % 7

    def take(self, s, tokens):
        c = self.m.cache
        if c.length[s] == 0:
            self.seen[s] = []
        elif s not in self.seen:  # a fork
            self.seen[s] = list(self.prompt)
        c.grow([(s, len(tokens))])
        c.length[s] += len(tokens)
        self.seen[s] = self.seen[s][:c.length[s] - len(tokens)] + list(tokens)
        self.prompt = list(self.seen[s])
        return self.after(self.seen[s])

    def forward(self, batch):
        import torch
        return torch.tensor([self.take(s, t) for s, t in batch])

    def verify(self, batch, choose):
        out = []
        self.steps += 1
        for s, tokens, parents in batch:
            self.nodes = max(self.nodes, len(tokens))
            self.m.cache.grow([(s, len(tokens))])
            lines = want_of.lines(parents)
            chosen = [self.after(self.seen[s] + [tokens[j] for j in reversed(line)]) for line in lines]
            walk, token = want_of.accept(chosen, tokens, parents)
            self.take(s, [tokens[i] for i in walk])
            self.m.cache.shed(s)
            out.append([tokens[i] for i in walk[1:]] + [token])
        return out


def decoder(**cache):
    s = workload.shape("qwen3-tiny")
    m = paged.PagedDecoder.__new__(paged.PagedDecoder)
    m.s, m.fmt = dict(s), 1
    m.cache = paged.PagedCache(s["layers"], s["kv_heads"], s["head_dim"], **{**dict(pages=8, page=16, max_len=64, device="cpu"), **cache})
    return m


def test_generate_with_drafts_takes_fewer_steps(monkeypatch):
    m = decoder(pages=30)
    f = Fake(monkeypatch, m)
    prompts = [[1, 2, 3], [6], [4, 4]]
    plain = m.generate(prompts, 30)
    for draft in (1, 5, 100):
        f.steps = f.nodes = 0
        assert m.generate(prompts, 30, draft=draft) == plain
        assert 0 < f.steps < 30 and f.nodes <= draft + 1 and len(m.cache.free) == 30
    stop = plain[0][9]
    assert m.generate(prompts, 30, {stop}, draft=5) == m.generate(prompts, 30, {stop})


def test_drafts_give_way_where_pages_run_out(monkeypatch):
    """A pool that holds the answers and no guesses: they come one by one, as without drafts."""
    m = decoder(pages=3, max_seqs=3)
    f = Fake(monkeypatch, m)
    plain = m.generate([[1], [2], [3]], 15)
    assert m.generate([[1], [2], [3]], 15, draft=40) == plain
    m = decoder(max_len=20)
    f = Fake(monkeypatch, m)
    assert m.generate([[1]], 19, draft=40) == m.generate([[1]], 19)


def test_copies_of_an_answer(monkeypatch):
    m = decoder(pages=30, max_seqs=6)
    Fake(monkeypatch, m)
    one = m.generate([[1, 2, 3]], 9)
    got = m.generate([[1, 2, 3]], 9, copies=4)
    assert got == one * 4 and len(m.cache.free) == 30 and len(m.cache.ids) == 6
    with pytest.raises(nb.NekoError, match="no room"):
        m.generate([[1, 2, 3]], 9, copies=7)
    assert len(m.cache.free) == 30 and len(m.cache.ids) == 6
    for bad in (dict(copies=0), dict(draft=-1)):
        with pytest.raises(nb.NekoError):
            m.generate([[1]], 3, **bad)


def test_the_sampling_reference():
    """Tie, nucleus, smallest share and the ends of u in the tests' own definition."""
    x = [1.0, 3.0, 3.0, 2.0, -math.inf, math.nan]
    assert want_of.sample(x, 0.0, 0.0, 0, 1.0, 0.0) == (1, 1.0)
    for held in (True, False):
        assert [want_of.sample(x, u, 1.0, 2, 1.0, 0.0, held)[0] for u in (0.0, 0.49, 0.5, 0.99)] == [1, 1, 2, 2]
        assert want_of.sample(x, 0.999, 1.0, 1, 1.0, 0.0, held) == (1, 1.0)
        assert {want_of.sample(x, u / 50, 1.0, 0, 0.5, 0.0, held)[0] for u in range(50)} == {1, 2}
        assert {want_of.sample(x, u / 50, 1.0, 0, 1.0, 0.3, held)[0] for u in range(50)} == {1, 2, 3}
        assert want_of.sample([-math.inf, math.nan], 0.5, 1.0, 0, 1.0, 0.0, held) == (-1, 0.0)
        assert want_of.sample([5.0, math.inf, math.inf], 0.7, 1.0, 0, 1.0, 0.0, held)[0] == 2
    assert struct.calcsize("@2P2i") == C.sizeof(C.c_void_p) * 3


def test_parents_of_another_number_change_nothing(monkeypatch):
    m = decoder(pages=4)
    s, t = m.cache.open(), m.cache.open()
    with pytest.raises(nb.NekoError, match="a parent for each token"):
        m.verify([(s, [1, 2], [-1]), (t, [1], [-1, 0])], None)
    assert len(m.cache.free) == 4


def test_drafts_of_nothing():
    from nekochat_b200.paged import Drafts
    assert Drafts([]).tree(5) == ([], [])
    for kw in (dict(gram=0), dict(looks=0)):
        with pytest.raises(nb.NekoError, match="1 or more"):
            Drafts([1, 2], **kw)
