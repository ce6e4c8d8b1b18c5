"""PagedDecoder without a GPU: what forward refuses before it touches the device, and how generate feeds it."""
import types

import pytest

import nekochat_b200 as nb
from nekochat_b200 import paged, workload


def decoder(**cache):
    """A decoder without weights: enough for what happens before the first kernel."""
    s = workload.shape("qwen3-tiny")
    m = paged.PagedDecoder.__new__(paged.PagedDecoder)
    m.s, m.fmt = dict(s), 1
    m.cache = paged.PagedCache(s["layers"], s["kv_heads"], s["head_dim"], **{**dict(pages=8, page=16, max_len=64, device="cpu"), **cache})
    return m


@pytest.mark.parametrize("ids", [[-1], [3, "vocab"], [1 << 40]])
def test_tokens_outside_the_vocabulary_are_refused(ids):
    m = decoder()
    s = m.cache.open()
    with pytest.raises(nb.NekoError, match="vocabulary"):
        m.forward([(s, [m.s["vocab"] if t == "vocab" else t for t in ids])])
    assert m.cache.length[s] == 0 and not m.cache.held[s]  # nothing was taken


class Fake:
    """Stands in for the device: a step's "logits" are the next tokens themselves, the sum of all that a sequence has taken in."""

    def __init__(self, monkeypatch, m, vocab=1000):
        self.calls, self.m, self.seen, self.vocab = [], m, {}, vocab
        monkeypatch.setattr(paged, "ops", types.SimpleNamespace(argmax=lambda x: x, status=lambda: None))
        monkeypatch.setattr(m, "forward", self.forward, raising=False)

    def forward(self, batch):
        import torch
        rows = sum(len(t) for _, t in batch)
        assert 0 < rows <= paged.MAX_ROWS and all(len(t) for _, t in batch)
        self.calls.append([(s, len(t)) for s, t in batch])
        self.m.cache.grow([(s, len(t)) for s, t in batch])
        for s, t in batch:
            self.m.cache.length[s] += len(t)
            self.seen[s] = (self.seen.get(s, 0) + sum(t)) % self.vocab
        return torch.tensor([self.seen[s] for s, _ in batch])

    def want(self, prompt, max_new, stop=()):
        out, total = [], sum(prompt) % self.vocab
        while len(out) < max_new and total not in stop:
            out.append(total)
            total = 2 * total % self.vocab
        return out


def test_generate_gives_back_what_it_opened(monkeypatch):
    m = decoder(max_seqs=3)
    Fake(monkeypatch, m)
    with pytest.raises(nb.NekoError, match="in use"):
        m.generate([[1]] * 4, 2)
    assert len(m.cache.ids) == 3 and not m.cache.held
    assert [len(o) for o in m.generate([[1]] * 3, 2)] == [2, 2, 2]
    with pytest.raises(nb.NekoError, match="empty prompt"):
        m.generate([[1], []], 2)
    assert len(m.cache.ids) == 3 and len(m.cache.free) == 8


def test_generate_makes_as_many_tokens_as_asked(monkeypatch):
    m = decoder()
    f = Fake(monkeypatch, m)
    assert m.generate([[1], [2]], 0) == [[], []] and not f.calls
    assert m.generate([], 3) == []
    f.seen.clear()
    assert m.generate([[5], [7]], 3) == [f.want([5], 3), f.want([7], 3)]


def test_generate_takes_long_prompts_in_pieces(monkeypatch):
    m = decoder(pages=2000, max_len=20000)
    f = Fake(monkeypatch, m)
    prompts = [[3] * 5000, [1] * 10, [2] * 9001, [4]]
    assert m.generate(prompts, 4) == [f.want(p, 4) for p in prompts]
    assert max(sum(n for _, n in c) for c in f.calls) == paged.MAX_ROWS
    assert len(m.cache.free) == 2000
    f.seen.clear()
    stop = f.want([3], 3)[2]
    assert m.generate([[3], [1] * 4500], 6, {stop}) == [f.want([3], 6, {stop}), f.want([1] * 4500, 6, {stop})]
