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
