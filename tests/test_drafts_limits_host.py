"""Refusals and bookkeeping of the drafting operators that need no GPU."""
import pytest

import nekochat_b200 as nb
from nekochat_b200 import ops, paged


def test_a_tree_without_masks_is_refused():
    """Not taken for plain paged attention."""
    import torch
    i = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros((1, 1, 16, 32), dtype=torch.float16)
    for mask in (None, [1]):
        with pytest.raises(nb.NekoError, match="mask"):
            ops.paged_tree_attention(torch.zeros(1, 1, 32), pool, pool, i[None], i, mask)


def test_pages_held_already_do_not_pay_for_others():
    """A sequence with pages behind its tokens (a step that failed left them) lends none to another's growth."""
    c = paged.PagedCache(1, 1, 32, pages=10, page=16, max_seqs=3, max_len=128, device="cpu")
    a, b = c.open(), c.open()
    c.grow([(a, 100)])
    assert len(c.held[a]) == 7 and len(c.free) == 3
    with pytest.raises(nb.NekoError, match="pages wanted"):
        c.grow([(a, 1), (b, 64)])
    assert len(c.held[a]) == 7 and not c.held[b] and len(c.free) == 3
    assert not c.fits([(a, 1), (b, 64)]) and c.fits([(a, 1), (b, 48)])
    c.grow([(a, 1), (b, 48)])
    assert len(c.held[b]) == 3 and not c.free
    c.close(a), c.close(b)
    assert sorted(c.free) == list(range(10))
