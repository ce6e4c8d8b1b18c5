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
