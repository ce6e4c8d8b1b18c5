"""neko_op_tree_masks with one of its outputs only, and with row starts that are out of order."""
import numpy as np
import pytest

from tests import drafts_reference as want_of
from tests.test_gpu_cache_edges import ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def call(torch, parent, q_start, max_new, mask, words, depth):
    import nekochat_b200 as nb
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = nb.lib().neko_op_tree_masks(ptr(parent), ptr(q_start), q_start.numel() - 1, parent.numel(), max_new, ptr(mask), words, ptr(depth),
                                     torch.cuda.current_stream().cuda_stream)
    assert rc == 0, nb.lib().neko_last_error()


@pytest.mark.parametrize("starts,tokens", [([2, 5, 5, 9], 12), ([0, 1], 3000), ([7, 7], 40), ([700, 900], 20000)])
def test_either_output_alone(torch, starts, tokens):
    """Rows of no sequence are zeros in it, whatever `words` says without a mask."""
    n, words = 200, 4
    parent = np.full(tokens, -1, np.int32)
    for a, b in zip(starts, starts[1:]):
        parent[a:b] = np.arange(-1, b - a - 1)
    mask, depth = np.zeros((tokens, words), np.uint64), np.zeros(tokens, np.int32)
    bits, deep = want_of.masks([parent[a:b].tolist() for a, b in zip(starts, starts[1:])], words)
    mask[starts[0]:starts[-1]], depth[starts[0]:starts[-1]] = bits, deep
    parent, at = torch.from_numpy(parent).cuda(), ints(torch, *starts)
    for w in (0, 4):
        got = torch.full((tokens,), -7, dtype=torch.int32, device="cuda")
        call(torch, parent, at, n, None, w, got)
        assert np.array_equal(got.cpu().numpy(), depth), w
    got = torch.full((tokens, words), -7, dtype=torch.int64, device="cuda")
    call(torch, parent, at, n, got, words, None)
    assert np.array_equal(got.cpu().numpy().view(np.uint64), mask)


@pytest.mark.parametrize("starts,good", [([0, 100, 300, 400], [(0, 100), (300, 400)]), ([100, 200, 150], [(100, 200)]),
                                         ([0, 64, -1], [(0, 64)]), ([0, 64, 2000, 64, 128], [(0, 64), (64, 128)]),
                                         ([0, 900, 10, 74], [(10, 74)]), ([500, 600, 0], [(500, 600)])])
def test_a_sequence_left_out_leaves_the_others(torch, starts, good):
    """Starts out of order: sequences that are there (and lie apart) have their masks and depths, all other rows are zeros."""
    from nekochat_b200 import NekoError, ops
    tokens, n = 700, 100
    parent = np.full(tokens, -1, np.int32)
    mask, depth = np.zeros((tokens, 2), np.uint64), np.zeros(tokens, np.int32)
    for a, b in good:
        parent[a:b] = np.arange(-1, b - a - 1)
        mask[a:b], depth[a:b] = want_of.masks([parent[a:b].tolist()], 2)
    d, at = torch.from_numpy(parent).cuda(), ints(torch, *starts)
    for _ in range(20):
        m, p = ops.tree_masks(d, at, n)
        assert np.array_equal(m.cpu().numpy().view(np.uint64), mask) and np.array_equal(p.cpu().numpy(), depth)
    with pytest.raises(NekoError, match="max_new"):
        ops.status()
