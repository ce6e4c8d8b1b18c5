"""neko_op_tree_masks with one of its outputs only, and with row starts that are out of order; what drafts that were not kept leave
of an 8-bit page."""
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


def test_what_is_not_kept_leaves_its_scale(torch):
    """8-bit pages: a node's values may raise its page's scale for the tokens before it and beside it, and the scale stays when the node is
    not kept. The tokens that are kept stand within half a step of the page's scale: 2^-4 of themselves, or half the least step,
    2^-10, of the scale; both once for each time that they are rounded (twice: as they come, and when the scale grows)."""
    from nekochat_b200 import ops
    ps, hd, ctx = 16, 64, 5
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn((ctx + 4, 1, hd), device="cuda", generator=g) for _ in range(2))
    big = 300.0
    k[ctx + 2] *= big  # node 2, a brother of node 3
    pool = torch.zeros((2, 2, 1, ps, hd), dtype=torch.float8_e4m3fn, device="cuda")
    scale, table = torch.ones((2, 2, 1), device="cuda"), ints(torch, 1, 0)[None]
    put = lambda rows, at, **how: ops.paged_append(k[rows], v[rows], pool[0], pool[1], table, ints(torch, at), k_scale=scale[0], v_scale=scale[1],  # noqa: E731
                                                   q_start=ints(torch, 0, k[rows].shape[0]), max_new=8, **how)
    put(slice(0, ctx), 0)
    before = scale.clone()
    parent = ints(torch, -1, 0, 0, 0)
    _, depth = ops.tree_masks(parent, ints(torch, 0, 4), 4)
    put(slice(ctx, ctx + 4), ctx, depth=depth)
    path, count, token = ops.tree_accept(ints(torch, 9, 1, 1, 8), ints(torch, 0, 3, 4, 9), parent, ints(torch, 0, 4), 4)
    assert path.tolist() == [[0, 3, 0, 0]] and count.tolist() == [2] and token.tolist() == [8]
    ops.paged_compact(pool, table, ints(torch, ctx), path, count, scale=scale)
    ops.status()
    assert scale[0, 1, 0] > 64 * before[0, 1, 0] and scale[1, 1, 0] <= 4 * before[1, 1, 0]
    keep = [*range(ctx + 1), ctx + 3]
    for i, x in enumerate((k, v)):
        got = pool[i, 1, 0, :len(keep)].double() * scale[i, 1, 0].double()
        want = x[keep, 0].double()
        assert ((got - want).abs() <= 2 * (2.0 ** -4 * want.abs() * 1.0625 + 2.0 ** -10 * scale[i, 1, 0])).all()


def test_drafts_on_8_bit_pages(torch):
    """The answers' lengths, their first tokens (before any guess) and the pages are those of one token at a time."""
    from nekochat_b200 import paged, workload
    m = paged.build("qwen3-tiny", kind="e4m3", page=16, pages=60, max_len=256, perturb=True, max_seqs=12)
    prompts = [workload.prompt(m.s, n, seed=i + 5).tolist() for i, n in enumerate((40, 1, 37))]
    plain, steps, verify = m.generate(prompts, 40), [], m.verify
    for draft in (1, 7, 70):
        del steps[:]
        m.verify = lambda *a: steps.append(1) or verify(*a)
        try:
            got = m.generate(prompts, 40, draft=draft)
        finally:
            del m.verify
        assert [len(x) for x in got] == [40] * 3 and [x[0] for x in got] == [x[0] for x in plain]
        assert all(0 <= t < m.s["vocab"] for x in got for t in x) and 0 < len(steps) < 40
        assert len(m.cache.free) == 60 and not m.cache.held
