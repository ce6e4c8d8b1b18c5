"""The paged operators where arguments, values and lengths are at their ends: what is left out is reported, what is not seen
has no effect, and memory outside is not touched. Definitions in 64 bits: paged_reference.py."""
import numpy as np
import pytest

from tests import paged_reference as ref
from tests.test_gpu_paged import Cache, append, attend, fresh_rows, starts  # noqa: F401

pytestmark = pytest.mark.gpu
ROUND = {"float32": 0.0, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def ints(torch, *a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.fixture(scope="module")
def native():
    from nekochat_b200 import model, workload
    s = workload.shape("qwen3-tiny")
    m = model.Model(s, 1, context=64, max_seqs=1, max_rows=16).load(workload.weights(s, 0, True))
    yield m
    m.close()


@pytest.mark.parametrize("rows", [3, 40])
def test_rows_left_out_are_reported_to_who_asks(torch, native, rows):
    """A sequence with more rows than max_new, and positions past the rotation table: the operators' own status says so,
    once, and a model's steps do not fail for it."""
    from nekochat_b200 import NekoError, ops, workload
    ops.status()
    rng = np.random.default_rng(rows)
    cache = Cache(torch, rng, [rows], 2, 16, 64, False)
    table = torch.from_numpy(cache.table).cuda()
    q, k, v = fresh_rows(torch, rng, rows, 4, 2, 64, torch.float32)
    held = dict(q_start=ints(torch, 0, rows))
    calls = [lambda: ops.paged_append(k, v, cache.k, cache.v, table, ints(torch, 0), max_new=rows - 1, **held),
             lambda: ops.paged_append(k, v, cache.k, cache.v, table, ints(torch, 0), max_new=rows, q=q,
                                      cs=ops.rope_table(rows - 1, 64, 1e4), **held),
             lambda: ops.paged_attention(q, cache.k, cache.v, table, ints(torch, rows), max_new=rows - 1, **held),
             lambda: ops.paged_attention(q[:-1], cache.k, cache.v, table, ints(torch, rows), max_new=rows, **held)]
    for call in calls:
        call()
        native.forward(workload.prompt(workload.shape("qwen3-tiny"), 3), 0)
        with pytest.raises(NekoError, match="max_new"):
            ops.status()
        ops.status()


@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("at", [2 ** 31 - 2, 2 ** 31 - 40, 2 ** 30, 2 ** 30 + 1])
def test_starts_past_every_table(torch, at, e4m3, n):
    """Positions that do not fit 31 bits: nothing is read from before the rotation table, nothing is stored, the queries are
    what they are without a rotation, and the status says so."""
    from nekochat_b200 import NekoError, ops
    rng = np.random.default_rng(122)
    cache = Cache(torch, rng, [9, 50], 2, 16, 64, e4m3)
    cache.fill(rng, [9, 50])
    q, k, v = fresh_rows(torch, rng, n, 4, 2, 64, torch.float32)
    gain = torch.rand(64, device="cuda") + 0.5
    args = dict(k_scale=cache.ks, v_scale=cache.vs, q_start=ints(torch, 0, n, n), max_new=n, q=q, q_gain=gain, k_gain=gain)
    table, start = torch.from_numpy(cache.table).cuda(), ints(torch, at, 50)
    before = [x.clone() for x in (cache.k, cache.v) + ((cache.ks, cache.vs) if e4m3 else ())]
    plain = ops.paged_append(k, v, cache.k, cache.v, table, start, **args)
    ops.status()
    turned = ops.paged_append(k, v, cache.k, cache.v, table, start, cs=ops.rope_table(600, 64, 1e4), **args)
    with pytest.raises(NekoError, match="positions past the rotation table"):
        ops.status()
    want = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * gain
    for got in (plain, turned):
        assert ((got - want).abs() <= 2e-6 * want.abs().amax(-1, keepdim=True)).all()
    for x, y in zip(before, (cache.k, cache.v, cache.ks, cache.vs)):
        assert torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8))
