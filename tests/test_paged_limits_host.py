"""Limits of the paged entries that come before any CUDA call."""
import numpy as np
import pytest

import nekochat_b200 as nb
from nekochat_b200 import ops
from tests.test_paged_host import APPEND, ATTEND, call  # noqa: F401


@pytest.mark.parametrize("over", [dict(tokens=1 << 30, max_new=1 << 30, n_head=16), dict(tokens=(1 << 31) - 1, max_new=(1 << 31) - 1, n_head=8),
                                  dict(tokens=1 << 28, max_new=1 << 28, n_head=8 * 48), dict(tokens=1 << 24, max_new=1 << 24, n_head=8 * 100)])
def test_refused_rows(over):
    """Rows of a KV head that 31 bits or the reciprocal of the group do not hold (the second is a whole call's of one head)."""
    assert call("neko_op_paged_attention", ATTEND, ops._ATTEND, **over) == -6
    assert b"rows" in nb.lib().neko_last_error()


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 12, 24, 48, 100, 127])
def test_rows_are_divided_exactly(group):
    """x * ceil(2^32 / group) >> 32 is x / group for every x that is not refused: where it first is not, the call is refused."""
    inv = -(-(1 << 32) // group)
    excess = inv * group - (1 << 32)
    top = min((1 << 31) - 1025, ((1 << 32) - 1) // excess if excess else 1 << 40)
    rng = np.random.default_rng(group)
    xs = np.unique(np.concatenate([rng.integers(0, top + 1, 200000), np.arange(top - 3 * group, top + 1), np.arange(3 * group)]))
    for near in (xs, np.minimum(xs // group * group + group - 1, top)):
        assert all(int(x) * inv >> 32 == int(x) // group for x in near)


def test_refused_lengths_of_an_append():
    """New tokens that take more pages than a grid counts; a max_new that is only loose is not refused (it fails later, without
    a GPU)."""
    assert call("neko_op_paged_append", APPEND, ops._APPEND, tokens=1 << 21, max_new=1 << 21) == -6
    assert b"pages of new tokens" in nb.lib().neko_last_error()
    assert call("neko_op_paged_append", APPEND, ops._APPEND, tokens=0, max_new=1 << 30) == 0


@pytest.mark.parametrize("theta,rot,original", [(1e4, 128, 4096), (1e4, 128, 65536), (1e4, 128, 131072), (1e4, 64, 1 << 20), (1e6, 128, 32768),
                                                (5e5, 48, 8192), (10.0, 16, 4096)])
@pytest.mark.parametrize("factor,fast,slow", [(4.0, 32.0, 1.0), (8.0, 16.0, 2.0)])
def test_yarn_ramps_between_its_two_speeds(theta, rot, original, factor, fast, slow):
    """Every pair's speed from the method's formulas: a pair that still turns more than beta_slow times is not fully slowed.
    The table holds cosines and sines in f32, half a unit of 1 each: 6e-8 of the gain, taken twice."""
    import math
    half = rot // 2
    table = ops.rope_table(7, rot, theta, "yarn", factor, original, fast, slow, device="cpu").numpy().astype(np.float64)
    where = lambda turns: rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(where(fast)), 0), min(math.ceil(where(slow)), rot - 1)
    gain = 0.1 * math.log(factor) + 1
    for j in range(half):
        speed = theta ** (-2 * j / rot)
        kept = 1.0 if j <= low else 0.0 if j >= high else 1 - (j - low) / (high - low)
        w = speed * kept + speed / factor * (1 - kept)
        turns = speed * original / (2 * math.pi)
        assert not (turns > fast * 1.2) or kept > 0.9, "a fast pair keeps its speed"
        assert not (turns > slow * theta ** (2 / rot)) or kept > 0, "a pair above beta_slow turns is slowed in part at most"
        for pos in range(7):
            assert abs(table[pos, j, 0] - gain * math.cos(pos * w)) <= 1.2e-7 * gain
            assert abs(table[pos, j, 1] - gain * math.sin(pos * w)) <= 1.2e-7 * gain


def test_an_infinite_cap_is_refused():
    """cap tanh(z / cap) has no value there (no cap is 0)."""
    assert call("neko_op_paged_attention", ATTEND, ops._ATTEND, tokens=2, softcap=float("inf")) == -1
    assert b"softcap" in nb.lib().neko_last_error()
