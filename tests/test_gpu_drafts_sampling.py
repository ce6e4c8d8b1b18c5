"""neko_op_sample_rows where its ranges end: batches of every size (one to eight CTAs a row), the largest vocabularies with weights that
are all alike, temperatures down to the least f32, the lowest finite logits, shares that are no numbers. Tokens are equal to the
definition's (drafts_reference.py), probabilities within one rounding to f32 and what 64 bits leave: 2^-23."""
import math

import numpy as np
import pytest

from tests import drafts_reference as want_of

pytestmark = pytest.mark.gpu
LOWEST = -np.finfo(np.float32).max


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def definition(x, u, params):
    return zip(*(want_of.sample(x[r], u[r], *params) for r in range(len(x))))


def check(torch, x, u, params, rows):
    """Rows of x and numbers u, repeated to each of the batches' sizes."""
    from nekochat_b200 import ops
    n, d = len(x), torch.from_numpy(x).cuda()
    want, p = (np.array(y) for y in definition(d.float().cpu().numpy(), u, params))
    for count in rows:
        pick = np.arange(count) % n
        token, prob = ops.sample_rows(d[torch.from_numpy(pick).cuda()], torch.from_numpy(u[pick]).cuda(), *params)
        wrong = np.flatnonzero(token.cpu().numpy() != want[pick])
        assert not len(wrong), (count, params, wrong[:4], token.cpu().numpy()[wrong[:4]], want[pick][wrong[:4]])
        assert (np.abs(prob.cpu().numpy() - p[pick]) <= 2.0 ** -23 * p[pick]).all(), (count, params)


def rows_of(rng, kind, V):
    x = np.zeros((5, V), np.float32)
    if kind == "peak":  # one above the others, which are alike
        x -= np.array([0.125, 0.1, 0.5, 1e-3, 2.0], np.float32)[:, None]
        x[np.arange(5), rng.integers(0, V, 5)] = 0
    elif kind == "near":  # within one step of max - x
        x = -rng.random((5, V)).astype(np.float32) / 80
    elif kind == "ties":
        x = np.round(rng.standard_normal((5, V)) * 2).astype(np.float32)
    elif kind == "normal":
        x = (rng.standard_normal((5, V)) * 2).astype(np.float32)
    return x


@pytest.mark.parametrize("V", [50257, 131073, 151936, 262144])
@pytest.mark.parametrize("kind", ["flat", "peak", "near", "ties", "normal"])
def test_a_row_in_batches_of_every_size(torch, kind, V):
    """What the other rows are, how many and on how many CTAs a row runs changes nothing."""
    rng = np.random.default_rng(V)
    x = rows_of(rng, kind, V)
    u = np.array([0.0, 0.37, 0.5, 0.93, 1 - 2.0 ** -20])
    for params in ((0.8, 0, 0.9, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 5000, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (1.0, 0, 1.0, 0.3)):
        check(torch, x, u, params, (1, 5, 40, 120, 200, 320))


@pytest.mark.parametrize("T", [1e30, 100.0, 1e-30, 6e-32, 1.9e-32, 1e-33, 1e-35, 1e-38, 1e-45])
@pytest.mark.parametrize("top", [0.0, 1e-25, -3e-22, 5.0])
def test_temperatures_at_the_ends(torch, T, top):
    """Tokens within some temperatures of the largest, and others far from it. The temperature is that of f32."""
    rng = np.random.default_rng(5)
    t = float(np.float32(T))
    for V in (7, 3000, 40000):
        x = np.float64(top) - np.minimum(t * rng.random((5, V)) * 60, 1e30) * (rng.random((5, V)) < 0.9)
        x[rng.random((5, V)) < 0.3] = -5.0 if T < 1 else -np.inf
        x[2:, 0] = top
        x = x.astype(np.float32)
        u = np.array([0.0, 0.37, 0.5, 0.93, 1 - 2.0 ** -20])
        for params in ((t, 0, 1.0, 0.0), (t, 0, 0.9, 0.0), (t, 5, 0.9, 0.0), (t, 0, 1.0, 0.05), (t, 2000, 0.8, 0.0)):
            check(torch, x, u, params, (5, 200))


@pytest.mark.parametrize("T", [1.0, 1e29, 1e30, 3e34, 1e36])
def test_the_lowest_values(torch, T):
    """Rows just above the lowest finite value, beside tokens that cannot be taken and places outside the row."""
    rng = np.random.default_rng(6)
    t = float(np.float32(T))
    for V in (1, 13, 3001, 30005):
        x = LOWEST + np.abs(rng.standard_normal((5, V))) * np.array([t, 2 * t, 2e31, 2e31, 1e36])[:, None]
        x[3] = LOWEST
        x[4] = LOWEST + 3 * t
        x[:3][rng.random((3, V)) < 0.5] = -np.inf
        x[2][rng.random(V) < 0.2] = np.nan
        x[:, V // 2] = LOWEST
        x = x.astype(np.float32)
        u = np.array([0.0, 0.37, 0.5, 0.93, 1 - 2.0 ** -20])
        for params in ((t, 0, 1.0, 0.0), (t, 0, 0.9, 0.0), (t, 5, 0.9, 0.0), (t, 0, 1.0, 0.05), (t, 2000, 0.8, 0.0)):
            check(torch, x, u, params, (5, 200))


def test_shares_that_are_no_numbers(torch):
    """top_p and min_p that are no numbers leave all tokens, as a number and as a row's."""
    from nekochat_b200 import ops
    x = torch.randn((64, 900), device="cuda")
    u = torch.rand(64, dtype=torch.float64, device="cuda")
    nan = torch.full((64,), math.nan, device="cuda")
    for k in (0, 40):
        token, prob = ops.sample_rows(x, u, 0.9, k)
        for p, m in ((nan, 0.0), (1.0, nan), (math.nan, 0.0), (1.0, math.nan), (math.nan, math.nan)):
            got = ops.sample_rows(x, u, 0.9, k, p, m)
            assert torch.equal(got[0], token) and torch.equal(got[1], prob)


def unrounded(x, u, t, top_p):
    """Token in extended precision and how far, relative to the sums, the draw and the cut are from where they would change."""
    w = np.exp((x.astype(np.longdouble) - x.max()) / np.longdouble(np.float32(t)))
    down = np.argsort(-x.astype(np.float64), kind="stable")
    room = np.longdouble(1)
    if top_p < 1:
        mass = np.cumsum(w[down])
        want = np.longdouble(np.float32(top_p)) * mass[-1]
        n = int(np.searchsorted(mass, want)) + 1
        room = min(abs(mass[n - 1] - want), abs(want - (mass[n - 2] if n > 1 else 0))) / mass[-1]
        down = down[:n]
    kept = np.sort(down)
    mass = np.cumsum(w[kept])
    want = np.longdouble(u) * mass[-1]
    i = int(np.searchsorted(mass, want, side="right"))
    room = min(room, abs(mass[i] - want) / mass[-1], (abs(want - mass[i - 1]) if i else np.longdouble(1)) / mass[-1])
    return int(kept[i]), float(room), float(w[kept[i]] / mass[-1])


@pytest.mark.parametrize("V", [1000, 50257, 262144])
def test_tokens_of_unrounded_weights(torch, V):
    """Against weights that are not rounded to 2^-44 of the largest. Each is off by 2^-45 at most (and 2^-50 of itself, 64 bits), so a sum
    of V of them, of which the largest is 1, by less than V 2^-45 + 2^-50 of itself; a token may differ only where its border is
    nearer than two such errors (the sum's and the target's)."""
    from nekochat_b200 import ops
    rng = np.random.default_rng(V)
    rows = 24
    x = (rng.standard_normal((rows, V)) * 2).astype(np.float32)
    u = rng.random(rows)
    off, checked = V * 2.0 ** -44 + 2.0 ** -48, 0
    for t, top_p in ((0.7, 1.0), (1.0, 0.9), (1.5, 0.97)):
        token, prob = ops.sample_rows(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(), t, 0, top_p)
        for r in range(rows):
            want, room, p = unrounded(x[r], u[r], t, top_p)
            if room > off:
                checked += 1
                assert int(token[r]) == want, (r, t, top_p)
                assert abs(float(prob[r]) - p) <= (2.0 ** -23 + off) * p
    assert checked > 2 * rows
