"""Sampling at the ends of its ranges.

Where u leaves one right answer: at 0 (and below, and NaN) the first
token kept, whatever stands behind it. No rounding decides that, so no other
token counts. A kept token's weight, relative to the row's largest, is at least
e^-60. A log-probability is ln(w / sum) rounded to fp32 once (2^-24 of it) from
weights of 2^-50 and a sum of at most 2^20 of them, far inside 2^-20."""
import math

import numpy as np
import pytest
import torch

from tests import engine
from tests.test_gpu_sample import check as check_filters
from tests.test_gpu_sample import settings

em = engine.load()
pytestmark = pytest.mark.gpu

# (rows, vocabulary): one workgroup a row with the row in LDS and without, and a
# row over several workgroups.
SPREADS = [(3, 3000), (2, 32000), (300, 40000), (1, 50001), (5, 100003)]


def weights(x, T):
    with np.errstate(all="ignore"):
        z = (x.astype(np.float64) - float(x.max())) / float(np.float32(T))
        return np.where(z >= -60, np.exp(z), 0.0)


def two_or_three(R, V, rng):
    """Rows of a few tokens 38 to 55 apart, the lightest first: within a wave's
    run of a row (another thread's, the next lane's, the same thread's) and far
    behind it; and a whole row far below one token."""
    x = np.full((R, V), -np.inf, np.float32)
    heavy = [1, 2, 40, 1500, V - 1, V // 2 + 3]
    for r in range(R):
        at = heavy[r % len(heavy)]
        x[r, 0], x[r, at] = 0.0, 38.0 + 17.0 * rng.random()
        if r % 3 == 1:
            x[r, at + 1 if at + 1 < V else at - 1] = x[r, at] + 1.0
    whole = rng.normal(0, 0.5, V).astype(np.float32)
    x[R - 1] = whole
    x[R - 1, min(777, V - 1)] = 45.0
    return x


def draw(x, u, T=1.0, **kw):
    R = x.shape[0]
    one = lambda v, t=torch.float32: torch.full((R,), v, dtype=t, device="cuda")
    kw = {k: one(v, torch.int32 if k == "top_k" else torch.float32) for k, v in kw.items()}
    tok, lp = em.sample(torch.from_numpy(x).cuda(), one(u), temperature=one(T), **kw)
    return tok.cpu().numpy(), lp.cpu().numpy()


def check(x, tok, lp, w, want, r):
    assert tok[r] == want, (r, tok[r], want)
    l = math.log(w[want] / w.sum())
    assert abs(lp[r] - l) <= 2.0 ** -24 * abs(l) + 2.0 ** -20, (r, lp[r], l)


@pytest.mark.parametrize("u", [0.0, -1.0, math.nan])
@pytest.mark.parametrize("R, V", SPREADS)
def test_the_first_token_kept(R, V, u):
    x = two_or_three(R, V, np.random.default_rng(R + V))
    for T, kw in ((1.0, {}), (1.0, dict(min_p=0.0)), (0.9, dict(top_p=1.0)), (1.0, dict(top_k=0))):
        tok, lp = draw(x, u, T, **kw)
        for r in range(R):
            w = weights(x[r], T)
            check(x, tok, lp, w, int(np.flatnonzero(w)[0]), r)


@pytest.mark.parametrize("R, V", SPREADS)
def test_the_first_token_of_a_long_top_k(R, V):
    """More tokens kept than the short list holds."""
    x = two_or_three(R, V, np.random.default_rng(R * V))
    k = 200
    light = 1 + np.arange(k)  # behind the first, as light or lighter
    x[:, light] = np.where(x[:, light] == -np.inf, -1.0, x[:, light]).astype(np.float32)
    tok, lp = draw(x, 0.0, top_k=k)
    for r in range(R):
        order = np.lexsort((np.arange(V), -x[r]))[:k]
        w = np.zeros(V)
        w[order] = weights(x[r], 1.0)[order]
        check(x, tok, lp, w, int(np.flatnonzero(w)[0]), r)


@pytest.mark.parametrize("k", [2, 3, 40, 128])
@pytest.mark.parametrize("R, V", SPREADS + [(1, 1 << 20)])
def test_the_first_token_of_a_short_top_k(R, V, k):
    """Tokens kept of 2^-55 to 2^-81 of the largest have a weight too."""
    x = two_or_three(R, V, np.random.default_rng(R * V + k))
    if R == 1:
        x[0] = np.where(np.arange(V) == V // 3, 0.0, np.where(np.arange(V) == V - 9, 41.0, -30.0))
    for u in (0.0, 2.0 ** -90):  # below every share but the first's
        tok, lp = draw(x, u, top_k=k)
        for r in range(R):
            order = np.lexsort((np.arange(V), -x[r]))[:k]
            w = np.zeros(V)
            w[order] = weights(x[r], 1.0)[order]
            check(x, tok, lp, w, int(np.flatnonzero(w)[0]), r)


@pytest.mark.parametrize("T", [0.3, 1.0])
@pytest.mark.parametrize("V", [32000, 50001])
def test_the_first_token_before_a_far_likelier_one(V, T):
    rng = np.random.default_rng(V)
    x = rng.normal(0, 2, (16, V)).astype(np.float32)
    for r in range(16):
        x[r, rng.integers(1, 1900)] += np.float32(45.0 * T)
    tok, lp = draw(x, 0.0, T)
    for r in range(16):
        w = weights(x[r], T)
        z = (x[r].astype(np.float64) - float(x[r].max())) / float(np.float32(T))
        first = int(np.flatnonzero(w)[0])
        # No token before it stands at the border of what counts.
        assert (np.abs(z[:first + 1] + 60) > 1e-3).all()
        check(x, tok, lp, w, first, r)


@pytest.mark.parametrize("R, V", [(2, 50001), (9, 100003)])
@pytest.mark.parametrize("part", range(16))
def test_top_p_ends_in_every_part_of_the_weights(part, R, V):
    """One token of weight 1 and the rest around 2^-(2 part + 1) of it, half of
    whose weight top-p keeps: the border lies in each sixteenth of the 2^-32
    that the histogram of a row over several workgroups covers."""
    rng = np.random.default_rng(part + V)
    x = (-math.log(2) * (2 * part + 2 * rng.random((R, V)))).astype(np.float32)
    at = rng.integers(0, V, R)
    x[np.arange(R), at] = 0.5
    rest = np.exp(x.astype(np.float64) - 0.5).sum(1) - 1
    p = ((1 + rest / 2) / (1 + rest)).astype(np.float32)
    for u in (0.0, 0.37, 0.999):
        check_filters(x, np.full(R, u, np.float32), settings(R, rng, p=p))


@pytest.mark.parametrize("u", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("kw", [{}, dict(top_k=2), dict(top_k=200), dict(min_p=1e-30)], ids=str)
@pytest.mark.parametrize("R, V", SPREADS)
def test_u_from_one_is_one_less_2_to_minus_53(R, V, kw, u):
    """A last token of e^-30 of the sum (2^-43) is drawn by it, one of e^-40
    (2^-58) not: both far from the border."""
    x = np.full((R, V), -np.inf, np.float32)
    heavy = (np.arange(R) * 37) % (V - 1)
    far = np.where(np.arange(R) % 2 == 0, 30.0, 40.0)
    behind = np.minimum(heavy + 1 + (np.arange(R) * 997) % V, V - 1)
    x[np.arange(R), heavy] = 5.0
    x[np.arange(R), behind] = (5.0 - far).astype(np.float32)
    tok, lp = draw(x, u, **kw)
    for r in range(R):
        want = int(behind[r] if far[r] == 30.0 else heavy[r])
        check(x, tok, lp, weights(x[r], 1.0), want, r)


@pytest.mark.parametrize("p", [0.6, 0.9, 0.999])
@pytest.mark.parametrize("R, V", SPREADS)
def test_the_first_token_top_p_keeps(R, V, p):
    """Rows of two or three tokens, and rows of many whose kept tokens are a
    list or the row itself: the first of them at u = 0."""
    rng = np.random.default_rng(R + 3 * V)
    x = two_or_three(R, V, rng)
    x[::2] = rng.normal(0, 1.0, (len(x[::2]), V)).astype(np.float32)
    x[::4, rng.integers(0, V, 5)] += 12.0
    tok, lp = draw(x, 0.0, top_p=p)
    for r in range(R):
        w = weights(x[r], 1.0)
        order = np.lexsort((np.arange(V), -x[r]))
        run = np.cumsum(w[order])
        kept = order[:int((run < float(np.float32(p)) * run[-1]).sum()) + 1]
        want = int(kept.min())
        assert want != int(kept[-1]) or kept.size < 200  # not the border's own
        only = np.zeros(V)
        only[kept] = w[kept]
        assert tok[r] == want, (r, tok[r], want)
        l = math.log(only[want] / only.sum())
        assert abs(lp[r] - l) <= 2.0 ** -24 * abs(l) + 2.0 ** -20, (r, lp[r], l)
