"""Sampling (csrc/sample.hip) against its definition in 64 bits. Tokens are
equal; where u lies within 2^-30 of a border of the cumulative weights (which
sums of integers of 2^-42 and finer settle otherwise than 64-bit floats may) the
tokens on both sides count. A log-probability is rounded to fp32 once and its
sum holds integers of 2^-42: within 2^-24 of it and 2^-20."""
import math

import numpy as np
import pytest
import torch

from tests import engine

em = engine.load()
pytestmark = pytest.mark.gpu


def reference(x, u, T, k, p, mp):
    """(tokens that are right, logprob of each) of one row."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    V = x.size
    top = x.max()
    if top == -np.inf:
        return [-1], [-math.inf]
    if not T > 0:
        return [int(np.argmax(x))], [0.0]
    with np.errstate(all="ignore"):
        z = np.where(x == top, 0.0, x - top)  # top may be +inf
        w = np.exp(np.where(z == -np.inf, -np.inf, z / T))
    w = np.where(x == -np.inf, 0.0, w)
    order = np.lexsort((np.arange(V), -x))
    order = order[x[order] > -np.inf]
    if k > 0:
        order = order[:k]
    if p < 1:
        run = np.cumsum(w[order])
        n = 1 if p <= 0 else int((run < p * run[-1]).sum()) + 1
        order = order[:n]
    if mp > 0:
        order = order[w[order] >= min(float(mp), 1.0)]
    kept = np.sort(order)
    run = np.cumsum(w[kept])
    u = 0.0 if not u > 0 else min(float(u), 1 - 2.0 ** -53)
    tokens = sorted({int(kept[min(int((run <= v * run[-1]).sum()), kept.size - 1)])
                     for v in (u, u - 2.0 ** -30, u + 2.0 ** -30)})
    return tokens, [math.log(w[t] / run[-1]) if w[t] else -math.inf for t in tokens]


def settings(R, rng, T=None, k=None, p=None, mp=None):
    def arr(v, dt):
        return None if v is None else np.broadcast_to(np.asarray(v, dt), (R,)).copy()
    return (arr(T, np.float32), arr(k, np.int32), arr(p, np.float32), arr(mp, np.float32))


def check(x, u, st, stride=None):
    R, V = x.shape
    T, k, p, mp = st
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()
    xd = torch.from_numpy(x).cuda()
    if stride:
        wide = torch.full((R, stride), 1e30, device="cuda")
        wide[:, :V] = xd
        xd = wide[:, :V]
    args = dict(temperature=dev(T), top_k=dev(k), top_p=dev(p), min_p=dev(mp))
    tok, lp = em.sample(xd, dev(u), **args)
    tok2, lp2 = em.sample(xd, dev(u), **args)
    assert torch.equal(tok, tok2) and torch.equal(lp.view(torch.int32), lp2.view(torch.int32))
    tok, lp = tok.cpu().numpy(), lp.cpu().numpy()
    for r in range(R):
        want, wl = reference(x[r], float(u[r]), float(T[r]) if T is not None else 1.0,
                             int(k[r]) if k is not None else 0,
                             float(p[r]) if p is not None else 1.0,
                             float(mp[r]) if mp is not None else 0.0)
        assert tok[r] in want, (r, tok[r], want)
        l = wl[want.index(tok[r])]
        if l == -math.inf:
            assert lp[r] == -math.inf
        else:
            assert abs(lp[r] - l) <= 2.0 ** -24 * abs(l) + 2.0 ** -20, (r, lp[r], l)
    return tok


def logits(R, V, rng, spread=2.0):
    x = rng.normal(0, spread, (R, V)).astype(np.float32)
    for r in range(R):
        x[r, rng.integers(0, V, 6)] += rng.uniform(0, 9, 6).astype(np.float32)
    return x


VOCABS = [1, 2, 3, 63, 64, 255, 256, 257, 1000, 1023, 1025, 4095, 4097, 8191, 32000, 50001]


@pytest.mark.parametrize("V", VOCABS)
def test_each_filter(V):
    rng = np.random.default_rng(V)
    R = 24
    x = logits(R, V, rng)
    u = rng.random(R).astype(np.float32)
    for kw in (dict(), dict(T=0.0), dict(T=0.7), dict(k=1), dict(k=5, T=1.3), dict(k=V), dict(k=V + 1),
               dict(p=0.9), dict(p=0.0), dict(p=1e-7), dict(p=0.999999), dict(mp=0.1),
               dict(mp=1.0), dict(k=50, p=0.95, T=0.8), dict(k=20, p=0.5, mp=0.05, T=1.5)):
        check(x, u, settings(R, rng, **kw))


@pytest.mark.parametrize("R, V", [(1, 131072), (3, 100003), (2, 1 << 20), (300, 1000), (1, 160001)])
def test_sizes_and_mixed_rows(R, V):
    rng = np.random.default_rng(R + V)
    x = logits(R, V, rng, 2.5)
    u = rng.random(R).astype(np.float32)
    for i in range(2 if V < 1 << 20 else 1):
        T = np.where(rng.random(R) < 0.2, 0.0, rng.uniform(0.3, 2.0, R)).astype(np.float32)
        k = np.where(rng.random(R) < 0.5, 0, rng.integers(1, 200, R)).astype(np.int32)
        p = np.where(rng.random(R) < 0.4, 1.0, rng.uniform(0.1, 1.0, R)).astype(np.float32)
        mp = np.where(rng.random(R) < 0.6, 0.0, rng.uniform(0, 0.2, R)).astype(np.float32)
        check(x, u, (T, k, p, mp))
    check(x, u, settings(R, rng, p=0.9))
    check(x, u, settings(R, rng))


@pytest.mark.parametrize("V", [10, 257, 5000, 32000, 70001])
def test_ties(V):
    """Few distinct logits: the filters cut inside a run of equal ones, whose
    lowest indices stay."""
    rng = np.random.default_rng(V)
    R = 16
    x = rng.integers(0, 3, (R, V)).astype(np.float32)
    x[0] = 1.0
    x[1] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    u = rng.random(R).astype(np.float32)
    u[:2] = 0.999999
    for kw in (dict(), dict(T=0.0), dict(k=1), dict(k=3), dict(k=V // 2), dict(p=0.5), dict(p=0.03),
               dict(k=V // 2 + 1, p=0.7), dict(mp=0.5), dict(T=math.inf, k=4)):
        check(x, u, settings(R, rng, **kw))


def test_numbers_at_the_ends():
    V = 3000
    rng = np.random.default_rng(5)
    x = logits(12, V, rng)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 7] = np.nan
    x[3, [5, 900]] = np.inf
    x[4, :] = -np.inf
    x[4, 2999] = -3.4e38
    x[5, :2990] = -np.inf
    x[6] = -3.4028235e38
    x[7] *= 1e38 / 20
    x[8] *= 1e-38
    x[9, 0] = 3.4028235e38
    x[10] = np.finfo(np.float32).min
    u = np.full(12, 0.6, np.float32)
    for kw in (dict(), dict(T=0.0), dict(k=3), dict(k=100), dict(p=0.7), dict(mp=0.2),
               dict(T=1e-30), dict(T=1e30), dict(T=math.inf), dict(T=math.nan), dict(T=-1.0),
               dict(p=math.nan), dict(mp=math.nan), dict(p=-1.0), dict(mp=7.0), dict(k=-3)):
        check(x, u, settings(12, rng, **kw))


def test_u_at_the_ends():
    x = logits(7, 999, np.random.default_rng(6))
    u = np.array([0, -1, math.nan, 1, 2, 1 - 2.0 ** -24, 2.0 ** -40], np.float32)
    for kw in (dict(), dict(k=3), dict(p=0.8), dict(mp=0.3)):
        check(x, u, settings(7, None, **kw))


def test_strided_rows():
    rng = np.random.default_rng(7)
    x = logits(5, 777, rng)
    u = rng.random(5).astype(np.float32)
    for stride in (778, 1001, 4096):
        check(x, u, settings(5, rng, k=20, p=0.9), stride)


def test_every_token_by_its_share():
    """u over a fine grid draws every token as often as its weight says."""
    V, R = 50, 4096
    x = np.tile(np.random.default_rng(8).normal(0, 1.5, V).astype(np.float32), (R, 1))
    u = ((np.arange(R) + 0.5) / R).astype(np.float32)
    tok = check(x, u, settings(R, None, T=0.9))
    w = np.exp((x[0].astype(np.float64) - x[0].max()) / np.float32(0.9))
    share = np.bincount(tok, minlength=V) / R
    assert np.abs(share - w / w.sum()).max() <= 1.0 / R  # borders fall between grid points
    assert (np.diff(tok) >= 0).all()


def test_graph_and_streams():
    rng = np.random.default_rng(9)
    x = torch.from_numpy(logits(6, 20011, rng)).cuda()
    p = torch.full((6,), 0.9, device="cuda")
    us = [torch.rand((6,), device="cuda") for _ in range(5)]
    want = [em.sample(x, u, top_p=p)[0].clone() for u in us]
    u = us[0].clone()
    tok = torch.empty((6,), dtype=torch.int32, device="cuda")
    lp = torch.empty((6,), device="cuda")
    scratch = torch.empty((max(1, em.sample_scratch_bytes(6, 20011)),), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        em.sample(x, u, top_p=p, tokens=tok, logprobs=lp, scratch=scratch)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        em.sample(x, u, top_p=p, tokens=tok, logprobs=lp, scratch=scratch)
    for v, w in zip(us, want):
        u.copy_(v)
        tok.fill_(-5)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(tok, w)
        assert torch.equal(em.sample(x, u, top_p=p)[0], w)
    got = [em.sample(x, v, top_p=p, stream=side)[0] for v in us]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_python_checks():
    x = torch.zeros((2, 10), device="cuda")
    u = torch.zeros((2,), device="cuda")
    for kw in (dict(logits=x.half()), dict(logits=x[0]), dict(logits=x.t()), dict(u=u[:1]),
               dict(u=u.cpu()), dict(top_k=u), dict(temperature=u.double()),
               dict(tokens=u), dict(scratch=u)):
        with pytest.raises(em.InvalidArgument):
            em.sample(**{**dict(logits=x, u=u), **kw})


# Rows that are spread over workgroups (few of a large vocabulary), rows done by
# one workgroup from memory (many) and from LDS (up to 32765 logits).
SPREADS = [(1, 9000), (3, 20000), (2, 50021), (100, 40007), (300, 33000), (200, 30000)]


@pytest.mark.parametrize("R, V", SPREADS)
def test_masked_runs_and_every_setting(R, V):
    """Long runs of -inf and NaN, where whole threads have nothing to draw."""
    rng = np.random.default_rng(R * V)
    R = min(R, 100) if V > 35000 else R
    x = logits(R, V, rng, 1.5)
    x[:, V // 4:V // 2] = -np.inf
    x[0, :] = -np.inf
    x[0, [3, V // 2 + 7, V - 1]] = [1.0, 2.0, 0.5]
    if R > 2:
        x[1, V // 2:] = np.nan
        x[2, :-2] = -np.inf
    u = rng.random(R).astype(np.float32)
    step = max(1, R // 12)
    x, u = x[::step].copy(), u[::step].copy()
    x = np.concatenate([x, np.repeat(x[-1:], R - x.shape[0], 0)])
    u = np.concatenate([u, np.repeat(u[-1:], R - u.shape[0], 0)])
    for kw in (dict(), dict(T=0.0), dict(T=math.inf), dict(T=0.2, p=0.9), dict(T=5.0, p=0.5),
               dict(k=40), dict(k=128, p=0.9), dict(k=129), dict(k=2000, p=0.3, mp=0.01),
               dict(p=0.99, mp=0.02), dict(mp=0.3), dict(p=0.0), dict(T=1e-3, p=0.999)):
        check(x, u, settings(R, rng, **kw))


@pytest.mark.parametrize("R, V", [(5, 40000), (300, 40000)])
def test_ties_across_workgroups(R, V):
    """Runs of equal logits over the borders between the workgroups' shares."""
    rng = np.random.default_rng(V + R)
    x = np.full((R, V), -2.0, np.float32)
    x[:, ::7] = 1.0
    x[0] = rng.integers(0, 40, V) * 0.25
    x[1, 10000:30000] = 3.0
    x[-1] = 0.5
    u = rng.random(R).astype(np.float32)
    u[-1] = 0.99999
    n = 4  # rows of their own; the rest repeat
    x[n:-1] = x[2]
    u[n:-1] = u[2]
    for kw in (dict(), dict(T=0.0), dict(k=3), dict(k=100), dict(k=5000), dict(p=0.5), dict(p=0.9),
               dict(k=6000, p=0.7), dict(mp=0.5)):
        check(x, u, settings(R, rng, **kw))


@pytest.mark.parametrize("V", [5000, 40000])
def test_more_infinities_than_are_kept(V):
    """Of tokens of infinite logits top-k keeps the first, which share the weight."""
    rng = np.random.default_rng(V)
    x = logits(4, V, rng)
    for r, n in enumerate((1, 150, 1500, V)):
        x[r, np.sort(rng.permutation(V)[:n])] = np.inf
    for u in (0.0, 0.3, 0.77, 0.9999):
        for kw in (dict(), dict(k=140), dict(k=600), dict(k=1200, p=0.5), dict(p=0.7), dict(mp=0.5)):
            check(x, np.full(4, u, np.float32), settings(4, rng, **kw))


def test_rows_together_or_alone_agree():
    """A row's draw does not depend on how many rows share the call."""
    rng = np.random.default_rng(11)
    x = np.repeat(logits(4, 60013, rng), 100, 0)
    u = np.tile(rng.random(100).astype(np.float32), 4)
    p = np.full(400, 0.8, np.float32)
    many = em.sample(torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda(),
                     top_p=torch.from_numpy(p).cuda())[0].cpu()
    for r in (0, 57, 123, 250, 399):
        one = em.sample(torch.from_numpy(x[r:r + 1]).cuda(), torch.from_numpy(u[r:r + 1]).cuda(),
                        top_p=torch.from_numpy(p[:1]).cuda())[0].cpu()
        assert int(one[0]) == int(many[r])
