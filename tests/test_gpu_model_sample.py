"""em_model_sample: the forward pass with the token drawn on the GPU. forward()
on the same tokens gives the same logits bit for bit (the same kernels and
graph nodes up to where they are written), so its token is em_sample's on
them, eagerly and replayed, whatever settings a captured step was made with."""
import ctypes

import numpy as np
import pytest
import torch

from tests import engine, inputs

em = engine.load()
pytestmark = pytest.mark.gpu


def model(q8=False, vocab=1000, heads=4, kv_heads=2, dim=64, hidden=96, layers=2, seq_len=40, seed=1):
    kv = dim // heads * kv_heads
    w = lambda *shape: inputs.normal(shape, 0.5 / np.sqrt(shape[0]) * 4, seed + sum(shape))
    one = lambda n: inputs.uniform((n,), 0.8, 1.2, seed + n)
    weights = {"token_embedding": inputs.normal((vocab, dim), 1.0, seed), "rms_final": one(dim),
               "wcls": w(dim, vocab),
               "layers": [{"rms_att": one(dim), "wqkv": w(dim, dim + 2 * kv), "wo": w(dim, dim),
                           "rms_ffn": one(dim), "w13": w(dim, 2 * hidden), "w2": w(hidden, dim)}
                          for _ in range(layers)]}
    cfg = dict(dim=dim, hidden_dim=hidden, n_layers=layers, n_heads=heads, n_kv_heads=kv_heads,
               vocab_size=vocab, seq_len=seq_len)
    return em.Model(cfg, weights, q8=q8)


def draw(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    one = lambda v, t=torch.float32: torch.tensor([v], dtype=t, device="cuda")
    tok, lp = em.sample(torch.from_numpy(logits)[None].cuda(), one(u), one(temperature),
                        one(top_k, torch.int32) if top_k > 0 else None, one(top_p), one(min_p))
    return int(tok), float(lp)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=20), dict(top_p=0.6),
            dict(top_k=5, top_p=0.9, min_p=0.01), dict(min_p=0.2, temperature=1.5)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("vocab", [1000, 40000])
def test_draws_from_the_logits_forward_returns(q8, vocab):
    m = model(q8, vocab)
    prompt = [5, 9, 2, 77, 31]
    u = inputs.uniform((64,), 0.0, 1.0, 3)
    want = draw(m.forward(prompt, 0), float(u[0]), top_p=0.9)
    assert m.sample(prompt, 0, float(u[0]), top_p=0.9) == want
    token, pos = want[0], len(prompt)
    for i in range(24):  # eager, captured and replayed steps of both kinds
        kw = SETTINGS[i % len(SETTINGS)]
        logits = m.forward(token, pos)
        got = m.sample(token, pos, float(u[i + 1]), **kw)
        assert got == draw(logits, float(u[i + 1]), **kw), (i, kw)
        assert np.array_equal(logits, m.forward(token, pos))
        token, pos = got[0], pos + 1
    m.close()


def test_rejections_leave_the_cache():
    m = model()
    first = m.forward([1, 2, 3], 0)
    for args, err in ((([1], 9, 0.5), em.OutOfRange), (([1000], 3, 0.5), em.OutOfRange),
                      (([1] * 41, 0, 0.5), em.OutOfRange)):
        with pytest.raises(err):
            m.sample(*args)
    tok = ctypes.c_int()
    L = em.lib()
    assert L.em_model_sample(None, None, 1, 0, 1.0, 0, 1.0, 0.0, 0.5, None, None) == em.EM_EINVAL
    assert L.em_model_sample(m.h, None, 0, 0, 1.0, 0, 1.0, 0.0, 0.5, ctypes.addressof(tok),
                             None) == em.EM_EINVAL
    one = np.array([1], np.int32)
    assert L.em_model_sample(m.h, one.ctypes.data, 1, 3, 1.0, 0, 1.0, 0.0, 0.5, None,
                             None) == em.EM_EINVAL
    assert L.em_model_sample(m.h, one.ctypes.data, 1, 3, 0.0, 0, 1.0, 0.0, 0.5,
                             ctypes.addressof(tok), None) == em.EM_OK
    assert tok.value == int(np.argmax(m.forward([1], 3)))
    assert np.array_equal(first, m.forward([1, 2, 3], 0))


def test_greedy_stream_is_the_argmax_stream():
    m = model(vocab=2000)
    a = b = 7
    for pos in range(30):
        a = int(np.argmax(m.forward(a, pos)))
    for pos in range(30):
        b = m.sample(b, pos, 0.9, temperature=0.0)[0]
    assert a == b
