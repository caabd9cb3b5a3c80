"""The paged-cache and sampling operators' refusals, on the host before any
HIP call: every bad argument has a message, and nothing to do is no error."""
import ctypes

import pytest

from tests import engine

em = engine.load()
P = 4096  # a pointer that no refused call follows


def shape(**kw):
    a = dict(n_heads=8, n_kv_heads=2, head_size=64, page_size=16, n_pages=10, max_pages=4,
             dtype="bf16")
    a.update(kw)
    return em.paged_shape(**a)


def batch(n_seqs=2, row_start=P, lengths=P, page_table=P, table_stride=4):
    return em.PagedBatch(n_seqs, row_start, lengths, page_table, table_stride)


def code(rc):
    return rc, em.lib().em_last_error().decode()


def append(s=None, b=None, rows=3, q=P, qs=768, k=P, ks=768, v=P, vs=768, freq=P, rotary=64,
           halves=0, q_out=P, os_=512, kc=P, vc=P):
    return code(em.lib().em_paged_append(ctypes.byref(s or shape()), ctypes.byref(b or batch()),
                                         rows, q, qs, k, ks, v, vs, freq, rotary, halves, q_out,
                                         os_, kc, vc, None))


def attention(s=None, b=None, rows=3, q=P, qs=768, kc=P, vc=P, out=P, os_=512, scale=0.0,
              window=0, scratch=P):
    return code(em.lib().em_paged_attention(ctypes.byref(s or shape()), ctypes.byref(b or batch()),
                                            rows, q, qs, kc, vc, out, os_, scale, window, scratch,
                                            None))


def sample(rows=2, vocab=100, logits=P, stride=100, u=P, settings=True, tokens=P, logprobs=None,
           scratch=P):
    st = em.Sampling()
    return code(em.lib().em_sample(rows, vocab, logits, stride, u,
                                   ctypes.byref(st) if settings else None, tokens, logprobs,
                                   scratch, None))


BAD_SHAPES = [
    (dict(n_heads=0), "multiple of n_kv_heads"), (dict(n_kv_heads=0), "multiple of n_kv_heads"),
    (dict(n_kv_heads=3), "multiple of n_kv_heads"), (dict(n_heads=8192), "4096 heads"),
    (dict(head_size=60), "multiple of 8"), (dict(head_size=264), "at most 256"),
    (dict(head_size=0), "head_size"), (dict(page_size=0), "positive"),
    (dict(n_pages=0), "positive"), (dict(max_pages=0), "positive"),
    (dict(page_size=1 << 16, max_pages=1 << 15), "2^30 positions"),
    (dict(dtype=7), "cache type"), (dict(slot_stride=132), "multiples of 8"),
    (dict(head_stride=56), "smaller than head_size"), (dict(slot_stride=0), "smaller"),
    (dict(page_stride=0), "smaller"), (dict(page_stride=1 << 58), "2^34"),
]


@pytest.mark.parametrize("kw, why", BAD_SHAPES, ids=lambda x: str(x))
def test_shapes_that_cannot_run(kw, why):
    s = shape(**kw)
    with pytest.raises(em.InvalidArgument, match=why.replace("^", r"\^")):
        em.paged_check(s)
    for rc, msg in (append(s), attention(s)):
        assert rc == em.EM_EINVAL and why in msg
    assert em.paged_attention_scratch_floats(s, 2, 3) == 0


@pytest.mark.parametrize("call", [append, attention])
def test_batches_that_cannot_run(call):
    for b, rows, why in ((batch(n_seqs=-1), 3, "sequences"), (batch(row_start=None), 3, "null"),
                         (batch(lengths=None), 3, "null"), (batch(page_table=None), 3, "null"),
                         (batch(table_stride=3), 3, "table_stride"),
                         (batch(), (1 << 22) + 1, "2^22 rows")):
        rc, msg = call(b=b, rows=rows)
        assert rc == em.EM_EINVAL and why in msg
    assert call(rows=0)[0] == em.EM_OK
    assert call(b=batch(n_seqs=0))[0] == em.EM_OK


def test_append_arguments():
    for kw, why in ((dict(rotary=60), "rotary"), (dict(rotary=-8), "rotary"),
                    (dict(rotary=72), "rotary"), (dict(freq=None), "null"), (dict(k=None), "null"),
                    (dict(v=None), "null"), (dict(q_out=None), "null"), (dict(kc=None), "null"),
                    (dict(vc=None), "null"), (dict(qs=766), "strides"), (dict(qs=508), "strides"),
                    (dict(ks=124), "strides"), (dict(vs=130), "strides"),
                    (dict(os_=500), "strides"), (dict(q=P + 4), "aligned"),
                    (dict(k=P + 8), "aligned"), (dict(v=P + 8), "aligned"),
                    (dict(freq=P + 4), "aligned"), (dict(kc=P + 2), "aligned"),
                    (dict(vc=P + 2), "aligned"), (dict(q_out=P + 4), "aligned")):
        rc, msg = append(**kw)
        assert rc == em.EM_EINVAL and why in msg, kw


def test_attention_arguments():
    for kw, why in ((dict(window=-1), "window"), (dict(window=(1 << 30) + 1), "window"),
                    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
                    (dict(scale=3e38), "scale"), (dict(q=None), "null"),
                    (dict(kc=None), "null"), (dict(vc=None), "null"), (dict(out=None), "null"),
                    (dict(qs=500), "strides"), (dict(os_=514), "strides"), (dict(q=P + 4), "aligned"),
                    (dict(kc=P + 8), "aligned"), (dict(out=P + 4), "aligned")):
        rc, msg = attention(**kw)
        assert rc == em.EM_EINVAL and why in msg, kw
    if em.paged_attention_scratch_floats(shape(), 2, 3):
        assert "null" in attention(scratch=None)[1]
        assert "aligned" in attention(scratch=P + 4)[1]


def test_sampling_arguments():
    for kw, why in ((dict(vocab=0), "vocabulary"), (dict(vocab=(1 << 20) + 1, stride=1 << 21),
                                                    "vocabulary"),
                    (dict(rows=(1 << 20) + 1), "rows"), (dict(stride=99), "stride"),
                    (dict(settings=False), "settings"), (dict(logits=None), "null"),
                    (dict(u=None), "null"), (dict(tokens=None), "null")):
        rc, msg = sample(**kw)
        assert rc == em.EM_EINVAL and why in msg, kw
    assert sample(rows=0)[0] == em.EM_OK
    assert em.sample_scratch_bytes(2, 1 << 21) == 0
    if em.sample_scratch_bytes(2, 100):
        assert "null" in sample(scratch=None)[1]
        assert "aligned" in sample(scratch=P + 8)[1]


def test_no_device_is_reported():
    if em.available():
        pytest.skip("a GPU is present")
    for rc, _ in (append(), attention(), sample()):
        assert rc == em.EM_ENODEV
