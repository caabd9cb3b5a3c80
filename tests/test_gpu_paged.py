"""The paged-cache operators (csrc/paged.hip, csrc/paged_attention.hip)
against their definitions in 64 bits (paged_ref.py, which derives the
attention's tolerance).

Append: a rotated value is two products and a sum of fp32 with a cosine and
sine each off by half a step (2^-24): within 4 2^-24 (|x0| + |x1|), then half a
step of the cache's type, or the type's least subnormal step."""
import numpy as np
import pytest
import torch

from tests import engine
from tests.paged_ref import EPS, Batch

em = engine.load()
pytestmark = pytest.mark.gpu


def freq(n, base=10000.0):
    return (base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().cuda()


# ---- append ------------------------------------------------------------------

def check_append(b, f, halves, **kw):
    want_q, want_k, want_v = b.ref_append(f, halves)
    before = torch.full((b.rows, b.H * b.D), -7.0, device="cuda")
    b.cuda()
    kc0, vc0 = b.kc.clone(), b.vc.clone()
    got = em.paged_append(b.shape, *b.batch(), b.q(), b.k(), b.v(), b.kc, b.vc, freq=f,
                          halves=halves, q_out=before, **kw)
    torch.cuda.synchronize()
    got = got.double().cpu()
    left = torch.isnan(want_q)
    assert torch.equal(got[left], torch.full_like(got[left], -7.0))
    top = float(b.qkv.abs().max()) * 2
    assert ((got - want_q)[~left].abs() <= 4 * 2.0 ** -24 * top).all()
    for cache, old, want in ((b.kc, kc0, want_k), (b.vc, vc0, want_v)):
        c, old = cache.double().cpu(), old.double().cpu()
        same = want == old
        assert torch.equal(c[same], old[same])  # gaps and other slots as they were
        tol = want.abs() * EPS[b.dtype] + 4 * 2.0 ** -24 * top * (1 + EPS[b.dtype]) + 2.0 ** -25
        assert ((c - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads, kv, D, ps, rotary, halves, layout", [
    (6, 6, 48, 16, 48, False, "slots"), (8, 2, 64, 1, 64, True, "slots"),
    (14, 2, 64, 17, 32, True, "heads"), (4, 4, 128, 24, 64, False, "wide"),
    (20, 4, 80, 32, 40, True, "wide"), (3, 1, 256, 8, 256, True, "heads"),
    (5, 5, 8, 5, 8, False, "slots"), (4, 2, 96, 16, 0, False, "slots")])
def test_append(dtype, heads, kv, D, ps, rotary, halves, layout):
    b = Batch(em, heads, kv, D, ps, [(0, 1), (37, 3), (5, 0), (1000, 1), (0, 41), (15, 1)], dtype,
              layout, seed=D + ps, lead=2, tail=3)
    check_append(b, freq(rotary // 2), halves)


def test_append_far_positions():
    """Angles of positions past 2^24, where fp32 steps are radians."""
    b = Batch(em, 2, 1, 64, 1 << 12, [(0, 2), (0, 2), (0, 1)], "f32", seed=3, spare_columns=0)
    b.max_pages = b.shape.max_pages = 1 << 18
    b.table = torch.full((3, 1 << 18), -1, dtype=torch.int32)
    for s, n in enumerate(((1 << 30) - 5, (1 << 24) + 3, 1 << 29)):
        b.lengths[s] = n
        b.table[s, (n - 1) >> 12] = s
        b.table[s, (n - 2) >> 12] = s
    check_append(b, freq(32), True)


def test_append_in_place_and_without_queries():
    b = Batch(em, 8, 2, 64, 16, [(3, 5), (40, 1)], "bf16", seed=5)
    f = freq(32)
    want, want_k, _ = b.ref_append(f, True)
    b.cuda()
    qkv = b.qkv.clone()
    q = qkv[:, :512]
    got = em.paged_append(b.shape, *b.batch(), q, b.k(), b.v(), b.kc, b.vc, freq=f, halves=True,
                          q_out=q)
    assert got.data_ptr() == q.data_ptr()
    assert (q.double().cpu() - want).abs().max() <= 4 * 2.0 ** -24 * 2 * float(b.qkv.abs().max())
    assert torch.equal(qkv[:, 512:], b.qkv[:, 512:])
    k1 = b.kc.clone()
    b.kc.normal_()
    rest = b.kc.clone()
    assert em.paged_append(b.shape, *b.batch(), None, b.k(), b.v(), b.kc, b.vc, freq=f,
                           halves=True) is None
    changed = b.kc != rest
    assert torch.equal(b.kc[changed], k1[changed]) and int(changed.sum()) > 0.9 * 6 * 128


def test_append_where_nothing_is_stored():
    """Positions that do not exist and pages that hold nothing."""
    b = Batch(em, 4, 2, 64, 8, [(10, 6), (0, 4), (30, 2), (0, 1)], "f32", seed=6, spare_columns=0)
    b.table[0, 1] = -1            # positions 8 .. 15 of sequence 0: a hole
    b.lengths[1] = 2              # its first two rows at -2, -1
    b.table[2, 3] = b.n_pages     # no such page
    b.table[2, 2] = 1 << 30
    b.lengths[3] = b.max_pages * 8 + 1  # its row past the table
    check_append(b, freq(32), False)


# ---- attention ---------------------------------------------------------------

def attend(b, scale=0.0, window=0, **kw):
    out = torch.full((b.rows, b.H * b.D + 8), -7.0, device="cuda")[:, :b.H * b.D]
    em.paged_attention(b.shape, *b.batch(), b.q(), b.kc, b.vc, out, scale=scale, window=window,
                       **kw)
    torch.cuda.synchronize()
    return out.double().cpu().numpy()


def check(b, scale=None, window=0, **kw):
    want, tol = b.ref_attention(scale, window)
    b.cuda()
    got = attend(b, 0.0 if scale is None else scale, window, **kw)
    nobody = np.isnan(want)
    assert (got[nobody] == -7.0).all()
    err = np.abs(got - want)[~nobody]
    assert (err <= tol[~nobody]).all(), (err.max(), tol[~nobody].min())
    assert np.array_equal(got, attend(b, 0.0 if scale is None else scale, window, **kw))
    return got


HEADS = [(6, 6, 48), (8, 2, 64), (32, 8, 128), (4, 4, 128), (20, 4, 80), (3, 1, 256), (14, 2, 64),
         (40, 1, 32), (5, 5, 8), (12, 2, 96), (7, 1, 200)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads, kv, D", HEADS)
def test_one_row_a_sequence(dtype, heads, kv, D):
    seqs = [(n - 1, 1) for n in (1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 128, 129, 300)]
    b = Batch(em, heads, kv, D, 16, seqs, dtype, seed=heads + D)
    check(b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads, kv, D", HEADS)
def test_chunks(dtype, heads, kv, D):
    seqs = [(0, 1), (0, 33), (129, 2), (7, 0), (65, 70), (200, 5), (0, 0), (31, 17)]
    b = Batch(em, heads, kv, D, 16, seqs, dtype, seed=heads * D, lead=1, tail=2)
    check(b)


@pytest.mark.parametrize("ps", [1, 2, 5, 8, 17, 24, 64, 100, 1000])
@pytest.mark.parametrize("layout", ["slots", "heads", "wide"])
def test_pages(ps, layout):
    for dtype in ("f32", "bf16"):
        b = Batch(em, 8, 2, 64, ps, [(0, 40), (333, 1), (97, 130), (12, 3)], dtype, layout,
                  seed=ps)
        check(b)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1 << 30])
def test_window(window):
    for dtype in ("f32", "f16", "bf16"):
        b = Batch(em, 8, 2, 64, 16, [(0, 40), (333, 1), (97, 130), (12, 3), (900, 1)], dtype,
                  seed=window % 1000)
        check(b, window=window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_long_contexts(dtype):
    """Contexts that are split over many workgroups, beside short ones."""
    b = Batch(em, 8, 2, 128, 64, [(9000, 1), (3, 1), (5000, 9), (0, 1)], dtype, seed=11)
    check(b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_long_chunk(dtype):
    b = Batch(em, 8, 8, 64, 32, [(700, 600)], dtype, seed=12)
    check(b)


def test_scale_and_large_scores():
    for scale in (1.0, -0.3, 1e-20, 3.0):
        b = Batch(em, 8, 2, 64, 16, [(333, 1), (50, 40)], "bf16", seed=13, q_scale=4.0)
        check(b, scale=scale)


def test_rows_that_see_nothing_and_holes():
    for dtype in ("f32", "bf16"):
        b = Batch(em, 8, 2, 64, 8, [(90, 6), (0, 4), (30, 40), (0, 3), (50, 1), (64, 5)], dtype,
                  seed=14, spare_columns=0)
        b.table[0, 2:9] = -1           # a hole in the middle
        b.table[1, 0] = -5             # nothing at all
        b.table[2, 0:4] = b.n_pages    # nothing before position 32: rows 30, 31 see nothing
        b.lengths[3] = 1               # rows at -2, -1, 0
        b.lengths[4] = b.max_pages * 8 + 20  # positions past the table are not there
        b.table[5, 8] = 1 << 30        # its own position's page is not there
        got = check(b)
        assert (got[6:10] == 0).all() and (got[10:12] == 0).all()
    check(Batch(em, 8, 2, 64, 8, [(90, 6), (30, 40)], "f32", seed=15), window=3)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see(dtype, bad):
    """Slots behind a sequence's end, other sequences' and, for the earlier
    rows of a chunk, the chunk's own later positions."""
    b = Batch(em, 8, 2, 64, 16, [(40, 1), (70, 33), (5, 4), (600, 40)], dtype, seed=16)
    # A position that only the last rows of its chunk see.
    late = {1: 100, 2: 8, 3: 637}
    want, tol = b.ref_attention()
    kv, vv = b.view(b.kc), b.view(b.vc)
    used = torch.zeros((b.n_pages, b.ps), dtype=torch.bool)
    for s, (p, n) in enumerate(b.seqs):
        for t in range(p + n):
            used[b.page(s, t), t % b.ps] = True
    kv[~used] = bad
    vv[~used] = bad
    for s, t in late.items():
        vv[b.page(s, t), t % b.ps, 0, 5] = bad
        kv[b.page(s, t), t % b.ps, 1, 3] = bad
    b.cuda()
    got = attend(b)
    for r in range(b.rows):
        s, pos = b.owner(r)
        if s in late and pos >= late[s]:
            assert not np.isfinite(got[r, 5::64][:4]).any()  # heads 0 .. 3: kv head 0
            continue
        assert (np.abs(got[r] - want[r]) <= tol[r]).all(), r


def test_scores_of_minus_infinity_have_no_weight():
    b = Batch(em, 4, 2, 64, 16, [(100, 1), (20, 20)], "f32", seed=17)
    b.q()[:, 0::64] = 1.0
    b.q()[:, 1:64] = 0.0
    kv = b.view(b.kc)
    for s, t in ((0, 0), (0, 77), (1, 3)):
        kv[b.page(s, t), t % b.ps, :, 0] = -float("inf")
    check(b)


def test_small_and_large_operands():
    """Scores formed from operands whose low bits a split into 16-bit terms
    drops, or whose products are near fp32's ends."""
    b = Batch(em, 4, 2, 64, 16, [(100, 1), (20, 20)], "f32", seed=18)
    b.qkv[:, :256] *= 2.0 ** -122
    b.kc *= 2.0 ** 118
    check(b)
    b = Batch(em, 4, 2, 64, 16, [(100, 1), (20, 20)], "bf16", seed=19)
    b.qkv[:, :256] *= 2.0 ** -122
    b.kc *= 2.0 ** 118
    check(b)
    b = Batch(em, 4, 2, 64, 16, [(100, 1), (20, 20)], "f32", seed=20)
    b.qkv[:, :256] *= 2.0 ** 110
    b.kc *= 2.0 ** -108
    b.vc *= 2.0 ** 100
    check(b)
    b = Batch(em, 4, 2, 64, 16, [(100, 1), (20, 20)], "f32", seed=21)
    b.vc *= 2.0 ** -120
    check(b)


def test_offsets_past_32_bits():
    """Pages whose elements lie past 2^31, bytes past 2^32."""
    b = Batch(em, 4, 2, 64, 16, [(40, 1), (20, 20)], "bf16", seed=22)
    want, tol = b.ref_attention()
    stride = (1 << 31) // 3
    stride -= stride % 8
    big = [torch.empty(((b.n_pages - 1) * stride + 16 * 128,), dtype=torch.bfloat16, device="cuda")
           for _ in range(2)]
    for dst, src in zip(big, (b.kc, b.vc)):
        dst.as_strided((b.n_pages, 16 * 128), (stride, 1)).copy_(src.view(b.n_pages, -1).cuda())
    assert (b.n_pages - 1) * stride > 1 << 31
    b.shape.page_stride = stride
    b.cuda()
    b.kc, b.vc = big
    got = attend(b)
    assert (np.abs(got - want) <= tol).all()
    k = torch.randn((b.rows, 128), device="cuda")
    em.paged_append(b.shape, *b.batch(), None, k, k, b.kc, b.vc)
    r = 0
    s, pos = b.owner(r)
    at = b.page(s, pos) * stride + pos % 16 * 128
    assert torch.equal(b.kc[at:at + 128], k[r].bfloat16())


def test_shared_pages_and_equal_sequences():
    """A prefix held once, and one sequence given twice: equal rows, equal bits."""
    b = Batch(em, 8, 2, 64, 16, [(64, 1), (64, 1), (30, 20), (30, 20)], "bf16", seed=23)
    b.table[1] = b.table[0]
    b.table[3, :2] = b.table[2, :2]
    b.table[3] = b.table[2]
    b.qkv[1] = b.qkv[0]
    b.qkv[22:42] = b.qkv[2:22]
    got = check(b)
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[2:22], got[22:42])


def test_many_sequences():
    """More sequences than a round of the row lookup, some of them empty."""
    seqs = [(i % 7, i % 3) for i in range(300)]
    b = Batch(em, 4, 1, 32, 4, seqs, "f32", seed=24)
    check(b)
    check_append(Batch(em, 4, 1, 32, 4, seqs, "f16", seed=25), freq(16), True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_long_and_short_sequences(dtype):
    """The plan over several rounds of 64 sequences: split ones of one row,
    chunks of many columns and empty ones among short ones."""
    seqs = [((37 * i) % 90, (1, 1, 0, 2, 1, 5, 1)[i % 7]) for i in range(150)]
    seqs[3], seqs[70], seqs[140], seqs[149] = (4000, 1), (2500, 12), (300, 40), (6000, 1)
    b = Batch(em, 16, 2, 64, 16, seqs, dtype, seed=43, lead=2, tail=1)
    check(b)
    check(b, window=1500)


@pytest.mark.parametrize("heads, kv, D", [(150, 1, 64), (260, 2, 24), (129, 1, 128)])
def test_more_heads_of_a_kv_head_than_a_tile(heads, kv, D):
    for dtype in ("f32", "f16", "bf16"):
        b = Batch(em, heads, kv, D, 16, [(0, 1), (333, 1), (97, 3), (700, 2)], dtype, seed=D)
        check(b)
        check(b, window=50)


def test_empty_batches():
    b = Batch(em, 4, 1, 32, 4, [(5, 0), (0, 0)], "f32", seed=26, tail=3)
    b.cuda()
    assert (attend(b) == -7.0).all()
    before = b.kc.clone()
    em.paged_append(b.shape, *b.batch(), b.q(), b.k(), b.v(), b.kc, b.vc)
    assert torch.equal(before, b.kc)


# ---- streams, graphs, refusals -------------------------------------------------

def test_another_stream():
    b = Batch(em, 8, 2, 64, 16, [(333, 1), (97, 130)], "bf16", seed=27)
    want, tol = b.ref_attention()
    b.cuda()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    outs = [em.paged_attention(b.shape, *b.batch(), b.q(), b.kc, b.vc, stream=s)
            for _ in range(4)]
    s.synchronize()
    for o in outs:
        assert (np.abs(o.double().cpu().numpy() - want) <= tol).all()


def test_two_streams_at_once():
    bs = [Batch(em, 8, 2, 64, 16, [(900 + i, 1), (97, 30)], "bf16", seed=28 + i) for i in (0, 1)]
    refs = [b.ref_attention() for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    for b in bs:
        b.cuda()
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (b, s) in enumerate(zip(bs, streams)):
            with torch.cuda.stream(s):
                outs[i].append(em.paged_attention(b.shape, *b.batch(), b.q(), b.kc, b.vc))
    torch.cuda.synchronize()
    for (want, tol), os_ in zip(refs, outs):
        for o in os_:
            assert (np.abs(o.double().cpu().numpy() - want) <= tol).all()


def test_graph_serves_other_lengths():
    """One capture of append and attention, replayed while the batch's device
    arrays change, beside an eager call on the same caches."""
    b = Batch(em, 8, 2, 64, 16, [(400, 1), (300, 1), (200, 1)], "bf16", seed=30)
    b.cuda()
    f = freq(32)
    out = torch.zeros((3, 512), device="cuda")
    q_out = torch.zeros((3, 512), device="cuda")
    scratch = torch.empty((max(1, em.paged_attention_scratch_floats(b.shape, 3, 3)),), device="cuda")

    def step():
        em.paged_append(b.shape, *b.batch(), b.q(), b.k(), b.v(), b.kc, b.vc, freq=f, halves=True,
                        q_out=q_out)
        em.paged_attention(b.shape, *b.batch(), q_out, b.kc, b.vc, out, scratch=scratch)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for lens in ([400, 300, 200], [1, 17, 90], [350, 2, 401], [33, 64, 128]):
        b.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        kc = b.kc.clone()
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(kc, b.kc)
        assert bool((got != 0).any(1).all())


def test_python_checks():
    b = Batch(em, 8, 2, 64, 16, [(33, 1), (7, 3)], "bf16", seed=31).cuda()
    ok = dict(row_start=b.starts, lengths=b.lengths, page_table=b.table, q=b.q(), key_cache=b.kc,
              value_cache=b.vc)
    for kw in (dict(row_start=b.starts[:-1]), dict(row_start=b.starts.long()),
               dict(lengths=b.lengths.cpu()), dict(page_table=b.table[:, :1]),
               dict(page_table=b.table[:1]), dict(q=b.q().double()), dict(q=b.q()[:, :100]),
               dict(q=b.q().t()), dict(key_cache=b.kc.float()), dict(value_cache=b.vc[:-8]),
               dict(value_cache=b.vc.cpu()), dict(scratch=torch.empty(1, device="cuda").int()),
               dict(out=torch.empty((3, 512), device="cuda"))):
        with pytest.raises(em.InvalidArgument):
            em.paged_attention(b.shape, **{**ok, **kw})
    need = em.paged_attention_scratch_floats(b.shape, 2, 4)
    if need:
        with pytest.raises(em.InvalidArgument, match="scratch"):
            em.paged_attention(b.shape, **ok, scratch=torch.empty(need - 1, device="cuda"))
    em.paged_attention(b.shape, **ok)


# ---- a run of them together ------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_serving_steps(dtype):
    """Prompts of three requests, then steps of one token each, the next
    token drawn from the attention's output as logits: every step's output
    against 64 bits on the caches as they are."""
    H, KV, D, ps = 8, 2, 64, 16
    b = Batch(em, H, KV, D, ps, [(0, 37), (0, 5), (0, 64)], dtype, seed=32, spare_columns=2)
    # Pages for the tokens to come.
    free = [p for p in range(b.n_pages) if p not in set(b.table.flatten().tolist())]
    b.table[0, 3] = free[0]
    b.table[2, 4] = free[1]
    b.cuda()
    f = freq(D // 2)
    g = torch.Generator(device="cuda").manual_seed(33)
    w = torch.randn((H * D, 100), generator=g, device="cuda")
    emb = torch.randn((100, (H + 2 * KV) * D), generator=g, device="cuda")
    for step in range(8):
        q = em.paged_append(b.shape, *b.batch(), b.q(), b.k(), b.v(), b.kc, b.vc, freq=f)
        rot, kc, vc = Batch.ref_append(b, f, False)
        assert (q.double().cpu() - rot).abs().max() <= 8 * 2.0 ** -24 * float(b.qkv.abs().max())
        b.qkv[:, :H * D] = q
        want, tol = b.ref_attention()
        out = em.paged_attention(b.shape, *b.batch(), b.q(), b.kc, b.vc)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all(), step
        last = out[(b.starts[1:] - 1).long()]
        logits = em.matmul(last.contiguous(), w)
        u = torch.rand((3,), generator=g, device="cuda")
        token, logprob = em.sample(logits, u, top_k=torch.full((3,), 5, dtype=torch.int32,
                                                               device="cuda"))
        kept = logits.topk(5, 1).indices
        assert bool((kept == token[:, None].long()).any(1).all()) and bool((logprob <= 0).all())
        # The next step: one row a sequence.
        b.qkv = emb[token.long()].contiguous()
        b.lengths += 1
        b.seqs = [(int(n) - 1, 1) for n in b.lengths]
        b.starts = torch.arange(4, dtype=torch.int32, device="cuda")
        b.rows = 3


def test_agrees_with_the_contiguous_cache():
    """A sequence whose pages lie in order is em_attention's cache."""
    H, KV, D, n = 8, 2, 64, 200
    b = Batch(em, H, KV, D, 50, [(190, 10)], "f32", seed=34)
    b.table[0, :4] = torch.arange(4, dtype=torch.int32)
    want, tol = b.ref_attention()
    b.cuda()
    s = em.attention_shape(H, KV, D, n)
    pos = torch.full((1,), 190, dtype=torch.int32, device="cuda")
    flat = em.attention(s, 10, pos, b.qkv, b.kc, b.vc)
    paged = em.paged_attention(b.shape, *b.batch(), b.q(), b.kc, b.vc)
    assert (np.abs((flat - paged).double().cpu().numpy()) <= 2 * tol).all()
