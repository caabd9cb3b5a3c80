"""Paged batches that the header defines and other tests do not reach: row
starts that leave the call's rows, operands of far apart sizes, against the 64-bit definitions of
paged_ref.py with the tolerances of test_gpu_paged.py."""
import math

import pytest
import torch

from tests import engine
from tests.paged_ref import Batch
from tests.test_gpu_paged import check, check_append, freq

em = engine.load()
pytestmark = pytest.mark.gpu


class Cut(Batch):
    """A sequence whose rows are not all the call's has none."""

    def owner(self, r):
        s, pos = super().owner(r)
        st = self.starts.tolist()
        if s is not None and (st[s] < 0 or st[s + 1] > self.rows):
            return None, None
        return s, pos


SEQS = [(2000, 5), (900, 1), (0, 0), (3000, 40), (17, 3), (2500, 6)]


def cut(dtype, first, last, seed):
    b = Cut(em, 8, 2, 64, 16, SEQS, dtype, seed=seed, tail=2)
    if first:
        b.starts[0] = -first
    if last:
        b.rows -= 2 + last
        b.qkv = b.qkv[:b.rows].contiguous()
    return b


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("first, last", [(1, 0), (0, 1), (0, 5), (3, 4), (1 << 30, 6)])
def test_rows_that_are_not_the_calls(dtype, first, last):
    """Sequences at the batch's ends with rows before its first or behind its
    last: nobody's to both operators, and the sequences beside them, split ones
    among them, as they are without."""
    b = cut(dtype, first, last, 50 + last)
    check(b)
    check(b, window=700)
    check_append(cut(dtype, first, last, 60 + last), freq(32), True)


def test_no_row_is_the_calls():
    b = Cut(em, 8, 2, 64, 16, [(2000, 5)], "bf16", seed=70)
    b.rows = 4
    b.qkv = b.qkv[:4].contiguous()
    got = check(b)
    assert (got == -7.0).all()
    check_append(Cut(em, 8, 2, 64, 16, [(0, 0), (2000, 5)], "f32", seed=71, lead=1), freq(32), False)


def test_new_queries_hold_zeros_where_nothing_is_rotated():
    """Rows that are nobody's or at positions that do not exist, in memory that
    held something else before."""
    b = Batch(em, 8, 2, 64, 16, [(37, 3), (0, 4), (5, 1)], "bf16", seed=72, lead=2, tail=3,
              spare_columns=0)
    b.lengths[1] = 2                     # its first two rows at -2, -1
    b.lengths[2] = b.max_pages * 16 + 1  # its row past the table
    f = freq(32)
    want, _, _ = b.ref_append(f, True)
    left = torch.isnan(want)
    assert left.any(1).tolist() == [True] * 2 + [False] * 3 + [True] * 2 + [False] * 2 + [True] * 4
    b.cuda()
    for _ in range(8):
        old = [torch.full((b.rows, 512), float("nan"), device="cuda") for _ in range(4)]
        del old
        got = em.paged_append(b.shape, *b.batch(), b.q(), b.k(), b.v(), b.kc, b.vc, freq=f,
                              halves=True).double().cpu()
        assert (got[left] == 0).all()
        top = float(b.qkv.abs().max()) * 2
        assert ((got - want)[~left].abs() <= 4 * 2.0 ** -24 * top).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads, kv, D", [(4, 2, 64), (8, 1, 128), (3, 3, 80), (2, 1, 256)])
@pytest.mark.parametrize("small", [-16, -8, -3])
def test_small_query_dims_beside_a_large_one(dtype, heads, kv, D, small):
    """The large dims meet keys of zero, the small ones large keys: the scores
    are made of bits far below the column's largest."""
    b = Batch(em, heads, kv, D, 16, [(100, 1), (20, 40), (300, 1), (64, 3)], dtype, seed=80 - small)
    b.q()[:] *= 2.0 ** small
    b.q()[:, 3::D] = 2.0 ** 13
    b.kc *= 2.0 ** 13
    b.view(b.kc)[..., 3] = 0
    assert b.kc.isfinite().all()
    check(b)


def test_ordinary_queries_with_small_dims():
    """Dims of 0 and of a millionth of the others beside ordinary ones."""
    for dtype in ("f16", "bf16"):
        b = Batch(em, 8, 2, 128, 16, [(500, 1), (20, 40)], dtype, seed=90, q_scale=4.0)
        b.q()[:, 5::7] *= 1e-6
        b.q()[:, 6::7] = 0.0
        check(b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 20])
def test_many_small_weights(dtype, rows):
    """20000 positions of value 1 and weight e^-21 beside one of value 0: sums of
    equal terms, at most one rounding (2^-24) each, scores of one product (21
    2^-24 and as much in log2 units), and over fp16 2^-39 a weight."""
    n = 20000
    b = Batch(em, 8, 2, 64, 64, [(n, rows)], dtype, seed=91)
    b.q()[:] = 0.0
    b.q()[:, ::64] = 1.0
    kv, vv = b.view(b.kc), b.view(b.vc)
    kv[:], vv[:] = 0.0, 1.0
    kv[..., 0] = -21.0
    p = b.page(0, 0)
    kv[p, 0], vv[p, 0] = 0.0, 0.0
    b.cuda()
    got = em.paged_attention(b.shape, *b.batch(), b.q(), b.kc, b.vc, scale=1.0).double().cpu()
    for r in range(rows):
        s = (n + r) * math.exp(-21.0)
        want = s / (1 + s)
        tol = want * (n + r + 200) * 2.0 ** -24 + (n + r) * 2.0 ** -39 * (dtype == "f16")
        assert float((got[r] - want).abs().max()) <= tol


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads, kv, D", [(4, 2, 64), (8, 1, 128), (2, 1, 256)])
def test_values_near_the_types_largest(dtype, heads, kv, D):
    """An output is a mean of values, so it is finite where they are, though a
    sum of them is not; other heads' ordinary values stay as exact as ever."""
    b = Batch(em, heads, kv, D, 16, [(100, 1), (20, 40), (3000, 1), (4000, 12), (0, 1), (64, 70)],
              dtype, seed=93)
    vv = b.view(b.vc)
    big = (1.0 + torch.rand(vv.shape, generator=torch.Generator().manual_seed(94))) * 2.0 ** 126
    vv[..., 0, :] = big[..., 0, :].to(vv.dtype)
    check(b)
    b.q()[:] *= 20.0  # a few positions take all the weight
    b.qkv = b.qkv.cpu()
    for name in ("table", "starts", "lengths", "kc", "vc"):
        setattr(b, name, getattr(b, name).cpu())
    check(b)
