"""Paged batches that the header defines and other tests do not reach: row
starts that leave the call's rows, against the 64-bit definitions of
paged_ref.py with the tolerances of test_gpu_paged.py."""
import pytest

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
