"""lmc_kv_pages_fork at the ends of what its header accepts."""
import numpy as np
import pytest

from lmc_b200 import runtime as rt
from tests.test_gpu_kv_q4 import dev

pytestmark = pytest.mark.gpu

INVALID = -1


def forked(table, parent):
    """The table after a call with parents from -1 on, and its counts."""
    t = np.where(parent[:, None] < 0, -1, table[np.maximum(parent, 0)])
    return t, lambda n: np.bincount(t[t >= 0], minlength=n).astype(np.int32)


@pytest.mark.parametrize("n_seqs", [8192, 8193, 10923, 12800, 12801, 16383, 16384])
@pytest.mark.parametrize("width", [1, 3])
def test_fork_of_many_sequences(cuda, n_seqs, width):
    """Up to 16384 sequences: the stripes get narrower as the rows get more,
    and their parents and changes of count need room beside them."""
    rng = np.random.default_rng(n_seqs + width)
    n_pages = n_seqs * width // 2
    table = rng.integers(-1, n_pages, (n_seqs, width)).astype(np.int32)
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    parent = np.where(rng.random(n_seqs) < 0.3, np.arange(n_seqs), rng.integers(-1, n_seqs, n_seqs)).astype(np.int32)
    want, counts = forked(table, parent)
    dt, dr, dp = dev(cuda, table), dev(cuda, refs), dev(cuda, parent)
    rt.call("lmc_kv_pages_fork", dt.data_ptr(), n_seqs, width, dr.data_ptr(), n_pages, dp.data_ptr(), None)
    assert np.array_equal(dt.cpu().numpy(), want) and np.array_equal(dr.cpu().numpy(), counts(n_pages))
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("bad", [-2, -1000000, -2**31])
def test_fork_of_a_parent_below_minus_one(cuda, bad):
    """Only -1 gives a row's pages back: a row with any other negative parent
    stays as it is, in table and counts, and the status tells once.  The other
    rows are served, one of them from the row that stays."""
    table = np.array([[0, 1, -1], [2, 3, 4], [5, -1, -1], [2, 6, 7]], np.int32)
    refs = np.bincount(table[table >= 0], minlength=9).astype(np.int32)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    dp = dev(cuda, np.array([1, bad, -1, 3], np.int32))
    rt.call("lmc_kv_pages_fork", dt.data_ptr(), 4, 3, dr.data_ptr(), 9, dp.data_ptr(), None)
    assert rt.lib().lmc_device_status() == INVALID and b"kv pages" in rt.lib().lmc_last_error()
    assert rt.lib().lmc_device_status() == 0
    want, counts = forked(table, np.array([1, 1, -1, 3]))
    assert np.array_equal(dt.cpu().numpy(), want) and np.array_equal(dr.cpu().numpy(), counts(9))
