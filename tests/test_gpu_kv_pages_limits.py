"""lmc_kv_pages_fork at the ends of what its header accepts."""
import numpy as np
import pytest

from lmc_b200 import runtime as rt
from tests.test_gpu_kv_q4 import dev

pytestmark = pytest.mark.gpu


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
