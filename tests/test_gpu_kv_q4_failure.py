"""What the 4-bit attention reports and leaves behind when something went wrong
in a kernel."""
import numpy as np
import pytest

from lmc_b200 import runtime as rt
from tests.test_gpu_kv_q4 import Cache, INVALID, TIMEOUT, attend, dev, rows_of

pytestmark = pytest.mark.gpu


def test_both_errors_are_reported(cuda):
    """A page outside the pool and a wait that ran out, before the status is
    asked for: it tells one, then the other, then nothing."""
    rng = np.random.default_rng(2)
    c = Cache(cuda, rng, [40], 1, 64, 64, 16)
    c.dt[0, 1] = c.n_pages  # page 0 is read instead
    out = cuda.zeros((1, 64), device="cuda")
    c.decode(cuda, out, *(dev(cuda, rows_of(rng, (1, 64))) for _ in range(3)), dev(cuda, np.array([40], np.int32)), 1)
    rt.call("lmc_set_wait_limit", 2_000_000)  # 2 ms
    try:
        assert rt.lib().lmc_wait_selftest(2) == TIMEOUT
    finally:
        rt.call("lmc_set_wait_limit", 0)
    assert rt.lib().lmc_device_status() == INVALID and b"page id" in rt.lib().lmc_last_error()
    assert rt.lib().lmc_device_status() == 0


def test_lost_tiles_make_their_outputs_nan(cuda):
    """Calls where one tile of a kv head never arrives: the self-test reports
    the timeout only if that head is NaN in every sequence that has the tile
    and nothing else is wrong (parts of a warp, a CTA and several CTAs, with
    an earlier call's numbers in the workspace); the next call is right."""
    rt.call("lmc_set_wait_limit", 2_000_000)  # 2 ms
    try:
        assert rt.lib().lmc_wait_selftest(3) == TIMEOUT, rt.lib().lmc_last_error()
        assert rt.lib().lmc_device_status() == 0
    finally:
        rt.call("lmc_set_wait_limit", 0)
    attend(cuda, 61, [100, 20], 2, 4, 64, 128, 16)
