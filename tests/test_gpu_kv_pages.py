"""lmc_kv_pages_fork, _reserve and _compact against tests/kv_ref.py (one sequence at a
time): tables, counts and pools exactly, and the operators together with
appends and decode as a server runs them."""
import numpy as np
import pytest

from lmc_b200 import runtime as rt
from tests import kv_ref
from tests.conftest import rel_err
from tests.test_gpu_kv_q4 import dev, rows_of

pytestmark = pytest.mark.gpu

INVALID = -1


def state(rng, n_seqs, width, n_pages, fill, shared):
    """A random table: row b holds its first entries, some of them other rows' pages."""
    table = np.full((n_seqs, width), -1, np.int32)
    free = list(rng.permutation(n_pages))
    for b in range(n_seqs):
        used = rng.integers(0, int(width * fill) + 1)
        src = rng.integers(0, b) if b and rng.random() < shared else -1
        for j in range(used):
            if src >= 0 and table[src, j] >= 0:
                table[b, j] = table[src, j]
            elif free:
                table[b, j] = free.pop()
    return table, np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)


@pytest.mark.parametrize("n_seqs,width,n_pages", [(1, 1, 1), (2, 1, 3), (5, 128, 300), (33, 67, 900), (300, 40, 5000),
                                                  (5000, 3, 9000)])
def test_fork(cuda, n_seqs, width, n_pages):
    """Random parents (fan-out, cycles, frees, rows left alone), three times in
    a row on the same table."""
    rng = np.random.default_rng(n_seqs)
    table, refs = state(rng, n_seqs, width, n_pages, 0.9, 0.4)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    for _ in range(3):
        parent = np.where(rng.random(n_seqs) < 0.3, np.arange(n_seqs), rng.integers(-1, n_seqs, n_seqs)).astype(np.int32)
        dp = dev(cuda, parent)
        rt.call("lmc_kv_pages_fork", dt.data_ptr(), n_seqs, width, dr.data_ptr(), n_pages, dp.data_ptr(), None)
        kv_ref.fork(table, refs, parent)
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    assert rt.lib().lmc_device_status() == 0


def test_fork_of_a_parent_that_does_not_exist(cuda):
    rng = np.random.default_rng(1)
    table, refs = state(rng, 4, 8, 40, 0.9, 0.0)
    dt, dr, dp = dev(cuda, table), dev(cuda, refs), dev(cuda, np.array([0, 4, 0, 1 << 30], np.int32))
    rt.call("lmc_kv_pages_fork", dt.data_ptr(), 4, 8, dr.data_ptr(), 40, dp.data_ptr(), None)
    assert rt.lib().lmc_device_status() == INVALID and b"kv pages" in rt.lib().lmc_last_error()
    kv_ref.fork(table, refs, [0, 1, 0, 3])  # those rows stay
    assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    assert rt.lib().lmc_device_status() == 0


class Pool:
    def __init__(self, torch, rng, n_pools, n_pages, page_bytes):
        self.torch, self.page_bytes = torch, page_bytes
        self.host = rng.integers(0, 256, (n_pools, n_pages, page_bytes), dtype=np.uint8)
        self.dev = [dev(torch, p) for p in self.host]
        self.list = rt.pool_list(self.dev)

    def copied(self, pairs):
        old = self.host.copy()
        for s, d in pairs:
            self.host[:, d] = old[:, s]

    def check(self):
        for h, d in zip(self.host, self.dev):
            assert np.array_equal(d.cpu().numpy(), h)


def workspace(torch, n_seqs, n_pages):
    n = rt.lib().lmc_kv_pages_workspace_bytes(n_seqs, n_pages)
    return torch.full((n + 64,), 0xff, dtype=torch.uint8, device="cuda"), n


def reserve(torch, pool, dt, dr, pos, P, n_pages, stream=None):
    n_seqs, width = dt.shape
    ws, n = workspace(torch, n_seqs, n_pages)
    short = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    dp = dev(torch, np.asarray(pos, np.int32))
    rt.call("lmc_kv_pages_reserve", pool.list, len(pool.dev), pool.page_bytes, dt.data_ptr(), n_seqs, width, P, dr.data_ptr(),
            n_pages, dp.data_ptr(), short.data_ptr(), ws.data_ptr(), n, stream)
    assert (ws[n:] == 0xff).all()
    return int(short.cpu())


@pytest.mark.parametrize("n_seqs,width,n_pages,P,pools,page_bytes", [
    (1, 1, 1, 16, 1, 16), (4, 6, 30, 16, 3, 4096 + 16), (40, 9, 400, 32, 2, 80), (130, 17, 2500, 16, 2, 1152),
    (1500, 4, 7000, 16, 1, 16), (7, 12, 60, 64, 300, 48)])
def test_reserve(cuda, n_seqs, width, n_pages, P, pools, page_bytes):
    """Fresh pages, copies on write by several writers of one page, idle rows,
    pools whose pages end inside a copy's stride, more pools than one launch
    takes; several steps on the same table."""
    rng = np.random.default_rng(n_seqs + width)
    table, refs = state(rng, n_seqs, width, n_pages, 0.6, 0.7)
    pool = Pool(cuda, rng, pools, n_pages, page_bytes)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    for step in range(3):
        held = (table >= 0).sum(1)
        pos = np.where(rng.random(n_seqs) < 0.5, held, np.maximum(held - 1, 0)) * P + rng.integers(0, P, n_seqs)
        pos = np.where((rng.random(n_seqs) < 0.1) | (pos >= width * P), -1 - rng.integers(0, 9, n_seqs), pos)
        missing, pairs = kv_ref.reserve(table, refs, pos, P)
        assert reserve(cuda, pool, dt, dr, pos, P, n_pages) == missing
        pool.copied(pairs)
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
        pool.check()
    assert rt.lib().lmc_device_status() == 0


def test_reserve_all_or_nothing(cuda):
    """Five pages wanted, three free: the call says two are missing and changes
    nothing; after one sequence gives its pages back it goes through."""
    rng = np.random.default_rng(2)
    table = np.array([[0, 1, -1], [0, 1, -1], [0, 1, -1], [2, 3, -1], [4, -1, -1], [5, -1, -1]], np.int32)
    n_pages, P = 9, 16
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    pool = Pool(cuda, rng, 2, n_pages, 64)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    pos = [20, 21, 22, 32, 16, 16]  # two copies of page 1, three fresh pages
    assert reserve(cuda, pool, dt, dr, pos, P, n_pages) == 2
    assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    pool.check()
    parent = np.array([0, 1, 2, -1, 4, 5], np.int32)
    rt.call("lmc_kv_pages_fork", dt.data_ptr(), 6, 3, dr.data_ptr(), n_pages, dev(cuda, parent).data_ptr(), None)
    kv_ref.fork(table, refs, parent)
    pos[3] = -1
    missing, pairs = kv_ref.reserve(table, refs, pos, P)
    assert missing == 0 and len(pairs) == 2
    assert reserve(cuda, pool, dt, dr, pos, P, n_pages) == 0
    pool.copied(pairs)
    assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    pool.check()
    assert reserve(cuda, pool, dt, dr, pos, P, n_pages) == 0  # everything writable already: nothing changes
    assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)


def test_reserve_outside_the_table(cuda):
    rng = np.random.default_rng(3)
    table, n_pages = np.array([[0, -1], [9, -1], [1, -1]], np.int32), 6
    refs = np.array([1, 1, 0, 0, 0, 0], np.int32)
    pool = Pool(cuda, rng, 1, n_pages, 32)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    assert reserve(cuda, pool, dt, dr, [32, 3, 16], 16, n_pages) == 0
    assert rt.lib().lmc_device_status() == INVALID and b"kv pages" in rt.lib().lmc_last_error()
    table[2, 1], refs[2] = 2, 1  # the third sequence is served
    assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("n_seqs,width,n_pages,pools,page_bytes,fill", [
    (1, 1, 1, 1, 16, 1.0), (3, 8, 20, 2, 48, 0.5), (6, 16, 96, 24, 1152, 0.5), (50, 30, 1024, 2, 64, 0.6),
    (50, 30, 1025, 1, 64, 0.3), (200, 25, 9000, 1, 16, 0.5), (4, 4, 50, 2, 32, 0.0), (5, 8, 30, 300, 16, 0.7)])
def test_compact(cuda, n_seqs, width, n_pages, pools, page_bytes, fill):
    rng = np.random.default_rng(n_pages)
    table, refs = state(rng, n_seqs, width, n_pages, fill, 0.3)
    pool = Pool(cuda, rng, pools, n_pages, page_bytes)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    ws, n = workspace(cuda, n_seqs, n_pages)
    live = cuda.full((1,), -7, dtype=cuda.int32, device="cuda")
    for _ in range(2):  # the second call has nothing to move
        rt.call("lmc_kv_pages_compact", pool.list, pools, page_bytes, dt.data_ptr(), n_seqs, width, dr.data_ptr(), n_pages,
                live.data_ptr(), ws.data_ptr(), n, None)
        n_live, pairs = kv_ref.compact(table, refs)
        pool.copied(pairs)
        assert int(live.cpu()) == n_live and (ws[n:] == 0xff).all()
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
        pool.check()
    assert rt.lib().lmc_device_status() == 0


def test_compact_entry_without_a_count(cuda):
    """A table that names a free page: that entry stays, the status tells."""
    rng = np.random.default_rng(4)
    table, n_pages = np.array([[7, 1, 5, 99]], np.int32), 9
    refs = np.array([0, 1, 0, 0, 0, 0, 0, 1, 0], np.int32)
    pool = Pool(cuda, rng, 1, n_pages, 32)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    ws, n = workspace(cuda, 1, n_pages)
    live = cuda.zeros(1, dtype=cuda.int32, device="cuda")
    rt.call("lmc_kv_pages_compact", pool.list, 1, 32, dt.data_ptr(), 1, 4, dr.data_ptr(), n_pages, live.data_ptr(),
            ws.data_ptr(), n, None)
    assert rt.lib().lmc_device_status() == INVALID
    assert dt.cpu().numpy().tolist() == [[0, 1, 5, 99]] and int(live.cpu()) == 2
    pool.copied([(7, 0)])
    pool.check()


@pytest.mark.parametrize("kvd", [rt.KV_Q4, rt.KV_F16])
def test_samples_and_beams_share_a_prompt(cuda, kvd):
    """As a server runs them, all in one captured step: append a prompt, fork
    it to every slot, then steps of reserve, decode and a reorder of the
    beams, a compaction in between.  Every sequence's output is attention in
    64 bits over the rows of its own history."""
    rng = np.random.default_rng(21)
    B, Hkv, G, Dh, P, S, n_pages, prompt = 5, 2, 4, 64, 16, 96, 24, 37
    RB = rt.kv_row_bytes(kvd, Dh)
    pools = [cuda.full((n_pages, Hkv, P, RB), 0xff, dtype=cuda.uint8, device="cuda") for _ in range(2)]
    plist = rt.pool_list(pools)
    table = cuda.full((B, S // P), -1, dtype=cuda.int32, device="cuda")
    refs = cuda.zeros(n_pages, dtype=cuda.int32, device="cuda")
    ws, wsb = workspace(cuda, B, n_pages)
    short, live = (cuda.zeros(1, dtype=cuda.int32, device="cuda") for _ in range(2))
    values = (lambda x: kv_ref.q4_rows(x)[1]) if kvd == rt.KV_Q4 else (lambda x: x.astype(np.float16).astype(np.float64))

    def make_writable(pos):
        rt.call("lmc_kv_pages_reserve", plist, 2, Hkv * P * RB, table.data_ptr(), B, S // P, P, refs.data_ptr(), n_pages,
                pos.data_ptr(), short.data_ptr(), ws.data_ptr(), wsb, None)
        assert int(short.cpu()) == 0

    def fork(parent):
        d = dev(cuda, np.array(parent, np.int32))
        rt.call("lmc_kv_pages_fork", table.data_ptr(), B, S // P, refs.data_ptr(), n_pages, d.data_ptr(), None)

    # pages for the prompt in slot 2, its rows, then every slot a copy of slot 2
    for t in range(0, prompt, P):
        make_writable(dev(cuda, np.array([-1, -1, t, -1, -1], np.int32)))
    k, v = rows_of(rng, (prompt, Hkv * Dh)), rows_of(rng, (prompt, Hkv * Dh))
    dk, dv = dev(cuda, k), dev(cuda, v)
    seq, pos = dev(cuda, np.full(prompt, 2, np.int32)), cuda.arange(prompt, dtype=cuda.int32, device="cuda")
    rt.call("lmc_kv_append", dk.data_ptr(), dv.data_ptr(), Hkv * Dh, pools[0].data_ptr(), pools[1].data_ptr(), kvd,
            seq.data_ptr(), pos.data_ptr(), prompt, B, Hkv, Dh, S, table.data_ptr(), P, n_pages, None)
    hist = [[(k[t], v[t]) for t in range(prompt)]] * B
    fork([2] * B)
    assert int(refs.max()) == B and int((refs > 0).sum()) == 3
    awsb = rt.lib().lmc_attention_workspace_bytes(B, Hkv * G, Dh, S)
    aws = cuda.empty(awsb + 4, dtype=cuda.uint8, device="cuda")
    for step in range(30):
        q, kn, vn = rows_of(rng, (B, Hkv * G * Dh)), rows_of(rng, (B, Hkv * Dh)), rows_of(rng, (B, Hkv * Dh))
        d = [dev(cuda, a) for a in (q, kn, vn)]
        out = cuda.zeros((B, Hkv * G * Dh), device="cuda")
        pos = cuda.full((B,), prompt + step, dtype=cuda.int32, device="cuda")
        make_writable(pos)
        rt.call("lmc_attention_decode_paged", out.data_ptr(), *(t.data_ptr() for t in d), pools[0].data_ptr(),
                pools[1].data_ptr(), kvd, n_pages, table.data_ptr(), S // P, P, pos.data_ptr(), B, Hkv * G, Hkv, Dh,
                aws.data_ptr(), awsb, None)
        hist = [h + [(kn[b], vn[b])] for b, h in enumerate(hist)]
        for b in range(B):
            kk, vv = (values(np.stack([r[i] for r in hist[b]]).reshape(-1, Hkv, Dh)).transpose(1, 0, 2) for i in range(2))
            want, _ = kv_ref.attention(q[b].reshape(-1, Dh), kk, vv)
            assert rel_err(out[b].cpu().numpy().reshape(want.shape), want) < 1e-5, (step, b)
        if step % 3 == 1:
            parent = rng.integers(0, B, B)
            fork(parent)
            hist = [hist[p] for p in parent]
        if step % 7 == 3:
            rt.call("lmc_kv_pages_compact", plist, 2, Hkv * P * RB, table.data_ptr(), B, S // P, refs.data_ptr(), n_pages,
                    live.data_ptr(), ws.data_ptr(), wsb, None)
            r = refs.cpu().numpy()
            assert (r[:int(live.cpu())] > 0).all() and (r[int(live.cpu()):] == 0).all()
        t = table.cpu().numpy()
        assert np.array_equal(np.bincount(t[t >= 0], minlength=n_pages), refs.cpu().numpy())
    fork([-1] * B)
    assert int(refs.abs().sum()) == 0 and int(table.max()) == -1
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("n_seqs,width,n_pages,pinned", [(700, 80, 40000, 0), (60, 40, 50021, 33000), (60, 40, 16384, 16000),
                                                         (3, 5, 16385, 16384), (900, 60, 32769, 400)])
def test_pools_of_many_pages(cuda, n_seqs, width, n_pages, pinned):
    """Pools that the plans go through in several rounds; the first `pinned`
    pages have a count of their own that no table names."""
    rng = np.random.default_rng(n_pages + pinned)
    table, refs = state(rng, n_seqs, width, n_pages, 0.9, 0.4)
    if pinned:  # the tables' pages lie anywhere behind them
        free = pinned + rng.permutation(n_pages - pinned)
        names = np.unique(table[table >= 0])
        names = names[:len(free)]
        to = np.full(n_pages, -1, np.int32)
        to[names] = free[:len(names)]
        table = np.where(table >= 0, to[table], -1).astype(np.int32)
        refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
        refs[:pinned] = 1
    pool = Pool(cuda, rng, 1, n_pages, 16)
    dt, dr = dev(cuda, table), dev(cuda, refs)
    held = (table >= 0).sum(1)
    for step in range(2):
        pos = np.minimum(held + step, width - 1) * 16 + step
        missing, pairs = kv_ref.reserve(table, refs, pos, 16)
        assert reserve(cuda, pool, dt, dr, pos, 16, n_pages) == missing
        pool.copied(pairs)
        assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    pool.check()
    ws, n = workspace(cuda, n_seqs, n_pages)
    live = cuda.full((1,), -7, dtype=cuda.int32, device="cuda")
    rt.call("lmc_kv_pages_compact", pool.list, 1, 16, dt.data_ptr(), n_seqs, width, dr.data_ptr(), n_pages, live.data_ptr(),
            ws.data_ptr(), n, None)
    n_live, pairs = kv_ref.compact(table, refs)
    pool.copied(pairs)
    assert int(live.cpu()) == n_live and (ws[n:] == 0xff).all()
    assert np.array_equal(dt.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), refs)
    pool.check()
    assert rt.lib().lmc_device_status() == 0
