"""4-bit K/V rows (LMC_KV_Q4) and the page operators on the device against
tests/kv_ref.py: rows bit for bit, attention in 64 bits, page tables, counts
and pools exactly.

Attention's tolerance.  Scores: every product q_i * value is formed from
operands of at least 22 bits, summed in fp32 over at most 16 partial sums per
chain, so |ds| <= (2^-22 + 18 * 2^-24) * sum |q_i k_i| / sqrt(Dh) < 2^-19.5 *
size, size being the largest such sum; the exponential's argument then is off
by ds, its value by ds + 2^-21 relative (fp32 exp).  Sums over positions run in
chains of at most n / 4 fp32 additions.  The output is a weighted mean of
values |v| <= vmax, so elementwise |do| <= (2 |ds| + 2^-20 + (n / 4 + 16) *
2^-24) * vmax.  Norm-wise the repository's attention bound 1e-5 holds on top."""
import numpy as np
import pytest

from lmc_b200 import runtime as rt
from tests import kv_ref
from tests.conftest import rel_err

pytestmark = pytest.mark.gpu

INVALID, TIMEOUT = -1, -6
GUARD = 64  # bytes behind every cache that must stay as they were


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rows_of(rng, shape, kind="normal"):
    x = rng.normal(0, 1, shape)
    if kind == "outliers":
        x[..., ::17] *= 12
    return x.astype(np.float32)


def tolerance(size, n, vmax):
    return (2 * 2.0 ** -19.5 * size + 2.0 ** -20 + (n / 4 + 16) * 2.0 ** -24) * vmax


# ---- rows ------------------------------------------------------------------------------------
def stored(x, kvd):
    """fp32 rows -> (cache bytes, values) of a row form."""
    if kvd == rt.KV_Q4:
        return kv_ref.q4_rows(x)
    if kvd == rt.KV_Q8:
        m = np.abs(x).max(-1, keepdims=True)
        inv = np.divide(np.float32(127), m, out=np.zeros_like(m), where=m > 0)
        c = np.clip(np.rint(x * inv), -127, 127).astype(np.int8)
        sc = (m / np.float32(127)).astype(np.float32)
        tail = np.zeros(x.shape[:-1] + (16,), np.uint8)
        tail[..., :4] = np.ascontiguousarray(sc).view(np.uint8)
        return np.concatenate([c.view(np.uint8), tail], -1), c.astype(np.float32) * sc
    t = x.astype(np.float16 if kvd == rt.KV_F16 else np.float32)
    return np.ascontiguousarray(t).view(np.uint8), t.astype(np.float64)


def special_rows(Dh):
    """Rows where a quantizer goes wrong: zeros, constants, one value apart,
    the ends of fp32 and fp16, quotients that are exactly half a step, values
    that are not finite."""
    r = [np.zeros(Dh), np.full(Dh, -3.7), np.full(Dh, 1e-30), np.full(Dh, 3e38), np.full(Dh, -7e4), np.arange(Dh) % 2 * 1e-7,
         np.arange(Dh) - 5.0, np.arange(Dh) * 1e-40, np.linspace(-65504, 65504, Dh), np.linspace(-3e38, 3e38, Dh),
         np.linspace(1000, 1000.5, Dh), np.where(np.arange(Dh) == 3, 15.0, (np.arange(Dh) % 16) * 0.5),
         np.where(np.arange(Dh) % 64 == 1, 15.0, np.where(np.arange(Dh) % 64 == 2, 0.0, np.arange(Dh) % 15 + 0.5)),
         np.where(np.arange(Dh) % 64 == 1, 30.0, np.where(np.arange(Dh) % 64 == 2, 0.0, 2 * (np.arange(Dh) % 15) + 1 + 1e-6))]
    for bad in (np.inf, -np.inf, np.nan):
        x = np.linspace(-1, 1, Dh)
        x[Dh - 2] = bad
        r.append(x)
    return np.stack(r).astype(np.float32)


@pytest.mark.parametrize("Dh", [32, 64, 96, 128, 160, 192, 224, 256])
def test_special_rows_bit_for_bit(cuda, Dh):
    """Each special row through append and read: the bytes and the values of
    the format's definition, bytes behind the cache untouched."""
    x = special_rows(Dh)
    n = len(x)
    want, vals = kv_ref.q4_rows(x)
    RB = want.shape[-1]
    buf = cuda.full((2, n * RB + GUARD), 0xA5, dtype=cuda.uint8, device="cuda")
    base = [buf[i].clone() for i in range(2)]
    k, v = dev(cuda, x), dev(cuda, x[::-1])
    pos = cuda.arange(n, dtype=cuda.int32, device="cuda")
    seq = cuda.zeros(n, dtype=cuda.int32, device="cuda")
    rt.call("lmc_kv_append", k.data_ptr(), v.data_ptr(), Dh, base[0].data_ptr(), base[1].data_ptr(), rt.KV_Q4,
            seq.data_ptr(), pos.data_ptr(), n, 1, 1, Dh, n, None, 0, 0, None)
    for b, w in zip(base, (want, want[::-1])):
        got = b.cpu().numpy()
        assert (got[n * RB:] == 0xA5).all()
        got = got[:n * RB].reshape(n, RB)
        bad = np.flatnonzero((got[:, :Dh // 2] != w[:, :Dh // 2]).any(-1))
        assert not len(bad), (bad, got[bad[:1]], w[bad[:1]])
        a, e = (t[:, Dh // 2:].copy().view(np.float16) for t in (got, w))
        assert ((a == e) | (np.isnan(a) & np.isnan(e))).all()
    out = cuda.full((n, Dh), 9.0, device="cuda")
    rt.call("lmc_kv_read", out.data_ptr(), None, Dh, base[0].data_ptr(), None, rt.KV_Q4, seq.data_ptr(), pos.data_ptr(), n, 1,
            1, Dh, n, None, 0, 0, None)
    got = out.cpu().numpy().astype(np.float64)
    # d * code is exact in fp32; adding m rounds once: half a step, 2^-24
    assert (np.isnan(got) == np.isnan(vals)).all()
    ok = ~np.isnan(vals)
    assert (np.abs(got - vals)[ok] <= 2.0 ** -24 * np.abs(vals)[ok]).all()
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("kvd", [rt.KV_F32, rt.KV_F16, rt.KV_Q8, rt.KV_Q4])
@pytest.mark.parametrize("rows,Hkv,Dh,S,P,extra,shift", [
    (1, 1, 32, 1, 0, 0, 0), (37, 3, 64, 53, 0, 4, 0), (100, 2, 128, 64, 16, 0, 0), (65, 5, 96, 96, 32, 3, 1),
    (33, 1, 256, 128, 64, 0, 2), (29, 12, 160, 31, 0, 7, 3)])
def test_append_and_read(cuda, kvd, rows, Hkv, Dh, S, P, extra, shift):
    """Rows of three sequences in a shuffled order: row strides wider than a
    row, fp32 rows off the 16-byte boundary, padding rows, one side left out;
    rows that no call names keep their bytes."""
    rng = np.random.default_rng(rows + Dh)
    n_seqs = 3
    rows = min(rows, n_seqs * S)
    where = rng.permutation(n_seqs * S)[:rows]
    seq, pos = (where // S).astype(np.int32), (where % S).astype(np.int32)
    skip = rng.random(rows) < 0.2
    ld = Hkv * Dh + extra
    x = [rows_of(rng, (rows, ld), "outliers") for _ in range(2)]
    flat = []  # at an offset of `shift` floats
    for a in x:
        t = cuda.zeros(rows * ld + 8, device="cuda")
        t[shift:shift + rows * ld] = dev(cuda, a).flatten()
        flat.append(t)
    RB = rt.kv_row_bytes(kvd, Dh)
    if P:
        each = S // P
        n_pages = n_seqs * each + 2
        table = rng.permutation(n_pages)[:n_seqs * each].astype(np.int32).reshape(n_seqs, each)
        shape = (n_pages, Hkv, P, RB)
        dt = dev(cuda, table)
        pages = (dt.data_ptr(), P, n_pages)
    else:
        shape, pages = (n_seqs, Hkv, S, RB), (None, 0, 0)
    ref = [np.full(shape, 0x5A, np.uint8) for _ in range(2)]
    vals = []
    for side in range(2):
        w, val = stored(x[side][:, :Hkv * Dh].reshape(rows, Hkv, Dh), kvd)
        vals.append(val)
        for r in range(rows):
            if not skip[r]:
                at = (table[seq[r], pos[r] // P], slice(None), pos[r] % P) if P else (seq[r], slice(None), pos[r])
                ref[side][at] = w[r]
    dpos, dseq = dev(cuda, np.where(skip, -1 - pos, pos).astype(np.int32)), dev(cuda, seq)
    c = [cuda.full(shape, 0x5A, dtype=cuda.uint8, device="cuda") for _ in range(2)]
    ptr = [t.data_ptr() + 4 * shift for t in flat]
    tail = (kvd, dseq.data_ptr(), dpos.data_ptr(), rows, n_seqs, Hkv, Dh, S, *pages, None)
    rt.call("lmc_kv_append", ptr[0], None, ld, c[0].data_ptr(), None, *tail)
    assert (c[1] == 0x5A).all()
    rt.call("lmc_kv_append", ptr[0], ptr[1], ld, c[0].data_ptr(), c[1].data_ptr(), *tail)
    sized = slice(0, RB if kvd != rt.KV_Q8 else Dh + 4)  # an int8 row's last 12 bytes are not used
    for side in range(2):
        assert np.array_equal(c[side].cpu().numpy()[..., sized], ref[side][..., sized])
    out = [cuda.full((rows * ld + 8,), 7.0, device="cuda") for _ in range(2)]
    rt.call("lmc_kv_read", *(o.data_ptr() + 4 * shift for o in out), ld, c[0].data_ptr(), c[1].data_ptr(), *tail)
    for side in range(2):
        o = out[side].cpu().numpy()
        assert (o[:shift] == 7).all() and (o[shift + rows * ld:] == 7).all()
        o = o[shift:shift + rows * ld].reshape(rows, ld)
        assert (o[:, Hkv * Dh:] == 7).all() and (o[skip] == 7).all()
        want = vals[side].reshape(rows, -1)
        assert (np.abs(o[:, :Hkv * Dh] - want)[~skip] <= 2.0 ** -24 * np.abs(want)[~skip]).all()
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("kvd", [rt.KV_F32, rt.KV_F16, rt.KV_Q8, rt.KV_Q4])
def test_append_and_read_many_rows(cuda, kvd):
    """Enough rows for two a thread, the last ones alone; one in seven is
    padding."""
    rows, Hkv, Dh, S = 5001, 8, 128, 2600
    rng = np.random.default_rng(9)
    x = rows_of(rng, (2, rows, Hkv * Dh), "outliers")
    where = rng.permutation(2 * S)[:rows]
    seq, pos = (where // S).astype(np.int32), (where % S).astype(np.int32)
    skip = np.arange(rows) % 7 == 6
    RB = rt.kv_row_bytes(kvd, Dh)
    c = [cuda.full((2, Hkv, S, RB), 0x5A, dtype=cuda.uint8, device="cuda") for _ in range(2)]
    dx, out = dev(cuda, x), cuda.full((2, rows, Hkv * Dh), 7.0, device="cuda")
    dpos, dseq = dev(cuda, np.where(skip, -1, pos).astype(np.int32)), dev(cuda, seq)
    tail = (Hkv * Dh, c[0].data_ptr(), c[1].data_ptr(), kvd, dseq.data_ptr(), dpos.data_ptr(), rows, 2, Hkv, Dh, S, None, 0, 0,
            None)
    rt.call("lmc_kv_append", dx[0].data_ptr(), dx[1].data_ptr(), *tail)
    rt.call("lmc_kv_read", out[0].data_ptr(), out[1].data_ptr(), *tail)
    for side in range(2):
        w, val = stored(x[side].reshape(rows, Hkv, Dh), kvd)
        ref = np.full(c[side].shape, 0x5A, np.uint8)
        ref[seq[~skip], :, pos[~skip]] = w[~skip]
        sized = slice(0, RB if kvd != rt.KV_Q8 else Dh + 4)
        assert np.array_equal(c[side].cpu().numpy()[..., sized], ref[..., sized])
        o, want = out[side].cpu().numpy(), val.reshape(rows, -1)
        assert (o[skip] == 7).all() and (np.abs(o - want)[~skip] <= 2.0 ** -24 * np.abs(want)[~skip]).all()
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("kvd", [rt.KV_F16, rt.KV_Q4])
def test_rows_outside_the_cache_are_left_out(cuda, kvd):
    """A position at the context's end, a sequence that does not exist, a page
    outside the pool: that row is skipped, the others are stored, and the
    device status tells once."""
    Hkv, Dh, S, P, n_pages = 2, 64, 64, 16, 5
    rng = np.random.default_rng(4)
    x = rows_of(rng, (6, Hkv * Dh))
    seq = np.array([0, 0, 1, 2, -1, 1], np.int32)
    pos = np.array([3, S, 20, 0, 0, 40], np.int32)
    table = np.array([[0, 1, 2, 3], [4, 3, n_pages, -1]], np.int32)  # sequence 1: positions 32.. in page n_pages
    w, _ = stored(x.reshape(6, Hkv, Dh), kvd)
    RB = w.shape[-1]
    ref = np.full((n_pages, Hkv, P, RB), 1, np.uint8)
    ref[0, :, 3], ref[3, :, 4] = w[0], w[2]
    dk, ds, dp, dt = dev(cuda, x), dev(cuda, seq), dev(cuda, pos), dev(cuda, table)
    c = cuda.full(ref.shape, 1, dtype=cuda.uint8, device="cuda")
    tail = (kvd, ds.data_ptr(), dp.data_ptr(), 6, 2, Hkv, Dh, S, dt.data_ptr(), P, n_pages, None)
    rt.call("lmc_kv_append", dk.data_ptr(), None, Hkv * Dh, c.data_ptr(), None, *tail)
    assert rt.lib().lmc_device_status() == INVALID and b"kv rows" in rt.lib().lmc_last_error()
    assert rt.lib().lmc_device_status() == 0
    assert np.array_equal(c.cpu().numpy(), ref)
    out = cuda.full((6, Hkv * Dh), 3.0, device="cuda")
    rt.call("lmc_kv_read", out.data_ptr(), None, Hkv * Dh, c.data_ptr(), None, *tail)
    assert rt.lib().lmc_device_status() == INVALID
    got = out.cpu().numpy()
    assert (got[[1, 3, 4, 5]] == 3).all() and (got[[0, 2]] != 3).any()


# ---- attention -------------------------------------------------------------------------------
class Cache:
    """A 4-bit cache of `len(lens)` sequences with lens[b] rows each, its
    values, and everything behind the rows filled with 0xff (NaN scales)."""

    def __init__(self, torch, rng, lens, Hkv, Dh, S, P, kind="outliers", spare=2):
        B, RB = len(lens), kv_ref.row_bytes(Dh)
        self.Hkv, self.Dh, self.S, self.P, self.n_pages = Hkv, Dh, S, P, 0
        self.k, self.v = [], []  # values per sequence [Hkv][len][Dh]
        if P:
            each = S // P
            self.n_pages = B * each + spare
            self.table = rng.permutation(self.n_pages)[:B * each].astype(np.int32).reshape(B, each)
        raw = [np.full((self.n_pages, Hkv, P, RB) if P else (B, Hkv, S, RB), 0xff, np.uint8) for _ in range(2)]
        for b, n in enumerate(lens):
            for side, to in enumerate((self.k, self.v)):
                r, val = kv_ref.q4_rows(rows_of(rng, (Hkv, n, Dh), kind if side == 0 else "normal"))
                to.append(val)
                if P:
                    for t0 in range(0, n, P):
                        raw[side][self.table[b, t0 // P], :, :min(P, n - t0)] = r[:, t0:t0 + P]
                else:
                    raw[side][b, :, :n] = r
        self.raw = raw
        self.dk, self.dv = dev(torch, raw[0]), dev(torch, raw[1])
        self.dt = dev(torch, self.table) if P else None

    def decode(self, torch, out, q, kn, vn, pos, G, stream=None, ws=None, noalloc=False):
        B, H = q.shape[0], self.Hkv * G
        wsb = rt.lib().lmc_attention_workspace_bytes(B, H, self.Dh, self.S)
        if ws is None:  # exactly the bytes asked for, garbage behind and in them
            ws = torch.full((wsb + GUARD,), 0xff, dtype=torch.uint8, device="cuda")
        first = [t.data_ptr() for t in (out, q, kn, vn, self.dk, self.dv)] + [rt.KV_Q4]
        if noalloc:
            rt.call("lmc_attention_decode_noalloc", *first, pos.data_ptr(), B, H, self.Hkv, self.Dh, self.S, stream)
        elif self.P:
            rt.call("lmc_attention_decode_paged", *first, self.n_pages, self.dt.data_ptr(), self.S // self.P, self.P,
                    pos.data_ptr(), B, H, self.Hkv, self.Dh, ws.data_ptr(), wsb, stream)
        else:
            rt.call("lmc_attention_decode", *first, pos.data_ptr(), B, H, self.Hkv, self.Dh, self.S, ws.data_ptr(), wsb, stream)
        return ws, wsb

    def check(self, got, q, kn, vn, pos, G):
        """`got` and the cache after the call against 64 bits."""
        kn, vn = (a.reshape(len(pos), self.Hkv, self.Dh) for a in (kn, vn))
        ref = [r.copy() for r in self.raw]
        for b, p in enumerate(pos):
            if p < 0 or p >= self.S:
                assert (got[b] == 5).all()  # left as it was
                continue
            (kr, kv), (vr, vv) = kv_ref.q4_rows(kn[b]), kv_ref.q4_rows(vn[b])
            for side, r in enumerate((kr, vr)):
                if self.P:
                    ref[side][self.table[b, p // self.P], :, p % self.P] = r
                else:
                    ref[side][b, :, p] = r
            k = np.concatenate([self.k[b][:, :p], kv[:, None]], 1)
            v = np.concatenate([self.v[b][:, :p], vv[:, None]], 1)
            want, size = kv_ref.attention(q[b].reshape(-1, self.Dh), k, v)
            g = got[b].reshape(want.shape)
            assert rel_err(g, want) < 1e-5, (b, p, rel_err(g, want))
            assert np.abs(g - want).max() <= tolerance(size, p + 1, np.abs(v).max()), (b, p)
        assert np.array_equal(self.dk.cpu().numpy(), ref[0]) and np.array_equal(self.dv.cpu().numpy(), ref[1])


def attend(torch, seed, pos, Hkv, G, Dh, S, P, noalloc=False, kind="outliers", qscale=1.0):
    rng = np.random.default_rng(seed)
    B = len(pos)
    c = Cache(torch, rng, [p if 0 <= p < S else 0 for p in pos], Hkv, Dh, S, P, kind)
    q = rows_of(rng, (B, Hkv * G * Dh)) * np.float32(qscale)
    kn, vn = rows_of(rng, (B, Hkv * Dh)), rows_of(rng, (B, Hkv * Dh))
    out = torch.full((B, Hkv * G * Dh), 5.0, device="cuda")
    d = [dev(torch, a) for a in (q, kn, vn, np.array(pos, np.int32))]
    ws, wsb = c.decode(torch, out, d[0], d[1], d[2], d[3], G, noalloc=noalloc)
    assert (ws[wsb:] == 0xff).all()
    c.check(out.cpu().numpy(), q, kn, vn, pos, G)
    assert rt.lib().lmc_device_status() == 0


@pytest.mark.parametrize("Dh", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("pos,S,P", [([0], 1, 0), ([300, 7], 307, 0), ([95, 31, 0], 128, 16)])
def test_attention_head_sizes(cuda, Dh, pos, S, P):
    """Every head size, 1 to 301 positions; contexts of odd length (rows of
    20, 36, 56 ... bytes then start at any multiple of 4) and pages of 16."""
    attend(cuda, Dh, pos, 2, 4, Dh, S, P)


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 16, 33])
@pytest.mark.parametrize("Dh,P", [(64, 0), (128, 32)])
def test_attention_group_sizes(cuda, G, Dh, P):
    attend(cuda, G, [130, 64], 3 if G < 16 else 1, G, Dh, 160, P)


@pytest.mark.parametrize("Dh", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("G,P", [(6, 0), (5, 32), (12, 16)])
def test_attention_head_sizes_of_large_groups(cuda, Dh, G, P):
    """More than four query heads per kv head take another form of the kernel."""
    attend(cuda, Dh + G, [150, 63, 0], 2, G, Dh, 160, P)


@pytest.mark.parametrize("Hkv,G,Dh,S,P,pos", [(2, 4, 64, 2048, 16, [1500, 3]), (2, 8, 128, 512, 0, [400, 64, -1]),
                                              (1, 3, 96, 160, 32, [100]), (3, 5, 224, 64, 0, [40, 63])])
def test_attention_of_rows_off_the_16_byte_boundary(cuda, Hkv, G, Dh, S, P, pos):
    """q, the new rows and the output at any 4-byte address."""
    rng = np.random.default_rng(S + G)
    B = len(pos)
    c = Cache(cuda, rng, [max(p, 0) for p in pos], Hkv, Dh, S, P)
    host = [rows_of(rng, (B, Hkv * n * Dh)) for n in (G, 1, 1)]
    flat = []
    for i, a in enumerate(host):
        t = cuda.zeros(a.size + 8, device="cuda")
        t[i + 1:i + 1 + a.size] = dev(cuda, a).flatten()
        flat.append(t[i + 1:i + 1 + a.size].view(a.shape))
    o = cuda.full((B * Hkv * G * Dh + 8,), 5.0, device="cuda")
    out = o[3:3 + B * Hkv * G * Dh].view(B, -1)
    c.decode(cuda, out, *flat, dev(cuda, np.array(pos, np.int32)), G)
    c.check(out.cpu().numpy(), *host, pos, G)
    assert (o[:3] == 5).all() and (o[-5:] == 5).all()


@pytest.mark.parametrize("G", [1, 3, 4, 5, 8])
def test_attention_largest_queries(cuda, G):
    """Queries near the end of fp32: one position takes all the weight (its
    lead is far over the scores' rounding), so the output is its values."""
    rng = np.random.default_rng(40 + G)
    Dh, n = 64, 70
    c = Cache(cuda, rng, [n], 1, Dh, 128, 0, "normal")
    q = (rows_of(rng, (1, G * Dh)) * np.float32(3e37)).astype(np.float32)
    kn, vn = rows_of(rng, (1, Dh)), rows_of(rng, (1, Dh))
    out = cuda.full((1, G * Dh), 5.0, device="cuda")
    c.decode(cuda, out, *(dev(cuda, a) for a in (q, kn, vn, np.array([n], np.int32))), G)
    k = np.concatenate([c.k[0], kv_ref.q4_rows(kn.reshape(1, 1, Dh))[1]], 1)
    v = np.concatenate([c.v[0], kv_ref.q4_rows(vn.reshape(1, 1, Dh))[1]], 1)
    s = np.sort(q.reshape(G, Dh).astype(np.float64) @ k[0].T / 8)
    assert np.isfinite(q).all() and (s[:, -1] - s[:, -2] > 64 + 2.0 ** -19 * np.abs(s).max(-1)).all()
    want, _ = kv_ref.attention(q.reshape(G, Dh), k, v)
    assert np.abs(out.cpu().numpy().reshape(G, Dh) - want).max() <= 2.0 ** -20 * np.abs(v).max()


@pytest.mark.parametrize("G", [3, 4, 6, 9])
def test_attention_queries_that_are_not_finite(cuda, G):
    """An infinity or a NaN in a query makes its own head NaN and no other."""
    rng = np.random.default_rng(50 + G)
    Dh, n = 128, 90
    c = Cache(cuda, rng, [n], 2, Dh, 128, 0, "normal")
    q = rows_of(rng, (1, 2 * G * Dh))
    q[0, 1 * Dh + 5], q[0, (G + 2) * Dh + 77] = np.inf, np.nan
    kn, vn = rows_of(rng, (1, 2 * Dh)), rows_of(rng, (1, 2 * Dh))
    out = cuda.full((1, 2 * G * Dh), 5.0, device="cuda")
    c.decode(cuda, out, *(dev(cuda, a) for a in (q, kn, vn, np.array([n], np.int32))), G)
    got = out.cpu().numpy().reshape(2 * G, Dh)
    bad = np.zeros(2 * G, bool)
    bad[[1, G + 2]] = True
    assert np.isnan(got[bad]).all()
    k, v = (np.concatenate([x[0], kv_ref.q4_rows(y.reshape(2, 1, Dh))[1]], 1) for x, y in ((c.k, kn), (c.v, vn)))
    want, _ = kv_ref.attention(np.where(bad[:, None], 0, q.reshape(2 * G, Dh)), k, v)
    assert rel_err(got[~bad], want[~bad]) < 1e-5


@pytest.mark.parametrize("pos", list(range(0, 70)) + [127, 128, 129, 255, 256, 257, 511, 512, 1023])
def test_attention_every_length(cuda, pos):
    """Each length up to two tiles and the borders of longer ones."""
    attend(cuda, pos, [pos], 1, 2, 64, 1024, 0)


@pytest.mark.parametrize("Hkv,G,Dh,S,P,pos", [
    (12, 1, 64, 1024, 0, [700]), (4, 8, 64, 2048, 16, [2047, 0, 511, -1, 1200, 63, 64, 2048, 31]),
    (8, 4, 128, 4096, 64, [4095, 17, 2000]), (1, 8, 128, 8192, 256, [8000]), (8, 4, 128, 5003, 0, [5002, 1])])
def test_attention_of_ragged_batches(cuda, Hkv, G, Dh, S, P, pos):
    """The repository's model shapes, long and ragged, idle rows (position
    -1) and a position past the context, whose output rows stay as they were."""
    attend(cuda, S + Dh, pos, Hkv, G, Dh, S, P)


def test_attention_many_sequences(cuda):
    rng = np.random.default_rng(8)
    attend(cuda, 9, [int(p) for p in rng.integers(-1, 48, 700)], 1, 2, 32, 48, 16)


@pytest.mark.parametrize("kind,qscale", [("normal", 1e-6), ("normal", 30.0), ("outliers", 3000.0), ("normal", 0.0)])
def test_attention_scales_of_q(cuda, kind, qscale):
    """Flat and peaked softmax, queries far outside fp16's range, a zero
    query (the mean of the values)."""
    attend(cuda, 3, [200, 77], 2, 4, 128, 256, 0, kind=kind, qscale=qscale if qscale != 3000.0 else 2.0)
    if qscale == 3000.0:
        # scores in the thousands: one position takes all the weight, so the
        # output is that row's values however the scores round, if its lead is
        # more than 64 (2^-92 of the weight) over their rounding
        rng = np.random.default_rng(5)
        c = Cache(cuda, rng, [100], 1, 64, 128, 0, "normal")
        q = (rows_of(rng, (1, 64)) * np.float32(1e7)).astype(np.float32)
        kn, vn = rows_of(rng, (1, 64)), rows_of(rng, (1, 64))
        out = cuda.full((1, 64), 5.0, device="cuda")
        c.decode(cuda, out, *(dev(cuda, a) for a in (q, kn, vn, np.array([100], np.int32))), 1)
        k = np.concatenate([c.k[0], kv_ref.q4_rows(kn.reshape(1, 1, 64))[1]], 1)
        v = np.concatenate([c.v[0], kv_ref.q4_rows(vn.reshape(1, 1, 64))[1]], 1)
        s = np.sort(k[0] @ q[0].astype(np.float64) / 8)
        assert s[-1] - s[-2] > 64 + 2.0 ** -19 * np.abs(s).max()
        want, _ = kv_ref.attention(q, k, v)
        # one value d * code + m, multiplied by p = 1 and divided by the sum 1
        assert np.abs(out.cpu().numpy() - want).max() <= 2.0 ** -20 * np.abs(v).max()


@pytest.mark.parametrize("scale", [1e-7, 1e-4, 1.0, 1000.0, 60000.0])
def test_attention_scales_of_v(cuda, scale):
    """Values whose steps d are subnormal fp16 numbers, ordinary, near the
    end of fp16: the output keeps its relative accuracy."""
    rng = np.random.default_rng(6)
    Dh, n = 128, 150
    c = Cache(cuda, rng, [n], 2, Dh, 160, 0, "normal")
    c.k, c.v = [], []
    for side, (to, f) in enumerate(((c.k, 1.0), (c.v, scale))):
        # the last rows' values are larger: the running scale has to follow
        x = rng.uniform(-1, 1, (2, n, Dh)) * f * np.where(np.arange(n) < 100, 1e-2, 1.0)[:, None]
        r, val = kv_ref.q4_rows(x.astype(np.float32))
        c.raw[side][0, :, :n] = r
        to.append(val)
    c.dk, c.dv = dev(cuda, c.raw[0]), dev(cuda, c.raw[1])
    q, kn = rows_of(rng, (1, 4 * Dh)), rows_of(rng, (1, 2 * Dh))
    vn = (rng.uniform(-1, 1, (1, 2 * Dh)) * scale).astype(np.float32)
    out = cuda.full((1, 4 * Dh), 5.0, device="cuda")
    c.decode(cuda, out, *(dev(cuda, a) for a in (q, kn, vn, np.array([n], np.int32))), 2)
    c.check(out.cpu().numpy(), q, kn, vn, [n], 2)


def test_attention_values_that_are_not_finite(cuda):
    """A group stored from an infinity reads back as NaN: as a key it makes
    the heads that read it NaN, as a value only its group's dims; past a
    sequence's end, and in other heads, it changes nothing."""
    rng = np.random.default_rng(7)
    Hkv, G, Dh, n = 2, 2, 128, 40
    c = Cache(cuda, rng, [n, n], Hkv, Dh, 64, 0, "normal")
    bad = rows_of(rng, (1, 128))
    bad[0, 70] = np.inf
    r, val = kv_ref.q4_rows(bad)
    c.raw[0][0, 1, 9] = r[0]   # sequence 0, head 1: a key
    c.raw[1][1, 0, 11] = r[0]  # sequence 1, head 0: a value, dims 64..127
    c.raw[0][:, :, n + 1:] = r[0]
    c.raw[1][:, :, n + 1:] = r[0]
    c.k[0][1, 9], c.v[1][0, 11] = val[0], val[0]
    c.dk, c.dv = dev(cuda, c.raw[0]), dev(cuda, c.raw[1])
    q, kn, vn = rows_of(rng, (2, Hkv * G * Dh)), rows_of(rng, (2, Hkv * Dh)), rows_of(rng, (2, Hkv * Dh))
    out = cuda.full((2, Hkv * G * Dh), 5.0, device="cuda")
    c.decode(cuda, out, *(dev(cuda, a) for a in (q, kn, vn, np.array([n, n], np.int32))), G)
    got = out.cpu().numpy().reshape(2, Hkv, G, Dh)
    assert np.isnan(got[0, 1]).all() and np.isfinite(got[0, 0]).all()
    assert np.isnan(got[1, 0, :, 64:]).all() and np.isfinite(got[1, 0, :, :64]).all() and np.isfinite(got[1, 1]).all()
    for b, h in ((0, 0), (1, 1)):
        k = np.concatenate([c.k[b][h], kv_ref.q4_rows(kn[b].reshape(Hkv, Dh)[h])[1][None]])
        v = np.concatenate([c.v[b][h], kv_ref.q4_rows(vn[b].reshape(Hkv, Dh)[h])[1][None]])
        want, _ = kv_ref.attention(q[b].reshape(Hkv, G, Dh)[h], k[None], v[None])
        assert rel_err(got[b, h], want) < 1e-5


@pytest.mark.parametrize("Hkv,G,Dh,S,pos", [(12, 1, 64, 1024, [700, 90]), (8, 4, 128, 4096, [3000])])
def test_attention_noalloc(cuda, Hkv, G, Dh, S, pos):
    for seed in (1, 2):
        attend(cuda, seed, pos, Hkv, G, Dh, S, 0, noalloc=True)


def test_attention_page_outside_the_pool(cuda):
    """Page ids outside the pool are not followed, the new row is not written
    through one, and the device status tells."""
    rng = np.random.default_rng(2)
    c = Cache(cuda, rng, [40, 40], 1, 64, 64, 16)
    c.dt[0, 1], c.dt[1, 2] = c.n_pages, -1
    before = [c.dk.clone(), c.dv.clone()]
    q, kn, vn = (dev(cuda, rows_of(rng, (2, 64))) for _ in range(3))
    out = cuda.zeros((2, 64), device="cuda")
    c.decode(cuda, out, q, kn, vn, dev(cuda, np.array([40, 40], np.int32)), 1)
    assert rt.lib().lmc_device_status() == INVALID and b"page id" in rt.lib().lmc_last_error()
    assert rt.lib().lmc_device_status() == 0
    for now, was in zip((c.dk, c.dv), before):  # only sequence 0's new row changed
        was[c.table[0, 2], :, 8] = now[c.table[0, 2], :, 8]
        assert cuda.equal(now, was)


def test_attention_wait_that_runs_out(cuda):
    """A wait for copies that never come ends within the limit, is reported
    once, and the next call's result is right."""
    rt.call("lmc_set_wait_limit", 2_000_000)  # 2 ms
    try:
        assert rt.lib().lmc_wait_selftest(2) == TIMEOUT and b"4-bit attention" in rt.lib().lmc_last_error()
        assert rt.lib().lmc_device_status() == 0
    finally:
        rt.call("lmc_set_wait_limit", 0)
    attend(cuda, 60, [100, 20], 2, 4, 64, 128, 16)


def test_attention_from_several_threads(cuda):
    """Calls of different group sizes (shared memory of different sizes, one
    kernel) from three threads at once, each on its own stream."""
    import threading
    todo, errors = [], []
    for i, G in enumerate((1, 4, 2)):
        rng = np.random.default_rng(70 + G)
        c = Cache(cuda, rng, [90, 33], 2, 64, 128, 0)
        q, kn, vn = (rows_of(rng, (2, n * 64)) for n in (2 * G, 2, 2))
        out = cuda.full((2, 2 * G * 64), 5.0, device="cuda")
        d = [dev(cuda, a) for a in (q, kn, vn, np.array([90, 33], np.int32))]
        todo.append((c, q, kn, vn, out, d, G, cuda.cuda.Stream()))
    wsb = rt.lib().lmc_attention_workspace_bytes(2, 8, 64, 128)
    spaces = [cuda.full((wsb + GUARD,), 0xff, dtype=cuda.uint8, device="cuda") for _ in todo]
    cuda.cuda.synchronize()

    def run(job, ws):
        c, _, _, _, out, d, G, stream = job
        try:
            for _ in range(300):
                c.decode(cuda, out, d[0], d[1], d[2], d[3], G, stream=stream.cuda_stream, ws=ws)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=a) for a in zip(todo, spaces)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    cuda.cuda.synchronize()
    assert not errors, errors
    for c, q, kn, vn, out, _, G, _ in todo:
        c.check(out.cpu().numpy(), q, kn, vn, [90, 33], G)


def test_attention_captured_and_replayed(cuda):
    """The call in a CUDA graph, replayed while positions move on: each
    replay attends one row more and appends at the new position; a second
    graph with its own workspace on another stream gives the same."""
    rng = np.random.default_rng(3)
    Hkv, G, Dh, S, P, B = 2, 4, 64, 256, 16, 3
    start = [5, 100, 30]
    c = [Cache(cuda, np.random.default_rng(11), start, Hkv, Dh, S, P) for _ in range(2)]
    q, kn, vn = rows_of(rng, (B, Hkv * G * Dh)), rows_of(rng, (B, Hkv * Dh)), rows_of(rng, (B, Hkv * Dh))
    d = [dev(cuda, a) for a in (q, kn, vn)]
    outs, graphs, poss, keep = [], [], [], []
    for i in range(2):
        out, pos = cuda.full((B, Hkv * G * Dh), 5.0, device="cuda"), dev(cuda, np.array(start, np.int32))
        wsb = rt.lib().lmc_attention_workspace_bytes(B, Hkv * G, Dh, S)
        ws = cuda.full((wsb + GUARD,), 0xff, dtype=cuda.uint8, device="cuda")
        s = cuda.cuda.Stream()
        g = cuda.cuda.CUDAGraph()
        cuda.cuda.synchronize()
        with cuda.cuda.stream(s):
            g.capture_begin()
            c[i].decode(cuda, out, *d, pos, G, stream=s.cuda_stream, ws=ws)
            pos += 1
            g.capture_end()
        outs.append(out), graphs.append((g, s)), poss.append(pos), keep.append(ws)
    for step in range(3):
        for g, s in graphs:
            with cuda.cuda.stream(s):
                g.replay()
        cuda.cuda.synchronize()
        pos = [p + step for p in start]
        assert cuda.equal(outs[0], outs[1])
        c[0].check(outs[0].cpu().numpy(), q, kn, vn, pos, G)
        for b, p in enumerate(pos):  # the appended row is now one of the cached ones
            for side, x in enumerate((kn, vn)):
                r, val = kv_ref.q4_rows(x[b].reshape(Hkv, Dh))
                to = (c[0].k, c[0].v)[side]
                to[b] = np.concatenate([to[b], val[:, None]], 1)
                c[0].raw[side][c[0].table[b, p // P], :, p % P] = r
    assert rt.lib().lmc_device_status() == 0


def test_attention_same_result_each_time(cuda):
    """The same call twice gives the same bits (no order of arrival in it)."""
    rng = np.random.default_rng(12)
    c = Cache(cuda, rng, [3000, 1500, 40], 4, 128, 4096, 64)
    d = [dev(cuda, rows_of(rng, s)) for s in ((3, 4 * 4 * 128), (3, 512), (3, 512))]
    pos = dev(cuda, np.array([3000, 1500, 40], np.int32))
    outs = []
    for _ in range(5):
        out = cuda.zeros((3, 4 * 4 * 128), device="cuda")
        c.decode(cuda, out, *d, pos, 4)
        outs.append(out)
    assert all(cuda.equal(o, outs[0]) for o in outs)


def test_attention_one_page_past_2_gib(cuda):
    """One page of 2^24 positions, whose rows end past 2^31 bytes.  All rows
    are zeros (score 0, value 0) but three: one at each end and the new one,
    their scores around 17 (e^17 is the number of the others), so the output
    is sum p v over the three, p = e^s / (sum of the three + 2^24 - 3).

    Tolerance: at most 64 workspace slots share an item, so 63 CTAs of four
    warps have its 2^19 tiles of 32 rows, 2081 a warp.  Each tile's sum of p is
    added to the warp's with a rounding of at most half a step, 2^-24 of the
    sum, 2081 * 2^-24 = 1.3e-4 in all (nothing is lost of sum p v, whose other
    terms are zeros); the rest is below 1e-5 as everywhere."""
    Dh, P = 256, 1 << 24
    RB = kv_ref.row_bytes(Dh)
    rng = np.random.default_rng(14)
    q = rng.normal(size=(1, Dh)).astype(np.float32)
    kx = (q * (17.0 * 16 / (q * q).sum()) + 0.05 * rng.normal(size=(3, Dh))).astype(np.float32)
    vx = rows_of(rng, (3, Dh))
    (kr, k), (vr, v) = kv_ref.q4_rows(kx), kv_ref.q4_rows(vx)
    pools = [cuda.zeros((1, 1, P, RB), dtype=cuda.uint8, device="cuda") for _ in range(2)]
    at = [3, P - 7, P - 1]
    for pool, r in zip(pools, (kr, vr)):
        for i in range(2):
            pool[0, 0, at[i]] = dev(cuda, r[i])
    out = cuda.full((1, Dh), 5.0, device="cuda")
    wsb = rt.lib().lmc_attention_workspace_bytes(1, 1, Dh, P)
    ws = cuda.full((wsb + GUARD,), 0xff, dtype=cuda.uint8, device="cuda")
    dq, dk, dv = dev(cuda, q), dev(cuda, kx[2:]), dev(cuda, vx[2:])
    pos, tab, seq = (dev(cuda, np.array([i], np.int32)) for i in (P - 1, 0, 0))
    rt.call("lmc_attention_decode_paged", out.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), pools[0].data_ptr(),
            pools[1].data_ptr(), rt.KV_Q4, 1, tab.data_ptr(), 1, P, pos.data_ptr(), 1, 1, 1, Dh, ws.data_ptr(), wsb, None)
    for pool, r in zip(pools, (kr, vr)):
        assert np.array_equal(pool[0, 0, P - 1].cpu().numpy(), r[2]) and not pool[0, 0, P - 6:P - 1].any()
        assert not pool[0, 0, 4:1000].any()
    s = k @ q[0].astype(np.float64) / 16
    p = np.exp(s)
    want = p @ v / (p.sum() + P - 3)
    assert 10 < s.min() and s.max() < 25 and rel_err(out.cpu().numpy()[0], want) < 2081 * 2.0 ** -24 + 1e-5
    vals = cuda.zeros((1, Dh), device="cuda")
    rt.call("lmc_kv_read", vals.data_ptr(), None, Dh, pools[0].data_ptr(), None, rt.KV_Q4, seq.data_ptr(), pos.data_ptr(), 1, 1, 1,
            Dh, P, tab.data_ptr(), P, 1, None)
    assert rel_err(vals.cpu().numpy(), k[2:]) < 1e-7
    assert (ws[wsb:] == 0xff).all() and rt.lib().lmc_device_status() == 0


def test_attention_offsets_past_32_bits(cuda):
    """A pool of more than 4 GiB: pages near its end hold the sequence."""
    Hkv, Dh, P = 8, 256, 64
    page = Hkv * P * kv_ref.row_bytes(Dh)
    n_pages = (1 << 32) // page + 70
    rng = np.random.default_rng(13)
    small = Cache(cuda, rng, [100], Hkv, Dh, 128, P, "normal", spare=0)
    big = [cuda.zeros((n_pages, Hkv, P, kv_ref.row_bytes(Dh)), dtype=cuda.uint8, device="cuda") for _ in range(2)]
    at = [n_pages - 1, n_pages - 33]
    for j, p in enumerate(at):
        for pool, src in zip(big, (small.dk, small.dv)):
            pool[p] = src[int(small.table[0, j])]
    q, kn, vn = rows_of(rng, (1, Hkv * Dh)), rows_of(rng, (1, Hkv * Dh)), rows_of(rng, (1, Hkv * Dh))
    out = cuda.full((1, Hkv * Dh), 5.0, device="cuda")
    full = small.dk, small.dv, small.dt, small.n_pages
    small.dk, small.dv, small.dt, small.n_pages = big[0], big[1], dev(cuda, np.array([at], np.int32)), n_pages
    small.decode(cuda, out, *(dev(cuda, a) for a in (q, kn, vn, np.array([100], np.int32))), 1)
    for j, p in enumerate(at):  # back into the small pools, to be compared whole
        for pool, dst in zip(big, full[:2]):
            dst[int(small.table[0, j])] = pool[p]
    small.dk, small.dv, small.dt, small.n_pages = full
    small.check(out.cpu().numpy(), q, kn, vn, [100], 1)
    vals = cuda.zeros((1, Hkv * Dh), device="cuda")
    one, zero = dev(cuda, np.array([100], np.int32)), dev(cuda, np.array([0], np.int32))
    tab = dev(cuda, np.array([at], np.int32))
    rt.call("lmc_kv_read", vals.data_ptr(), None, Hkv * Dh, big[0].data_ptr(), None, rt.KV_Q4, zero.data_ptr(), one.data_ptr(),
            1, 1, Hkv, Dh, 128, tab.data_ptr(), P, n_pages, None)
    assert rel_err(vals.cpu().numpy().reshape(Hkv, Dh), kv_ref.q4_rows(kn.reshape(Hkv, Dh))[1]) < 1e-7
    assert rt.lib().lmc_device_status() == 0
