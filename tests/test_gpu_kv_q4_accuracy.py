"""Decode attention over 4-bit rows where its number formats could lose bits:
against 64 bits on the values that the rows stand for.

Every output is sum p v / sum p.  With ds the bound on a score's error, a
weight p is off by at most 2 ds + 2^-20 relative to it (ds of its own and of
the maximum, fp32 exponential, p d in 22 bits), and the sums over n positions
by (n / 4 + 16) 2^-24 (chains of at most n / 4 fp32 additions).  A value is
taken as (m + 7.5 d) + d (2 c - 15) / 2, two terms of at most the row's largest
|value| in its group, so per group |do| <= rel * 2 * sum p vmax / sum p with
rel = 2 ds + 2^-20 + (n / 4 + 16) 2^-24 and vmax the row's largest |value| there."""
import numpy as np
import pytest

from lmc_b200 import runtime as rt
from tests import kv_ref
from tests.conftest import rel_err
from tests.test_gpu_kv_q4 import Cache, dev, rows_of

pytestmark = pytest.mark.gpu


def decode(torch, q, k, v):
    """q [H][Dh], k and v [Hkv][n][Dh] fp32, the last row the new one ->
    (out, values of the stored k, of the stored v)."""
    (H, Dh), (Hkv, n, _) = q.shape, k.shape
    c = Cache(torch, np.random.default_rng(0), [0], Hkv, Dh, n, 0)
    for side, (x, vals) in enumerate(((k, c.k), (v, c.v))):
        r, val = kv_ref.q4_rows(x)
        c.raw[side][0, :, :n - 1] = r[:, :n - 1]
        vals[0] = val
    c.dk, c.dv = dev(torch, c.raw[0]), dev(torch, c.raw[1])
    out = torch.full((1, H * Dh), 5.0, device="cuda")
    new = [np.ascontiguousarray(x[:, -1].reshape(1, -1)) for x in (k, v)]
    c.decode(torch, out, *(dev(torch, a) for a in (q.reshape(1, -1), *new, np.array([n - 1], np.int32))), H // Hkv)
    assert rt.lib().lmc_device_status() == 0
    return out.cpu().numpy().reshape(H, Dh), c.k[0], c.v[0]


def check(out, q, k, v, ds, norm=True, least=0.0):
    """Per group of 64 dims against the bound above; ds [H] or a number, `least`
    what a weight may be off by at least."""
    (H, Dh), G = q.shape, q.shape[0] // k.shape[0]
    n = k.shape[1]
    for h in range(H):
        kk, vv = k[h // G], v[h // G]
        s = kk @ q[h].astype(np.float64) / np.sqrt(Dh)
        p = np.exp(s - s.max())
        p /= p.sum()
        rel = 2 * np.broadcast_to(ds, H)[h] + 2.0 ** -20 + (n / 4 + 16) * 2.0 ** -24
        for g in range(0, Dh, 64):
            x, want = vv[:, g:g + 64], p @ vv[:, g:g + 64]
            worst = np.abs(out[h, g:g + 64] - want).max()
            assert worst <= rel * 2 * (p @ np.abs(x).max(-1)) + least * np.abs(x).max(-1).sum(), (h, g, worst / (p @ np.abs(x).max(-1)), rel)
            if norm:  # the repository's attention bound
                assert rel_err(out[h, g:g + 64], want) < 1e-5, (h, g, rel_err(out[h, g:g + 64], want))


def keys_with_zero(rng, Hkv, n, Dh, step):
    """Keys whose groups run from -8 to 7 steps (powers of two), so that m =
    -8 d exactly, code 8 is exactly 0, and small numbers are stored as 0."""
    step = np.broadcast_to(step, (Hkv, n, Dh)).astype(np.float32)
    k = (rng.normal(0, 2.5, (Hkv, n, Dh)) * step).astype(np.float32)
    k = np.clip(k, -8 * step, 7 * step)
    k[..., 0::64], k[..., 1::64] = -8 * step[..., 0::64], 7 * step[..., 1::64]
    return k


@pytest.mark.parametrize("G", [1, 4, 5, 8, 9])
@pytest.mark.parametrize("Dh", [64, 96, 128, 256])
def test_scores_of_zero_keys_are_zero(cuda, G, Dh):
    """Keys that are exactly 0 wherever q is not: every score is 0 (ds = 0),
    the output the mean of the values, however large q and its sum are.  The
    rows' steps d are 1 and 64."""
    rng = np.random.default_rng(G + Dh)
    n = 90
    k = np.zeros((1, n, Dh), np.float32)
    step = np.where(np.arange(n) % 2, 64, 1)
    k[..., 0::64], k[..., 1::64] = -8 * step[:, None], 7 * step[:, None]
    q = rng.uniform(512, 1024, (G, Dh)).astype(np.float32)
    q[:, 0::64] = q[:, 1::64] = 0
    v = rows_of(rng, (1, n, Dh))
    out, kv, vv = decode(cuda, q, k, v)
    assert not (kv[:, :, None] * q).any()
    check(out, q, kv, vv, 0.0)


@pytest.mark.parametrize("G", [1, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("where,r", [("groups", 1000), ("groups", 30000), ("within", 30), ("within", 100), ("within", 1000)])
def test_queries_of_unequal_channels(cuda, G, where, r):
    """Channels of q that are r times larger, where the keys are r times
    smaller (one group of 64 dims) or 0 (every 16th dim).

    q is held to a whole number of at least 2^29 for the largest |q| of a
    group, so a channel is off by at most 2^-30 of that; m + 8 d is 0 here, and
    what is left of a score are at most 8 fp32 roundings (the whole numbers'
    sum, times d, the groups added up, the scale, the difference to the
    maximum), each of at most 2^-24 of sum |q k|."""
    rng = np.random.default_rng(G + r)
    Dh, n, Hkv = 128, 200, 2
    big = np.arange(Dh) >= 64 if where == "groups" else np.arange(Dh) % 16 == 5
    step = 0.25 * np.where(big, 1 / 2.0 ** np.round(np.log2(r)), 1) if where == "groups" else 0.25
    k = keys_with_zero(rng, Hkv, n, Dh, step)
    if where == "within":
        k[..., big] = 0
    q = rows_of(rng, (Hkv * G, Dh)) * np.where(big, r, 1).astype(np.float32)
    v = rows_of(rng, (Hkv, n, Dh))
    out, kv, vv = decode(cuda, q, k, v)
    kk, a = np.repeat(np.abs(kv), G, 0), np.abs(q.astype(np.float64))
    held = sum(2.0 ** -30 * a[:, g:g + 64].max(-1) * kk[:, :, g:g + 64].sum(-1).max(-1) for g in (0, 64))
    size = np.einsum("hnd,hd->hn", kk, a).max(-1)
    check(out, q, kv, vv, (held + 8 * 2.0 ** -24 * size) / np.sqrt(Dh))


def scores_bound(q, k):
    """ds of ordinary queries: products of at least 22 bits and 18 fp32
    roundings of at most 2^-24 of sum |q k|, as in the other attention tests."""
    G = q.shape[0] // k.shape[0]
    size = np.einsum("hnd,hd->hn", np.abs(np.repeat(k, G, 0)), np.abs(q.astype(np.float64))).max(-1)
    return (2.0 ** -22 + 18 * 2.0 ** -24) * size / np.sqrt(q.shape[1])


@pytest.mark.parametrize("G", [1, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("Dh,large,small", [(128, 3e3, 3e-3), (128, 3e3, 3e-4), (128, 9e4, 3e-4), (96, 9e4, 3e-4), (256, 9e4, 3e-4)])
def test_value_groups_of_unequal_size(cuda, G, Dh, large, small):
    """Groups of a head's values that are far larger than the next: each
    keeps its own accuracy."""
    rng = np.random.default_rng(G + Dh)
    n, Hkv = 150, 2
    q, k = rows_of(rng, (Hkv * G, Dh)), rows_of(rng, (Hkv, n, Dh))
    for order in ((large, small), (small, large)):
        v = rng.uniform(-0.5, 0.5, (Hkv, n, Dh)) * np.where(np.arange(Dh) // 64 % 2, order[1], order[0])
        out, kv, vv = decode(cuda, q, k, v.astype(np.float32))
        check(out, q, kv, vv, scores_bound(q, kv))


@pytest.mark.parametrize("G", [1, 4, 5, 8])
@pytest.mark.parametrize("at", [3, 100])
def test_large_value_of_a_row_without_weight(cuda, G, at):
    """A row whose values are 1e7 times the others' and whose weight is below
    e^-45 for one head of each group, 1 for the next: the heads that do not
    see it keep their accuracy."""
    rng = np.random.default_rng(G)
    n, Hkv, Dh = 150, 1, 128
    q, k = rows_of(rng, (G, Dh)), rows_of(rng, (Hkv, n, Dh)) * np.float32(0.3)
    # the row's key along q of head 0, downwards (and so that no other head has it as its maximum)
    k[0, at] = -q[0] * (60 * np.sqrt(Dh) / (q[0] @ q[0]))
    v = rng.uniform(-0.5, 0.5, (Hkv, n, Dh)) * 3e-4
    v[0, at] *= 1e8
    out, kv, vv = decode(cuda, q, k.astype(np.float32), v.astype(np.float32))
    s = kv[0] @ q[0].astype(np.float64) / np.sqrt(Dh)
    assert s[at] < s.max() - 45
    check(out, q, kv, vv, scores_bound(q, kv))


@pytest.mark.parametrize("G", [1, 5])
@pytest.mark.parametrize("step", [0.1, 0.67, 3.0])
@pytest.mark.parametrize("late", [0.0, 3e-4])
def test_maximum_that_rises_in_every_tile(cuda, G, step, late):
    """Scores that rise by `step` from one tile of 64 positions to the next
    over the 140 tiles that a warp has, the values large in the warp's first
    tile and small or 0 in the others: the scale of p d goes down with the
    weight, by no more and no less.

    Rows of keys are constant fp16 numbers x (d = 0, one product with sum q),
    whose scores are off by at most 8 fp32 roundings of sum |q k| = x.  Weights
    below 2^-126 are 0 in fp32 (steps of 0.67 and 3: e^-93 and e^-417 for the
    large values), which takes at most 2^-126 |v| of each position."""
    rng = np.random.default_rng(G)
    Dh, S, tiles = 32, 1 << 22, 4 * 140  # (a context whose shares are that long: up to 1041 tiles a CTA)
    n = 64 * tiles
    x = (np.arange(n) // 64 * step).astype(np.float16).astype(np.float32)
    v = rng.uniform(-0.5, 0.5, (n, Dh)) * np.where(np.arange(n) // 64 % 140 == 0, 3e3, late)[:, None]
    q = np.full((G, Dh), np.sqrt(Dh) / Dh, np.float32)
    (kr, k), (vr, vv) = kv_ref.q4_rows(np.repeat(x[:, None], Dh, 1)), kv_ref.q4_rows(v.astype(np.float32))
    caches = [cuda.zeros((1, 1, S, kv_ref.row_bytes(Dh)), dtype=cuda.uint8, device="cuda") for _ in range(2)]
    for c, r in zip(caches, (kr, vr)):
        c[0, 0, :n - 1] = dev(cuda, r[:-1])
    out = cuda.full((G, Dh), 5.0, device="cuda")
    wsb = rt.lib().lmc_attention_workspace_bytes(1, G, Dh, S)
    ws = cuda.full((wsb,), 0xff, dtype=cuda.uint8, device="cuda")
    d = [dev(cuda, a) for a in (q, np.repeat(x[-1:], Dh), v[-1].astype(np.float32), np.array([n - 1], np.int32))]
    rt.call("lmc_attention_decode", out.data_ptr(), *(t.data_ptr() for t in d[:3]), *(c.data_ptr() for c in caches), rt.KV_Q4,
            d[3].data_ptr(), 1, G, 1, Dh, S, ws.data_ptr(), wsb, None)
    assert rt.lib().lmc_device_status() == 0
    check(out.cpu().numpy(), q, k[None], vv[None], 8 * 2.0 ** -24 * x.max(), norm=False, least=2.0 ** -126)


@pytest.mark.parametrize("G", [1, 4, 5, 8])
@pytest.mark.parametrize("offset,r", [(100, 1), (100, 100), (100, 1000), (0, 100), (0, 1000)])
def test_queries_of_unequal_channels_over_keys_of_one_sign(cuda, G, offset, r):
    """Keys around 100, or from 0 on, that are small in every 16th channel, where q
    is r times larger: d (q . codes) and m sum(q) are large against the score and
    cancel.  What is left is of the size of the products q k, as above."""
    rng = np.random.default_rng(G + r + offset)
    Dh, n, Hkv = 128, 300, 2
    big = np.arange(Dh) % 16 == 5
    k = offset + rng.normal(0, 1, (Hkv, n, Dh)) if offset else np.abs(rng.normal(0, 1, (Hkv, n, Dh)))
    k[..., big] *= 1.0 / r if offset else 0.0
    q = rows_of(rng, (Hkv * G, Dh)) * np.where(big, 0.3 * r, 0.3).astype(np.float32)
    v = rows_of(rng, (Hkv, n, Dh))
    out, kv, vv = decode(cuda, q, k.astype(np.float32), v)
    kk, a = np.repeat(np.abs(kv), G, 0), np.abs(q.astype(np.float64))
    held = sum(2.0 ** -30 * a[:, g:g + 64].max(-1) * kk[:, :, g:g + 64].sum(-1).max(-1) for g in (0, 64))
    size = np.einsum("hnd,hd->hn", kk, a).max(-1)
    check(out, q, kv, vv, (held + 8 * 2.0 ** -24 * size) / np.sqrt(Dh))
