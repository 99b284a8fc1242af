"""What the entry points of the 4-bit and paged cache refuse, before they touch a
device, and the format's sizes (no GPU needed)."""
import ctypes

import numpy as np
import pytest

from lmc_b200 import runtime as rt
from tests import kv_ref

P = ctypes.c_void_p(4096)  # never dereferenced: the checks fail first
ODD = ctypes.c_void_p(4100)
INVALID, UNSUPPORTED = -1, -2


def status(name, *args):
    rc = getattr(rt.lib(), name)(*args)
    return rc, rt.lib().lmc_last_error()


def test_row_sizes():
    for Dh, size in ((32, 20), (64, 36), (96, 56), (128, 72), (160, 92), (192, 108), (224, 128), (256, 144)):
        assert rt.kv_row_bytes(rt.KV_Q4, Dh) == kv_ref.row_bytes(Dh) == size


def test_reference_rows_hold_their_values():
    """The reference quantizer: packing and unpacking agree, and a code is
    never more than half a step off (the rounding of m widens it by at most
    2^-11 |m|, values outside the codes' range by what d's rounding leaves:
    2^-11 x 15 d)."""
    rng = np.random.default_rng(1)
    for Dh in (32, 64, 96, 128, 256):
        x = rng.normal(0, 3, (50, Dh)).astype(np.float32)
        rows, vals = kv_ref.q4_rows(x)
        assert rows.shape == (50, kv_ref.row_bytes(Dh))
        assert np.array_equal(kv_ref.q4_values(rows, Dh), vals)
        for g in range(0, Dh, 64):
            p = x[:, g:g + 64]
            step = (p.max(-1) - p.min(-1)) / 15 * (1 + 2.0 ** -9)
            slack = 2.0 ** -11 * (np.abs(p).max(-1) + 15 * step)
            assert (np.abs(vals[:, g:g + 64] - p).max(-1) <= step / 2 + slack).all()


ROWS = dict(k=P, v=P, ld=256, kc=P, vc=P, kv=rt.KV_Q4, seq=P, pos=P, rows=4, n_seqs=2, Hkv=2, Dh=128, S=64,
            pages=None, page=0, n_pages=0)


@pytest.mark.parametrize("name", ["lmc_kv_append", "lmc_kv_read"])
@pytest.mark.parametrize("change,code,word", [
    (dict(k=None, v=None), INVALID, b"null"), (dict(kc=None), INVALID, b"null"), (dict(vc=None), INVALID, b"null"),
    (dict(pos=None), INVALID, b"null"), (dict(kv=4), UNSUPPORTED, b"kv dtype 4"), (dict(kv=-1), UNSUPPORTED, b"kv dtype"),
    (dict(rows=-1), INVALID, b"rows=-1"), (dict(n_seqs=0), INVALID, b"n_seqs=0"), (dict(Hkv=0), INVALID, b"Hkv=0"),
    (dict(Dh=48), INVALID, b"Dh=48"), (dict(Dh=0), INVALID, b"Dh=0"), (dict(Dh=-32), INVALID, b"Dh=-32"),
    (dict(Dh=288, ld=600), INVALID, b"Dh=288"), (dict(S=0), INVALID, b"S=0"), (dict(ld=255), INVALID, b"ld=255"),
    (dict(Hkv=2 ** 28, ld=2 ** 31 - 1), INVALID, b"ld>=Hkv"), (dict(kc=ODD), INVALID, b"16-byte"),
    (dict(vc=ODD), INVALID, b"16-byte"), (dict(rows=2 ** 30, Hkv=8, ld=2048), INVALID, b"in one call"),
    (dict(pages=P, page=24, n_pages=4), INVALID, b"pages"), (dict(pages=P, page=8, n_pages=4), INVALID, b"pages"),
    (dict(pages=P, page=16, n_pages=0), INVALID, b"pages"), (dict(pages=P, page=128, n_pages=4), INVALID, b"pages"),
    (dict(pages=P, page=16, n_pages=4, S=72), INVALID, b"pages")])
def test_rows_refusals(name, change, code, word):
    rc, msg = status(name, *{**ROWS, **change}.values(), None)
    assert rc == code and word in msg, (rc, msg)


def test_no_rows_is_no_work():
    for name in ("lmc_kv_append", "lmc_kv_read"):
        assert status(name, *{**ROWS, "rows": 0}.values(), None)[0] == 0


def test_attention_refusals_of_4_bit_caches():
    """A cache off a 16-byte boundary; other refusals as for the other row
    forms (a workspace that is too small, a head size that is no multiple
    of 32)."""
    dec = lambda kc, vc, Dh, ws: ("lmc_attention_decode", P, P, P, P, kc, vc, rt.KV_Q4, P, 2, 8, 2, Dh, 4096, P, ws, None)
    for args, word in ((dec(ODD, P, 128, 1 << 30), b"16-byte"), (dec(P, ODD, 128, 1 << 30), b"16-byte"),
                       (dec(P, P, 128, 8), b"workspace"), (dec(P, P, 80, 1 << 30), b"Dh=80"), (dec(P, P, 0, 1 << 30), b"Dh=0"),
                       (dec(P, P, -32, 1 << 30), b"Dh=-32"), (dec(P, P, 288, 1 << 30), b"Dh=288")):
        rc, msg = status(*args)
        assert rc == INVALID and word in msg, (rc, msg)
    rc, msg = status("lmc_attention_decode_noalloc", P, P, P, P, ODD, P, rt.KV_Q4, P, 1, 8, 2, 128, 256, None)
    assert rc == INVALID and b"16-byte" in msg
    rc, msg = status("lmc_attention_decode_paged", P, P, P, P, P, P, rt.KV_Q4, 8, P, 4, 24, P, 1, 8, 2, 128, P, 0, None)
    assert rc == INVALID and b"attention_paged" in msg


def test_attention_refuses_contexts_too_long_for_4_bit_rows():
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        rc, msg = status("lmc_attention_decode", P, P, P, P, P, P, rt.KV_Q4, P, 1, 1, 1, 32, n, P, 1 << 40, None)
        assert rc == UNSUPPORTED and b"2^30" in msg, (rc, msg)


def test_page_operator_refusals():
    one = (ctypes.c_void_p * 1)(4096)
    null, odd = (ctypes.c_void_p * 2)(4096, None), (ctypes.c_void_p * 2)(4096, 4104)
    ws = rt.lib().lmc_kv_pages_workspace_bytes(4, 100)
    assert ws > 0 and rt.lib().lmc_kv_pages_workspace_bytes(-1, 100) == 0
    fork = lambda **k: ("lmc_kv_pages_fork", *{**dict(t=P, n=4, w=8, r=P, np=100, p=P), **k}.values(), None)
    res = lambda **k: ("lmc_kv_pages_reserve", *{**dict(h=one, k=1, by=4096, t=P, n=4, w=8, ps=16, r=P, np=100, pos=P,
                                                        sh=P, ws=P, wb=ws), **k}.values(), None)
    com = lambda **k: ("lmc_kv_pages_compact", *{**dict(h=one, k=1, by=4096, t=P, n=4, w=8, r=P, np=100, nl=P, ws=P,
                                                        wb=ws), **k}.values(), None)
    cases = [(fork(t=None), b"null"), (fork(r=None), b"null"), (fork(p=None), b"null"), (fork(n=0), b"0 sequences"),
             (fork(n=16385), b"16384"), (fork(w=0), b"x 0 entries"), (fork(np=0), b"0 pages"),
             (res(pos=None), b"null"), (res(sh=None), b"null"), (res(ws=None), b"null"), (res(ps=24), b"24 positions"),
             (res(ps=8), b"8 positions"), (res(n=-1), b"-1 sequences"), (com(nl=None), b"null"), (com(np=-5), b"-5 pages")]
    for f in (res, com):
        cases += [(f(h=None), b"pools"), (f(k=0), b"0 pools"), (f(by=0), b"0 bytes"), (f(by=4088), b"multiple of 16"),
                  (f(h=null, k=2), b"pool 1"), (f(h=odd, k=2), b"pool 1"), (f(wb=ws - 1), b"workspace"), (f(t=None), b"null"),
                  (f(r=None), b"null")]
    for args, word in cases:
        rc, msg = status(*args)
        assert rc == INVALID and word in msg, (args, rc, msg)


def test_reserve_of_too_many_sequences_is_refused():
    one, ws = (ctypes.c_void_p * 1)(4096), rt.lib().lmc_kv_pages_workspace_bytes(65537, 9)
    rc, msg = status("lmc_kv_pages_reserve", one, 1, 4096, P, 65537, 8, 16, P, 9, P, P, P, ws, None)
    assert rc == INVALID and b"65537 sequences" in msg, (rc, msg)


def test_page_pools_too_large_are_refused():
    one, n = (ctypes.c_void_p * 1)(4096), (1 << 30) + 1
    ws = rt.lib().lmc_kv_pages_workspace_bytes(4, n)
    assert ws > 16 << 30
    for args in (("lmc_kv_pages_reserve", one, 1, 4096, P, 4, 8, 16, P, n, P, P, P, ws, None),
                 ("lmc_kv_pages_compact", one, 1, 4096, P, 4, 8, P, n, P, P, ws, None)):
        rc, msg = status(*args)
        assert rc == INVALID and b"1073741825 pages" in msg, (rc, msg)


def test_model_load_takes_4_bit_rows_and_refuses_unknown_ones():
    h = ctypes.c_void_p()
    rc, msg = status("lmc_model_load", b"/nonexistent.gguf", 1, rt.KV_Q4, ctypes.byref(h))
    assert rc == -5 and b"cannot open" in msg
    rc, msg = status("lmc_model_load", b"/nonexistent.gguf", 1, 4, ctypes.byref(h))
    assert rc == INVALID and b"kv dtype" in msg


def test_oracle_rounds_4_bit_rows_like_the_format(orc):
    """The oracle's 4-bit rows (a C restatement) hold the values of the
    format's definition in tests/kv_ref.py, special rows included."""
    from tests.test_gpu_kv_q4 import rows_of, special_rows
    rng = np.random.default_rng(5)
    for Dh in (32, 64, 96, 128, 256):
        x = np.concatenate([special_rows(Dh), rows_of(rng, (200, Dh), "outliers")])
        want = kv_ref.q4_rows(x)[1]
        got = orc.kv_round_rows(x, rt.KV_Q4).astype(np.float64)
        # the oracle stores the value as fp32: half a step
        assert (np.isnan(got) == np.isnan(want)).all()
        ok = ~np.isnan(want)
        assert (np.abs(got - want)[ok] <= 2.0 ** -24 * np.abs(want)[ok]).all()
