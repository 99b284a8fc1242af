"""4-bit K/V rows and attention over them in 64 bits, and the page operators one
sequence at a time: what the tests of the 4-bit paged cache compare with."""
import numpy as np


def row_bytes(Dh):
    return Dh // 2 + 4 * -(-Dh // 64)


def q4_rows(x):
    """fp32 [..., Dh] -> (row bytes uint8 [..., row_bytes], the values they
    stand for as float64).  Every rounding that LMC_KV_Q4 names: m =
    fp16(min), d = fp16((max - m) / 15) in fp32 steps, saturated; the code is
    the nearest whole number to the 64-bit quotient."""
    x = np.asarray(x, np.float32)
    Dh = x.shape[-1]
    codes, tail, vals = [], [], []
    for g in range(0, Dh, 64):
        p = x[..., g:g + 64]
        fine = np.isfinite(p).all(-1, keepdims=True)
        p = np.where(fine, p, np.float32(0))
        m = np.clip(p.min(-1, keepdims=True), -65504, 65504).astype(np.float16)
        with np.errstate(over="ignore"):
            w = np.maximum(p.max(-1, keepdims=True) - m.astype(np.float32), np.float32(0))
            d = np.minimum(w / np.float32(15), np.float32(65504)).astype(np.float16)
        d64, m64 = d.astype(np.float64), m.astype(np.float64)
        c = np.clip(np.rint((p.astype(np.float64) - m64) / np.where(d64 > 0, d64, 1)), 0, 15)
        c = np.where(d64 > 0, c, 0).astype(np.uint8)
        d = np.where(fine, d, np.float16(np.nan))
        m = np.where(fine, m, np.float16(0))
        codes.append(c)
        tail.append(np.concatenate([d, m], -1))
        vals.append(d.astype(np.float64) * c + m.astype(np.float64))
    c = np.concatenate(codes, -1)
    packed = (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)
    t = np.ascontiguousarray(np.concatenate(tail, -1)).view(np.uint8)
    return np.concatenate([packed, t], -1), np.concatenate(vals, -1)


def q4_values(rows, Dh):
    """Row bytes -> the float64 values they stand for."""
    c = rows[..., :Dh // 2]
    c = np.stack([c & 15, c >> 4], -1).reshape(c.shape[:-1] + (Dh,)).astype(np.float64)
    t = np.ascontiguousarray(rows[..., Dh // 2:]).view(np.float16).astype(np.float64)
    d, m = (np.repeat(t[..., k::2], 64, -1)[..., :Dh] for k in (0, 1))
    return d * c + m


def attention(q, k, v):
    """q [H][Dh], k and v [Hkv][n][Dh] in 64 bits -> (out [H][Dh], the largest
    sum of |q_i k_ti| / sqrt(Dh) over the scores)."""
    H, Dh = q.shape
    G = H // k.shape[0]
    out, size = np.empty((H, Dh)), 0.0
    for h in range(H):
        kk, vv = k[h // G], v[h // G]
        s = kk @ q[h].astype(np.float64) / np.sqrt(Dh)
        size = max(size, float((np.abs(kk) @ np.abs(q[h].astype(np.float64))).max() / np.sqrt(Dh)))
        p = np.exp(s - s.max())
        out[h] = p @ vv / p.sum()
    return out, size


def fork(table, refs, parent):
    old = table.copy()
    for b, p in enumerate(parent):
        if p < len(table):
            table[b] = -1 if p < 0 else old[p]
    refs[:] = np.bincount(table[table >= 0], minlength=len(refs))


def reserve(table, refs, pos, P):
    """-> (missing, [(source, destination)] of the pages copied)."""
    t, r, copies = table.copy(), refs.copy(), []
    free, want = [i for i in range(len(r)) if r[i] == 0], 0
    for b, p in enumerate(pos):
        if p < 0 or p // P >= t.shape[1]:
            continue
        e = t[b, p // P]
        if e >= 0 and r[e] <= 1:
            continue
        want += 1
        new = free[want - 1] if want <= len(free) else -1
        if e >= 0:
            copies.append((e, new))
            r[e] -= 1
        t[b, p // P] = new
        if new >= 0:
            r[new] = 1
    if want > len(free):
        return want - len(free), []
    table[:], refs[:] = t, r
    return 0, copies


def compact(table, refs):
    """-> (pages in use, [(source, destination)])."""
    n = int((refs > 0).sum())
    holes = [i for i in range(n) if refs[i] == 0]
    moved = list(zip([i for i in range(n, len(refs)) if refs[i] > 0], holes))
    for s, d in moved:
        refs[d], refs[s] = refs[s], 0
        table[table == s] = d
    return n, moved
