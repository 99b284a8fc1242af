"""Serving with a 4-bit, paged KV cache: the operators' cases, plain forms and exact values.

  decode   one token per sequence: its K/V row is quantized into the cache and attention runs
           over the rows of 4-bit codes (lmc_attention_decode, lmc_attention_decode_paged)
  append   a prompt's K/V rows quantized into the cache, and read back (lmc_kv_append, lmc_kv_read)
  fork     sequences become copies of others, page by page, or give their pages back (lmc_kv_pages_fork)
  reserve  before a step: every sequence gets a page of its own to write in (lmc_kv_pages_reserve)
  compact  pages in use move to the lowest ids (lmc_kv_pages_compact)

A 4-bit row (LMC_KV_Q4) of Dh values is Dh / 2 bytes of codes (dim 2 i in the low half of byte i)
followed, for each group of 64 dims (the last may have 32), by two fp16 numbers d and m; a value is
d * code + m.
"""
import math

import numpy as np
import torch

own = False

GROUP = 64
CODES = 15
F16_MAX = 65504.0
KV_F16, KV_Q4 = 1, 3


# ---- the row format -------------------------------------------------------------------------
def row_bytes(dh):
    return dh // 2 + 4 * -(-dh // GROUP)


def group_sizes(dh):
    return [min(GROUP, dh - g) for g in range(0, dh, GROUP)]


def quantize(x):
    """fp32 [..., Dh] -> packed rows uint8 [..., row_bytes].  m = fp16(min), d = fp16((max - m) / 15)
    (fp32 steps, saturated at the largest fp16), code = the whole number nearest to (x - m) / d
    in 0..15, decided in 64 bits; a group with a value that is not finite has d = NaN."""
    dh, codes, tail = x.shape[-1], [], []
    for part in torch.split(x, group_sizes(dh), -1):
        fine = torch.isfinite(part).all(-1, keepdim=True)
        part = torch.where(fine, part, 0.0)
        lo, hi = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
        m = lo.clamp(-F16_MAX, F16_MAX).half()
        width = (hi - m.float()).clamp(min=0.0)
        d = (width / torch.full_like(width, CODES)).clamp(max=F16_MAX).half()  # (a number would be multiplied by 1 / 15)
        c = torch.round((part.double() - m.double()) / torch.where(d > 0, d, 1.0).double()).clamp(0, CODES)
        codes.append(torch.where(d > 0, c, 0.0).to(torch.uint8))
        tail.append(torch.cat([torch.where(fine, d, float("nan")), torch.where(fine, m, 0.0)], -1))
    c = torch.cat(codes, -1)
    packed = c[..., 0::2] | (c[..., 1::2] << 4)
    return torch.cat([packed, torch.cat(tail, -1).contiguous().view(torch.uint8)], -1)


def dequantize(rows, dh):
    """packed rows uint8 [..., row_bytes] -> fp32 [..., Dh]."""
    c = rows[..., : dh // 2]
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    dm = rows[..., dh // 2:].contiguous().view(torch.float16).float()
    d, m = (dm[..., k::2].repeat_interleave(GROUP, -1)[..., :dh] for k in (0, 1))
    return d * c + m


# ---- cases ----------------------------------------------------------------------------------
def listed():
    return [
        # GPT-2 Small's heads, one sequence in the middle of its context: the smallest step of a chat
        dict(name="decode gpt2 b1", op="decode", batch=1, hkv=12, group=1, dh=64, ctx=1024, page=0, lo=700, hi=700),
        # the TinyLlama shape, 64 users of different lengths in a paged pool
        dict(name="decode tinyllama b64", op="decode", batch=64, hkv=4, group=8, dh=64, ctx=2048, page=16, lo=1, hi=2048),
        # the 8B shape, one user with a very long context
        dict(name="decode 8b long", op="decode", batch=1, hkv=8, group=4, dh=128, ctx=131072, page=64, lo=131071, hi=131071),
        # the 8B shape, a full server: 128 users up to 4096 positions
        dict(name="decode 8b b128", op="decode", batch=128, hkv=8, group=4, dh=128, ctx=4096, page=32, lo=1, hi=4096),
        # one prompt of odd length in a paged pool
        dict(name="append tinyllama 509", op="append", seqs=1, rows=509, hkv=4, dh=64, ctx=2048, page=16),
        # a batch of prompts in contiguous caches
        dict(name="append 8b 16x2000", op="append", seqs=16, rows=2000, hkv=8, dh=128, ctx=2048, page=0),
        # a beam search's reorder of 5 beams
        dict(name="fork 5 beams", op="fork", seqs=5, table=128, used=47, mode="beam"),
        # 256 slots: finished sequences freed, their slots given to new samples of the others
        dict(name="fork 256 slots", op="fork", seqs=256, table=2048, used=1800, mode="mixed"),
        # 4 samples of one prompt about to write for the first time (GPT-2: 12 layers)
        dict(name="reserve 4 samples", op="reserve", seqs=4, fan=4, pools=24, hkv=12, dh=64, page=16, prompt=203),
        # 128 samples of 16 prompts (the 8B shape: 32 layers)
        dict(name="reserve 128 samples", op="reserve", seqs=128, fan=8, pools=64, hkv=8, dh=128, page=16, prompt=500),
        # a small pool after a burst of requests
        dict(name="compact 96 pages", op="compact", seqs=6, pages=96, pools=24, hkv=12, dh=64, page=16, live=41),
        # a server's pool shrunk before its memory is given to something else
        dict(name="compact 1024 pages", op="compact", seqs=64, pages=1024, pools=64, hkv=8, dh=128, page=16, live=600),
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "append", "fork", "reserve", "compact"])
    if op == "decode":
        page = rng.choice([0, 16, 32, 64, 256])
        ctx = log_int(rng, 16, 131072)
        ctx = -(-ctx // page) * page if page else ctx
        hkv, dh = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([32, 64, 64, 96, 128, 128, 160, 256])
        most = max(1, min(256, 128 * 4096 * 8 * 128 // (2 * ctx * hkv * dh)))
        hi = rng.randint(max(1, ctx // 2), ctx)
        return dict(op="decode", batch=log_int(rng, 1, most), hkv=hkv, group=rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), dh=dh,
                    ctx=ctx, page=page, lo=rng.choice([1, hi]), hi=hi)
    if op == "append":
        page = rng.choice([0, 16, 128])
        ctx = log_int(rng, 16, 8192)
        ctx = -(-ctx // page) * page if page else ctx
        hkv, dh = rng.choice([1, 2, 3, 4, 8, 12]), rng.choice([32, 64, 96, 128, 256])
        most = max(1, min(64, 16 * 2000 * 8 * 128 // (ctx * hkv * dh)))
        return dict(op="append", seqs=log_int(rng, 1, most), rows=rng.randint(1, ctx), hkv=hkv, dh=dh, ctx=ctx, page=page)
    if op == "fork":
        table = log_int(rng, 1, 2048)
        return dict(op="fork", seqs=log_int(rng, 2, 256), table=table, used=rng.randint(1, table), mode=rng.choice(["beam", "mixed"]))
    page, hkv, dh, pools = rng.choice([16, 32]), rng.choice([1, 2, 3, 4]), rng.choice([32, 64, 128]), rng.choice([2, 12, 24, 44, 64])
    if op == "reserve":
        fan = rng.choice([1, 2, 3, 5, 8])
        return dict(op="reserve", seqs=fan * log_int(rng, 1, 128 // fan), fan=fan, pools=pools, hkv=hkv, dh=dh, page=page, prompt=rng.randint(1, 500))
    pages = log_int(rng, 8, 1024)
    return dict(op="compact", seqs=log_int(rng, 1, 64), pages=pages, pools=pools, hkv=hkv, dh=dh, page=page, live=rng.randint(1, pages))


# ---- what is known of a case without its inputs ---------------------------------------------
def lengths(c):
    """Positions in the cache after the step, per sequence: spread from lo to hi in an order of
    their own, one slot of a ragged batch of 8 or more idle (0)."""
    n = c["batch"]
    v = [c["lo"] + (c["hi"] - c["lo"]) * ((b * 37) % n) // max(1, n - 1) for b in range(n)]
    v = [min(max(x, 1), c["hi"]) for x in v] if n > 1 else [c["hi"]]
    if n >= 8 and c["lo"] != c["hi"]:
        v[n // 2] = 0
    return v


def append_positions(c):
    """Row r of sequence s goes to position r; every 64th row from row 50 on is padding (-1)."""
    r = np.tile(np.arange(c["rows"], dtype=np.int32), (c["seqs"], 1))
    r[:, 50::64] = -1
    return r.reshape(-1)


def parents(c):
    n = c["seqs"]
    p = [(b * 3 + 1) % max(1, n // 2) for b in range(n)]
    if c["mode"] == "mixed":  # every third slot stays, every fifth is freed
        p = [b if b % 3 == 0 else -1 if b % 5 == 1 else p[b] for b in range(n)]
    return p


def family_prompt(c, f):
    """Positions of family f's prompt: every fourth family's ends with its last page full."""
    n = max(1, c["prompt"] - 7 * f)
    return -(-n // c["page"]) * c["page"] if f % 4 == 3 else n


def page_elems(c):
    return c["hkv"] * c["page"] * c["dh"]


def work(c):
    if c["op"] == "decode":
        n, hq, rb = lengths(c), c["hkv"] * c["group"] * c["dh"], row_bytes(c["dh"])
        live, rows = sum(1 for x in n if x), sum(n)
        new = live * c["hkv"] * (8 * c["dh"] + 2 * rb)  # the new K and V rows: fp32 read, 4 bits written
        back = live * c["hkv"] * 8 * c["dh"]  # their values, read back
        table = 4 * sum(-(-x // c["page"]) for x in n) if c["page"] else 0
        return {"bytes": 2 * (rows - live) * c["hkv"] * rb + live * 8 * hq + new + back + table, "flops": 4 * rows * hq}
    if c["op"] == "append":
        rows = int((append_positions(c) >= 0).sum())
        return {"bytes": rows * c["hkv"] * (16 * c["dh"] + 4 * row_bytes(c["dh"])), "flops": 8 * rows * c["hkv"] * c["dh"]}
    if c["op"] == "fork":  # the rows that change, read at their parent and written; a count per page
        changed = sum(1 for b, p in enumerate(parents(c)) if p != b)
        kept = sum(1 for b, p in enumerate(parents(c)) if p != b and p >= 0)
        return {"bytes": 4 * c["table"] * (changed + kept) + 8 * c["seqs"] * c["used"], "flops": c["table"] * changed}
    if c["op"] == "reserve":
        fam = c["seqs"] // c["fan"]
        copies = sum(c["fan"] - 1 for f in range(fam) if family_prompt(c, f) % c["page"])
        return {"bytes": 4 * copies * page_elems(c) * c["pools"] + 16 * c["seqs"], "flops": c["seqs"]}
    live = c["live"]  # about live * (1 - live / pages) of the live pages lie above the lowest `live` ids
    moved = live * (c["pages"] - live) / c["pages"]
    return {"bytes": 4 * moved * page_elems(c) * c["pools"] + 8 * c["pages"], "flops": c["pages"]}


# ---- inputs ---------------------------------------------------------------------------------
def page_table(c, n_seqs, g):
    """A table [n_seqs][ctx / page] of distinct pages in a random order, a few pages to spare."""
    each = c["ctx"] // c["page"]
    n_pages = n_seqs * each + 3
    perm = torch.randperm(n_pages, generator=g, device="cuda")[: n_seqs * each]
    return perm.view(n_seqs, each).int().contiguous(), n_pages


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case=c, stream=torch.cuda.current_stream().cuda_stream)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["op"] in ("decode", "append"):
        n_seqs = c["batch"] if c["op"] == "decode" else c["seqs"]
        hkv, dh, ctx, page, rb = c["hkv"], c["dh"], c["ctx"], c["page"], row_bytes(c["dh"])
        # keys have a few large channels, values have not
        big = 1.0 + 6.0 * (torch.rand(hkv, 1, dh, generator=g, device="cuda") < 0.03)
        s["pages"], n_pages = page_table(c, n_seqs, g) if page else (None, 0)
        shape = (n_pages, hkv, page, rb) if page else (n_seqs, hkv, ctx, rb)
        s["n_pages"], s["n_seqs"] = n_pages, n_seqs
        # bytes that no row was written to hold anything (0xff: a NaN for a scale)
        s["kc"], s["vc"] = (torch.full(shape, 255, dtype=torch.uint8, device="cuda") for _ in range(2))
        if c["op"] == "decode":
            n = lengths(c)
            s["pos"] = ints([x - 1 for x in n])
            for b, x in enumerate(n):
                if x > 1:  # every row before the new one
                    k, v = quantize(normal(hkv, x - 1, dh) * big), quantize(normal(hkv, x - 1, dh))
                    if page:
                        full, ids = -(-(x - 1) // page), s["pages"][b].long()
                        for cache, r in ((s["kc"], k), (s["vc"], v)):
                            t = torch.full((hkv, full * page, rb), 255, dtype=torch.uint8, device="cuda")
                            t[:, : x - 1] = r
                            cache[ids[:full]] = t.view(hkv, full, page, rb).transpose(0, 1)
                    else:
                        s["kc"][b, :, : x - 1], s["vc"][b, :, : x - 1] = k, v
            h = hkv * c["group"]
            s["q"] = normal(n_seqs, h * dh)
            s["k"], s["v"] = (normal(n_seqs, hkv, dh) * big[:, 0]).view(n_seqs, -1), normal(n_seqs, hkv * dh)
            s["out"], s["rows"] = torch.zeros(n_seqs, h * dh, device="cuda"), n_seqs
            s["seq"] = torch.arange(n_seqs, dtype=torch.int32, device="cuda")
            # enough for the split-context scratch of any of the library's plans
            s["ws"] = torch.empty(n_seqs * h * 64 * (dh + 2), device="cuda")
        else:
            s["pos"] = torch.from_numpy(append_positions(c)).cuda()
            s["seq"] = torch.arange(n_seqs, dtype=torch.int32, device="cuda").repeat_interleave(c["rows"]).contiguous()
            s["rows"] = n_seqs * c["rows"]
            s["k"], s["v"] = (normal(s["rows"], hkv, dh) * big[:, 0]).view(s["rows"], -1), normal(s["rows"], hkv * dh)
        s["ko"], s["vo"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    # page operators: the table and the pages' use counts lie in one buffer, kept as they were
    # before the call (`before`), since each pass starts from there
    n = c["seqs"]
    if c["op"] == "fork":
        wide = c["table"]
        n_pages = n * c["used"] + 5
        table = torch.full((n, wide), -1, dtype=torch.int32, device="cuda")
        table[:, : c["used"]] = torch.randperm(n_pages, generator=g, device="cuda")[: n * c["used"]].view(n, -1).int()
        table[1::2, : c["used"] // 2] = table[0: n - 1: 2, : c["used"] // 2]  # pairs share a prompt
        s["parent"] = ints(parents(c))
    elif c["op"] == "reserve":
        fam, P = n // c["fan"], c["page"]
        wide = max(family_prompt(c, f) for f in range(fam)) // P + 2
        each = [-(-family_prompt(c, f) // P) for f in range(fam)]
        n_pages = sum(each) + n + 5
        perm = torch.randperm(n_pages, generator=g, device="cuda").int()
        table = torch.full((n, wide), -1, dtype=torch.int32, device="cuda")
        at = 0
        for f in range(fam):
            table[f * c["fan"]:(f + 1) * c["fan"], : each[f]] = perm[at: at + each[f]]
            at += each[f]
        s["pos"] = ints([family_prompt(c, b // c["fan"]) for b in range(n)])
        s["short"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    else:
        n_pages, live = c["pages"], c["live"]
        wide = -(-2 * live // n) + 1
        table = torch.full((n * wide,), -1, dtype=torch.int32, device="cuda")
        ids = torch.randperm(n_pages, generator=g, device="cuda")[:live].int()
        table[:live] = ids  # every live page once, then some of them shared
        table[live: live + live // 3] = ids[: live // 3]
        table = table.view(wide, n).t().contiguous()
        s["n_live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    flat = table.reshape(-1).long()
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda").scatter_add_(0, flat.clamp(min=0), (flat >= 0).int())
    s["before"] = torch.cat([table.reshape(-1), refs])
    s["now"] = s["before"].clone()
    s["pages"], s["refs"], s["n_pages"], s["wide"] = s["now"][: n * wide].view(n, wide), s["now"][n * wide:], n_pages, wide
    s["ws"] = torch.empty(n_pages * 4 + n * 4 + 64, dtype=torch.int32, device="cuda")
    if c["op"] != "fork":
        s["pools"] = torch.randn(c["pools"], n_pages, page_elems(c), generator=g, device="cuda", dtype=torch.float16)
    return s


# ---- the plain forms ------------------------------------------------------------------------
def where_rows(s):
    """(first index, slot) of each row of a cache: its page or sequence, and its position there."""
    c, pos, seq = s["case"], s["pos"].long(), s["seq"].long()
    ok = pos >= 0
    pos, seq = pos[ok], seq[ok]
    if c["page"]:
        return ok, s["pages"][seq, pos // c["page"]].long(), pos % c["page"]
    return ok, seq, pos


def plain_append(s):
    """The new rows quantized into the caches; their values."""
    c = s["case"]
    ok, first, slot = where_rows(s)
    for cache, x, to in ((s["kc"], s["k"], s["ko"]), (s["vc"], s["v"], s["vo"])):
        r = quantize(x.view(-1, c["hkv"], c["dh"])[ok])
        cache[first, :, slot] = r
        to[ok] = dequantize(r, c["dh"]).flatten(1)
    return s["ko"], s["vo"]


def plain_decode(s):
    c = s["case"]
    ko, vo = plain_append(s)
    n, hkv, dh, ctx = c["batch"], c["hkv"], c["dh"], c["ctx"]
    top = min(ctx, -(-c["hi"] // max(1, c["page"])) * max(1, c["page"]))  # no sequence is longer
    rows = []
    for cache in (s["kc"], s["vc"]):
        if c["page"]:
            ids = s["pages"][:, : top // c["page"]].long()
            rows.append(cache[ids].transpose(1, 2).reshape(n, hkv, top, -1))
        else:
            rows.append(cache[:, :, :top])
    seen = torch.arange(top, device="cuda") <= s["pos"][:, None]  # [n, top]
    k, v = (torch.where(seen[:, None, :, None], dequantize(r, dh), 0.0) for r in rows)
    q = s["q"].view(n, hkv, c["group"], dh)
    w = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(dh)
    w = w.masked_fill(~seen[:, None, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-3e38))
    o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    live = s["pos"] >= 0
    s["out"][live] = o.reshape(n, -1)[live]
    return [s["out"], ko, vo]


def plain_fork(s):
    s["now"].copy_(s["before"])
    t, p = s["pages"].clone(), s["parent"].long()
    changed = (p != torch.arange(len(p), device="cuda"))[:, None]
    new = torch.where(p[:, None] < 0, -1, t[p.clamp(min=0)])
    for entries, sign in ((t, -1), (new, 1)):
        s["refs"].scatter_add_(0, entries.flatten().long().clamp(min=0), (sign * (changed & (entries >= 0)).int()).flatten())
    s["pages"].copy_(new)
    return [s["pages"], s["refs"]]


def plain_reserve(s):
    s["now"].copy_(s["before"])
    c, pos, refs = s["case"], s["pos"].long(), s["refs"]
    b = torch.arange(c["seqs"], device="cuda")
    j = pos // c["page"]
    e = s["pages"][b, j].long()
    same = (e[:, None] == e[None, :]) & (e >= 0)[:, None]
    rank = (same & (b[None, :] < b[:, None])).sum(1)  # writers of the same page before this one
    copy = (e >= 0) & (rank < refs[e.clamp(min=0)] - 1)  # the last holder keeps the page
    need = copy | (e < 0)
    free = torch.argsort((refs != 0).int(), stable=True)  # free ids first, lowest first
    short = (need.sum() - (refs == 0).sum()).clamp(min=0)
    s["short"][0] = short
    need, copy = need & (short == 0), copy & (short == 0)
    new = free[(torch.cumsum(need.int(), 0) - 1).clamp(0, len(free) - 1)]
    src, dst = e[copy], new[copy]
    s["pools"][:, dst] = s["pools"][:, src]
    refs.scatter_add_(0, new, need.int())
    refs.scatter_add_(0, e.clamp(min=0), -copy.int())
    s["pages"][b, j] = torch.where(need, new, e).int()
    return [s["pages"], refs, s["short"], s["pools"]]


def plain_compact(s):
    s["now"].copy_(s["before"])
    refs = s["refs"]
    ids, live = torch.arange(len(refs), device="cuda"), refs > 0
    n_live = live.sum()
    s["n_live"][0] = n_live
    src, dst = ids[live & (ids >= n_live)], ids[~live & (ids < n_live)]
    to = ids.clone()
    to[src] = dst
    s["pools"][:, dst] = s["pools"][:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    t = s["pages"].long()
    s["pages"].copy_(torch.where(t < 0, -1, to[t.clamp(min=0)]))
    return [s["pages"], refs, s["n_live"], s["pools"]]


# ---- the framework's calls ------------------------------------------------------------------
def own_read(rt, s):
    c = s["case"]
    rt.call("lmc_kv_read", s["ko"].data_ptr(), s["vo"].data_ptr(), c["hkv"] * c["dh"], s["kc"].data_ptr(), s["vc"].data_ptr(), KV_Q4,
            s["seq"].data_ptr(), s["pos"].data_ptr(), s["rows"], s["n_seqs"], c["hkv"], c["dh"], c["ctx"],
            rt.ptr(s["pages"]), c["page"], s["n_pages"], s["stream"])
    return [s["ko"], s["vo"]]


def own_append(s):
    from lmc_b200 import runtime as rt
    c = s["case"]
    rt.call("lmc_kv_append", s["k"].data_ptr(), s["v"].data_ptr(), c["hkv"] * c["dh"], s["kc"].data_ptr(), s["vc"].data_ptr(), KV_Q4,
            s["seq"].data_ptr(), s["pos"].data_ptr(), s["rows"], s["n_seqs"], c["hkv"], c["dh"], c["ctx"],
            rt.ptr(s["pages"]), c["page"], s["n_pages"], s["stream"])
    return own_read(rt, s)


def own_decode(s):
    from lmc_b200 import runtime as rt
    c = s["case"]
    h = c["hkv"] * c["group"]
    first = [s["out"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["kc"].data_ptr(), s["vc"].data_ptr(), KV_Q4]
    last = [s["ws"].data_ptr(), s["ws"].numel() * 4, s["stream"]]
    if c["page"]:
        rt.call("lmc_attention_decode_paged", *first, s["n_pages"], s["pages"].data_ptr(), c["ctx"] // c["page"], c["page"],
                s["pos"].data_ptr(), c["batch"], h, c["hkv"], c["dh"], *last)
    else:
        rt.call("lmc_attention_decode", *first, s["pos"].data_ptr(), c["batch"], h, c["hkv"], c["dh"], c["ctx"], *last)
    return [s["out"]] + own_read(rt, s)


def own_fork(s):
    from lmc_b200 import runtime as rt
    s["now"].copy_(s["before"])
    rt.call("lmc_kv_pages_fork", s["pages"].data_ptr(), s["case"]["seqs"], s["wide"], s["refs"].data_ptr(), s["n_pages"],
            s["parent"].data_ptr(), s["stream"])
    return [s["pages"], s["refs"]]


def pool_list(rt, s):
    """The pools' addresses, as a program that owns one buffer per layer keeps them."""
    if "list" not in s:
        s["list"] = rt.pool_list([p for p in s["pools"]])
    return s["list"]


def own_reserve(s):
    from lmc_b200 import runtime as rt
    c = s["case"]
    s["now"].copy_(s["before"])
    rt.call("lmc_kv_pages_reserve", pool_list(rt, s), c["pools"], page_elems(c) * 2, s["pages"].data_ptr(), c["seqs"], s["wide"], c["page"],
            s["refs"].data_ptr(), s["n_pages"], s["pos"].data_ptr(), s["short"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel() * 4, s["stream"])
    return [s["pages"], s["refs"], s["short"], s["pools"]]


def own_compact(s):
    from lmc_b200 import runtime as rt
    c = s["case"]
    s["now"].copy_(s["before"])
    rt.call("lmc_kv_pages_compact", pool_list(rt, s), c["pools"], page_elems(c) * 2, s["pages"].data_ptr(), c["seqs"], s["wide"],
            s["refs"].data_ptr(), s["n_pages"], s["n_live"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel() * 4, s["stream"])
    return [s["pages"], s["refs"], s["n_live"], s["pools"]]


def run(s):
    op = s["case"]["op"]
    if own:
        return {"decode": own_decode, "append": own_append, "fork": own_fork, "reserve": own_reserve, "compact": own_compact}[op](s)
    return {"decode": plain_decode, "append": plain_append, "fork": plain_fork, "reserve": plain_reserve, "compact": plain_compact}[op](s)


# ---- exact values ---------------------------------------------------------------------------
def exact_row_values(x, dh):
    """The values that 4-bit rows of x [..., Dh] stand for, in 64 bits: every rounding that the
    format names, taken one by one."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for g0 in range(0, dh, GROUP):
        p = x[..., g0: g0 + GROUP].double()
        m = p.min(-1, keepdim=True).values.float().half().double()
        width = (p.max(-1, keepdim=True).values - m).float()  # fp32 difference of two fp32 numbers
        d = (width.clamp(min=0) / torch.tensor(15.0, device=x.device)).half().double()
        near = torch.floor((p - m) / d.clamp(min=1e-30) + 0.5)
        tie = ((p - m) / d.clamp(min=1e-30) + 0.5) == near
        near = torch.where(tie & (near % 2 == 1), near - 1, near)  # a tie goes to the even code
        out[..., g0: g0 + GROUP] = torch.where(d > 0, near.clamp(0, 15) * d + m, m)
    return out


def exact_cache_values(rows, dh):
    b = rows.long()
    i = torch.arange(dh, device=rows.device)
    code = (b[..., i // 2] >> (4 * (i % 2))) & 15
    t = rows[..., dh // 2:].contiguous().view(torch.float16).double()
    return t[..., 2 * (i // GROUP)] * code + t[..., 2 * (i // GROUP) + 1]


def exact_decode(c, s):
    n, hkv, dh, G = c["batch"], c["hkv"], c["dh"], c["group"]
    new = [exact_row_values(s[x].view(n, hkv, dh), dh) for x in ("k", "v")]
    out = torch.zeros(n, hkv * G, dh, dtype=torch.float64, device="cuda")
    for b, x in enumerate(lengths(c)):
        if not x:
            new[0][b] = new[1][b] = 0
            continue
        for h in range(hkv):
            vals = []
            for cache, nv in zip((s["kc"], s["vc"]), new):
                if c["page"]:
                    full = -(-x // c["page"])
                    r = cache[s["pages"][b, :full].long(), h].reshape(full * c["page"], -1)[: x - 1]
                else:
                    r = cache[b, h, : x - 1]
                vals.append(torch.cat([exact_cache_values(r, dh), nv[b, h][None]]))
            q = s["q"][b].view(hkv, G, dh)[h].double()
            a = torch.softmax((q @ vals[0].T) * dh ** -0.5, -1)
            out[b, h * G:(h + 1) * G] = a @ vals[1]
    return [out.view(n, -1), new[0].view(n, -1), new[1].view(n, -1)]


def exact_pages(c, s):
    """The page operators, one sequence and one page at a time, on the host."""
    n, wide = c["seqs"], s["wide"]
    flat = s["before"].cpu().numpy().copy()
    t, refs = flat[: n * wide].reshape(n, wide), flat[n * wide:]
    if c["op"] == "fork":
        old = t.copy()
        for b, p in enumerate(parents(c)):
            t[b] = -1 if p < 0 else old[p]
        refs = np.bincount(t[t >= 0], minlength=len(refs))
        return [t, refs]
    pools = s["pools"].clone()
    if c["op"] == "reserve":
        free = [i for i in range(len(refs)) if refs[i] == 0]
        for b in range(n):
            j = family_prompt(c, b // c["fan"]) // c["page"]
            e = t[b, j]
            if e >= 0 and refs[e] == 1:
                continue
            p = free.pop(0)
            if e >= 0:
                pools[:, p] = s["pools"][:, e]
                refs[e] -= 1
            t[b, j], refs[p] = p, 1
        return [t, refs, np.zeros(1, np.int32), pools]
    n_live = int((refs > 0).sum())
    holes = [i for i in range(n_live) if refs[i] == 0]
    moved = {}
    for p in range(n_live, len(refs)):
        if refs[p] > 0:
            moved[p] = holes.pop(0)
            pools[:, moved[p]] = s["pools"][:, p]
            refs[moved[p]], refs[p] = refs[p], 0
    t = np.array([[moved.get(x, x) for x in row] for row in t.tolist()], np.int32)
    return [t, refs, np.array([n_live], np.int32), pools]


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "decode":
        return exact_decode(c, s)
    if c["op"] == "append":
        got = []
        for x in ("k", "v"):
            v = torch.cat([exact_row_values(p, c["dh"]) for p in s[x].view(s["rows"], c["hkv"], c["dh"]).split(8192)])
            v[s["pos"] < 0] = 0
            got.append(v.flatten(1))
        return got
    return exact_pages(c, s)
