"""Operators of the 8-bit key-value cache, as a serving program calls them: what is timed, and with what inputs.

The cache holds pages of 256 tokens: codes [pages][layers][K, V][kv heads][256][head dim] in 8 bits (e4m3 or int8), one fp32
scale per (token, kv head) of K and of V, and for every block of `block` tokens the per-channel bounds of its keys.  A conversation
slot owns a list of page ids.  A case names one of four uses:

  store   the rows of some tokens go into the cache (quantised, bounds of their blocks renewed) and are read back
  attend  attention of one new token per row over all of its slot's tokens
  pick    the blocks of a row's context that a cheap score selects, per kv head
  blocks  attention of one new token per row over given blocks

`run` with `own` calls the framework; without it, it computes the same from elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 256
LARGEST = {"e4m3": 448.0, "int8": 127.0}  # of a code
TINY = 2.0 ** -100                        # rows whose largest value is below this are stored as zeros
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, kind, rows, lo, hi, qh=16, kvh=2, hd=256, fmt="e4m3", dtype="fp16", block=64, **more):
    c = dict(kind=kind, rows=rows, lo=lo, hi=hi, qh=qh, kvh=kvh, hd=hd, fmt=fmt, dtype=dtype, block=block, **more)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # a decode step of 16 conversations appends one token each
        _case("store_step_16rows", "store", 16, 1000, 8000, prompt=0),
        # a page of text as a prompt, into an empty slot of a model with more kv heads
        _case("store_prompt_419", "store", 419, 0, 0, 32, 8, 128, "int8", "bf16", 32, prompt=1),
        # a full piece of a long prompt
        _case("store_piece_1024", "store", 1024, 7000, 7000, prompt=1),
        # one user, the first words: launches are everything
        _case("attend_1row_100", "attend", 1, 100, 100, gate=0, idle=0),
        # one user with a long document
        _case("attend_1row_48000", "attend", 1, 48000, 48000, gate=1, idle=0),
        # the benchmark's load: 16 ragged slots of 1K to 48K tokens, gated as the model's attention is
        _case("attend_16rows_e4m3", "attend", 16, 1024, 49152, gate=1, idle=0),
        # a full server of another head layout in int8; some rows are empty or not in use
        _case("attend_64rows_int8", "attend", 64, 256, 4096, 32, 8, 128, "int8", "bf16", gate=0, idle=1),
        # a small model without shared kv heads
        _case("attend_23rows_mha", "attend", 23, 40, 3001, 6, 6, 64, "int8", "fp16", gate=0, idle=1),
        # one user with a long document looks for 32 blocks
        _case("pick_1row_48000", "pick", 1, 48000, 48000, count=32, first=1, last=2),
        # a loaded server with small blocks
        _case("pick_16rows", "pick", 16, 4096, 49152, block=16, count=128, first=1, last=4),
        # the benchmark's load over 2048 tokens each instead of the whole context
        _case("blocks_16rows", "blocks", 16, 4096, 49152, gate=1, count=32),
        # one user, ten query heads per kv head, small blocks in int8
        _case("blocks_1row_int8", "blocks", 1, 20000, 20000, 20, 2, 128, "int8", "bf16", 16, gate=0, count=100),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "pick", "blocks"])
    hd = rng.choice([64, 128, 256])
    kvh = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 6, 7, 8, 8, 8, 12, 16])
    fmt, dtype, block = rng.choice(["e4m3", "int8"]), rng.choice(["fp16", "bf16"]), rng.choice([16, 32, 64, 128, 256])
    if kind == "store":
        prompt = rng.randint(0, 1)
        rows = _log_int(rng, 1, 1024 if prompt else 64)
        while rows * kvh * hd > 1024 * 2 * 256 or rows * kvh * hd * block > 1024 * 2 * 256 * 64:
            rows = max(1, rows // 2)
            if rows == 1:
                break
        at = _log_int(rng, 1, 20000) - 1
        return _case(None, kind, rows, at, at if prompt else at + _log_int(rng, 1, 8000), kvh * group, kvh, hd, fmt, dtype, block, prompt=prompt)
    rows = _log_int(rng, 1, 64)
    most = max(64, min(60000, 200_000 * 512 // (rows * kvh * hd)))  # keeps a case below the largest listed one
    lo = _log_int(rng, 1, most)
    hi = max(lo, _log_int(rng, max(1, most // 20), most))
    more = {}
    if kind in ("attend", "blocks"):
        more["gate"] = rng.randint(0, 1)
    if kind == "attend":
        more["idle"] = rng.randint(0, 1)
    if kind in ("pick", "blocks"):
        more["count"] = min(_log_int(rng, 4, 512), max(4, 4096 // block), -(-hi // block) + 3)
    if kind == "pick":
        more["first"], more["last"] = rng.randint(0, 1), rng.randint(0, 2)
    return _case(None, kind, rows, lo, hi, kvh * group, kvh, hd, fmt, dtype, block, **more)


# ---------------------------------------------------------------------------------------------- inputs
def _lengths(case, gen):
    n = case["rows"]
    if n == 1:
        return torch.tensor([case["hi"]])
    u = (torch.randperm(n, generator=gen) + torch.rand(n, generator=gen)) / n  # one from each of n equal parts of the log range
    lo, hi = max(1, case["lo"]), max(1, case["hi"])
    return (lo * (hi / lo) ** u.double()).round().long().clamp(lo, hi)


def _quantise(x, fmt):
    """[..., hd] in fp32 -> codes (bytes) and the scale of every row."""
    top = torch.tensor(LARGEST[fmt], device=x.device)
    a = x.abs().amax(-1)
    inv = torch.where(a < TINY, torch.zeros_like(a), torch.div(top.expand_as(a), a))
    scale = torch.where(a < TINY, torch.zeros_like(a), torch.div(a, top.expand_as(a)))
    y = (x * inv[..., None]).clamp(-LARGEST[fmt], LARGEST[fmt])
    y = y.to(torch.float8_e4m3fn) if fmt == "e4m3" else y.round().to(torch.int8)
    return y.view(torch.uint8), scale


def _values(codes, fmt):
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float()


def _bounds_of(k):
    """[..., tokens, hd] keys in fp32, NaN where a token is not counted -> lo8, hi8, scale of the block."""
    gone = k.isnan()
    lo = torch.where(gone, torch.full_like(k, math.inf), k).amin(-2)
    hi = torch.where(gone, torch.full_like(k, -math.inf), k).amax(-2)
    b = torch.maximum(lo.abs(), hi.abs()).amax(-1)
    f = torch.full_like(b, 127.0)
    inv = torch.where(b < TINY, torch.zeros_like(b), torch.div(f, b))
    lo8 = torch.floor(lo * inv[..., None]).clamp_min(-127).to(torch.int8)
    hi8 = torch.ceil(hi * inv[..., None]).clamp_max(127).to(torch.int8)
    return lo8, hi8, torch.where(b < TINY, torch.zeros_like(b), torch.div(b, f))


def _fill(codes, scales, bounds, fmt, block, dev, gen):
    """A cache whose keys drift from block to block, as those of a text do."""
    pages, _, _, kvh, _, hd = codes.shape
    step = max(1, (1 << 27) // (kvh * PAGE * hd))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        k = torch.randn(n, kvh, PAGE // block, block, hd, device=dev, generator=gen)
        k += 0.7 * torch.randn(n, kvh, PAGE // block, 1, hd, device=dev, generator=gen)
        c, s = _quantise(k, fmt)
        codes[p:p + n, :, 0] = c.view(n, 1, kvh, PAGE, hd)
        scales[p:p + n, :, 0] = s.view(n, 1, kvh, PAGE)
        lo8, hi8, sb = _bounds_of(_values(c, fmt) * s[..., None])
        bounds[p:p + n, :, :, :, :hd] = lo8.view(torch.uint8)[:, None]
        bounds[p:p + n, :, :, :, hd:2 * hd] = hi8.view(torch.uint8)[:, None]
        bounds[p:p + n, :, :, :, 2 * hd:2 * hd + 4].view(torch.float32)[..., 0] = sb[:, None]
        v = torch.randn(n, kvh, PAGE, hd, device=dev, generator=gen) * (0.3 + torch.rand(n, kvh, PAGE, 1, device=dev, generator=gen))
        c, s = _quantise(v, fmt)
        codes[p:p + n, :, 1] = c[:, None]
        scales[p:p + n, :, 1] = s[:, None]


def prepare(case, seed):
    dev = torch.device("cuda")
    gc = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    n, kvh, qh, hd, block, dt = case["rows"], case["kvh"], case["qh"], case["hd"], case["block"], TYPES[case["dtype"]]
    lens = _lengths(case, gc)
    if case["kind"] == "store" and case["prompt"]:  # rows of one slot, newest first as the engine keeps a piece
        slots, pos = torch.zeros(n, dtype=torch.long), case["lo"] + torch.arange(n - 1, -1, -1)
        ctx = torch.tensor([case["lo"] + n])
    else:
        slots = torch.randperm(n + 2, generator=gc)[:n]
        pos = lens.clone() - 1
        ctx = torch.zeros(n + 2, dtype=torch.long)
        ctx[slots] = lens
    if case.get("idle") and n > 4:  # an empty conversation, rows that are not in use, and one of a single token
        lens[1], lens[n // 2] = 0, 1
        slots[n - 2:] = -1
    need = (ctx + PAGE - 1) // PAGE
    hi = max(1, case["hi"])
    room = n if case["kind"] == "store" and case["prompt"] else 0  # pages for the longest context of each of the n parts, whatever the seed
    pages = (hi + room) // PAGE + 2 if room or n == 1 else sum(int(max(1, case["lo"]) ** (1 - i / n) * hi ** (i / n)) // PAGE + 2 for i in range(1, n + 1))
    most = (hi + room) // PAGE + 2
    table = torch.full((len(ctx), most), -1, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=gc).int(), 0
    for s, k in enumerate(need.tolist()):
        table[s, :k] = order[at:at + k]
        at += k
    st = dict(case=case, slots=slots.int().to(dev), pos=pos.int().to(dev), lens=lens.int().to(dev), table=table.to(dev), max_len=max(1, int(lens.max())))
    st["codes"] = torch.zeros(pages, 1, 2, kvh, PAGE, hd, dtype=torch.uint8, device=dev)
    st["scales"] = torch.zeros(pages, 1, 2, kvh, PAGE, device=dev)
    st["bounds"] = torch.zeros(pages, 1, kvh, PAGE // block, 2 * hd + 16, dtype=torch.uint8, device=dev)
    _fill(st["codes"], st["scales"], st["bounds"], case["fmt"], block, dev, gen)
    if case["kind"] == "store":
        st["k"], st["v"] = (torch.randn(n, kvh, hd, device=dev, generator=gen).to(dt) for _ in range(2))
        st["ko"], st["vo"] = torch.zeros_like(st["k"]), torch.zeros_like(st["v"])
    else:
        st["q"] = (1.5 * torch.randn(n, qh, hd, device=dev, generator=gen)).to(dt)
        st["y"] = torch.randn(n, qh, hd, device=dev, generator=gen).to(dt)
        st["gate"] = torch.randn(n, qh, hd, device=dev, generator=gen).to(dt) if case.get("gate") else None
    if case["kind"] in ("pick", "blocks"):
        st["ids"] = torch.full((n, kvh, case["count"]), -1, dtype=torch.int32, device=dev)
    if case["kind"] == "blocks":  # a random choice, with the newest block always in it
        nb = (lens + block - 1) // block
        key = torch.rand(n, kvh, int(nb.max()), generator=gc)
        idx = torch.arange(int(nb.max()))
        key[(idx >= nb[:, None])[:, None].expand_as(key)] = -1
        key[(idx == nb[:, None] - 1)[:, None].expand_as(key)] = 2
        k = min(case["count"], int(nb.max()))
        val, ids = key.topk(k, -1)
        ids = torch.where(val < 0, torch.full_like(ids, 1 << 30), ids).sort(-1).values
        st["ids"][:, :, :k] = torch.where(ids == 1 << 30, torch.full_like(ids, -1), ids).int().to(dev)
    if own:  # the handle and the workspace, which a server makes once
        from qwental_b200.kv8 import Kv8Cache
        st["cache"] = Kv8Cache(st["codes"], st["scales"], st["table"], st["bounds"], format=case["fmt"])
        st["work"] = torch.empty(st["cache"].work_bytes(n, qh, st["max_len"]), dtype=torch.uint8, device=dev)
    return st


# ---------------------------------------------------------------------------------------------- one pass
def run(st):
    kind = st["case"]["kind"]
    if own:
        c = st["cache"]
        if kind == "store":
            c.put(st["k"], st["v"], st["slots"], st["pos"])
            c.get(st["ko"], st["vo"], st["slots"], st["pos"])
            return _stored(st, st["ko"], st["vo"])
        if kind == "attend":
            c.attn(st["q"], st["lens"], st["slots"], st["y"], max_len=st["max_len"], gate=st["gate"], work=st["work"])
            return st["y"]
        if kind == "pick":
            c.pick(st["q"], st["lens"], st["slots"], st["ids"], max_len=st["max_len"], first=st["case"]["first"], last=st["case"]["last"], work=st["work"])
            return st["ids"]
        c.attn(st["q"], st["lens"], st["slots"], st["y"], max_len=st["max_len"], gate=st["gate"], blocks=st["ids"], work=st["work"])
        return st["y"]
    return {"store": _store, "attend": _attend, "pick": _pick, "blocks": _blocks}[kind](st)


def _stored(st, k, v):
    hd = st["case"]["hd"]
    return dict(k=k, v=v, scales=st["scales"], lo_hi=st["bounds"][..., :2 * hd].view(torch.int8), bound=st["bounds"][..., 2 * hd:2 * hd + 4].view(torch.float32))


def _store(st):
    case, codes, scales, bounds = st["case"], st["codes"], st["scales"], st["bounds"]
    fmt, block, hd, kvh = case["fmt"], case["block"], case["hd"], case["kvh"]
    slots, pos = st["slots"].long(), st["pos"].long()
    page, off = st["table"][slots, pos // PAGE].long(), pos % PAGE
    for kv, x in ((0, st["k"]), (1, st["v"])):
        c, s = _quantise(x.float(), fmt)
        codes[page, 0, kv, :, off] = c
        scales[page, 0, kv, :, off] = s
    # bounds of the blocks that got rows, over their tokens up to the newest one written
    b, sub = pos // block, off // block
    newest = torch.where((slots[:, None] == slots) & (b[:, None] == b), pos, torch.zeros_like(pos)).amax(1) % block
    h = torch.arange(kvh, device=pos.device)
    kc = codes.view(-1, 1, 2, kvh, PAGE // block, block, hd)[page[:, None], 0, 0, h, sub[:, None]]
    ks = scales.view(-1, 1, 2, kvh, PAGE // block, block)[page[:, None], 0, 0, h, sub[:, None]]
    k = _values(kc, fmt) * ks[..., None]
    k = torch.where((torch.arange(block, device=pos.device) > newest[:, None])[:, None, :, None], torch.full_like(k, math.nan), k)
    lo8, hi8, sb = _bounds_of(k)
    bounds[page, 0, :, sub] = torch.cat([lo8.view(torch.uint8), hi8.view(torch.uint8), sb[..., None].contiguous().view(torch.uint8),
                                         torch.zeros(*sb.shape, 12, dtype=torch.uint8, device=pos.device)], -1)
    kv = [(_values(codes[page, 0, i, :, off], fmt) * scales[page, 0, i, :, off][..., None]).to(st["k"].dtype) for i in (0, 1)]
    return _stored(st, *kv)


def _softmax_av(st, q, k, v, valid):
    """q [n, kvh, G, hd], k and v [n, kvh, T, hd], valid [n, kvh, T] -> rows as the program's buffer holds them."""
    s = torch.matmul(q, k.transpose(-1, -2)) * q.shape[-1] ** -0.5
    s = torch.where(valid[:, :, None], s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = torch.where(valid.any(-1)[:, :, None, None], o, torch.zeros_like(o)).reshape(q.shape[0], -1, q.shape[-1])
    if st["gate"] is not None:
        o = o / (1 + torch.exp(-st["gate"].float()))
    return torch.where((st["slots"] >= 0)[:, None, None], o.to(st["y"].dtype), st["y"])


def _split_heads(st):
    q = st["q"].float()
    return q.view(q.shape[0], st["case"]["kvh"], -1, q.shape[-1])


def _attend(st):
    case, fmt = st["case"], st["case"]["fmt"]
    pages = (st["max_len"] + PAGE - 1) // PAGE
    page = st["table"][st["slots"].clamp_min(0).long(), :pages].clamp_min(0).long()
    n, kvh, hd = case["rows"], case["kvh"], case["hd"]
    kv = [(_values(st["codes"][page, 0, i], fmt) * st["scales"][page, 0, i][..., None]).transpose(1, 2).reshape(n, kvh, pages * PAGE, hd) for i in (0, 1)]
    valid = (torch.arange(pages * PAGE, device=page.device) < st["lens"][:, None])[:, None].expand(n, kvh, -1)
    return _softmax_av(st, _split_heads(st), kv[0], kv[1], valid)


def _blocks(st):
    case, fmt, block = st["case"], st["case"]["fmt"], st["case"]["block"]
    n, kvh, hd, per = case["rows"], case["kvh"], case["hd"], PAGE // block
    ids = st["ids"].long()
    b = ids.clamp_min(0)
    page = torch.gather(st["table"][st["slots"].clamp_min(0).long()], 1, (b // per).view(n, -1)).view_as(b).clamp_min(0).long()
    h = torch.arange(kvh, device=b.device)[:, None]
    kv = []
    for i in (0, 1):
        c = st["codes"].view(-1, 1, 2, kvh, per, block, hd)[page, 0, i, h, b % per]
        s = st["scales"].view(-1, 1, 2, kvh, per, block)[page, 0, i, h, b % per]
        kv.append((_values(c, fmt) * s[..., None]).view(n, kvh, -1, hd))
    valid = (ids >= 0)[..., None] & (b[..., None] * block + torch.arange(block, device=b.device) < st["lens"][:, None, None, None])
    return _softmax_av(st, _split_heads(st), kv[0], kv[1], valid.view(n, kvh, -1))


def _pick(st):
    case, block, hd, kvh = st["case"], st["case"]["block"], st["case"]["hd"], st["case"]["kvh"]
    per, most = PAGE // block, (st["max_len"] + block - 1) // block
    q = _split_heads(st)
    a = q.abs().amax(-1)
    f = torch.full_like(a, 127.0)
    none = (a < TINY) | ~a.isfinite()
    q8 = (q * torch.where(none, torch.zeros_like(a), torch.div(f, a))[..., None]).round()
    sq = torch.where(none, torch.zeros_like(a), torch.div(a, f))
    blk = torch.arange(most, device=q.device)
    page = st["table"][st["slots"].clamp_min(0).long()][:, blk // per].clamp_min(0).long()
    rec = st["bounds"][page, 0, :, blk % per].transpose(1, 2)  # [n, kvh, blocks, record]
    lo, hi = rec[..., :hd].contiguous().view(torch.int8).float(), rec[..., hd:2 * hd].contiguous().view(torch.int8).float()
    sb = rec[..., 2 * hd:2 * hd + 4].contiguous().view(torch.float32)[..., 0]
    # sums of whole numbers below 2^24: exact in fp32
    i = torch.matmul(q8.clamp_min(0), hi.transpose(-1, -2)) + torch.matmul(q8.clamp_max(0), lo.transpose(-1, -2))
    s = torch.where(i == 0, i, (sq[..., None] * sb[:, :, None]) * i)
    s = torch.where(sb[:, :, None] == math.inf, torch.full_like(s, math.inf), s).amax(2)
    nblk = ((st["lens"] + block - 1) // block)[:, None, None]
    forced = (blk < case["first"]) | (blk >= nblk - case["last"])
    rank = torch.where(blk >= nblk, 0, torch.where(forced, 2, 1))  # by class first, then by score, then by index
    order = s.sort(dim=-1, descending=True, stable=True).indices
    order = torch.gather(order, -1, torch.gather(rank.expand_as(s), -1, order).sort(dim=-1, descending=True, stable=True).indices)[..., :case["count"]]
    ids = torch.where(order < nblk, order, torch.full_like(order, 1 << 30)).sort(-1).values
    ids = torch.where(ids == 1 << 30, torch.full_like(ids, -1), ids).int()
    out = torch.full_like(st["ids"], -1)
    out[..., :ids.shape[-1]] = ids
    return torch.where((st["slots"] >= 0)[:, None, None], out, st["ids"])


# ---------------------------------------------------------------------------------------------- work and definition
def work(case):
    n, kvh, qh, hd, block = case["rows"], case["kvh"], case["qh"], case["hd"], case["block"]
    if case["kind"] == "store":
        codes = n * kvh * 2 * (hd + 4)
        touched = -(-n // block) + 1 if case["prompt"] else n
        return dict(bytes=n * kvh * 2 * hd * 2 * 2 + 2 * codes + touched * kvh * (block * (hd + 4) / (1 if case["prompt"] else 2) + 2 * hd + 4), flops=n * kvh * 2 * hd * 6)
    lens = _lengths(case, torch.Generator().manual_seed(0)).double()
    rows = n * qh * hd * 2 * (3 if case.get("gate") else 2)
    if case["kind"] == "pick":
        blocks = float((lens / block).ceil().sum())
        return dict(bytes=blocks * kvh * (2 * hd + 4) + rows / 2 + n * kvh * case["count"] * 4, flops=blocks * qh * 4 * hd)
    tokens = float(lens.sum()) if case["kind"] == "attend" else float(torch.minimum(lens, torch.tensor(float(case["count"] * block))).sum())
    return dict(bytes=tokens * kvh * 2 * (hd + 4) + rows, flops=tokens * qh * hd * 4)


def _decode64(codes, scales, fmt):
    b = codes.long()
    if fmt == "int8":
        v = torch.where(b > 127, b - 256, b).double()
    else:  # sign, 4 bits of exponent (bias 7), 3 bits of mantissa
        e, m = (b >> 3) & 15, (b & 7).double()
        v = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e.double() - 7))
        v = torch.where(b > 127, -v, v)
    return v * scales.double()[..., None]


def _nearest64(x, fmt):
    """The value of the nearest code, ties to even, for |x| up to the largest."""
    if fmt == "int8":
        return x.round()
    step = 2.0 ** (torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (x / step).round() * step


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "store":
        got = []
        for x in (st["k"].double(), st["v"].double()):
            s = x.abs().amax(-1, keepdim=True) / LARGEST[case["fmt"]]
            got.append(torch.where(s > 0, _nearest64(x / s.clamp_min(1e-300), case["fmt"]) * s, torch.zeros_like(x)))
        return dict(k=got[0], v=got[1], scales=None, lo_hi=None, bound=None)
    if case["kind"] == "pick":
        return None  # whole numbers
    n, kvh, qh, hd, block = case["rows"], case["kvh"], case["qh"], case["hd"], case["block"]
    y = st["y"].double().clone()
    lens, slots = st["lens"].tolist(), st["slots"].tolist()
    for r in range(n):
        if slots[r] < 0:
            continue
        y[r] = 0
        if lens[r] <= 0:
            continue
        pg = st["table"][slots[r], :(lens[r] + PAGE - 1) // PAGE].long()
        for h in range(kvh):
            k, v = (_decode64(st["codes"][pg, 0, i, h].reshape(-1, hd)[:lens[r]], st["scales"][pg, 0, i, h].reshape(-1)[:lens[r]], case["fmt"]) for i in (0, 1))
            if case["kind"] == "blocks":
                ids = [b for b in st["ids"][r, h].tolist() if b >= 0]
                t = torch.cat([torch.arange(b * block, min(lens[r], (b + 1) * block)) for b in ids]).to(k.device)
                k, v = k[t], v[t]
            g = slice(h * (qh // kvh), (h + 1) * (qh // kvh))
            y[r, g] = torch.softmax(st["q"][r, g].double() @ k.T / math.sqrt(hd), -1) @ v
        if st["gate"] is not None:
            y[r] *= torch.sigmoid(st["gate"][r].double())
    return y
