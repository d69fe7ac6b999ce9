"""The 8-bit key-value cache on the GPU against plain numpy statements (tests/kv8_ref.py): stored codes, scales, bounds and chosen blocks bit for bit,
attention against 64 bits within what its roundings allow; rows that are empty, not in use, out of the cache; strides; streams, graphs, batches."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from qwental_b200 import kv8  # noqa: E402
from tests import kv8_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
PAGE = 256
NP = {torch.float16: np.float16}


def host(t):
    return t.float().cpu().numpy() if t.dtype == torch.bfloat16 else t.cpu().numpy()


class Rig:
    """A cache of random pages for slots of the given lengths, as tensors and as numpy arrays.  Page entries past a slot's tokens name no page, rows
    past its last token hold codes that are no numbers and scales that are NaN."""

    def __init__(self, lens, kvh=2, hd=256, fmt="e4m3", block=64, layers=2, layer=1, seed=0, spare=1):
        rng = np.random.default_rng(seed)
        self.rng, self.kvh, self.hd, self.fmt, self.block, self.layer = rng, kvh, hd, fmt, block, layer
        n = len(lens)
        self.lens = np.asarray(lens, np.int32)
        need = [(max(0, x) + PAGE - 1) // PAGE for x in lens]
        pages, self.max_pages = sum(need) + spare, max(need) + 1
        self.slots = rng.permutation(n + 2)[:n].astype(np.int32)
        self.table = np.full((n + 2, self.max_pages), -7, np.int32)
        order = rng.permutation(pages)
        at = 0
        for i, k in enumerate(need):
            self.table[self.slots[i], :k] = order[at:at + k]
            at += k
        codes = rng.integers(0, 256, (pages, layers, 2, kvh, PAGE, hd), np.uint8)
        if fmt == "e4m3":
            codes[(codes & 0x7f) == 0x7f] = 0x3c
        else:
            codes[codes == 0x80] = 5
        scales = (rng.uniform(0.2, 1, (pages, layers, 2, kvh, PAGE)) * (1 / 200 if fmt == "e4m3" else 1 / 70)).astype(np.float32)
        for i, x in enumerate(lens):
            if x > 0 and x % PAGE:
                p = self.table[self.slots[i], need[i] - 1]
                codes[p, :, :, :, x % PAGE:] = 0xff
                scales[p, :, :, :, x % PAGE:] = np.nan
        self.codes, self.scales = codes, scales
        self.bounds = np.zeros((pages, layers, kvh, PAGE // block, 2 * hd + 16), np.uint8)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        self.t = dict(codes=dev(codes), scales=dev(scales), bounds=dev(self.bounds), table=dev(self.table))
        self.cache = kv8.Kv8Cache(self.t["codes"], self.t["scales"], self.t["table"], self.t["bounds"], format=fmt, status=self.status)

    def kv(self, i, head, lens=None):
        """float64 keys and values of row i's slot"""
        n = int(self.lens[i] if lens is None else lens)
        pg = self.table[self.slots[i], :(n + PAGE - 1) // PAGE]
        return [ref.values(self.codes[pg, self.layer, j, head].reshape(-1, self.hd)[:n], self.fmt) *
                self.scales[pg, self.layer, j, head].reshape(-1)[:n, None].astype(np.float64) for j in (0, 1)]

    def fill_bounds(self):
        for i, n in enumerate(self.lens):
            for b in range((n + self.block - 1) // self.block):
                p, sub = self.table[self.slots[i], b * self.block // PAGE], b % (PAGE // self.block)
                m = min(self.block, n - b * self.block)
                rows = slice(sub * self.block, sub * self.block + m)
                for h in range(self.kvh):
                    lo, hi, s = ref.bounds(self.codes[p, self.layer, 0, h, rows], self.scales[p, self.layer, 0, h, rows], self.fmt)
                    self.bounds[p, self.layer, h, sub] = np.concatenate([lo.view(np.uint8), hi.view(np.uint8), s.reshape(1).view(np.uint8), np.zeros(12, np.uint8)])
        self.t["bounds"].copy_(torch.from_numpy(self.bounds))

    def idx(self, a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()

    def randn(self, *shape, dtype=torch.float16, scale=1.0):
        return torch.from_numpy((self.rng.standard_normal(shape) * scale).astype(np.float32)).to(dtype).cuda()


def check_attention(rig, q, y, dtype, gate=None, blocks=None, rows=None, scale=None, lens=None):
    """Every row of y against 64 bits."""
    G = q.shape[1] // rig.kvh
    qn, yn = host(q).astype(np.float64), host(y).astype(np.float64)
    gn = host(gate).astype(np.float64) if gate is not None else None
    half = torch.finfo(dtype).eps / 2
    for r in (range(len(rig.lens)) if rows is None else rows):
        for h in range(rig.kvh):
            k, v = rig.kv(r, h, None if lens is None else lens[r])
            if blocks is not None:
                n = len(k)
                t = np.concatenate([np.arange(b * rig.block, min(n, (b + 1) * rig.block)) for b in blocks[r, h] if b >= 0] + [np.zeros(0, int)]).astype(int)
                k, v = k[t], v[t]
            g = slice(h * G, (h + 1) * G)
            want, spread = ref.attend(qn[r, g], k, v, rig.hd ** -0.5 if scale is None else scale, None if gn is None else gn[r, g])
            tol = ref.tolerance(want, half, spread, np.abs(v).max() if len(v) else 0.0, rig.hd, max(1, len(k)))
            d = np.abs(yn[r, g] - want)
            assert (d <= tol).all(), (r, h, int(rig.lens[r]), float((d / tol).max()), float(d.max()))


# ------------------------------------------------------------------------------------------------ rows in and out
@pytest.mark.parametrize("hd,kvh,block", [(256, 2, 64), (128, 3, 16), (64, 1, 256), (64, 5, 32), (128, 8, 128)])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_go_in_bit_for_bit_and_come_back(hd, kvh, block, fmt, dtype):
    """One new token for some slots, then a run of rows of one slot, newest first: codes, scales, bounds, and nothing else changes."""
    rig = Rig([1, 700, 256, 64, 300, 17], kvh, hd, fmt, block, seed=hd + kvh)
    c, rng = rig.cache, rig.rng
    run = np.arange(299, 139, -1)
    for slots, pos in ((rig.slots, rig.lens - 1), (np.full(len(run), rig.slots[4]), run), (np.full(1, rig.slots[1]), np.array([3]))):
        n = len(slots)
        k, v = rig.randn(n, kvh, hd, dtype=dtype, scale=3.0), rig.randn(n, kvh, hd, dtype=dtype, scale=0.1)
        k[0, 0] = 0
        if n > 3:
            v[1, 0] = 0
            v[1, 0, 5] = -2.0
            k[2, kvh - 1, 1:] = 0
        c.put(k, v, rig.idx(slots), rig.idx(pos), layer=rig.layer)
        page, off = rig.table[slots, pos // PAGE], pos % PAGE
        for j, x in ((0, k), (1, v)):
            cc, ss = ref.quantise(host(x), fmt)
            for r in range(n):
                rig.codes[page[r], rig.layer, j, :, off[r]] = cc[r]
                rig.scales[page[r], rig.layer, j, :, off[r]] = ss[r]
        for r in range(n):
            if any(slots[i] == slots[r] and pos[i] // block == pos[r] // block and pos[i] > pos[r] for i in range(n)):
                continue
            first = off[r] // block * block
            for h in range(kvh):
                lo, hi, s = ref.bounds(rig.codes[page[r], rig.layer, 0, h, first:off[r] + 1], rig.scales[page[r], rig.layer, 0, h, first:off[r] + 1], fmt)
                rig.bounds[page[r], rig.layer, h, off[r] // block] = np.concatenate([lo.view(np.uint8), hi.view(np.uint8), s.reshape(1).view(np.uint8), np.zeros(12, np.uint8)])
        assert np.array_equal(rig.t["codes"].cpu().numpy(), rig.codes)
        assert np.array_equal(rig.t["scales"].cpu().numpy().view(np.uint32), rig.scales.view(np.uint32))
        assert np.array_equal(rig.t["bounds"].cpu().numpy(), rig.bounds)
        ko, vo = torch.zeros_like(k), torch.zeros_like(v)
        c.get(ko, vo, rig.idx(slots), rig.idx(pos), layer=rig.layer)
        for j, x in ((0, ko), (1, vo)):
            want = np.stack([ref.values(rig.codes[page[r], rig.layer, j, :, off[r]], fmt).astype(np.float32) * rig.scales[page[r], rig.layer, j, :, off[r], None] for r in range(n)])
            assert torch.equal(x.cpu(), torch.from_numpy(want).to(dtype))
    assert int(rig.status) == 0


def test_rows_that_hold_no_numbers_and_tiny_ones():
    """An infinity or a NaN makes its row NaN and the block's scale infinite; rows below 2^-100 are zeros."""
    rig = Rig([256], 2, 128, "int8", 64, layers=1, layer=0)
    n = 40
    k = rig.randn(n, 2, 128, dtype=torch.bfloat16)
    k[3, 0, 100] = float("inf")
    k[4, 0, 1] = float("nan")
    k[5] = 1e-38
    pos = np.arange(n)
    rig.cache.put(k, k.clone(), rig.idx(np.full(n, rig.slots[0])), rig.idx(pos))
    p = rig.table[rig.slots[0], 0]
    s = rig.t["scales"].cpu().numpy()[p, 0, 0]
    assert np.isnan(s[0, [3, 4]]).all() and (s[:, 5] == 0).all() and np.isfinite(s[1, :5]).all()
    b = rig.t["bounds"].cpu().numpy()[p, 0, :, 0, 256:260].copy().view(np.float32)[:, 0]
    assert np.isposinf(b[0]) and np.isfinite(b[1]) and b[1] > 0
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    rig.cache.get(ko, vo, rig.idx(np.full(n, rig.slots[0])), rig.idx(pos))
    assert ko[3, 0].isnan().all() and vo[4, 0].isnan().all() and (ko[5] == 0).all() and ko[3, 1].isfinite().all()
    # a slot of those 40 tokens: the head with the NaN rows is NaN, the other is not
    y = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device="cuda")
    rig.cache.attn(rig.randn(1, 4, 128, dtype=torch.bfloat16), rig.idx([40]), rig.idx(rig.slots), y, max_len=256)
    assert y[0, :2].isnan().all() and y[0, 2:].isfinite().all()
    rig.cache.attn(rig.randn(1, 4, 128, dtype=torch.bfloat16), rig.idx([3]), rig.idx(rig.slots), y, max_len=256)
    assert y.isfinite().all()


def test_the_later_of_two_rows_for_one_position_stays_and_unused_rows_are_passed_over():
    rig = Rig([300, 20], 2, 64, "e4m3", 16, layers=1, layer=0)
    s0, s1 = int(rig.slots[0]), int(rig.slots[1])
    slots = np.array([s0, s1, s0, -1, s0, s1, s0])
    pos = np.array([290, 7, 290, 5, -3, 7, 289])
    k, v = rig.randn(7, 2, 64), rig.randn(7, 2, 64)
    before = rig.t["codes"].clone()
    rig.cache.put(k, v, rig.idx(slots), rig.idx(pos))
    ko, vo = torch.full_like(k, 9.0), torch.full_like(k, 9.0)
    rig.cache.get(ko, vo, rig.idx(slots), rig.idx(pos))
    assert (ko[[3, 4]] == 9).all() and (vo[[3, 4]] == 9).all()
    assert torch.equal(ko[0], ko[2]) and torch.equal(ko[1], ko[5])
    for r in (2, 5, 6):
        cc, ss = ref.quantise(host(k[r]), "e4m3")
        assert np.array_equal(host(ko[r]), (ref.values(cc, "e4m3").astype(np.float32) * ss[:, None]).astype(np.float16))
    changed = (rig.t["codes"] != before).any(-1).sum().item()
    assert changed <= 3 * 2 * 2
    assert int(rig.status) == 0


@pytest.mark.parametrize("hd,kvh", [(64, 5), (128, 1), (256, 2)])
def test_a_cache_without_bounds_stores_the_same_codes(hd, kvh):
    rig = Rig([900, 70], kvh, hd, "int8", 64, layers=1, layer=0, seed=3)
    plain = kv8.Kv8Cache(rig.t["codes"].clone(), rig.t["scales"].clone(), rig.t["table"], format="int8", status=rig.status)
    s0, s1 = int(rig.slots[0]), int(rig.slots[1])
    slots = np.array([s0] * 600 + [s1] * 3 + [-1, s0, s0])
    pos = np.concatenate([np.arange(850, 250, -1), [0, 69, 0], [3, -1, 300]])  # (positions 0 and 300 twice)
    n = len(slots)
    k, v = rig.randn(n, kvh, hd, dtype=torch.bfloat16), rig.randn(n, kvh, hd, dtype=torch.bfloat16)
    for c in (rig.cache, plain):
        c.put(k, v, rig.idx(slots), rig.idx(pos))
    for a, b in zip(rig.cache.tensors[:2], plain.tensors[:2]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    cc, ss = ref.quantise(host(k), "int8")
    for r in (0, 599, 601, 602, n - 1):
        assert np.array_equal(plain.tensors[0].cpu().numpy()[rig.table[slots[r], pos[r] // PAGE], 0, 0, :, pos[r] % PAGE], cc[r])
    with pytest.raises(kv8.Kv8Error, match="bounds"):
        plain.pick(rig.randn(2, kvh, hd), rig.idx(rig.lens), rig.idx(rig.slots), torch.zeros(2, kvh, 3, dtype=torch.int32, device="cuda"), max_len=900)
    bad = rig.idx([99, s0])
    plain.put(k[:2].contiguous(), v[:2].contiguous(), bad, rig.idx([0, 10 ** 6]))
    assert int(rig.status) & 0xf00 == 0x200


@pytest.mark.parametrize("kvh,n", [(100, 300), (1, 256), (1, 257), (2, 128), (2, 129), (2, 1000), (300, 40)])
def test_many_rows_at_once_and_one_by_one(kvh, n):
    """Rows of several slots in mixed order, some for the same place, some not in use, in one call and one by one in the order of their positions: the same codes, scales and
    bounds, however the call shares them out (few or many rows for the heads); a captured call leaves the same when it is replayed with other rows."""
    block, slots, hd = 32, 5, 64
    rng = np.random.default_rng(n)
    cell = rng.permutation(slots * 256)[:n]
    sl, ps = (cell // 256).astype(np.int32), (cell % 256).astype(np.int32)
    sl[3::17], ps[5::19] = -1, -1
    ps[n // 2], sl[n // 2] = ps[0], sl[0]  # the same place twice
    x = [torch.from_numpy(rng.standard_normal((n, kvh, hd)).astype(np.float16)).cuda() for _ in range(2)]
    idx = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731

    def new():
        t = [torch.zeros(slots, 1, 2, kvh, PAGE, hd, dtype=torch.uint8, device="cuda"), torch.zeros(slots, 1, 2, kvh, PAGE, device="cuda"),
             torch.zeros(slots, 1, kvh, PAGE // block, 2 * hd + 16, dtype=torch.uint8, device="cuda")]
        return t, kv8.Kv8Cache(t[0], t[1], torch.arange(slots, dtype=torch.int32, device="cuda").view(slots, 1), t[2], format="int8")

    want, c = new()
    for i in sorted(range(n), key=lambda i: (ps[i], i)):
        c.put(x[0][i:i + 1], x[1][i:i + 1], idx(sl[i:i + 1]), idx(ps[i:i + 1]))
    got, c = new()
    c.put(x[0], x[1], idx(sl), idx(ps))
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    again, c = new()
    s, p, k, v = torch.full((n,), -1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros_like(x[0]), torch.zeros_like(x[1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.put(k, v, s, p)
    g.replay()  # no row is in use
    assert not any(t.any() for t in again)
    s.copy_(idx(sl)), p.copy_(idx(ps)), k.copy_(x[0]), v.copy_(x[1])
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(again, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_rows_outside_the_cache_are_dropped_and_reported():
    rig = Rig([300], 2, 128, "int8", 64, layers=1, layer=0)
    n_slots = rig.table.shape[0]
    s = int(rig.slots[0])
    free = int([i for i in range(n_slots) if i != s][0])  # its entries are -7
    for slot, p in ((n_slots, 0), (2 ** 31 - 1, 0), (s, rig.max_pages * PAGE), (s, 2 ** 31 - 1), (free, 0)):
        rig.status.zero_()
        before = [rig.t[x].clone() for x in ("codes", "scales", "bounds")]
        k = rig.randn(1, 2, 128)
        rig.cache.put(k, k, rig.idx([slot]), rig.idx([p]))
        assert int(rig.status) & 0xf00 == 0x200
        for a, b in zip(before, ("codes", "scales", "bounds")):
            assert torch.equal(a.view(torch.uint8), rig.t[b].view(torch.uint8))
        rig.status.zero_()
        ko = torch.zeros_like(k)
        vo = torch.zeros_like(k)
        rig.cache.get(ko, vo, rig.idx([slot]), rig.idx([p]))
        assert ko.isnan().all() and vo.isnan().all() and int(rig.status) & 0xf00 == 0x200


def test_a_full_piece_and_strided_rows():
    """1024 rows of two slots cut out of a wider tensor at an odd place, heads far apart."""
    rig = Rig([900, 900], 2, 256, "e4m3", 64, layers=1, layer=0)
    big = rig.randn(1024, 3, 2 * 256 + 1 + 256)
    k, v = big[:, 0:2, 1:257], big[:, 1:3, 513:769]
    slots = np.repeat(rig.slots, 512)
    pos = np.concatenate([np.arange(512), np.arange(300, 812)])
    perm = rig.rng.permutation(1024)
    rig.cache.put(k, v, rig.idx(slots[perm]), rig.idx(pos[perm]))
    for x, j in ((k, 0), (v, 1)):
        cc, ss = ref.quantise(host(x), "e4m3")
        page, off = rig.table[slots[perm], pos[perm] // PAGE], pos[perm] % PAGE
        assert np.array_equal(rig.t["codes"].cpu().numpy()[page, 0, j, :, off], cc)
        assert np.array_equal(rig.t["scales"].cpu().numpy()[page, 0, j, :, off], ss)
    out = torch.zeros(1024, 2, 2, 260, dtype=torch.float16, device="cuda")
    rig.cache.get(out[:, 0, :, 2:258], out[:, 1, :, 4:260], rig.idx(slots[perm]), rig.idx(pos[perm]))
    assert (out[:, 0, :, :2] == 0).all() and (out[:, 0, :, 258:] == 0).all() and (out[:, 1, :, :4] == 0).all()
    cc, ss = ref.quantise(host(k), "e4m3")
    assert np.array_equal(host(out[:, 0, :, 2:258]), (ref.values(cc, "e4m3").astype(np.float32) * ss[..., None]).astype(np.float16))


# ------------------------------------------------------------------------------------------------ attention
LENS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 512, 700, 1025, 2049, 3001]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("hd,kvh,G,dtype,gate", [(256, 2, 8, torch.float16, 1), (256, 1, 16, torch.bfloat16, 0), (256, 3, 1, torch.float16, 0), (128, 8, 4, torch.bfloat16, 0),
                                                 (128, 2, 10, torch.float16, 1), (128, 1, 9, torch.float16, 0), (64, 6, 1, torch.float16, 0), (64, 1, 7, torch.bfloat16, 1), (64, 2, 16, torch.float16, 0)])
def test_attention_over_all_tokens(hd, kvh, G, dtype, gate, fmt):
    rig = Rig(LENS, kvh, hd, fmt, seed=hd + G)
    n, qh = len(LENS), kvh * G
    q = rig.randn(n, qh, hd, dtype=dtype, scale=1.5)
    g = rig.randn(n, qh, hd, dtype=dtype) if gate else None
    y = torch.full_like(q, 7.0)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=rig.layer, max_len=3001, gate=g)
    check_attention(rig, q, y, dtype, g)
    assert (y[0] == 0).all() and int(rig.status) == 0


def test_one_long_row_and_many_short_ones():
    rig = Rig([48000], 2, 256, "e4m3", seed=3)
    q = rig.randn(1, 16, 256, scale=1.5)
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=48128)
    check_attention(rig, q, y, torch.float16)
    lens = np.random.default_rng(5).integers(0, 400, 200)
    rig = Rig(lens, 1, 64, "int8", seed=4)
    q = rig.randn(200, 4, 64)
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=400)
    check_attention(rig, q, y, torch.float16)


def test_many_rows_of_one_slot():
    """1024 rows, each over the slot's tokens up to its own position (a prompt's piece)."""
    rig = Rig([1100], 2, 128, "int8", layers=1, layer=0, seed=8)
    n = 1024
    lens = np.arange(n) + 50
    q = rig.randn(n, 4, 128)
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(lens), rig.idx(np.full(n, rig.slots[0])), y, max_len=1100)
    slot, rig.slots, rig.lens = rig.slots[0], np.full(n, rig.slots[0], np.int32), lens
    check_attention(rig, q, y, torch.float16, rows=[0, 1, 200, 206, 207, 461, 462, 1000, 1023])


@pytest.mark.parametrize("qs,vs,ks", [(1e4, 1.0, 1.0), (1e-6, 1.0, 1.0), (1.0, 1e-30, 1.0), (1.0, 1e30, 1e-20), (30.0, 1e-5, 5.0)])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attention_at_the_ends_of_the_ranges(qs, vs, ks, fmt):
    """Scales of values and keys far from 1 and far from one another (one token's values 2^-40 of the others'), queries of every size in bf16."""
    rig = Rig([300, 77], 1, 128, fmt, layers=1, layer=0, seed=6)
    rig.scales[:, :, 0] *= np.float32(ks)
    rig.scales[:, :, 1] *= np.float32(vs)
    rig.scales[:, :, 1, :, ::7] *= np.float32(2.0 ** -40)
    rig.scales[:, :, 1, :, 3] = 0
    rig.t["scales"].copy_(torch.from_numpy(rig.scales))
    q = rig.randn(2, 8, 128, dtype=torch.bfloat16, scale=qs)
    q[0, 2] = 0
    y = torch.zeros_like(q)
    sc = 0.05 / max(qs * ks, 1e-3)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=300, scale=sc)
    check_attention(rig, q, y, torch.bfloat16, scale=sc)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_query_that_holds_no_numbers_spoils_its_head_alone(bad):
    rig = Rig([300, 1], 2, 128, "e4m3", layers=1, layer=0, seed=12)
    rig.codes[:, :, 0] &= 0x7f  # keys of one sign: a query of -infinity has no score but -infinity
    rig.t["codes"].copy_(torch.from_numpy(rig.codes))
    q = rig.randn(2, 12, 128)
    q[0, 7, 5] = bad
    q[1, 0, 127] = bad
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=300)
    gone = torch.zeros(2, 12, dtype=torch.bool)
    gone[0, 7] = gone[1, 0] = True
    assert torch.equal(y.isnan().all(-1).cpu(), gone) and torch.equal(y.isnan().any(-1).cpu(), gone)


def test_a_single_token_that_wins_everything():
    """Scores far apart: the row is that token's value."""
    rig = Rig([500, 500], 1, 64, "int8", layers=1, layer=0, seed=9)
    q = rig.randn(2, 2, 64, scale=60.0)
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=500, scale=1.0)
    check_attention(rig, q, y, torch.float16, scale=1.0)


def test_a_row_is_the_same_alone_and_in_any_call():
    lens = [700, 5000, 31, 12000, 256, 0]
    for kvh, G, hd in ((2, 8, 256), (1, 5, 64)):
        rig = Rig(lens, kvh, hd, "e4m3", seed=77)
        q = rig.randn(len(lens), kvh * G, hd)
        y = torch.zeros_like(q)
        rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=12000)
        for rows in ([0], [1], [3], [4, 2], [3, 0, 5]):
            z = torch.zeros_like(q[rows])
            rig.cache.attn(q[rows], rig.idx(rig.lens[rows]), rig.idx(rig.slots[rows]), z, layer=1, max_len=int(max(lens[r] for r in rows)) + 1)
            assert torch.equal(z, y[rows])


def test_rows_not_in_use_stay_and_others_do_not_matter():
    rig = Rig([100, 200, 300, 400], 2, 128, "int8", seed=1)
    q = rig.randn(4, 8, 128)
    y = rig.randn(4, 8, 128)
    before = y.clone()
    slots, lens = rig.slots.copy(), rig.lens.copy()
    slots[1] = -1
    lens[2] = -5
    rig.cache.attn(q, rig.idx(lens), rig.idx(slots), y, layer=1, max_len=400)
    assert torch.equal(y[1], before[1]) and (y[2] == 0).all()
    check_attention(rig, q, y, torch.float16, rows=[0, 3])
    assert int(rig.status) == 0


def test_rows_outside_the_cache_are_nan_and_reported():
    rig = Rig([600, 600, 600, 600], 2, 64, "e4m3", seed=2)
    q = rig.randn(4, 4, 64)
    y = torch.zeros_like(q)
    table = rig.table.copy()
    table[rig.slots[1], 1] = rig.codes.shape[0]      # one page past the pool
    table[rig.slots[2], 0] = -1
    rig.t["table"].copy_(torch.from_numpy(table))
    slots = rig.slots.copy()
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(slots), y, layer=1, max_len=600)
    assert y[1].isnan().all() and y[2].isnan().all() and int(rig.status) & 0xf00 == 0x200
    check_attention(rig, q, y, torch.float16, rows=[0, 3])
    rig.t["table"].copy_(torch.from_numpy(rig.table))
    rig.status.zero_()
    slots[0] = 6      # no such slot
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(slots), y, layer=1, max_len=599)  # and every row is longer than the call allows
    assert y.isnan().all() and int(rig.status) & 0xf00 == 0x200


def test_strided_queries_gates_and_results():
    """Rows as slices of a projection's output: [q | gate] per head, heads in another order, odd places; the bytes around the results stay."""
    rig = Rig([0, 77, 700, 300], 2, 128, "int8", seed=4)
    x = rig.randn(4, 16, 2 * 128 + 3)
    q, gate = x[:, 8:, 1:129], x[:, 8:, 130:258]
    out = torch.full((4, 128 + 5, 8), 3.0, dtype=torch.float16, device="cuda")
    wide = torch.full((8, 4, 140), 3.0, dtype=torch.float16, device="cuda")
    y = wide.transpose(0, 1)[:, :, 7:135]
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=700, gate=gate)
    check_attention(rig, q, y, torch.float16, gate)
    assert (wide[:, :, :7] == 3).all() and (wide[:, :, 135:] == 3).all()
    flat = rig.randn(4 * 8 * 128 + 8)
    z = torch.zeros(4, 8, 128, dtype=torch.float16, device="cuda")
    q2 = flat[4:4 + 4 * 8 * 128].view(4, 8, 128)  # 8-byte aligned rows
    rig.cache.attn(q2, rig.idx(rig.lens), rig.idx(rig.slots), z, layer=1, max_len=700)
    check_attention(rig, q2, z, torch.float16)
    q3 = rig.randn(4, 1, 128).expand(4, 8, 128)  # one query for all heads
    rig.cache.attn(q3, rig.idx(rig.lens), rig.idx(rig.slots), z, layer=1, max_len=700)
    check_attention(rig, q3, z, torch.float16)
    del out


# ------------------------------------------------------------------------------------------------ chosen blocks
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("hd,kvh,G,block,count", [(256, 2, 8, 64, 12), (128, 1, 10, 16, 40), (64, 3, 2, 256, 3), (128, 2, 4, 32, 1), (256, 1, 1, 128, 30), (64, 2, 16, 16, 37)])
def test_attention_over_given_blocks(hd, kvh, G, block, count, fmt):
    lens = [1, 16, 17, 100, 256, 300, 700, 2000, 3001, 0]
    rig = Rig(lens, kvh, hd, fmt, block, seed=block + hd)
    rng = rig.rng
    blocks = np.full((len(lens), kvh, count), -1, np.int32)
    for r, n in enumerate(lens):
        nb = (n + block - 1) // block
        for h in range(kvh):
            k = min(nb, int(rng.integers(0, count + 1))) if (r + h) % 3 else min(nb, count)
            blocks[r, h, :k] = rng.permutation(nb)[:k] if h % 2 else np.sort(rng.permutation(nb)[:k])
    q = rig.randn(len(lens), kvh * G, hd, scale=1.5)
    y = torch.full_like(q, 7.0)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=3001, blocks=rig.idx(blocks))
    check_attention(rig, q, y, torch.float16, blocks=blocks)
    assert int(rig.status) == 0


def test_blocks_outside_a_row_are_nan_and_reported():
    rig = Rig([600, 600, 64], 1, 64, "e4m3", 32, seed=2)
    q = rig.randn(3, 4, 64)
    y = torch.zeros_like(q)
    blocks = np.array([[[0, 5, 19]], [[3, 2 ** 31 - 1, -1]], [[2, -1, -1]]], np.int32)  # the first of row 0: 600 tokens are blocks 0 to 18
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=600, blocks=rig.idx(blocks))
    assert y.isnan().all() and int(rig.status) & 0xf00 == 0x200


PICKS = [(256, 2, 8, 64, 12, 1, 2), (128, 1, 10, 16, 40, 0, 0), (64, 3, 2, 256, 3, 0, 1), (128, 2, 4, 32, 1, 0, 1), (256, 1, 1, 128, 30, 2, 2), (64, 2, 16, 16, 257, 1, 4)]


@pytest.mark.parametrize("hd,kvh,G,block,count,first,last", PICKS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_blocks_are_chosen_as_stated(hd, kvh, G, block, count, first, last, dtype):
    lens = [1, 16, 17, 100, 256, 300, 700, 2000, 5001, 0, 33]
    rig = Rig(lens, kvh, hd, "e4m3", block, seed=block + hd)
    rig.codes[:, :, 0] = np.where(rig.rng.random(rig.codes[:, :, 0].shape) < 0.3, rig.codes[:, :, 0], 0x18)  # keys that are alike: scores that are equal
    rig.fill_bounds()
    tie = rig.bounds[rig.table[rig.slots[8], 0]].copy()
    rig.bounds[rig.table[rig.slots[8], 3:9]] = tie  # six pages of the same blocks
    p = rig.table[rig.slots[7], 1]
    rig.bounds[p, 1, 0, 0, 2 * hd:2 * hd + 4] = np.float32(np.inf).reshape(1).view(np.uint8)  # a block with a row that holds no numbers
    rig.bounds[p, 1, 0, -1, 2 * hd:2 * hd + 4] = 0
    rig.t["bounds"].copy_(torch.from_numpy(rig.bounds))
    q = rig.randn(len(lens), kvh * G, hd, dtype=dtype, scale=2.0)
    q[3, 0] = 0
    q[4, 0, 3] = float("inf")
    q[5, G - 1] = 1e-3
    slots = rig.slots.copy()
    slots[10] = -1
    blocks = torch.full((len(lens), kvh, count), 77, dtype=torch.int32, device="cuda")
    rig.cache.pick(q, rig.idx(rig.lens), rig.idx(slots), blocks, layer=1, max_len=5001, first=first, last=last)
    got, qn = blocks.cpu().numpy(), host(q).astype(np.float32)
    assert (got[10] == 77).all()
    for r, n in enumerate(lens[:10]):
        nb = (n + block - 1) // block
        b = np.arange(nb)
        for h in range(kvh):
            recs = rig.bounds[rig.table[rig.slots[r], b * block // PAGE], 1, h, b % (PAGE // block)]
            want = ref.pick(qn[r, h * G:(h + 1) * G], recs, hd, nb, count, first, last) if nb else np.full(count, -1)
            assert np.array_equal(got[r, h], want), (r, h, n)
    assert int(rig.status) == 0


def test_choice_among_many_blocks_and_equal_ones():
    """60000 blocks of 16 tokens in a slot that uses few pages over and over: every score comes many times, the lowest numbers win."""
    rig = Rig([16 * 40], 1, 64, "int8", 16, layers=1, layer=0, seed=11)
    rig.fill_bounds()
    pages = rig.table[rig.slots[0], :2]
    n = 60000
    table = np.resize(pages, (rig.table.shape[0], n // 16 + 1)).astype(np.int32)
    c = kv8.Kv8Cache(rig.t["codes"], rig.t["scales"], torch.from_numpy(table).cuda(), rig.t["bounds"], format="int8", status=rig.status)
    q = rig.randn(1, 3, 64)
    recs = rig.bounds[table[0, np.arange(n) // 16], 0, 0, np.arange(n) % 16]
    for count in (1, 37, 1000, 5000):
        blocks = torch.zeros(1, 1, count, dtype=torch.int32, device="cuda")
        c.pick(q, rig.idx([n * 16 - 3]), rig.idx([0]), blocks, max_len=n * 16, first=1, last=0)
        assert np.array_equal(blocks.cpu().numpy()[0, 0], ref.pick(host(q)[0].astype(np.float32), recs, 64, n, count, 1, 0))


def test_choice_outside_the_cache_is_reported():
    rig = Rig([600, 600, 600], 1, 64, "e4m3", 32, seed=2)
    rig.fill_bounds()
    table = rig.table.copy()
    table[rig.slots[1], 1] = 10 ** 6
    rig.t["table"].copy_(torch.from_numpy(table))
    q = rig.randn(3, 2, 64)
    blocks = torch.full((3, 1, 30), 5, dtype=torch.int32, device="cuda")
    rig.cache.pick(q, rig.idx([600, 600, 700]), rig.idx(rig.slots), blocks, layer=1, max_len=600, last=0)
    got = blocks.cpu().numpy()[:, 0]
    assert np.array_equal(got[0], np.r_[np.arange(19), np.full(11, -1)]) and int(rig.status) & 0xf00 == 0x200
    assert np.array_equal(got[1], np.r_[np.arange(8), np.arange(16, 19), np.full(19, -1)]) and (got[2] == -1).all()


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("fmt,hd,G,block", [("e4m3", 256, 8, 64), ("int8", 128, 6, 16)])
def test_a_conversation(fmt, hd, G, block):
    """As a serving loop uses them: prompts in pieces, then steps of put, pick and attention over the choice; every step against 64 bits on the codes
    that are in the cache, and a choice of everything against attention over all tokens."""
    kvh, n = 2, 3
    prompts = [500, 130, 3]
    rig = Rig([700, 300, 200], kvh, hd, fmt, block, seed=21)
    rig.t["codes"].fill_(0xff)
    rig.t["scales"].fill_(float("nan"))
    c, slots = rig.cache, rig.idx(rig.slots)
    for i, m in enumerate(prompts):
        for a in range(0, m, 200):
            b = min(m, a + 200)
            k, v = rig.randn(b - a, kvh, hd), rig.randn(b - a, kvh, hd)
            c.put(k, v, rig.idx(np.full(b - a, rig.slots[i])), rig.idx(np.arange(a, b)), layer=1)
    lens = np.array(prompts)
    for step in range(40):
        k, v, q = rig.randn(n, kvh, hd), rig.randn(n, kvh, hd), rig.randn(n, kvh * G, hd, scale=1.5)
        c.put(k, v, slots, rig.idx(lens), layer=1)
        lens = lens + 1
        few = torch.empty(n, kvh, 6, dtype=torch.int32, device="cuda")
        c.pick(q, rig.idx(lens), slots, few, layer=1, max_len=700, first=1, last=1)
        y, all_y, full = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
        c.attn(q, rig.idx(lens), slots, y, layer=1, max_len=700, blocks=few)
        if step % 13:
            continue
        c.attn(q, rig.idx(lens), slots, all_y, layer=1, max_len=700)
        every = torch.empty(n, kvh, 700 // block + 1, dtype=torch.int32, device="cuda")
        c.pick(q, rig.idx(lens), slots, every, layer=1, max_len=700)
        c.attn(q, rig.idx(lens), slots, full, layer=1, max_len=700, blocks=every)
        rig.codes, rig.scales = rig.t["codes"].cpu().numpy(), rig.t["scales"].cpu().numpy()
        check_attention(rig, q, y, torch.float16, blocks=few.cpu().numpy(), lens=lens)
        check_attention(rig, q, all_y, torch.float16, lens=lens)
        check_attention(rig, q, full, torch.float16, lens=lens)
        rig.lens = lens.astype(np.int32)
        rig.fill_bounds()
        for r in range(n):
            nb = (int(lens[r]) + block - 1) // block
            b = np.arange(nb)
            for h in range(kvh):
                recs = rig.bounds[rig.table[rig.slots[r], b * block // PAGE], 1, h, b % (PAGE // block)]
                assert np.array_equal(few.cpu().numpy()[r, h], ref.pick(host(q)[r, h * G:(h + 1) * G].astype(np.float32), recs, hd, nb, 6, 1, 1))
    assert int(rig.status) == 0


def test_offsets_past_32_bits():
    """A pool of over 4 GB of codes: the last pages."""
    kvh, hd = 2, 256
    pages = (1 << 32) // (2 * kvh * PAGE * hd) + 40
    codes = torch.zeros(pages, 1, 2, kvh, PAGE, hd, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(pages, 1, 2, kvh, PAGE, device="cuda")
    bounds = torch.zeros(pages, 1, kvh, 4, 2 * hd + 16, dtype=torch.uint8, device="cuda")
    table = torch.arange(pages - 8, pages, dtype=torch.int32, device="cuda").flip(0).view(2, 4).contiguous()
    c = kv8.Kv8Cache(codes, scales, table, bounds, format="int8")
    rng = np.random.default_rng(0)
    n = 900
    x = [torch.from_numpy(rng.standard_normal((n, kvh, hd)).astype(np.float16)).cuda() for _ in range(2)]
    idx = lambda a: torch.from_numpy(np.asarray(a, np.int32)).cuda()  # noqa: E731
    c.put(x[0], x[1], idx([1] * n), idx(np.arange(n)))
    q = torch.from_numpy(rng.standard_normal((1, 16, hd)).astype(np.float16)).cuda()
    y = torch.zeros_like(q)
    c.attn(q, idx([n]), idx([1]), y, max_len=n)
    deq = []
    for t in x:
        cc, ss = ref.quantise(host(t), "int8")
        deq.append(ref.values(cc, "int8") * ss[..., None].astype(np.float64))
    for h in range(kvh):
        want, spread = ref.attend(host(q)[0, h * 8:h * 8 + 8].astype(np.float64), deq[0][:, h], deq[1][:, h], hd ** -0.5)
        assert (np.abs(host(y)[0, h * 8:h * 8 + 8] - want) <= ref.tolerance(want, 2.0 ** -11, spread, np.abs(deq[1][:, h]).max(), hd, n)).all()
    ids = torch.zeros(1, kvh, 20, dtype=torch.int32, device="cuda")
    c.pick(q, idx([n]), idx([1]), ids, max_len=n)
    assert np.array_equal(ids.cpu().numpy()[0, 0], np.r_[np.arange(15), np.full(5, -1)])
    assert not codes[:1000].any()


# ------------------------------------------------------------------------------------------------ streams, graphs, batches
def test_streams_and_captured_graphs():
    """Calls on two streams at once with workspaces of their own; a step captured once and replayed with other lengths, slots and rows, next to another graph."""
    rig = Rig([700, 300, 1500], 2, 256, "e4m3", seed=31)
    rig.fill_bounds()
    n, L = 3, rig.layer
    slots = rig.idx(rig.slots)
    q = [rig.randn(n, 16, 256) for _ in range(2)]
    lens = [rig.idx(rig.lens), rig.idx(rig.lens // 2)]
    want = []
    for i in range(2):
        y, ids = torch.zeros_like(q[i]), torch.zeros(n, 2, 5, dtype=torch.int32, device="cuda")
        rig.cache.pick(q[i], lens[i], slots, ids, layer=L, max_len=1500)
        rig.cache.attn(q[i], lens[i], slots, y, layer=L, max_len=1500, blocks=ids)
        want.append((y, ids))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    work = [torch.empty(rig.cache.work_bytes(n, 16, 1500), dtype=torch.uint8, device="cuda") for _ in range(2)]
    got = [(torch.zeros_like(q[i]), torch.zeros_like(want[i][1])) for i in range(2)]
    torch.cuda.synchronize()
    with pytest.raises(kv8.Kv8Error, match="workspace"):
        rig.cache.attn(q[0], lens[0], slots, got[0][0], layer=L, max_len=1500, stream=streams[0].cuda_stream)
    for _ in range(20):
        for i in range(2):
            rig.cache.pick(q[i], lens[i], slots, got[i][1], layer=L, max_len=1500, work=work[i], stream=streams[i].cuda_stream)
            rig.cache.attn(q[i], lens[i], slots, got[i][0], layer=L, max_len=1500, blocks=got[i][1], work=work[i], stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
    # graphs: one per workspace, replayed in turn on one stream
    graphs, qq, ll = [], [], []
    for i in range(2):
        qi, li = q[i].clone(), lens[i].clone()
        y, ids = got[i]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            rig.cache.pick(qi, li, slots, ids, layer=L, max_len=1500, work=work[0])
            rig.cache.attn(qi, li, slots, y, layer=L, max_len=1500, blocks=ids, work=work[0])
        graphs.append(g)
        qq.append(qi)
        ll.append(li)
    for swap in (0, 1):
        for i in range(2):
            qq[i].copy_(q[i ^ swap])
            ll[i].copy_(lens[i ^ swap])
            got[i][0].zero_()
        for i in range(2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], want[i ^ swap][0]) and torch.equal(got[i][1], want[i ^ swap][1])


def test_calls_of_few_and_of_many_rows_from_two_threads():
    """What a call needs of a kernel that another call uses too (its shared memory grows with the rows) does not depend on who comes last; the same for a
    captured call of many rows, replayed after a call of few."""
    import threading
    rig = Rig([300] * 64, 1, 64, "int8", seed=7)
    big = np.tile(np.arange(64), 16)
    lens, slots = rig.idx(rig.lens[big]), rig.idx(rig.slots[big])
    q = rig.randn(1024, 4, 64)
    want = torch.zeros_like(q)
    rig.cache.attn(q, lens, slots, want, layer=1, max_len=512)
    counts = (1024, 200)  # both of more tasks than the variant for few takes
    got = [torch.zeros_like(q) for _ in counts]
    work = [torch.empty(rig.cache.work_bytes(1024, 4, 512), dtype=torch.uint8, device="cuda") for _ in counts]
    streams = [torch.cuda.Stream() for _ in counts]
    graph, y = torch.cuda.CUDAGraph(), torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rig.cache.attn(q, lens, slots, y, layer=1, max_len=512)
    errors = []

    def run(i):
        try:
            n = counts[i]
            c = kv8.Kv8Cache(rig.t["codes"], rig.t["scales"], rig.t["table"], rig.t["bounds"], format="int8")
            for _ in range(200):
                c.attn(q[:n], lens[:n], slots[:n], got[i][:n], layer=1, max_len=512, work=work[i], stream=streams[i].cuda_stream)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    graph.replay()
    torch.cuda.synchronize()
    assert not errors, errors
    for g, n in list(zip(got, counts)) + [(y, 1024)]:
        assert torch.equal(g[:n], want[:n])


def test_buffers_of_other_places_are_refused():
    rig = Rig([100], 1, 64, "int8", layers=1, layer=0)
    a = kv8.RowsStruct()
    pinned = torch.zeros(1 << 12, dtype=torch.uint8)  # pageable host memory
    x = rig.randn(1, 1, 64)
    i = rig.idx([0])
    a.k, a.v, a.slots, a.pos, a.nb, a.k_row, a.k_head, a.v_row, a.v_head = pinned.data_ptr(), x.data_ptr(), i.data_ptr(), i.data_ptr(), 1, 64, 64, 64, 64
    err = C.create_string_buffer(256)
    L = kv8.bind()
    before = rig.t["codes"].clone()
    assert L.qw_kv8_put(C.byref(rig.cache.c), C.byref(a), None, err, 256) == -3 and b"not device memory" in err.value
    torch.cuda.synchronize()
    assert torch.equal(before, rig.t["codes"])


class View:
    """A torch tensor's memory as a buffer a batch can bind (an upload into a Buf, and back)."""

    def __init__(self, gpu, t):
        self.t, self.raw = t, t.contiguous().cpu().view(torch.uint8).numpy()
        self.buf = gpu.buf_from(self.raw.reshape(-1))

    def read(self):
        return torch.from_numpy(self.buf.download(np.uint8, self.raw.size)).view(self.t.dtype).reshape(self.t.shape)


@pytest.fixture(scope="module")
def gpu():
    from qwental_b200.gpu import Gpu
    g = Gpu()
    yield g
    g.close()


@pytest.mark.parametrize("graphs", [False, True])
def test_batches_give_the_same_bytes(gpu, graphs):
    """The families kv8_put, kv8_get, kv8_pick and kv8_attn in one batch, launched and replayed as a graph, against the calls on a stream."""
    from qwental_b200.gpu import GpuError
    rig = Rig([700, 300, 64], 2, 128, "int8", 32, seed=51)
    rig.fill_bounds()
    n, qh, L = 3, 12, rig.layer
    c = rig.cache
    k, v, q, gate = rig.randn(n, 2, 128), rig.randn(n, 2, 128), rig.randn(n, qh, 128), rig.randn(n, qh, 128)
    before = {x: View(gpu, rig.t[x]) for x in rig.t}
    slots, pos, lens = rig.idx(rig.slots), rig.idx(rig.lens - 1), rig.idx(rig.lens)
    ko, vo, y, ids = torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(q), torch.zeros(n, 2, 9, dtype=torch.int32, device="cuda")
    c.put(k, v, slots, pos, layer=L)
    c.get(ko, vo, slots, pos, layer=L)
    c.pick(q, lens, slots, ids, layer=L, max_len=700, first=1, last=1)
    c.attn(q, lens, slots, y, layer=L, max_len=700, gate=gate, blocks=ids)
    dense = torch.zeros_like(q)
    c.attn(q, lens, slots, dense, layer=L, max_len=700)
    B = {x: View(gpu, t) for x, t in dict(k=k, v=v, q=q, gate=gate, slots=slots, pos=pos, lens=lens, ko=torch.zeros_like(k), vo=torch.zeros_like(v), y=torch.zeros_like(q),
                                          dense=torch.zeros_like(q), ids=torch.zeros_like(ids)).items()}
    work = gpu.buf(c.work_bytes(n, qh, 700))
    fam = {f: gpu.compile(f, f + "_t") for f in ("kv8_put", "kv8_get", "kv8_pick", "kv8_attn")}

    def sizes(**over):
        s = kv8.SizesStruct(*[getattr(c.c, f) for f in ("pages", "layers", "kvh", "hd", "format", "block", "slots", "max_pages")], n, L, 0, qh, 700, 9, 1, 1, 128 ** -0.5)
        for f, x in over.items():
            setattr(s, f, x)
        return bytes(s)

    def rows(b, f, x, z, **over):
        b.kernel(fam[f]).buf(0, before["codes"].buf).buf(1, before["scales"].buf).buf(2, before["bounds"].buf).buf(3, before["table"].buf)
        b.buf(4, B[x].buf).buf(5, B[z].buf).buf(6, B["slots"].buf).buf(7, B["pos"].buf).bytes(8, np.array([256, 128, 256, 128], np.int64)).bytes(15, sizes(**over)).dispatch((1,), (1,))

    def attend(b, out, gated, **over):
        b = b.kernel(fam["kv8_attn"]).buf(0, before["codes"].buf).buf(1, before["scales"].buf).buf(3, before["table"].buf).buf(4, B["q"].buf)
        none = gpu_none()
        gpu.L.qw_batch_buf(b.b, 5, C.byref(B["gate"].buf.b) if gated else none, 0)
        gpu.L.qw_batch_buf(b.b, 9, C.byref(B["ids"].buf.b) if gated else none, 0)
        b.buf(6, B[out].buf).buf(7, B["lens"].buf).buf(8, B["slots"].buf).buf(10, work).bytes(11, np.array([qh * 128, 128] * 3, np.int64)).bytes(15, sizes(**over)).dispatch((1,), (1,))

    def choose(b, **over):
        b.kernel(fam["kv8_pick"]).buf(0, before["codes"].buf).buf(1, before["scales"].buf).buf(2, before["bounds"].buf).buf(3, before["table"].buf).buf(4, B["q"].buf)
        b.buf(7, B["lens"].buf).buf(8, B["slots"].buf).buf(9, B["ids"].buf).buf(10, work).bytes(11, np.array([qh * 128, 128], np.int64)).bytes(15, sizes(**over)).dispatch((1,), (1,))

    def gpu_none():
        from qwental_b200.lib import QwBuf
        return C.byref(QwBuf())

    gpu.L.qw_gpu_set_graphs(gpu.g, graphs)
    try:
        for _ in range(3 if graphs else 1):
            b = gpu.batch()
            rows(b, "kv8_put", "k", "v")
            rows(b, "kv8_get", "ko", "vo")
            choose(b)
            attend(b, "y", True)
            attend(b, "dense", False)
            b.end()
        for x in ("codes", "scales", "bounds"):
            assert torch.equal(before[x].read().view(torch.uint8), rig.t[x].cpu().view(torch.uint8)), x
        for x, t in dict(ko=ko, vo=vo, y=y, dense=dense, ids=ids).items():
            assert torch.equal(B[x].read(), t.cpu()), x
        # refusals: sizes that do not fit the buffers, a layer that is not there, and a row of a slot that is not there
        for bad in (dict(pages=c.c.pages + 1), dict(max_pages=c.c.max_pages + 1), dict(layer=2), dict(nb=4), dict(hd=256), dict(max_len=10 ** 6), dict(kvh=3), dict(dtype=5)):
            for what in ("put", "pick", "attn"):
                if what == "put" and "max_len" in bad:
                    continue
                b = gpu.batch()
                if what == "put":
                    rows(b, "kv8_put", "k", "v", **bad)
                elif what == "pick":
                    choose(b, **bad)
                else:
                    attend(b, "y", True, **bad)
                with pytest.raises(GpuError):
                    b.end()
        B["slots"].buf.upload(np.array([99, 0, 0], np.int32))
        b = gpu.batch()
        rows(b, "kv8_get", "ko", "vo")
        with pytest.raises(GpuError, match="rejected"):
            b.end()
        B["slots"].buf.upload(rig.slots)
        b = gpu.batch()
        rows(b, "kv8_get", "ko", "vo")
        b.end()
    finally:
        gpu.L.qw_gpu_set_graphs(gpu.g, False)
