"""Attention over the 8-bit key-value cache where its arithmetic can go wrong, against 64 bits: value rows that are zero or far apart in size, elements of a
query far apart, weights far below the largest; rows in which every token and every chunk counts; empty rows, scores beyond the range, lists of
blocks that are too long."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
from qwental_b200 import kv8  # noqa: E402
from tests import kv8_ref as ref  # noqa: E402
from tests.test_gpu_kv8 import PAGE, Rig, host  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
LN2 = np.log(2.0)


def set_rows(rig, i, j, codes=None, scales=None, head=slice(None)):
    """Keys (j = 0) or values (j = 1) of the first tokens of row i's slot: codes [n, hd], scales [n], for every head."""
    n = len(codes if codes is not None else scales)
    for p0 in range(0, n, PAGE):
        p, m = rig.table[rig.slots[i], p0 // PAGE], min(PAGE, n - p0)
        if codes is not None:
            rig.codes[p, rig.layer, j, head, :m] = codes[p0:p0 + m].view(np.uint8)
        if scales is not None:
            rig.scales[p, rig.layer, j, head, :m] = scales[p0:p0 + m]


def upload(rig):
    rig.t["codes"].copy_(torch.from_numpy(rig.codes))
    rig.t["scales"].copy_(torch.from_numpy(rig.scales))


def one_code(fmt):
    return 1 if fmt == "int8" else 0x38  # stands for 1


def scored_by_channel_0(rig, i, s, fmt):
    """Keys whose score with a query of ones in channel 0 is s[t], at softmax scale 1: one product each."""
    codes = np.zeros((len(s), rig.hd), np.uint8)
    codes[:, 0] = np.where(s < 0, 0xff if fmt == "int8" else 0xb8, one_code(fmt))
    set_rows(rig, i, 0, codes, np.abs(s).astype(np.float32))


def queries_of_channel_0(rig, n, heads, dtype):
    q = torch.zeros(n, heads, rig.hd, dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    return q


# ------------------------------------------------------------------------------------------------ values that are zero, or far apart in size
@pytest.mark.parametrize("fmt,dtype,value", [("int8", F16, 65504.0), ("e4m3", F16, 65504.0), ("int8", F16, 1e4), ("int8", F16, 1e3), ("int8", BF16, 1e6), ("e4m3", BF16, 1e30)])
@pytest.mark.parametrize("n,zeros,hd,G", [(600, 32, 64, 2), (3000, 96, 128, 5), (3000, 32, 256, 12), (70000, 224, 64, 9)])
def test_rows_of_zeros_before_large_values_count(n, zeros, hd, G, fmt, dtype, value):
    """A row whose values are zero has its part of the softmax's sum, whatever comes later: tokens of zeros in the first steps of a chunk (of 2, 4 or 8 steps), then in
    the chunk's last step one of a higher score and large values.
    Tolerance: a score is one product, times the row's scale, the query's power of two and the softmax scale (three roundings of 2^-24), joined with log2 of the value's
    scale (one more, and log2's own 2^-22) and a maximum (one more): 6 2^-24 (|s'| + |lv| + 15) + 2^-22 |lv| in the exponent, twice (a weight and the sum); exponentials
    2^-22 each; sums and the join's products at most 300 roundings of 2^-23; then half a step of the result."""
    wins = [0.0, 5.0, 7.5, 10.0, 13.0, 16.5, 25.0]  # by so much the large row's score is higher, in powers of two
    chunk = 64 if n <= 2048 else 128 if n <= 65536 else 256
    rig = Rig([n] * len(wins), 1, hd, fmt, layers=1, layer=0, seed=n)
    v_one = rig.rng.integers(1, 120, hd).astype(np.uint8)
    v_one[0] = 127 if fmt == "int8" else 0x7e  # the largest code
    largest = ref.LARGEST[fmt]
    vs = np.float32(value / largest)
    for i, d in enumerate(wins):
        s = np.full(n, -60.0)
        s[chunk:chunk + zeros] = 0
        s[2 * chunk - 1] = d * LN2
        scored_by_channel_0(rig, i, s, fmt)
        scales = np.full(n, vs * np.float32(2.0 ** -10), np.float32)
        codes = np.tile(v_one, (n, 1))
        scales[chunk:chunk + zeros] = 0
        codes[chunk:chunk + zeros] = 0
        scales[2 * chunk - 1] = vs
        set_rows(rig, i, 1, codes, scales)
    upload(rig)
    q = queries_of_channel_0(rig, len(wins), G, dtype)
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=n, scale=1.0)
    got = host(y).astype(np.float64)
    for i, d in enumerate(wins):
        k, v = rig.kv(i, 0)
        want, _ = ref.attend(host(q)[i].astype(np.float64), k, v, 1.0)
        lv = abs(np.log2(vs))
        rel = 2 * LN2 * (6 * 2.0 ** -24 * (d + lv + 15) + 2.0 ** -22 * lv) + 2.0 ** -21 + 300 * 2.0 ** -23
        tol = np.abs(want) * (rel + torch.finfo(dtype).eps / 2 * (1 + rel))
        off = np.abs(got[i] - want)
        assert (off <= tol).all(), (d, float((off / tol).max()), got[i, 0, :2], want[0, :2])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_a_row_of_nothing_but_zero_values_is_zero(fmt):
    """300,000 tokens' worth of nothing: the sum of the weights stays a number (chunks of 256, 2^18 tokens and more)."""
    n = 270_000
    rig = Rig([16 * PAGE], 1, 64, fmt, layers=1, layer=0, seed=1)
    rig.codes[:, :, 1] = 0
    rig.scales[:, :, 1] = 0
    upload(rig)
    table = np.resize(rig.table[rig.slots[0], :16], (rig.table.shape[0], n // PAGE + 1)).astype(np.int32)
    c = kv8.Kv8Cache(rig.t["codes"], rig.t["scales"], torch.from_numpy(table).cuda(), format=fmt)
    q = rig.randn(1, 3, 64)
    y = torch.full_like(q, 5.0)
    c.attn(q, rig.idx([n]), rig.idx([0]), y, max_len=n)
    assert (y == 0).all()


# ------------------------------------------------------------------------------------------------ queries and weights over a wide range
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype,top,rest", [(F16, 60000.0, 0.05), (F16, 60000.0, 2e-4), (BF16, 1e4, 0.01), (BF16, 3e5, 1e-3), (BF16, 1e20, 1e12)])
@pytest.mark.parametrize("hd,G", [(64, 7), (128, 2), (256, 16)])
def test_small_elements_of_a_query_count_beside_a_large_one(hd, G, dtype, top, rest, fmt):
    """One channel of the queries is far above the others and all keys are zero there, so that the others alone make the scores.
    Values are not negative and every row of them has one channel, so a result's relative error is that of the weights: twice (hd + 8) 2^-23 of sum |q k| in the scores
    (a weight and the sum), 2^-17 for exponentials, sums and log2 of the values' scales, then half a step of the result."""
    n = 300
    rig = Rig([n, 77], 1, hd, fmt, layers=1, layer=0, seed=hd + G)
    rig.codes[:, :, 0, :, :, 5] = 0
    for i in (0, 1):
        m = int(rig.lens[i])
        codes = np.zeros((m, hd), np.uint8)
        codes[np.arange(m), np.arange(m) % hd] = rig.rng.integers(0x60, 0x7f, m)
        set_rows(rig, i, 1, codes)
    upload(rig)
    q = rig.randn(2, G, hd, dtype=dtype, scale=rest)
    q[:, :, 5] = top
    y = torch.zeros_like(q)
    sc = 2.0 / (rest * hd ** 0.5)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=n, scale=sc)
    got, qn = host(y).astype(np.float64), host(q).astype(np.float64)
    for i in (0, 1):
        k, v = rig.kv(i, 0)
        want, spread = ref.attend(qn[i], k, v, float(np.float32(sc)))
        rel = 4 * (hd + 8) * 2.0 ** -23 * spread + 2.0 ** -17
        tol = np.abs(want) * (rel + torch.finfo(dtype).eps / 2 * (1 + rel)) + 2.0 ** -25
        off = np.abs(got[i] - want)
        assert (off <= tol).all(), (i, float((off / tol).max()))


@pytest.mark.parametrize("below", [12, 20, 26, 28])
@pytest.mark.parametrize("n,hd,G", [(200, 64, 3), (1500, 128, 8), (3000, 256, 11)])
def test_weights_far_below_the_largest_count(n, hd, G, below):
    """The first token of every chunk has almost all of the chunk's weight and values in channel 0 alone; the others, 2^-below of it each, have theirs in channel 1.
    A weight w, the largest 2^15, is held as two fp16 numbers: to 2^-22 of itself, or to 2^-25 where that is more, so 2^-12 of itself at 2^-13 (28 below)."""
    rig = Rig([n], 1, hd, "int8", layers=1, layer=0, seed=n)
    chunk = 32 if n <= 512 else 64 if n <= 2048 else 128
    s = np.full(n, -below * LN2)
    s[::chunk] = 0
    scored_by_channel_0(rig, 0, s, "int8")
    codes = np.zeros((n, hd), np.uint8)
    codes[:, 1] = 100
    codes[::chunk] = 0
    codes[::chunk, 0] = 100
    set_rows(rig, 0, 1, codes, np.full(n, 0.25, np.float32))
    upload(rig)
    q = queries_of_channel_0(rig, 1, G, BF16)
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=n, scale=1.0)
    k, v = rig.kv(0, 0)
    want, _ = ref.attend(host(q)[0].astype(np.float64), k, v, 1.0)
    rel = 2 * LN2 * 6 * 2.0 ** -24 * (below + 17) + max(2.0 ** -22, 2.0 ** (below - 40)) + 2.0 ** -16
    off = np.abs(host(y)[0] - want)
    assert (off <= np.abs(want) * (rel + 2.0 ** -8 * (1 + rel))).all(), (float((off / want.clip(1e-30)).max()), host(y)[0, 0, :2], want[0, :2])


@pytest.mark.parametrize("hd,G,dtype", [(64, 4, F16), (128, 1, F16), (64, 8, F16), (256, 6, F16), (128, 16, F16)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_weights_are_held_to_more_than_eleven_bits(hd, G, dtype, fmt):
    """Values of one size and both signs at almost equal weights, whose sum nearly cancels: what is left is far below the rounding of a weight to fp16.
    Tolerance, of the value: exponents of at most 16, with three roundings of 2^-24 of a score of up to 1.5 and two more of 2^-24 of 16, times ln 2: 25.5 2^-24; an exponential
    2^-22, a weight's two parts 2^-22, partial sums that stay below a few weights: under 2^-18 together.  With the high parts alone a weight is off by up to
    2^-11, 2^-12.5 in the mean, and the sum by about 2^-12.5 / sqrt(40) = 2^-15.2."""
    n = 40
    rig = Rig([n], 1, hd, fmt, layers=1, layer=0, seed=hd)
    s = rig.rng.uniform(0.2, 1.0, n // 2).repeat(2)
    s[1::2] *= 1 + 2.0 ** -14
    scored_by_channel_0(rig, 0, s, fmt)
    codes = np.zeros((n, hd), np.uint8)
    codes[0::2] = 100 if fmt == "int8" else 0x70
    codes[1::2] = 256 - 100 if fmt == "int8" else 0xf0
    set_rows(rig, 0, 1, codes, np.ones(n, np.float32))
    upload(rig)
    q = queries_of_channel_0(rig, 1, G, dtype)
    q[0, :, 0] = 1 - torch.arange(G, device="cuda") / 32
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=n, scale=1.0)
    k, v = rig.kv(0, 0)
    want, _ = ref.attend(host(q)[0].astype(np.float64), k, v, 1.0)
    off = np.abs(host(y)[0] - want)
    assert np.abs(want).max() < 2.0 ** -12 * np.abs(v).max()
    assert (off <= np.abs(v).max() * 2.0 ** -18 + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all(), float(off.max() / np.abs(v).max())


# ------------------------------------------------------------------------------------------------ every token counts
LONG = [31, 513, 2048, 2049, 4097, 5000, 8193, 20000, 48001, 65536, 65537, 70001]


@pytest.mark.parametrize("hd,kvh,G,fmt,dtype,lens", [(256, 1, 8, "e4m3", F16, LONG), (256, 2, 3, "int8", F16, LONG), (256, 1, 16, "int8", BF16, LONG), (128, 1, 8, "int8", F16, LONG),
                                                     (64, 1, 12, "e4m3", F16, [5000, 9001]), (128, 3, 1, "e4m3", F16, [20000]), (256, 1, 5, "int8", F16, [131073])])
def test_every_token_of_a_long_row_counts(hd, kvh, G, fmt, dtype, lens):
    """Token t has values in channel t % hd alone, and none are negative: a token, a step or a chunk that is lost, or counted twice, moves its channels by its share of
    at least hd / tokens, and a result's relative error is that of its weights: in the scores twice (hd + 8) 2^-23 of sum |q k| (a weight and the sum), 2^-17 for
    exponentials, log2, sums and joins; then half a step of the result."""
    rig = Rig(lens, kvh, hd, fmt, layers=1, layer=0, seed=hd + G)
    for i, n in enumerate(lens):
        codes = np.zeros((n, hd), np.uint8)
        codes[np.arange(n), np.arange(n) % hd] = rig.rng.integers(0x70, 0x7f, n)
        set_rows(rig, i, 1, codes)
    upload(rig)
    qh = kvh * G
    q = rig.randn(len(lens), qh, hd, dtype=dtype, scale=0.3)
    y = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=max(lens))
    got, qn = host(y).astype(np.float64), host(q).astype(np.float64)
    for i in range(len(lens)):
        for h in range(kvh):
            k, v = rig.kv(i, h)
            g = slice(h * G, (h + 1) * G)
            want, spread = ref.attend(qn[i, g], k, v, hd ** -0.5)
            rel = 4 * (hd + 8) * 2.0 ** -23 * spread + 2.0 ** -17
            tol = np.abs(want) * (rel + torch.finfo(dtype).eps / 2 * (1 + rel)) + 2.0 ** -25
            off = np.abs(got[i, g] - want)
            assert (off <= tol).all(), (lens[i], h, float((off / tol).max()))


# ------------------------------------------------------------------------------------------------ results that are zero, and such that are no numbers
def test_an_empty_row_is_zero_whatever_its_gate_and_its_list_hold():
    rig = Rig([0, 300, 0], 2, 128, "int8", 64, seed=3)
    q, gate = rig.randn(3, 8, 128), rig.randn(3, 8, 128)
    gate[0] = float("nan")
    gate[2, 3] = float("-inf")
    gate[1, 1, 7] = float("nan")  # of a row in use: its results are not numbers
    blocks = np.tile(np.arange(6, dtype=np.int32), (3, 2, 1))
    blocks[1, :, 5] = -1
    for more in (dict(), dict(blocks=rig.idx(blocks))):
        y = torch.full_like(q, 7.0)
        rig.status.zero_()
        rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=300, gate=gate, **more)
        assert (y[0] == 0).all() and (y[2] == 0).all() and y[1, 1, 7].isnan() and int(y[1].isnan().sum()) == 1 and int(rig.status) == 0


def test_a_list_of_no_valid_blocks_is_zero_whatever_the_gate():
    rig = Rig([300], 1, 64, "int8", 64, seed=3)
    q, y = rig.randn(1, 2, 64), rig.randn(1, 2, 64)
    rig.cache.attn(q, rig.idx([300]), rig.idx(rig.slots), y, layer=1, max_len=300, blocks=rig.idx(np.full((1, 1, 4), -1)), gate=torch.full_like(q, float("nan")))
    assert (y == 0).all()


def test_scores_that_all_overflow_are_no_numbers():
    """Scores of minus infinity alone leave nothing to divide by; one that is a number decides alone."""
    rig = Rig([300, 300], 1, 64, "int8", layers=1, layer=0, seed=3)
    for i in (0, 1):
        s = np.full(300, -1e30)
        if i:
            s[123] = 0
        scored_by_channel_0(rig, i, s, "int8")
    upload(rig)
    q = queries_of_channel_0(rig, 2, 3, BF16) * 1e20
    blocks = rig.idx(np.tile(np.arange(5), (2, 1, 1)))
    for more in (dict(), dict(blocks=blocks)):
        y = torch.zeros_like(q)
        rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, max_len=300, scale=1.0, **more)
        assert y[0].isnan().all()
        want = torch.from_numpy(rig.kv(1, 0)[1][123]).to(BF16)
        assert (y[1].cpu().float() - want.float()).abs().max() <= 2.0 ** -7 * want.float().abs().max()


@pytest.mark.parametrize("block", [16, 32, 64, 256])
def test_a_list_longer_than_its_row_has_blocks(block):
    """A number beyond the row's last block is found wherever it stands in the list, in the head whose list it is; -1 behind the last is fine."""
    n, kvh = 2 * block, 2
    rig = Rig([n] * 6 + [3 * block - 5], kvh, 64, "e4m3", block, seed=2)
    lists = [[0, 1, 7, -1], [7, 0, 1, -1], [0, -1, -1, 7], [1, 0, -1, -1], [0, 1, -1, 2], [0, 1, 0, -1], [2, 1, 0, 3]]
    blocks = np.array([[x, [0, 1, -1, -1]] for x in lists], np.int32)
    q = rig.randn(7, 2 * kvh, 64)
    y = torch.zeros_like(q)
    for r in range(7):
        rig.status.zero_()
        rig.cache.attn(q[r:r + 1], rig.idx([rig.lens[r]]), rig.idx(rig.slots[r:r + 1]), y[r:r + 1], layer=1, max_len=3 * block, blocks=rig.idx(blocks[r:r + 1]))
        assert (int(rig.status) & 0xf00 == 0x200) == (r != 3), r
        assert bool(y[r, :2].isnan().all()) == (r != 3) and y[r, 2:].isfinite().all(), r
    many = torch.zeros_like(q)
    rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), many, layer=1, max_len=3 * block, blocks=rig.idx(blocks))
    assert torch.equal(many.view(torch.int16), y.view(torch.int16))


def test_results_in_place_of_the_queries_or_of_the_gate():
    rig = Rig([0, 77, 700, 5000], 2, 128, "int8", seed=4)
    q, gate = rig.randn(4, 8, 128), rig.randn(4, 8, 128)
    y = torch.zeros_like(q)
    call = lambda q, g, y: rig.cache.attn(q, rig.idx(rig.lens), rig.idx(rig.slots), y, layer=1, max_len=5000, gate=g)  # noqa: E731
    call(q, gate, y)
    a, b = q.clone(), gate.clone()
    call(a, gate, a)
    call(q, b, b)
    assert torch.equal(a, y) and torch.equal(b, y)


# ------------------------------------------------------------------------------------------------ refusals that need a device
def test_keys_and_values_are_not_read_back_into_one_place():
    """k and v that share memory are refused before anything is launched; side by side, or in turn in one tensor, they are fine."""
    n, kvh, hd = 5, 2, 64
    rig = Rig([300], kvh, hd, "int8", layers=1, layer=0)
    slots, pos = rig.idx(np.full(n, rig.slots[0])), rig.idx(np.arange(n) * 3)
    flat = torch.zeros(8 * n * kvh * hd, dtype=torch.float16, device="cuda")
    kw, vw = flat[:n * kvh * hd].view(n, kvh, hd), flat[n * kvh * hd:2 * n * kvh * hd].view(n, kvh, hd)
    rig.cache.get(kw, vw, slots, pos)
    want = kw.clone(), vw.clone()

    def at(start, row, head):
        return flat.as_strided((n, kvh, hd), (row, head, 1), start)

    full = kvh * hd
    for a, b in ((at(0, full, hd), at(0, full, hd)), (at(0, full, hd), at(hd - 1, full, hd)), (at(0, full, hd), at((n - 1) * full + hd, full, hd)), (at(0, 2 * full, hd), at(full - 1, 2 * full, hd)),
                 (at(0, 2 * full, hd), at(2 * full - 1, 2 * full, hd)), (at(0, hd, n * hd), at(3 * hd + 1, hd, n * hd)), (at(0, full, hd), at(full, 2 * full, hd))):
        flat.fill_(7)
        with pytest.raises(kv8.Kv8Error, match="on one another"):
            rig.cache.get(a, b, slots, pos)
        assert (flat == 7).all()
    for a, b in ((at(0, 2 * full, hd), at(full, 2 * full, hd)), (at(full, 2 * full, hd), at(0, 2 * full, hd)), (at(0, full, hd), at(n * full, full, hd)), (at(0, hd, 2 * n * hd), at(n * hd, hd, 2 * n * hd)),
                 (at(0, 2 * full, 2 * hd), at(hd, 2 * full, 2 * hd)), (at(0, full, hd), at(n * full, 2 * full, hd))):
        flat.fill_(7)
        rig.cache.get(a, b, slots, pos)
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
