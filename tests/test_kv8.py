"""The 8-bit key-value cache without a GPU: what the calls refuse (before they touch a device), where rows lie, what lies outside, and the families."""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from qwental_b200 import kv8  # noqa: E402
from tests import kv8_ref as ref  # noqa: E402

SIZES = dict(pages=5, layers=2, kvh=3, hd=128, format=0, block=32, slots=4, max_pages=6)


def cache(**over):
    d = dict(codes=4096, scales=4096, bounds=4096, page_table=4096, status=None, **SIZES)
    d.update(over)
    return kv8.CacheStruct(**d)


def rows(**over):
    d = dict(k=4096, v=4096, slots=4096, pos=4096, k_row=384, k_head=128, v_row=384, v_head=128, nb=2, layer=1, dtype=0)
    d.update(over)
    return kv8.RowsStruct(**d)


def attn(**over):
    d = dict(q=4096, gate=None, y=4096, lens=4096, slots=4096, blocks=None, work=4096, work_bytes=1 << 30, q_row=768, q_head=128, y_row=768, y_head=128, scale=0.1,
             nb=2, layer=1, dtype=1, qh=6, max_len=1000, nblocks=0)
    d.update(over)
    return kv8.AttnStruct(**d)


def pick(**over):
    d = dict(q=4096, lens=4096, slots=4096, blocks=4096, work=4096, work_bytes=1 << 30, q_row=768, q_head=128, nb=2, layer=1, dtype=1, qh=6, max_len=1000, nblocks=8, first=1, last=2)
    d.update(over)
    return kv8.PickStruct(**d)


def call(name, c, a):
    L = kv8.bind()
    err = C.create_string_buffer(256)
    rc = getattr(L, name)(C.byref(c), C.byref(a), None, err, 256)
    return rc, err.value.decode()


BAD_CACHE = [(dict(hd=96), "head dimension"), (dict(hd=0), "head dimension"), (dict(format=2), "format"), (dict(block=8), "block"), (dict(block=48), "block"),
             (dict(block=512), "block"), (dict(pages=0), "at least one"), (dict(kvh=0), "at least one"), (dict(slots=0), "at least one"), (dict(kvh=32768, pages=1, layers=1), "kv heads"), (dict(max_pages=0), "at least one"),
             (dict(pages=1 << 21), "2^31"), (dict(layers=1 << 31, pages=1 << 31), "2^31"), (dict(max_pages=1 << 24), "2^31"), (dict(codes=None), "null pointer"), (dict(scales=None), "null pointer"),
             (dict(page_table=None), "null pointer"), (dict(codes=4097), "16-byte"), (dict(scales=4100), "16-byte"), (dict(bounds=4104), "16-byte")]


@pytest.mark.parametrize("over,msg", BAD_CACHE)
@pytest.mark.parametrize("name,args", [("qw_kv8_put", rows), ("qw_kv8_get", rows), ("qw_kv8_attn", attn), ("qw_kv8_pick", pick)])
def test_a_bad_cache_is_refused(name, args, over, msg):
    rc, m = call(name, cache(**over), args())
    assert rc == -1 and msg in m and m.startswith(name), m


@pytest.mark.parametrize("name", ["qw_kv8_put", "qw_kv8_get"])
@pytest.mark.parametrize("over,msg", [(dict(nb=0), "1 to 1024"), (dict(nb=1025), "1 to 1024"), (dict(layer=2), "layer"), (dict(dtype=2), "type"), (dict(k=None), "null"),
                                      (dict(v=None), "null"), (dict(slots=None), "null"), (dict(pos=None), "null")])
def test_bad_rows_are_refused(name, over, msg):
    rc, m = call(name, cache(), rows(**over))
    assert rc == -1 and msg in m


@pytest.mark.parametrize("over", [dict(k_row=0), dict(v_row=0), dict(k_head=0), dict(v_head=0)])
def test_rows_read_back_onto_one_another_are_refused(over):
    rc, m = call("qw_kv8_get", cache(), rows(**over))
    assert rc == -1 and "on one another" in m
    rc, m = call("qw_kv8_put", cache(), rows(**over))  # one row for many places is fine
    assert rc != -1


@pytest.mark.parametrize("over,code,msg", [(dict(nb=0), -1, "1 to 1024"), (dict(layer=2), -1, "layer"), (dict(dtype=7), -1, "type"), (dict(qh=0), -1, "query heads"), (dict(qh=7), -1, "query heads"),
                                           (dict(qh=51), -1, "query heads"), (dict(max_len=0), -1, "max_len"), (dict(max_len=6 * 256 + 1), -1, "max_len"), (dict(q=None), -1, "null"),
                                           (dict(y=None), -1, "null"), (dict(lens=None), -1, "null"), (dict(slots=None), -1, "null"), (dict(work=None), -1, "null"),
                                           (dict(work=4104), -1, "16-byte"), (dict(blocks=4096), -1, "no number"), (dict(scale=0.0), -1, "scale"), (dict(scale=-1.0), -1, "scale"),
                                           (dict(scale=float("nan")), -1, "scale"), (dict(scale=float("inf")), -1, "scale"), (dict(y_row=0), -1, "on one another"),
                                           (dict(y_head=0), -1, "on one another"), (dict(work_bytes=16), -2, "too small")])
def test_bad_attention_is_refused(over, code, msg):
    rc, m = call("qw_kv8_attn", cache(), attn(**over))
    assert rc == code and msg in m


@pytest.mark.parametrize("over,code,msg", [(dict(nb=2000), -1, "1 to 1024"), (dict(layer=9), -1, "layer"), (dict(dtype=7), -1, "type"), (dict(qh=7), -1, "query heads"), (dict(max_len=0), -1, "max_len"),
                                           (dict(nblocks=0), -1, "at least one"), (dict(first=7, last=2), -1, "first + last"), (dict(first=0xffffffff, last=2), -1, "first + last"),
                                           (dict(blocks=None), -1, "null"), (dict(work=4097), -1, "16-byte"), (dict(work_bytes=100), -2, "too small")])
def test_a_bad_choice_is_refused(over, code, msg):
    rc, m = call("qw_kv8_pick", cache(), pick(**over))
    assert rc == code and msg in m


@pytest.mark.parametrize("name,args,fields", [("qw_kv8_put", rows, "k v slots pos"), ("qw_kv8_get", rows, "k v slots pos"), ("qw_kv8_attn", attn, "q y gate lens slots"),
                                              ("qw_kv8_pick", pick, "q lens slots blocks")])
def test_pointers_between_elements_are_refused(name, args, fields):
    for f in fields.split():
        for off in (1, 2) if f in ("slots", "pos", "lens", "blocks") else (1,):
            rc, m = call(name, cache(), args(**{f: 4096 + off}))
            assert rc == -1 and "boundary" in m, f
    rc, m = call("qw_kv8_attn", cache(), attn(blocks=4098, nblocks=2))
    assert rc == -1 and "boundary" in m
    for over in (dict(page_table=4098), dict(status=4097)):
        rc, m = call(name, cache(**over), args())
        assert rc == -1 and "4-byte" in m


def test_results_closer_than_a_row_is_long_are_refused():
    for name, args, fields in (("qw_kv8_get", rows, "k_row k_head v_row v_head"), ("qw_kv8_attn", attn, "y_row y_head")):
        for f in fields.split():
            for x in (127, -127, 1):
                rc, m = call(name, cache(), args(**{f: x}))
                assert rc == -1 and "on one another" in m
    for name, args, over in (("qw_kv8_put", rows, dict(k_row=1, k_head=3)), ("qw_kv8_attn", attn, dict(q_row=1, gate_head=0)), ("qw_kv8_pick", pick, dict(q_head=1))):
        assert "on one another" not in call(name, cache(), args(**over))[1]  # what is read may overlap


def test_more_tokens_than_a_call_takes_are_refused():
    big = dict(pages=1000, max_pages=1 << 22, kvh=64, layers=1, hd=64)
    rc, m = call("qw_kv8_attn", cache(**big), attn(layer=0, qh=64, nb=1024, max_len=(1 << 30) - 1, q_head=64, y_head=64))
    assert rc == -1 and "more tokens" in m


def test_a_choice_needs_bounds():
    rc, m = call("qw_kv8_pick", cache(bounds=None), pick())
    assert rc == -1 and "bounds" in m


def test_good_arguments_need_a_device():
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    for name, args in (("qw_kv8_put", rows()), ("qw_kv8_get", rows()), ("qw_kv8_attn", attn()), ("qw_kv8_pick", pick())):
        rc, m = call(name, cache(), args)
        assert rc == -3 and "device" in m


def test_sizes_and_workspaces():
    L = kv8.bind()
    n = (C.c_size_t * 3)()
    assert L.qw_kv8_bytes(C.byref(cache()), n) == 0
    assert list(n) == [5 * 2 * 2 * 3 * 256 * 128, 5 * 2 * 2 * 3 * 256 * 4, 5 * 2 * 3 * 8 * (256 + 16)]
    assert L.qw_kv8_bytes(C.byref(cache(hd=100)), n) == -1
    w = L.qw_kv8_attn_work(C.byref(cache()), 2, 6, 1000, 0)
    assert w > 0 and w == L.qw_kv8_attn_work(C.byref(cache()), 1, 6, 1000, 0) * 2
    assert call("qw_kv8_attn", cache(), attn(work_bytes=w - 1))[0] == -2
    assert 0 < L.qw_kv8_attn_work(C.byref(cache()), 2, 6, 1000, 3) <= w  # fewer tokens
    assert L.qw_kv8_attn_work(C.byref(cache()), 2, 6, 1000, 1 << 30) <= w  # never more blocks than there are
    assert L.qw_kv8_attn_work(C.byref(cache()), 2, 5, 1000, 0) == 0 and L.qw_kv8_attn_work(C.byref(cache()), 2, 6, 10000, 0) == 0
    assert L.qw_kv8_pick_work(C.byref(cache()), 2, 1000) >= 2 * 3 * 32 * 4 and L.qw_kv8_pick_work(C.byref(cache()), 2, 0) == 0


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
def test_a_workspace_for_everything_serves_chosen_blocks(block):
    """Blocks are gone over as a whole, so a list of them may need more chunks than the row's tokens: 70 tokens are three of 32, one block of 256 is eight."""
    L = kv8.bind()
    c = cache(block=block, pages=1000, max_pages=1000, layers=1)
    for n in (1, 15, 16, 17, 70, 255, 256, 257, 500, 512, 513, 600, 2047, 2048, 2049, 2100, 65535, 65536, 65537, 70001):
        w = L.qw_kv8_attn_work(C.byref(c), 2, 6, n, 0)
        for k in (1, 2, 3, 5, 8, 100, 129, 4096, 1 << 20):
            assert 0 < L.qw_kv8_attn_work(C.byref(c), 2, 6, n, k) <= w, (n, k)
        assert call("qw_kv8_attn", c, attn(layer=0, max_len=n, work_bytes=w, blocks=4096, nblocks=-(-n // block)))[0] != -2
        assert call("qw_kv8_attn", c, attn(layer=0, max_len=n, work_bytes=w))[0] != -2


def test_rows_lie_where_the_layout_says_and_nothing_outside_is_touched():
    """The kernels' own index arithmetic (kv8.h), on the host."""
    L = kv8.bind()
    c = cache()
    at = np.arange(5 * 2 * 2 * 3 * 256).reshape(5, 2, 2, 3, 256)
    for page in range(5):
        for layer in range(2):
            for kv in range(2):
                for head in range(3):
                    for pos in (0, 1, 255, 256, 1535):
                        assert L.qw_kv8_row_index(C.byref(c), 3, pos, page, layer, kv, head) == at[page, layer, kv, head, pos % 256]
    for slot, pos, page in ((-1, 0, 0), (4, 0, 0), (2 ** 31 - 1, 0, 0), (0, -1, 0), (0, 1536, 0), (0, 2 ** 31 - 1, 0), (0, 0, -1), (0, 0, 5), (0, 0, 2 ** 31 - 1), (0, 0, -2 ** 31)):
        assert L.qw_kv8_row_index(C.byref(c), slot, pos, page, 0, 0, 0) == -1
    big = cache(pages=(2 ** 31 - 1) // (2 * 2 * 3 * 256), max_pages=2 ** 23 - 1)  # the last row of the largest pool
    last = big.pages - 1
    assert L.qw_kv8_row_index(C.byref(big), 0, 255, last, 1, 1, 2) == big.pages * 2 * 2 * 3 * 256 - 1
    assert L.qw_kv8_row_index(C.byref(big), 0, (2 ** 23 - 1) * 256 - 1, 0, 0, 0, 0) == 255


def test_python_face_checks_its_tensors():
    mk = lambda: (torch.zeros(3, 1, 2, 2, 256, 64, dtype=torch.uint8), torch.zeros(3, 1, 2, 2, 256), torch.zeros(2, 4, dtype=torch.int32))  # noqa: E731
    c, s, t = mk()
    kv8.Kv8Cache(c, s, t)
    b = torch.zeros(3, 1, 2, 4, 144, dtype=torch.uint8)
    assert kv8.Kv8Cache(c, s, t, b).c.block == 64
    for bad in ((c[..., :32], s, t), (c.float(), s, t), (c, s.double(), t), (c, s[..., :1], t), (c, s, t.long()), (c, s, t[0]), (c[:, :, :, :, ::2], s, t)):
        with pytest.raises(kv8.Kv8Error):
            kv8.Kv8Cache(*bad)
    for bad in (b[..., :80], b.float(), b[:, :, :, :3].contiguous(), torch.zeros(3, 1, 2, 32, 144, dtype=torch.uint8)):
        with pytest.raises(kv8.Kv8Error):
            kv8.Kv8Cache(c, s, t, bad)
    with pytest.raises(kv8.Kv8Error):
        kv8.Kv8Cache(c, s, t, b, block=32)
    with pytest.raises(kv8.Kv8Error):
        kv8.Kv8Cache(c, s, t, format="int4")
    k = kv8.Kv8Cache(c, s, t, b)
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    with pytest.raises(kv8.Kv8Error, match="no CPU path"):
        k.put(x, x, i, i)
    for bad in ((x.float(), x, i, i), (x, x.bfloat16(), i, i), (x[:1], x, i, i), (x, x, i.long(), i), (x, x, i, i[:1]), (x.transpose(1, 2), x, i, i), (x[:, :1], x, i, i)):
        with pytest.raises(kv8.Kv8Error):
            k.put(*bad)
    with pytest.raises(kv8.Kv8Error):
        k.attn(x, i, i, x.bfloat16(), max_len=10)
    with pytest.raises(kv8.Kv8Error):
        k.attn(x, i, i, x, max_len=10, blocks=torch.zeros(2, 1, 4, dtype=torch.int32))
    with pytest.raises(kv8.Kv8Error):
        k.work_bytes(1, 3, 10)


def test_families_are_registered():
    L = kv8.bind()
    fams = {L.qw_gpu_family_name(i).decode() for i in range(L.qw_gpu_family_count())}
    assert {"kv8_put", "kv8_get", "kv8_attn", "kv8_pick"} <= fams


def test_the_plain_statement_rounds_as_torch_does():
    """The tests' own e4m3 rounding against torch's conversion on the CPU, and both formats at their borders."""
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.standard_normal(20000) * 10.0 ** rng.uniform(-4, 2, 20000), ref.e4m3_values()[:127], (ref.e4m3_values()[:126] + ref.e4m3_values()[1:127]) / 2]).astype(np.float32)
    x = np.clip(x, -448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref._nearest_e4m3(x), want)
    for fmt in ("e4m3", "int8"):
        y = rng.standard_normal((50, 64)).astype(np.float32)
        y[3] = 0
        y[4] = 1e-38
        y[5, 7] = np.nan
        y[6, 9] = -np.inf
        c, s = ref.quantise(y, fmt)
        assert np.isnan(s[[5, 6]]).all() and (s[[3, 4]] == 0).all() and not (c[[5, 6]]).any() and not (ref.values(c[[3, 4]], fmt)).any()
        ok = np.r_[0:3, 7:50]
        back = ref.values(c[ok], fmt) * s[ok, None]
        a = np.abs(y[ok]).max(1, keepdims=True)
        assert (np.abs(back - y[ok]) <= (a / 127 / 2 if fmt == "int8" else np.maximum(np.abs(y[ok]) * 2.0 ** -4, a / 448 * 2.0 ** -10)) * (1 + 1e-5)).all()
