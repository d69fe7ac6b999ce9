"""The 8-bit key-value cache's host side without a GPU: arguments that would be taken for others, results that share memory, calls from several threads."""
import ctypes as C
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
from qwental_b200 import kv8  # noqa: E402
from tests.test_kv8 import attn, cache, call, pick, rows  # noqa: E402


def on_cpu():
    """A cache of CPU tensors (calls get as far as the device) with rows for it."""
    c = kv8.Kv8Cache(torch.zeros(3, 1, 2, 2, 256, 64, dtype=torch.uint8), torch.zeros(3, 1, 2, 2, 256), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(3, 1, 2, 4, 144, dtype=torch.uint8))
    return c, torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)


def test_a_list_without_room_is_not_a_call_without_a_list():
    c, x, i = on_cpu()
    none = torch.zeros(2, 2, 0, dtype=torch.int32)
    work = torch.zeros(1 << 20, dtype=torch.uint8)
    with pytest.raises(kv8.Kv8Error, match="one block at least"):
        c.attn(x, i, i, x.clone(), max_len=10, blocks=none, work=work)
    with pytest.raises(kv8.Kv8Error, match="one block at least"):
        c.pick(x, i, i, none, max_len=10, first=0, last=0, work=work)


def shares(nb, heads, hd, row, head):
    """By going over every pair of results."""
    at = sorted(int(x) for x in (np.arange(nb)[:, None] * row + np.arange(heads) * head).reshape(-1))
    return any(b - a < hd for a, b in zip(at, at[1:]))


def test_results_that_share_memory_are_refused_and_no_others():
    """Row and head strides together: 128 and 128 put (row 0, head 1) where (row 1, head 0) is."""
    rng = np.random.default_rng(3)
    cases = [(2, 3, 128, 128), (2, 3, 256, 128), (2, 3, 384, 128), (2, 3, 128, 256), (2, 3, 300, 128), (2, 3, 383, 128), (2, 3, -384, 128), (2, 3, -256, 128), (5, 3, 128, 640), (5, 3, 128, 512),
             (5, 3, 128, 639), (4, 3, 200, 400), (4, 3, 300, 450), (1, 3, 0, 128), (1, 3, 5, 128), (2, 3, 384, 0), (3, 3, 0, 384), (2, 3, 1 << 62, 128), (2, 3, -(1 << 63), 128), (1024, 3, 384, 128),
             (1024, 3, 383, 128), (1024, 3, 128, 131072), (1024, 3, 128, 131071)]
    cases += [(int(rng.integers(1, 12)), 3, int(rng.integers(-900, 900)), int(rng.integers(-900, 900))) for _ in range(3000)]
    for heads in (1, 3, 6):  # (rows of three kv heads; results of one, three or six query heads)
        for nb, _, row, head in cases if heads == 3 else cases[:23]:
            want = "on one another" if shares(nb, heads, 128, row, head) else None
            got = [call("qw_kv8_attn", cache(kvh=3 if heads > 1 else 1), attn(nb=nb, qh=heads, y_row=row, y_head=head))[1]]
            if heads == 3:
                got += [call("qw_kv8_get", cache(), rows(k=1 << 30, nb=nb, k_row=row, k_head=head, v_row=384, v_head=128))[1]]
                got += [call("qw_kv8_get", cache(), rows(v=1 << 30, nb=nb, v_row=row, v_head=head, k_row=384, k_head=128))[1]]
            assert all(("on one another" in m) == (want is not None) for m in got), (nb, heads, row, head, got)


def test_every_thread_gets_its_own_message(monkeypatch):
    """Two threads in calls of one cache at the same time: a refusal's text is that of its own call, and a call that succeeds in between does not clear it."""
    c, _, _ = on_cpu()
    c.index = 0
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    meet, said = threading.Barrier(3), {}

    def library(name, rc, late):  # stands in for a call that writes its message while others are under way
        def f(ref, args, stream, err, size):
            meet.wait(10)
            if late:
                meet.wait(10)
            err.value = name.encode()
            if not late:
                meet.wait(10)
            meet.wait(10)
            return rc
        return f

    def run(name, rc, late):
        try:
            c._call(library(name, rc, late), kv8.RowsStruct(), 0)
            said[name] = None
        except kv8.Kv8Error as e:
            said[name] = str(e)

    threads = [threading.Thread(target=run, args=x) for x in (("first", -1, False), ("second", -1, True), ("", 0, True))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert said == {"first": "first", "second": "second", "": None}


def test_a_thread_launches_under_its_own_family():
    """QW_PDL_OFF names families that are launched without the attribute; which one a launch is of is its thread's own."""
    code = """
import ctypes, threading
from qwental_b200 import lib
L = lib.load()
family, enabled = L._Z21qw_pdl_current_familyPKc, L._Z14qw_pdl_enabledv
family.argtypes, enabled.restype = [ctypes.c_char_p], ctypes.c_bool
off, on = ctypes.create_string_buffer(b"kv8_get"), ctypes.create_string_buffer(b"kv8_put")
family(off)
assert not enabled()
t = threading.Thread(target=lambda: (family(on), seen.append(enabled())))
seen = []
t.start()
t.join()
assert seen == [True] and not enabled(), (seen, enabled())
"""
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, QW_PDL_OFF="kv8_get", QW_PDL="1"), capture_output=True, text=True, timeout=120,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(kv8.__file__))))
    assert r.returncode == 0, r.stderr[-800:]


def test_a_list_of_more_blocks_than_are_counted_is_refused():
    """Entries are counted in 32 bits, in steps of 32 or 512: with 2^32 - 1 of them a count would come round and never end."""
    for n in (0x80000000, 0xfffffe00, 0xffffffff):
        rc, m = call("qw_kv8_pick", cache(), pick(nblocks=n))
        assert rc == -1 and "2^31 - 1 blocks" in m
        rc, m = call("qw_kv8_attn", cache(), attn(blocks=4096, nblocks=n))
        assert rc == -1 and "2^31 - 1 blocks" in m
    for name, args in (("qw_kv8_pick", pick(nblocks=0x7fffffff)), ("qw_kv8_attn", attn(blocks=4096, nblocks=0x7fffffff)), ("qw_kv8_attn", attn(nblocks=0xffffffff))):
        assert "blocks" not in call(name, cache(), args)[1]


@pytest.mark.parametrize("bad", [1 << 32, (1 << 32) + 10, -1, -(1 << 32) + 10, 1 << 64])
def test_numbers_that_32_bits_do_not_hold_are_refused(bad):
    """They would arrive as others: a max_len of 2^32 + 10 as 10, layer 2^32 as layer 0."""
    c, x, i = on_cpu()
    ids, work = torch.zeros(2, 2, 3, dtype=torch.int32), torch.zeros(1 << 20, dtype=torch.uint8)
    calls = [lambda: c.put(x, x, i, i, layer=bad), lambda: c.get(x, x.clone(), i, i, layer=bad), lambda: c.attn(x, i, i, x.clone(), max_len=bad, work=work),
             lambda: c.attn(x, i, i, x.clone(), layer=bad, max_len=10, work=work), lambda: c.attn(x, i, i, x.clone(), max_len=bad),
             lambda: c.pick(x, i, i, ids, max_len=bad, work=work), lambda: c.pick(x, i, i, ids, layer=bad, max_len=10, work=work), lambda: c.pick(x, i, i, ids, max_len=10, first=bad, work=work),
             lambda: c.pick(x, i, i, ids, max_len=10, last=bad, work=work), lambda: c.work_bytes(bad, 2, 10), lambda: c.work_bytes(1, bad, 10), lambda: c.work_bytes(1, 2, bad),
             lambda: c.work_bytes(1, 2, 10, bad)]
    for f in calls:
        with pytest.raises(kv8.Kv8Error, match="32 bits"):
            f()


def test_a_page_table_that_32_bits_do_not_hold_is_refused():
    meta = lambda *s, dtype=torch.uint8: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    for shape in ((1, (1 << 32) + 5), ((1 << 32) + 5, 1)):
        with pytest.raises(kv8.Kv8Error, match="32 bits"):
            kv8.Kv8Cache(meta(3, 1, 2, 2, 256, 64), meta(3, 1, 2, 2, 256, dtype=torch.float32), meta(*shape, dtype=torch.int32))
