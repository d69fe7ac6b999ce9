"""The 8-bit key-value cache's host side without a GPU: arguments that would be taken for others, results that share memory, calls from several threads."""
import ctypes as C

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
