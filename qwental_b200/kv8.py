"""Python face of the 8-bit key-value cache (include/qw_kv8.h) for hosts that hold their memory as torch tensors: rows in and out,
attention of one new token per row, and the choice of blocks.  All work happens in libqw_gpu_cuda.so, on torch's current stream (or the
one that is given, as a cudaStream_t); nothing waits, and every call may be captured into a CUDA graph.  Tensors have to outlive the work on them: one that was made on
another stream than the call's is the caller's to record there.  Errors raise Kv8Error with the library's message.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import lib as _lib

PAGE = 256
FORMATS = {"e4m3": 0, "int8": 1}
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


class Kv8Error(RuntimeError):
    pass


def _raw_stream(index):
    """The cudaStream_t of torch's current stream (torch.cuda.current_stream() builds an object around it, 3 us)."""
    get = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return get(index) if get is not None else torch.cuda.current_stream(index).cuda_stream


def _in_32_bits(a, b=0, c=0, d=0):
    """ctypes would cut larger or negative numbers down to 32 bits without a word."""
    if not (0 <= a <= 0xffffffff and 0 <= b <= 0xffffffff and 0 <= c <= 0xffffffff and 0 <= d <= 0xffffffff):
        raise Kv8Error("a layer, length or number of blocks, rows or heads that 32 bits do not hold")


class CacheStruct(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("codes", "scales", "bounds", "page_table", "status")] + \
               [(n, C.c_uint32) for n in ("pages", "layers", "kvh", "hd", "format", "block", "slots", "max_pages")]


class RowsStruct(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "slots", "pos")] + [(n, C.c_int64) for n in ("k_row", "k_head", "v_row", "v_head")] + \
               [(n, C.c_uint32) for n in ("nb", "layer", "dtype", "reserved")]


class AttnStruct(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "gate", "y", "lens", "slots", "blocks", "work")] + [("work_bytes", C.c_size_t)] + \
               [(n, C.c_int64) for n in ("q_row", "q_head", "gate_row", "gate_head", "y_row", "y_head")] + [("scale", C.c_float)] + \
               [(n, C.c_uint32) for n in ("nb", "layer", "dtype", "qh", "max_len", "nblocks", "reserved")]


class PickStruct(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q", "lens", "slots", "blocks", "work")] + [("work_bytes", C.c_size_t), ("q_row", C.c_int64), ("q_head", C.c_int64)] + \
               [(n, C.c_uint32) for n in ("nb", "layer", "dtype", "qh", "max_len", "nblocks", "first", "last")]


class SizesStruct(C.Structure):
    """The sizes a batch's kv8 families take (bind 15)."""
    _fields_ = [(n, C.c_uint32) for n in ("pages", "layers", "kvh", "hd", "format", "block", "slots", "max_pages",
                                          "nb", "layer", "dtype", "qh", "max_len", "nblocks", "first", "last")] + [("scale", C.c_float)]


def bind():
    L = _lib.load()
    vp, sz, u = C.c_void_p, C.c_size_t, C.c_uint32
    P = C.POINTER
    for name, res, args in (("qw_kv8_bytes", C.c_int, [P(CacheStruct), P(sz * 3)]), ("qw_kv8_put", C.c_int, [P(CacheStruct), P(RowsStruct), vp, C.c_char_p, sz]),
                            ("qw_kv8_get", C.c_int, [P(CacheStruct), P(RowsStruct), vp, C.c_char_p, sz]),
                            ("qw_kv8_attn", C.c_int, [P(CacheStruct), P(AttnStruct), vp, C.c_char_p, sz]), ("qw_kv8_attn_work", sz, [P(CacheStruct), u, u, u, u]),
                            ("qw_kv8_pick", C.c_int, [P(CacheStruct), P(PickStruct), vp, C.c_char_p, sz]), ("qw_kv8_pick_work", sz, [P(CacheStruct), u, u]),
                            ("qw_kv8_row_index", C.c_int64, [P(CacheStruct), C.c_int64, C.c_int64, C.c_int64, u, u, u])):
        f = getattr(L, name)
        f.restype, f.argtypes = res, args
    return L


class Kv8Cache:
    """The tensors of one cache: codes uint8 [pages, layers, 2, kvh, 256, hd], scales float32 [pages, layers, 2, kvh, 256], page_table int32
    [slots, max_pages] and, for `pick` and chosen blocks, bounds uint8 [pages, layers, kvh, 256 / block, 2 hd + 16].  It keeps no copy: page ids may
    be written into page_table between calls, on the same stream."""

    def __init__(self, codes, scales, page_table, bounds=None, *, format="e4m3", block=None, status=None):
        self.L = bind()
        if format not in FORMATS:
            raise Kv8Error("unknown format %r" % (format,))
        if codes.dim() != 6 or codes.shape[2] != 2 or codes.shape[4] != PAGE or codes.dtype != torch.uint8:
            raise Kv8Error("codes are uint8 [pages, layers, 2, kv heads, 256, head dim]")
        pages, layers, _, kvh, _, hd = codes.shape
        if tuple(scales.shape) != (pages, layers, 2, kvh, PAGE) or scales.dtype != torch.float32:
            raise Kv8Error("scales are float32 [pages, layers, 2, kv heads, 256]")
        if page_table.dim() != 2 or page_table.dtype != torch.int32:
            raise Kv8Error("page_table is int32 [slots, max_pages]")
        if bounds is not None:
            if bounds.dim() != 5 or bounds.shape[3] < 1 or tuple(bounds.shape) != (pages, layers, kvh, bounds.shape[3], 2 * hd + 16) or bounds.dtype != torch.uint8:
                raise Kv8Error("bounds are uint8 [pages, layers, kv heads, 256 / block, 2 hd + 16]")
            if bounds.shape[3] > PAGE or PAGE % bounds.shape[3] or block not in (None, PAGE // bounds.shape[3]):
                raise Kv8Error("bounds are of another block size")
            block = PAGE // bounds.shape[3]
        if status is not None and (status.numel() < 1 or status.element_size() != 4):
            raise Kv8Error("status is one 32-bit word")
        _in_32_bits(*page_table.shape)
        self.tensors = (codes, scales, bounds, page_table, status)
        self.device = codes.device
        self.index = codes.get_device()
        for t in self.tensors:
            if t is not None and (t.device != self.device or not t.is_contiguous()):
                raise Kv8Error("a cache's tensors are contiguous and on one device")
        ptr = [None if t is None else t.data_ptr() for t in self.tensors]
        self.c = CacheStruct(*ptr, pages, layers, kvh, hd, FORMATS[format], block or 64, page_table.shape[0], page_table.shape[1])
        self.kvh, self.hd, self.slots, self.max_pages = kvh, hd, page_table.shape[0], page_table.shape[1]
        self._local = threading.local()  # a buffer for messages per thread: the library writes it while other threads run
        self._ref = C.byref(self.c)
        if self.L.qw_kv8_bytes(C.byref(self.c), (C.c_size_t * 3)()):
            raise Kv8Error("a cache of these sizes is not supported (head dim 64, 128 or 256; blocks of 16 to 256 tokens)")

    # ---- arguments
    def _index(self, t, nb, what):
        if t.dtype is not torch.int32 or t.shape != (nb,) or not t.is_contiguous() or t.get_device() != self.index:
            raise Kv8Error("%s is int32 [%d] on the cache's device" % (what, nb))
        return t.data_ptr()

    def _rows(self, t, nb, heads, dtype, what):
        if t.shape != (nb, heads, self.hd) or t.dtype is not dtype or t.get_device() != self.index:
            raise Kv8Error("%s is %s [%d, %d, %d] on the cache's device" % (what, dtype, nb, heads, self.hd))
        row, head, one = t.stride()
        if one != 1:
            raise Kv8Error("the last dimension of %s is contiguous" % what)
        return t.data_ptr(), row, head

    def _blocks(self, t, nb):
        if t.dtype is not torch.int32 or t.dim() != 3 or t.shape[0] != nb or t.shape[1] != self.kvh or not t.is_contiguous() or t.get_device() != self.index:
            raise Kv8Error("blocks are int32 [%d, %d, n] on the cache's device" % (nb, self.kvh))
        if t.shape[2] < 1:  # (its address is 0, which to the library is a call without a list)
            raise Kv8Error("a list has room for one block at least")
        _in_32_bits(t.shape[2])
        return t.data_ptr(), t.shape[2]

    def _work(self, work, need, stream):
        if work is None:
            if stream is not None:  # it would go back to torch's allocator while that stream still uses it
                raise Kv8Error("a call on a stream that is given needs a workspace that is given")
            work = torch.empty(max(16, need), dtype=torch.uint8, device=self.device)
        if work.get_device() != self.index or not work.is_contiguous():
            raise Kv8Error("the workspace is contiguous and on the cache's device")
        return work, work.data_ptr(), work.numel() * work.element_size()

    def _call(self, fn, args, stream):
        if self.index < 0:
            raise Kv8Error("the cache is not in device memory (this library has no CPU path)")
        if stream is None:
            stream = _raw_stream(self.index)
        err = getattr(self._local, "err", None)
        if err is None:
            err = self._local.err = C.create_string_buffer(256)
        if torch.cuda.current_device() == self.index:
            rc = fn(self._ref, C.byref(args), stream, err, 256)
        else:
            with torch.cuda.device(self.device):
                rc = fn(self._ref, C.byref(args), stream, err, 256)
        if rc:
            raise Kv8Error(err.value.decode())

    @staticmethod
    def _dtype(t, what):
        d = _DTYPES.get(t.dtype)
        if d is None:
            raise Kv8Error("%s is float16 or bfloat16" % what)
        return d

    # ---- calls
    def work_bytes(self, nb, qh, max_len, blocks=0):
        """A workspace that serves pick and attn for these sizes, over everything or any list of blocks; given `blocks`, over lists of so many only."""
        _in_32_bits(nb, qh, max_len, blocks)
        n = self.L.qw_kv8_attn_work(C.byref(self.c), nb, qh, max_len, blocks)
        if n == 0:
            raise Kv8Error("sizes that the calls refuse")
        return max(n, self.L.qw_kv8_pick_work(C.byref(self.c), nb, max_len))

    def _rows_call(self, fn, k, v, slots, pos, layer, stream):
        nb, dt = slots.shape[0], self._dtype(k, "k")
        _in_32_bits(nb, layer)
        kp, kr, kh = self._rows(k, nb, self.kvh, k.dtype, "k")
        vp, vr, vh = self._rows(v, nb, self.kvh, k.dtype, "v")
        self._call(fn, RowsStruct(kp, vp, self._index(slots, nb, "slots"), self._index(pos, nb, "pos"), kr, kh, vr, vh, nb, layer, dt), stream)

    def put(self, k, v, slots, pos, layer=0, stream=None):
        """Quantises rows k, v [nb, kvh, hd] into position pos[r] of slot slots[r], and renews the bounds of their blocks."""
        self._rows_call(self.L.qw_kv8_put, k, v, slots, pos, layer, stream)

    def get(self, k, v, slots, pos, layer=0, stream=None):
        """Reads rows back into k, v [nb, kvh, hd]."""
        self._rows_call(self.L.qw_kv8_get, k, v, slots, pos, layer, stream)

    def attn(self, q, lens, slots, y, layer=0, *, max_len, scale=None, gate=None, blocks=None, work=None, stream=None):
        """y [nb, qh, hd] = attention of q over the first lens[r] tokens of slot slots[r] (of the blocks [nb, kvh, n], if given), times sigmoid(gate)."""
        nb, qh, dt = lens.shape[0], q.shape[1] if q.dim() == 3 else 0, self._dtype(q, "q")
        _in_32_bits(nb, qh, layer, max_len)
        qp, qr, qd = self._rows(q, nb, qh, q.dtype, "q")
        yp, yr, yd = self._rows(y, nb, qh, q.dtype, "y")
        gp, gr, gd = (None, 0, 0) if gate is None else self._rows(gate, nb, qh, q.dtype, "gate")
        bp, nblocks = (None, 0) if blocks is None else self._blocks(blocks, nb)
        work, wp, size = self._work(work, self.L.qw_kv8_attn_work(self._ref, nb, qh, max_len, nblocks) if work is None else 0, stream)
        self._call(self.L.qw_kv8_attn, AttnStruct(qp, gp, yp, self._index(lens, nb, "lens"), self._index(slots, nb, "slots"), bp, wp, size, qr, qd, gr, gd, yr, yd,
                                                  self.hd ** -0.5 if scale is None else scale, nb, layer, dt, qh, max_len, nblocks), stream)
        return y

    def pick(self, q, lens, slots, blocks, layer=0, *, max_len, first=0, last=1, work=None, stream=None):
        """blocks [nb, kvh, n]: the block numbers with the best scores for q, ascending, the first `first` and the last `last` always among them."""
        nb, qh, dt = lens.shape[0], q.shape[1] if q.dim() == 3 else 0, self._dtype(q, "q")
        _in_32_bits(nb, qh, layer, max_len)
        _in_32_bits(first, last)
        qp, qr, qd = self._rows(q, nb, qh, q.dtype, "q")
        bp, nblocks = self._blocks(blocks, nb)
        work, wp, size = self._work(work, self.L.qw_kv8_pick_work(self._ref, nb, max_len) if work is None else 0, stream)
        self._call(self.L.qw_kv8_pick, PickStruct(qp, self._index(lens, nb, "lens"), self._index(slots, nb, "slots"), bp, wp, size, qr, qd, nb, layer, dt, qh, max_len, nblocks,
                                                  first, last), stream)
        return blocks
