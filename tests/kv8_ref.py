"""Plain numpy statements of the 8-bit key-value cache's operators (include/qw_kv8.h): codes bit for bit, attention in 64 bits, the choice of blocks
in whole numbers.  Test infrastructure."""
import numpy as np

PAGE, TINY = 256, np.float32(2.0 ** -100)
LARGEST = {"e4m3": np.float32(448), "int8": np.float32(127)}
_E4M3 = None


def e4m3_values():
    """What the 256 codes stand for; 0x7f and 0xff as 480, which the format's own tables call NaN."""
    global _E4M3
    if _E4M3 is None:
        b = np.arange(256)
        e, m = b >> 3 & 15, b & 7
        v = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
        _E4M3 = np.where(b > 127, -v, v)
    return _E4M3


def values(codes, fmt):
    """uint8 codes -> float64"""
    return e4m3_values()[codes] if fmt == "e4m3" else codes.view(np.int8).astype(np.float64)


def _nearest_e4m3(x):
    """fp32 within +-448 -> codes, to nearest, ties to even."""
    x = x.astype(np.float64)
    a = np.abs(x)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    r = np.round(a / step) * step  # (numpy rounds halves to even; a step is a code's spacing, so r is a code's value)
    code = np.searchsorted(e4m3_values()[:127], r).astype(np.uint8)
    assert np.array_equal(e4m3_values()[code], r)
    return code | (np.signbit(x).astype(np.uint8) << 7)


def quantise(x, fmt):
    """fp32 [..., hd] -> codes, scales as the cache holds them."""
    x = x.astype(np.float32)
    F = LARGEST[fmt]
    a = np.abs(x).max(-1)
    nan, zero = ~np.isfinite(a), a < TINY
    off = nan | zero
    safe = np.where(off, np.float32(1), a)
    inv = np.where(off, np.float32(0), F / safe)
    with np.errstate(invalid="ignore"):
        y = np.where(off[..., None], np.float32(0), np.clip(x * inv[..., None], -F, F))
    codes = _nearest_e4m3(y) if fmt == "e4m3" else np.rint(y).astype(np.int8).view(np.uint8)
    codes = np.where(off[..., None], np.uint8(0) if fmt == "int8" else codes & 0x80 * zero[..., None].astype(np.uint8), codes)
    scale = np.where(nan, np.float32(np.nan), np.where(zero, np.float32(0), safe / F))
    return codes.astype(np.uint8), scale.astype(np.float32)


def bounds(codes, scales, fmt):
    """codes [n, hd], scales [n] of a block's tokens -> lo8, hi8, scale."""
    with np.errstate(invalid="ignore"):
        k = values(codes, fmt).astype(np.float32) * scales[:, None]
    ok = ~np.isnan(scales)
    hd = codes.shape[1]
    lo = k[ok].min(0) if ok.any() else np.zeros(hd, np.float32)
    hi = k[ok].max(0) if ok.any() else np.zeros(hd, np.float32)
    b = np.maximum(np.abs(lo), np.abs(hi)).max()
    zero = b < TINY
    inv = np.float32(0) if zero else np.float32(127) / b
    lo8 = np.maximum(np.float32(-127), np.floor(lo * inv)).astype(np.int8)
    hi8 = np.minimum(np.float32(127), np.ceil(hi * inv)).astype(np.int8)
    return lo8, hi8, np.float32(np.inf) if not ok.all() else np.float32(0) if zero else b / np.float32(127)


def attend(q, k, v, scale, gate=None):
    """float64: q [G, hd], k and v [T, hd] -> y [G, hd] and how far scores computed in fp32 may be off (see tolerance)."""
    if len(k) == 0:
        return np.zeros(q.shape), 0.0
    s = scale * q @ k.T
    p = np.exp(s - s.max(1, keepdims=True))
    y = p @ v / p.sum(1, keepdims=True)
    if gate is not None:
        y = y / (1 + np.exp(-gate))
    return y, scale * (np.abs(q) @ np.abs(k).T).max()


def tolerance(ref, half_step, spread, vmax, hd, tokens):
    """How far a row computed in fp32 may be from `ref`, from the operations that round:
    scores: hd products summed, the row's scale and the softmax scale: (hd + 8) 2^-24 of sum |q k| (`spread`), which moves a weight by twice that;
    exponentials and the weights' 22 bits: 2^-20;  sums over the tokens: sqrt(tokens) + 16 steps of 2^-24 (they are added in groups);
    all of it times the largest value.  Then the last rounding: half a step of the result, or of the smallest normal number."""
    rel = 2 * (hd + 8) * 2.0 ** -24 * spread + 2.0 ** -20 + (tokens ** 0.5 + 16) * 2.0 ** -24
    return half_step * np.abs(ref) * (1 + 2.0 ** -8) + vmax * rel + 2.0 ** -25


def pick(q, recs, hd, n, count, first, last):
    """q fp32 [G, hd], recs uint8 [blocks, 2 hd + 16] in order of the blocks -> ids [count]."""
    a = np.abs(q).max(1)
    none = (a < TINY) | ~np.isfinite(a)
    inv = np.where(none, np.float32(0), np.float32(127) / np.where(none, np.float32(1), a)).astype(np.float32)
    sq = np.where(none, np.float32(0), a / np.float32(127)).astype(np.float32)
    with np.errstate(invalid="ignore"):
        q8 = np.where(none[:, None], 0, np.rint(q * inv[:, None])).astype(np.int64)
    lo, hi = recs[:n, :hd].copy().view(np.int8).astype(np.int64), recs[:n, hd:2 * hd].copy().view(np.int8).astype(np.int64)
    sb = recs[:n, 2 * hd:2 * hd + 4].copy().view(np.float32)[:, 0]
    i = np.maximum(q8, 0) @ hi.T + np.minimum(q8, 0) @ lo.T
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.where(i == 0, np.float32(0), (sq[:, None] * sb[None]).astype(np.float32) * i.astype(np.float32)).max(0)
    s = np.where(np.isposinf(sb), np.float32(np.inf), s)
    b = np.arange(n)
    forced = (b < first) | (b >= n - last)
    order = np.lexsort((b, -s, ~forced))  # forced ones, then by score, then by number
    ids = np.sort(order[:count])
    return np.concatenate([ids, np.full(count - len(ids), -1)]).astype(np.int32)
