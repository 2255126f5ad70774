"""Plain statements of the INT4 cache and its attention in 64 bits, for the tests of `ane_fieldfare_b200.attention`.

Nothing here calls the library.  A cache is the bytes of its pages; `unpack` says what they stand for."""
import numpy as np

GROUP = 64


def to_bf16(x):
    """float64 -> the nearest bf16 (ties to even), as float64.  NaN and infinities stay."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        f = x.astype(np.float32)
        # a second rounding is harmless only where the first was exact enough: nudge to odd
        back = f.astype(np.float64)
        bits = f.view(np.uint32).astype(np.int64)
        inexact = np.isfinite(x) & np.isfinite(back) & (back != x)
        toward = np.where(np.abs(back) > np.abs(x), -1, 0)
        bits = np.where(inexact, (bits + toward) | 1, bits)
        rounded = (bits + 0x7FFF + ((bits >> 16) & 1)) & 0xFFFF0000
        out = rounded.astype(np.uint32).view(np.float32).astype(np.float64)
    return np.where(np.isfinite(x), out, x)


def unpack(pages, kvHeads, dim, pageTokens):
    """pages uint8 [n][kvHeads][block] -> (keys, values) float64 [n * pageTokens][kvHeads][dim]."""
    n = pages.shape[0]
    codeBytes, wordBytes = pageTokens * dim // 2, pageTokens * dim // 16
    flat = np.ascontiguousarray(pages).reshape(n, kvHeads, 2, codeBytes + wordBytes)
    codes = flat[..., :codeBytes].reshape(n, kvHeads, 2, pageTokens, dim // 2)
    both = np.stack([codes & 15, codes >> 4], axis=-1).reshape(n, kvHeads, 2, pageTokens, dim).astype(np.float64)
    words = np.ascontiguousarray(flat[..., codeBytes:]).view(np.uint32).reshape(n, kvHeads, 2, pageTokens, dim // GROUP)
    scale = (words << 16).view(np.float32).astype(np.float64)
    bias = (words & 0xFFFF0000).astype(np.uint32).view(np.float32).astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        value = both * np.repeat(scale, GROUP, -1) + np.repeat(bias, GROUP, -1)
    value = value.transpose(2, 0, 3, 1, 4).reshape(2, n * pageTokens, kvHeads, dim)
    return value[0], value[1]


def quantized(x):
    """(codes, scale, bias, value) of heads [..., dim] (float64 holding bf16 numbers); NaN throughout a group that has no code."""
    g = x.reshape(x.shape[:-1] + (-1, GROUP))
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        low, high = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
        step = (high.astype(np.float32) - low.astype(np.float32)) / np.float32(15)
        scale = to_bf16(step)
        whole = np.isfinite(g).all(-1, keepdims=True) & np.isfinite(scale) & (scale < 3.4e38)
        inverse = np.where(scale > 0, np.float32(1) / scale.astype(np.float32), np.float32(0)).astype(np.float32)
        code = np.rint((g.astype(np.float32) - low.astype(np.float32)) * inverse)
        code = np.where(np.isnan(code), 0, np.clip(code, 0, 15)).astype(np.float64)
        value = np.where(whole, code * scale + low, np.nan)
    return np.where(whole, code, 0).reshape(x.shape), scale, low, value.reshape(x.shape)


def attention(q, keys, values, slotsOf, lengths, rows, window, sinks, scale):
    """q float64 [tokens][heads][dim]; slotsOf[r]: slots of request r's keys in order.  Returns (out, bound): the exact rows
    and, per element, how far 16-bit operands with 11 significant bits and 32-bit sums may take them, without the last
    rounding: every weight off by twice the roundings of its logit (2^-11 of sum |q k|, twice for the numerator and the
    sum), one rounding each of weight and value."""
    tokens, heads, dim = q.shape
    kvHeads = keys.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    first = 0
    for r, (n, m) in enumerate(zip(lengths, rows)):
        at = np.asarray(slotsOf[r][:n], dtype=np.int64)
        for i in range(m):
            p = n - m + i
            j = np.arange(n)
            seen = j <= p
            if window:
                seen &= (j > p - window) | (j < sinks)
            pick = at[seen]
            if not len(pick):
                continue
            for h in range(heads):
                k, v = keys[pick, h // (heads // kvHeads)], values[pick, h // (heads // kvHeads)]
                with np.errstate(invalid="ignore"):
                    s = scale * (k @ q[first + i, h])
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[first + i, h] = w @ v
                    size = w @ np.abs(v)
                    loud = scale * np.abs(k) @ np.abs(q[first + i, h])
                    bound[first + i, h] = 2.0 ** -10 * (1 + loud.max()) * size
        first += m
    return out, bound


def plan(old, new, table, free, count, pageTokens, rows):
    """The book-keeping, one page after the other; returns (table, free, count, rowStart, positions, slots)."""
    table, free = table.copy(), free.copy()
    pages = lambda n: -(-n // pageTokens)  # noqa: E731
    for r, (a, b) in enumerate(zip(old, new)):
        for i in range(pages(b), pages(a)):
            free[count] = table[r, i]
            count += 1
    start, positions, slots = [0], [], []
    for r, (a, b) in enumerate(zip(old, new)):
        for i in range(pages(a), pages(b)):
            count -= 1
            table[r, i] = free[count]
        for p in range(a, b):
            positions.append(p)
            slots.append(table[r, p // pageTokens] * pageTokens + p % pageTokens)
        start.append(len(positions))
    pad = rows - len(positions)
    return table, free, count, start, positions + [0] * pad, slots + [-1] * pad
