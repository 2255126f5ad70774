"""Plain statements in 64 bits of block means, block selection and attention over listed blocks, for the tests of
`ane_fieldfare_b200.attention`.  Nothing here calls the library."""
import numpy as np

BLOCK = 64


def exponent(x):
    """floor(log2) of the largest magnitude along the last dimension (kept), -2000 for none."""
    top = np.abs(x).max(-1, keepdims=True)
    return np.where(top > 0, np.frexp(np.where(np.isfinite(top), top, 1.0))[1] - 1, -2000)


def held(x, e):
    """x in whole numbers of 2^(e - 6), to the nearest (ties to even), at most 127 of them."""
    step = np.ldexp(1.0, np.asarray(e) - 6)
    return np.clip(np.rint(x / step), -127, 127) * step


def block_mean(keys):
    """keys [64][dim] of a head -> the mean as it is held."""
    if not np.isfinite(keys).all():
        return np.full(keys.shape[1], np.nan)
    mean = keys.sum(0) / BLOCK
    return held(mean, np.clip(exponent(mean), -60, 60))


def query(q):
    """Queries [group][dim] of a row that share a head -> as they are scored (times a power of two common to them)."""
    fine = np.isfinite(q).all(-1, keepdims=True)
    q = np.where(fine, q, 0.0)
    e = np.where(fine, np.maximum(exponent(q), -100), -2000)
    top = max(-100, e.max())
    e = np.maximum(e, top - 60)
    return held(q, e) * 2.0 ** -top


def choose(scores, seen, blocks, first, last):
    """Ids of one list, -1 behind; scores of the blocks 0 .. seen - 1 (NaN before all)."""
    if seen <= blocks:
        chosen = list(range(seen))
    else:
        middle = range(first, seen - last)
        key = {b: (0 if np.isnan(scores[b]) else 1, -scores[b] if not np.isnan(scores[b]) else 0.0, b) for b in middle}
        best = sorted(middle, key=lambda b: key[b])[:blocks - first - last]
        chosen = list(range(first)) + sorted(best) + list(range(seen - last, seen))
    return chosen + [-1] * (blocks - len(chosen))


def select(q, meansOf, lengths, rows, kvHeads, blocks, first, last, most=1 << 30):
    """q float64 [tokens][heads][dim]; meansOf[r] [blocks][kvHeads][dim] of request r; at most `most` blocks have room."""
    tokens, heads, dim = q.shape
    out = np.full((tokens, kvHeads, blocks), -1, dtype=np.int64)
    at = 0
    for r, (n, m) in enumerate(zip(lengths, rows)):
        for i in range(m):
            p = n - m + i
            seen = min(p // BLOCK + 1, most) if p >= 0 else 0
            for h in range(kvHeads):
                group = heads // kvHeads
                part = query(q[at + i, h * group:(h + 1) * group])
                means = meansOf[r][:max(0, seen - last), h]
                with np.errstate(invalid="ignore"):
                    scores = (part @ means.T).max(0) if len(means) else np.zeros(0)
                out[at + i, h] = choose(scores, seen, blocks, first, last)
        at += m
    return out


def attention_listed(q, keys, values, slotsOf, lengths, rows, ids, scale):
    """Attention over the keys of listed blocks up to the row's own, a block named twice counting twice; like
    attention_reference.attention (out, bound)."""
    tokens, heads, dim = q.shape
    kvHeads = keys.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    first = 0
    for r, (n, m) in enumerate(zip(lengths, rows)):
        at = np.asarray(slotsOf[r][:n], dtype=np.int64)
        for i in range(m):
            p = n - m + i
            for h in range(heads):
                g = h // (heads // kvHeads)
                j = np.concatenate([np.arange(b * BLOCK, b * BLOCK + BLOCK) for b in ids[first + i, g] if b >= 0] or [np.zeros(0, dtype=np.int64)])
                j = j[j <= p].astype(np.int64)
                if not len(j):
                    continue
                k, v = keys[at[j], g], values[at[j], g]
                with np.errstate(invalid="ignore"):
                    s = scale * (k @ q[first + i, h])
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[first + i, h] = w @ v
                    loud = scale * np.abs(k) @ np.abs(q[first + i, h])
                    bound[first + i, h] = 2.0 ** -10 * (1 + loud.max()) * (w @ np.abs(v))
        first += m
    return out, bound
