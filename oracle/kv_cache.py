"""The key/value cache in 8 bits in numpy and float64, one sequence and head at a time (the reference has no such cache: parity unpinned).

Caches are token-major here, (batch, heads, length, dim); `by_sixteen` gives the layout that values have in memory."""
import numpy as np

f64 = np.float64


def by_sixteen(ints):
    b, h, n, d = ints.shape
    return np.ascontiguousarray(ints.reshape(b, h, n // 16, 16, d).swapaxes(3, 4))


def by_token(values):
    b, h, n, d, _ = values.shape
    return np.ascontiguousarray(values.swapaxes(3, 4).reshape(b, h, n * 16, d))


def nearest(num, den):
    """num / den to the nearest integer, halves away from zero, 0 for a den of 0."""
    q = np.divide(num, den, out=np.zeros(np.broadcast_shapes(np.shape(num), np.shape(den))), where=den != 0)
    return np.where(q < 0, np.ceil(q - 0.5), np.floor(q + 0.5))


def finite(x):
    """Infinities as the largest finite numbers, NaN as 0."""
    return np.nan_to_num(np.asarray(x, dtype=f64), nan=0.0, posinf=65504.0, neginf=-65504.0)


def write(ints, absmax, x, pos, count):
    """In place: ints (batch, heads, length, dim) int8, absmax (batch, heads, blocks) fp16; x (batch, heads, tokens, dim) fp16, pos and count (batch)."""
    length = ints.shape[2]
    block = length // absmax.shape[2]
    x = finite(x)
    for b in range(ints.shape[0]):
        p, n = int(pos[b]), min(int(count[b]), x.shape[2])
        if p < 0:
            continue
        end = min(p + n, length)
        t = p
        while t < end:
            blk = t // block
            stop = min(end, (blk + 1) * block)
            new = x[b, :, t - p:stop - p]
            top = np.abs(new).max(axis=(1, 2))
            if t > blk * block:
                old = np.abs(absmax[b, :, blk]).astype(f64)
                top = np.maximum(top, old)
                part = ints[b, :, blk * block:t].astype(f64)
                ints[b, :, blk * block:t] = nearest(part * old[:, None, None], top[:, None, None]).astype(np.int8)
            ints[b, :, t:stop] = nearest(127 * new, top[:, None, None]).astype(np.int8)
            absmax[b, :, blk] = top.astype(np.float16)
            t = stop


def values_of(ints, absmax):
    block = ints.shape[2] // absmax.shape[2]
    return ints.astype(f64) * np.repeat(absmax.astype(f64), block, axis=2)[..., None] / 127


def read(ints, absmax, start, tokens):
    """float64 (batch, heads, tokens, dim)"""
    whole = values_of(ints, absmax)
    out = np.zeros(ints.shape[:2] + (tokens, ints.shape[3]))
    for b in range(ints.shape[0]):
        for i in range(tokens):
            if 0 <= start[b] + i < ints.shape[2]:
                out[b, :, i] = whole[b, :, start[b] + i]
    return out


def bucket_bias(table, mapping, rel, bidirectional):
    """table (buckets), rel integer array -> float64 (cuda/position_bucket.cu:38-54)"""
    far = np.where(rel < 0, -rel if bidirectional else 0, rel)
    index = mapping[np.minimum(far, len(mapping) - 1)] + np.where((rel < 0) & bidirectional, len(table) // 2, 0)
    return table.astype(f64)[index]


def attention(q, keys, values, key_absmax, value_absmax, lens, scale, causal, pos=None, mask=None, table=None, mapping=None, bidirectional=False):
    """(out, bound) in float64: the formula's result, and how far a result may be off whose scores are fp32 sums, whose probabilities are
    rounded to fp16 beside the largest product of a probability and its value's magnitude, and whose sums are fp32."""
    batch, heads, n, dim = q.shape
    group = heads // keys.shape[1]
    K, V = values_of(keys, key_absmax), values_of(values, value_absmax)
    block = keys.shape[2] // key_absmax.shape[2]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(batch):
        length = max(0, min(int(lens[b]), keys.shape[2]))
        first = length - n if pos is None else int(pos[b])
        for h in range(heads):
            k, v = K[b, h // group, :length], V[b, h // group, :length]
            s = np.repeat(value_absmax[b, h // group].astype(f64), block)[:length] / 127
            for i in range(n):
                at = first + i
                seen = np.ones(length, dtype=bool)
                if causal:
                    seen &= np.arange(length) <= at
                if mask is not None:
                    seen &= mask[b, min(i, mask.shape[1] - 1), :length]
                if not seen.any():
                    continue
                row = q[b, h, i].astype(f64)
                x = k[seen] @ row * scale
                bias = 0.0
                if table is not None:
                    bias = bucket_bias(table[h], mapping, at - np.arange(length)[seen], bidirectional)
                    x = x + bias
                p = np.exp(x - x.max())
                total = p.sum()
                out[b, h, i] = p @ v[seen] / total
                size = p @ np.abs(v[seen]) / total
                # exponent: fp32 chains of dim additions; the factor, the product, the bias and log2 of the magnitude (|.| <= 40) rounded once each
                off = ((np.abs(k[seen]) @ np.abs(row)) * abs(scale) * (dim + 8) * 2.0 ** -24 + (np.abs(x) + np.abs(bias) + 40) * 2.0 ** -22).max()
                count = seen.sum()
                bound[b, h, i] = size * (2.0 ** -11 + 2 * off + 2 * (count + 64) * 2.0 ** -24) + \
                    count * 127 * 2.0 ** -25 * (p * s[seen]).max() / total + np.abs(out[b, h, i]) * 2.0 ** -11 + 2.0 ** -25
    return out, bound
