"""Attention over fp16 keys and values, its gradients, and rotary positions in numpy and float64 (the reference has no such operators: parity unpinned), each with a
bound on what a result may be off, derived from the roundings on the way."""
import math

import numpy as np

from .kv_cache import bucket_bias

f64 = np.float64
E16, E32 = 2.0 ** -11, 2.0 ** -24           # half a step, relative
TINY = 2.0 ** -25                           # half a step of the smallest fp16 numbers


def buckets(rel, mapping, count, bidirectional):
    far = np.where(rel < 0, -rel if bidirectional else 0, rel)
    return mapping[np.minimum(far, len(mapping) - 1)] + np.where((rel < 0) & bidirectional, count // 2, 0)


def seen_by(n, length, keys, first, causal, mask):
    """(queries, length) bool; mask (rows, length) or None."""
    rel = first + np.arange(n)[:, None] - np.arange(length)[None]
    seen = np.broadcast_to(np.arange(length) < keys, (n, length)).copy()
    if causal:
        seen &= rel >= 0
    if mask is not None:
        seen &= mask
    return rel, seen


def attention(q, k, v, lens, first, scale, causal, mask=None, table=None, mapping=None, bidirectional=False, dout=None):
    """q (batch, heads, n, dim), k, v (batch, held, length, dim), lens and first (batch) integers, mask (batch, rows, length) or None.
    Without dout (out, bound); with it lists of (out, dq, dk, dv[, dtable]) and of their bounds.

    Roundings: scores are fp32 sums of dim products; exponents and exponentials fp32; probabilities and the scores' gradients rounded to fp16, the first beside a power of two that makes
    their row's largest 2^7 at least, the second beside one that brings 2 |dout| sqrt(dim) max |v| to 2^15; sums fp32; results fp16, D from what their rounding left too."""
    q, k, v = (np.asarray(x, f64) for x in (q, k, v))
    batch, heads, n, dim = q.shape
    length, group = k.shape[2], heads // max(k.shape[1], 1)
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    train = dout is not None
    if train:
        dout = np.asarray(dout, f64)
        grads = [np.zeros(q.shape), np.zeros(k.shape), np.zeros(k.shape)] + ([np.zeros(table.shape)] if table is not None else [])
        offs = [np.zeros(x.shape) for x in grads]
    for b in range(batch):
        keys = max(0, min(int(lens[b]), length))
        rel, seen = seen_by(n, length, keys, int(first[b]), causal, None if mask is None else mask[b])
        rel, seen = rel[:, :keys], seen[:, :keys]
        for h in range(heads):
            Q, K, V = q[b, h], k[b, h // group, :keys], v[b, h // group, :keys]
            with np.errstate(invalid="ignore", over="ignore"):
                x = Q @ K.T * scale
                size = np.abs(Q) @ np.abs(K).T * abs(scale)
            bias = np.zeros_like(x)
            if table is not None:
                bias = bucket_bias(table[h], mapping, rel, bidirectional)
                x = x + bias
            x = np.where(seen, x, -np.inf)
            top = x.max(1, initial=-np.inf, keepdims=True)
            p = np.exp(x - np.where(np.isfinite(top), top, 0))
            total = p.sum(1, keepdims=True)
            empty = total == 0
            p = p / np.where(empty, 1, total)
            Vs = np.where(seen.any(0)[:, None], V, 0)
            o = p @ Vs
            out[b, h] = o
            # relative error of a probability: chains of dim additions, the exponent's roundings (|x|, |bias| and the statistics), the exponential
            off = np.where(seen, size * (dim + 8) * E32 + (np.abs(np.where(seen, x, 0)) + np.abs(bias) + 32) * 2.0 ** -22, 0).max(1, initial=0, keepdims=True)
            weight = p @ np.abs(Vs)
            count = seen.sum(1, keepdims=True)
            bo = weight * (E16 + 2 * off + 2 * (count + 64) * E32) + count * 2.0 ** -32 * p.max(1, initial=0, keepdims=True) * np.abs(Vs).max(0, initial=0)[None] + np.abs(o) * E16 + TINY
            bound[b, h] = bo
            if not train:
                continue
            G = np.where(empty, 0, dout[b, h])
            dp = np.where(seen, G @ np.where(seen.any(0)[:, None], V, 0).T, 0)
            D = (G * o).sum(1, keepdims=True)           # of a result whose roundings were kept: fp32, but for 2^-11 of 2^-11
            least = count * 2.0 ** -32 * p.max(1, initial=0, keepdims=True) * np.abs(Vs).max(0, initial=0)[None]
            bD = weight * (2 * off + 2.0 ** -21 + 2 * (count + 64) * E32) + least + np.abs(o) * 2.0 ** -21 + 2.0 ** -36
            ds = p * (dp - D)
            e_p = p * (2 * off + 2.0 ** -21)                        # of a probability before it is rounded
            e_dp = (np.abs(G) @ np.abs(Vs).T) * (dim + 8) * E32
            e_D = (np.abs(G) * bD).sum(1, keepdims=True) + (np.abs(G) * np.abs(o)).sum(1, keepdims=True) * (dim + 8) * E32
            e_ds = np.where(seen, e_p * np.abs(dp - D) + p * (e_dp + e_D), 0)
            norms = np.sqrt((G ** 2).sum(1, keepdims=True))
            # ds is taken times 2^e, with 2 |do| sqrt(dim) max |v| 2^e in [1/2, 1], over the finite values of the sequence's keys, masked or not (|v| <= sqrt(dim) max |v|), and p
            # times 2^15: half a step of the smallest fp16 numbers, 2^-25, is 2^-25 2^-15 2^-e <= 2^-40 4 |do| sqrt(dim) max |v| of ds
            finite = np.abs(v[b, h // group, :keys])
            vtop = math.sqrt(dim) * np.where(np.isfinite(finite), finite, 0).max(initial=0)
            own = np.where(seen, 4 * norms * vtop * 2.0 ** -40, 0)
            gtop = np.sqrt((dout[b, h // group * group:(h // group + 1) * group] ** 2).sum(-1)).max(initial=0)
            all_ = np.where(seen, 4 * gtop * vtop * 2.0 ** -40, 0)
            c = abs(scale)
            rounded = np.abs(ds) * E16
            grads[0][b, h] = scale * ds @ K
            offs[0][b, h] = c * ((e_ds + rounded + own + np.abs(ds) * (keys + 64) * E32) @ np.abs(K))
            grads[1][b, h // group, :keys] += scale * ds.T @ Q
            offs[1][b, h // group, :keys] += c * ((e_ds + rounded + all_ + np.abs(ds) * (group * n + 64) * E32).T @ np.abs(Q))
            grads[2][b, h // group, :keys] += p.T @ G
            offs[2][b, h // group, :keys] += (e_p + p * E16 + np.where(seen, 2.0 ** -40, 0) + p * (group * n + 64) * E32).T @ np.abs(G)
            if table is not None:
                which = buckets(rel, mapping, table.shape[1], bidirectional)
                grads[3][h] += np.bincount(which.ravel(), ds.ravel(), table.shape[1])
                offs[3][h] += np.bincount(which.ravel(), (e_ds + np.abs(ds) * (batch * n + keys + 64) * E32).ravel(), table.shape[1])
    if not train:
        return out, bound
    return [out] + grads, [bound] + [o + np.abs(g) * E16 + TINY for g, o in zip(grads, offs)]


def rotary(x, positions, turns, magnitude, interleaved, inverse=False):
    """x (batch, heads, tokens, dim), positions (batch, tokens) integers, turns (pairs): (turned, bound).  Angles lose 2^-24 of a turn at most where they become fp32."""
    x = np.asarray(x, f64)
    r = 2 * len(turns)
    at = np.asarray(positions, f64)[:, None, :, None] * np.asarray(turns, f64)
    angle = 2 * math.pi * (at - np.round(at)) * (-1 if inverse else 1)
    cos, sin = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    one, other = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    out, bound = x.copy(), np.zeros(x.shape)
    a, b = x[..., one], x[..., other]
    out[..., one], out[..., other] = a * cos - b * sin, a * sin + b * cos
    # the angle's: 2 pi 2^-25 of its fp32 form, |position| turns 2^-53 of its fp64 one; cosine, products and sum in fp32
    lost = (np.abs(a) + np.abs(b)) * magnitude * (2 * math.pi * 2.0 ** -25 + np.abs(at) * 2 * math.pi * 2.0 ** -52 + 8 * E32)
    bound[..., one], bound[..., other] = lost, lost
    bound[..., :r] += np.abs(out[..., :r]) * E16 + TINY
    return out, bound
