"""Attention over fp16 queries, keys and values without scores in memory, with gradients.  What ``bmm``, a position bias, ``mask``, ``softmax`` and ``bmm`` do one after
another (the sequence of the reference's models), in one pass; for training, for chunks of a prompt and for single tokens over a cache of fp16.

    out = attention(q, k, v, causal=True)                               # (batch, heads, tokens, dim), any strides
    out = attention(q, k, v, lens=lens, pos=pos)                        # a decode step over the first lens keys of a buffer
    out = attention(q, k, v, pos=0, bias=pe.weight, mapping=mapping)    # with PositionEmbedding's biases, which get gradients too

Activations of this package are (batch, heads * dim_head, tokens): ``x.view(batch, heads, dim_head, tokens).transpose(2, 3)`` is what goes in, and the result and the
gradients have the same layout in memory.
"""
import math
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from ..library import cpmk          # (the launchers themselves: what the kernels layer checks is checked here)
from ._common import cur_stream, current_device
from .kv_cache import _each

MAX_DIM, MAX_DISTANCES = 256, 1024
_NO_MASK, _NO_TABLE = (None, 0, 0), (None, None, 0, 0, 0)


@lru_cache(maxsize=1024)
def _workspace(device, *sizes):         # (how keys are divided depends on the device's number of compute units; the call costs more than the look-up)
    return cpmk.attention_forward_workspace(*sizes)


_backward_workspace = lru_cache(maxsize=1024)(cpmk.attention_backward_workspace)


def _seen(mask):
    return mask.data_ptr(), mask.stride(0), mask.stride(1) if mask.size(1) > 1 else 0


def _forward(q, k, v, table, seen, rows, sizes, keep):
    """(result, what the backward pass needs besides it)"""
    out = torch.empty_like(q)
    batch, heads, kv_heads, tokens, _, length = sizes
    # (a number for each row, and one for each part of the keys, which are 256 at least)
    lse, rest = (torch.empty(batch * (heads * tokens + kv_heads * (length // 256 + 1)), dtype=torch.float32, device=q.device), torch.empty_like(out)) if keep else (None, None)
    size = _workspace(q.device.index, *sizes)
    space = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    cpmk.attention_forward(*sizes, q.data_ptr(), *q.stride(), k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), *rows, *table, *seen, out.data_ptr(), *out.stride(),
                           lse.data_ptr() if keep else None, rest.data_ptr() if keep else None, space.data_ptr() if size else None, cur_stream())
    return out, lse, rest


class OpAttention(torch.autograd.Function):
    """forward: one pass over the keys; backward: the probabilities computed again from what the forward pass kept of each row, the log
    of its sum and what its result's rounding left."""

    @staticmethod
    def forward(ctx, q, k, v, bias, mapping, mask, lens, pos, table, seen, rows, sizes):
        out, lse, rest = _forward(q, k, v, table, seen, rows, sizes, True)
        ctx.save_for_backward(q, k, v, bias, mapping, mask, out, lse, rest, lens, pos)       # (lens and pos too: the kernels look at them again)
        ctx.plain = (sizes, rows, table, seen)
        return out

    @staticmethod
    def backward(ctx, dout):
        assert not torch.is_grad_enabled(), "the gradients have no gradients"       # (create_graph; a wrapper that refuses it costs 10 us)
        q, k, v, bias, mapping, mask, out, lse, rest, lens, pos = ctx.saved_tensors
        sizes, rows, table, seen = ctx.plain
        # (addresses again: what was saved may have been packed and unpacked meanwhile)
        rows = (None if lens is None else lens.data_ptr(), rows[1], None if pos is None else pos.data_ptr(), *rows[3:])
        if bias is not None:
            table = (bias.data_ptr(), mapping.data_ptr(), *table[2:])
        if mask is not None:
            assert mask.stride(2) == 1 or mask.size(2) <= 1
            seen = _seen(mask)
        assert rest.stride() == out.stride()
        batch, heads, kv_heads, tokens, dim, length = sizes
        current_device(q.device)
        assert dout.dtype == torch.float16
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dbias = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[3] else None
        if batch * heads * dim == 0:
            return (dq, dk, dv, None if dbias is None else dbias.zero_()) + (None,) * 8
        size = _backward_workspace(batch, heads, kv_heads, tokens, length, 0 if dbias is None else mapping.size(0), table[4])
        space = torch.empty(max(size, 4), dtype=torch.uint8, device=q.device)
        cpmk.attention_backward(*sizes, q.data_ptr(), *q.stride(), k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), *rows, *table, *seen, out.data_ptr(), *out.stride(),
                                lse.data_ptr(), rest.data_ptr(), dout.data_ptr(), *dout.stride(), dq.data_ptr(), *dq.stride(), dk.data_ptr(), *dk.stride(), dv.data_ptr(), *dv.stride(),
                                None if dbias is None else dbias.data_ptr(), space.data_ptr(), cur_stream())
        return (dq, dk, dv, dbias) + (None,) * 8


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens=None, scale: float = None, causal: bool = True, pos=None, mask: torch.Tensor = None,
              bias: torch.Tensor = None, mapping: torch.Tensor = None, bidirectional: bool = False) -> torch.Tensor:
    """softmax(scale q k^T + position bias) v, with gradients to q, k, v and bias.  The arguments are those of QuantizedKV.attention.

    q (batch, heads, queries, dim), k and v (batch, kv heads, length, dim), heads a multiple of the kv heads (neighbouring ones share a head of keys); scale: dim ** -0.5.
    lens: the first lens keys of every sequence count (an int, or an int32 tensor with one for each; None: all).
    pos: the first query's position (int, int32 tensor, or None: the queries are the last of the lens keys; sequences padded at their end want pos=0 with their lens);
    causal: keys behind a query's position do not count.
    mask: bool (batch, length) or (batch, 1 or queries, length), True where a key counts.  A query without keys gives zeros, and no gradients.
    bias, mapping, bidirectional: PositionEmbedding's weight (heads, num_buckets) and the table of position_embedding_init.
    The result has the shape of q, and its layout where q is dense; so have the gradients theirs."""
    device = current_device(q.device)
    assert q.dtype == k.dtype == v.dtype == torch.float16 and k.device == device and v.device == device
    batch, heads, queries, dim = q.shape
    shape = k.shape
    assert v.shape == shape and len(shape) == 4 and shape[0] == batch and shape[3] == dim and dim <= MAX_DIM
    kv_heads, length = shape[1:3]
    assert (heads % kv_heads == 0) if kv_heads else heads == 0
    lens_each, keys = (None, length) if lens is None else _each(lens, batch, device)
    assert lens_each is not None or 0 <= keys <= length, "more keys than there are"
    pos_each, first = (None, -1) if pos is None else _each(pos, batch, device)
    assert pos is None or pos_each is not None or 0 <= first < 2 ** 30
    scale = max(dim, 1) ** -0.5 if scale is None else float(scale)
    assert math.isfinite(scale)
    seen, table = _NO_MASK, _NO_TABLE
    if mask is not None:
        assert mask.dtype == torch.bool and mask.device == device
        if mask.ndim == 2:
            mask = mask[:, None]
        assert mask.ndim == 3 and mask.shape[::2] == (batch, length) and mask.size(1) in (1, queries)
        assert mask.stride(2) == 1 or length <= 1
        seen = _seen(mask)
    if bias is not None:
        assert bias.dtype == torch.float16 and bias.ndim == 2 and bias.size(0) == heads and bias.size(1) > 0 and bias.is_contiguous() and bias.device == device
        assert mapping is not None and mapping.dtype == torch.int32 and mapping.ndim == 1 and mapping.is_contiguous() and mapping.device == device
        assert 0 < mapping.size(0) * (2 if bidirectional else 1) <= MAX_DISTANCES
        table = (bias.data_ptr(), mapping.data_ptr(), bias.size(1), mapping.size(0), int(bool(bidirectional)))
    rows = (lens_each, keys, pos_each, first, int(bool(causal)), scale)
    sizes = (batch, heads, kv_heads, queries, dim, length)
    # (an autograd function costs 5 us of the host's time, as much as a step's kernel; one with forward-mode tangents goes through it all the same, and is refused there)
    if getattr(forward_ad, "_current_level", 0) < 0 and not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (bias is not None and bias.requires_grad))):
        return _forward(q, k, v, table, seen, rows, sizes, False)[0]
    return OpAttention.apply(q, k, v, bias, mapping, mask, lens if lens_each is not None else None, pos if pos_each is not None else None, table, seen, rows, sizes)


def attentionTH(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens=None, scale: float = None, causal: bool = True, pos=None, mask: torch.Tensor = None,
                bias: torch.Tensor = None, mapping: torch.Tensor = None, bidirectional: bool = False) -> torch.Tensor:
    """Plain-torch formulation of the same, in fp32 (fp64 for fp64 tensors)."""
    batch, heads, queries, dim = q.shape
    kv_heads, length = k.size(1), k.size(2)
    wide = torch.promote_types(q.dtype, torch.float32)

    def each(x):
        return x.long() if isinstance(x, torch.Tensor) else torch.full((batch,), int(x), dtype=torch.long, device=q.device)
    lens = each(length if lens is None else lens).clamp(0, length)
    at = (lens - queries if pos is None else each(pos))[:, None] + torch.arange(queries, device=q.device)
    key, value = (x.to(wide).repeat_interleave(heads // kv_heads, 1) for x in (k, v))
    scores = torch.matmul(q.to(wide), key.transpose(2, 3)) * (dim ** -0.5 if scale is None else scale)
    index = torch.arange(length, device=q.device)
    rel = at[:, :, None] - index
    if bias is not None:
        far = rel.abs() if bidirectional else rel.clamp(min=0)
        bucket = mapping.long()[far.clamp(max=mapping.size(0) - 1)].clamp(max=bias.size(1))
        if bidirectional:
            bucket = bucket + torch.where(rel < 0, bias.size(1) // 2, 0)
        scores = scores + bias.to(wide)[:, bucket.clamp(0, bias.size(1) - 1)].transpose(0, 1)
    seen = (index < lens[:, None])[:, None].expand_as(rel)
    if causal:
        seen = seen & (rel >= 0)
    if mask is not None:
        seen = seen & (mask[:, None] if mask.ndim == 2 else mask)
    seen = seen[:, None]
    p = torch.softmax(scores.masked_fill(~seen, -1e30), 3) * seen
    return torch.matmul(p, value).to(q.dtype)
