"""Key/value cache in 8 bits with a magnitude for each block of tokens and head.  For inference: no gradients.

    cache = QuantizedKV.empty(batch, heads, length, dim_head)
    cache.write(k, v, 0)                              # a prompt: k, v (batch, heads, tokens, dim_head), any strides
    ctx = cache.attention(q, tokens)                  # its queries, causal
    for pos in range(tokens, ...):                    # decode
        cache.write(k, v, pos)
        ctx = cache.attention(q, pos + 1)

Activations of this package are (batch, heads * dim_head, tokens): ``k.view(batch, heads, dim_head, tokens).transpose(2, 3)`` is what goes
in, and a result for such queries has the same layout in memory.
"""
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from ..kernels.kv_cache import BLOCKS
from ..library import cpmk          # (the launchers themselves: what the kernels layer checks is checked here, and a layer of forty arguments costs 1 us)
from ._common import cur_stream, _device


def _check_gradients(x: torch.Tensor):
    assert not (x.requires_grad and torch.is_grad_enabled()), "the cache keeps no gradients"
    # (no level of forward mode is entered, as a rule, and none is a look at one number; tangents count under no_grad too)
    assert getattr(forward_ad, "_current_level", 0) < 0 or forward_ad.unpack_dual(x).tangent is None, "the cache keeps no gradients, nor those of forward mode"


def _check_tokens(x: torch.Tensor, device):
    assert x.dtype == torch.float16 and x.device == device
    _check_gradients(x)


@lru_cache(maxsize=1024)
def _workspace(device, *sizes):         # (how keys are divided depends on the device's number of compute units; the call costs more than the look-up)
    return cpmk.kv_attention_int8_workspace(*sizes)


def _each(x, batch, device):
    """(address, number) of something that is the same for every sequence or an int32 tensor with one value each."""
    if isinstance(x, torch.Tensor):
        assert x.dtype == torch.int32 and x.shape == (batch,) and x.is_contiguous() and x.device == device
        return x.data_ptr(), 0
    number = int(x)
    assert number == x, "positions and lengths are integers"
    return None, number


class QuantizedKV:
    """keys (batch, heads, length, dim) int8; values (batch, heads, length / 16, dim, 16) int8, sixteen tokens of a unit side by side;
    key_absmax, value_absmax (batch, heads, length / block) fp16: an integer q of a block stands for q * absmax / 127."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_absmax: torch.Tensor, value_absmax: torch.Tensor):
        assert keys.ndim == 4 and keys.dtype == torch.int8 and values.dtype == torch.int8
        batch, heads, length, dim = keys.shape
        assert dim % 16 == 0 and dim <= 256 and length % 16 == 0
        assert values.shape == (batch, heads, length // 16, dim, 16)
        assert key_absmax.ndim == 3 and key_absmax.shape[:2] == (batch, heads) and key_absmax.shape == value_absmax.shape
        assert key_absmax.dtype == torch.float16 and value_absmax.dtype == torch.float16
        blocks = key_absmax.size(2)
        assert blocks * max(BLOCKS) >= length and (length == 0 or (blocks > 0 and length % blocks == 0 and length // blocks in BLOCKS))
        for x in (keys, values, key_absmax, value_absmax):
            assert x.is_cuda and x.is_contiguous() and x.device == keys.device
        self.keys, self.values, self.key_absmax, self.value_absmax = keys, values, key_absmax, value_absmax
        self.batch, self.heads, self.length, self.dim = batch, heads, length, dim
        self.block = length // blocks if length else BLOCKS[0]

    @classmethod
    def empty(cls, batch: int, heads: int, length: int, dim: int, block: int = 64, device="cuda") -> "QuantizedKV":
        """A cache for at least `length` tokens of each sequence (rounded up to whole blocks), holding zeros."""
        assert block in BLOCKS and dim % 16 == 0 and 0 <= dim <= 256
        length = (length + block - 1) // block * block

        def zeros(*shape, dtype=torch.int8):
            return torch.zeros(shape, dtype=dtype, device=device)
        tops = (batch, heads, length // block)
        return cls(zeros(batch, heads, length, dim), zeros(batch, heads, length // 16, dim, 16), zeros(*tops, dtype=torch.float16),
                   zeros(*tops, dtype=torch.float16))

    def _here(self):
        here = _device() if _device is not None and torch.cuda.is_initialized() else torch.cuda.current_device()
        device = self.keys.device
        assert device.index == here, "the cache lies on another device than the current one"
        return device

    def write(self, k: torch.Tensor, v: torch.Tensor, pos, count=None) -> None:
        """k, v (batch, heads, tokens, dim) to the positions pos .. pos + tokens - 1 of every sequence; pos an int, or an int32 tensor with one for each.
        count: int32 tensor, how many tokens of each sequence are real (the first ones); None: all.

        With positions on the device a sequence at a negative one is left alone, and tokens that would come to lie behind the cache are dropped.
        What the sequence held behind the tokens written counts no longer."""
        device = self._here()
        _check_tokens(k, device)
        _check_tokens(v, device)
        assert k.ndim == 4 and k.shape == v.shape
        batch, heads, tokens, dim = k.shape
        assert batch == self.batch and heads == self.heads and dim == self.dim
        pos_each, pos = _each(pos, self.batch, device)
        assert pos_each is not None or 0 <= pos <= self.length - tokens, "tokens outside of the cache"
        count_each = None
        if count is not None:
            assert isinstance(count, torch.Tensor)
            count_each, _ = _each(count, self.batch, device)
        cpmk.kv_write_int8(batch, heads, tokens, dim, self.length, self.block, k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), pos_each, pos,
                           count_each, self.keys.data_ptr(), self.values.data_ptr(), self.key_absmax.data_ptr(), self.value_absmax.data_ptr(), cur_stream())

    def read(self, start=0, tokens: int = None, columns: bool = False):
        """Keys and values of the positions start .. start + tokens - 1 (start an int or an int32 tensor with one for each sequence; tokens: up to the
        cache's end) as fp16 (batch, heads, tokens, dim), zeros outside of the cache.  columns: laid out (batch, heads, dim, tokens) in memory."""
        device = self._here()
        from_each, first = _each(start, self.batch, device)
        if tokens is None:
            assert from_each is None, "how many tokens"
            tokens = self.length - first
        assert tokens >= 0 and -2 ** 31 <= first < 2 ** 31

        def buffer():
            shape = (self.batch, self.heads, self.dim, tokens) if columns else (self.batch, self.heads, tokens, self.dim)
            out = torch.empty(shape, dtype=torch.float16, device=device)
            return out.transpose(2, 3) if columns else out
        k, v = buffer(), buffer()
        cpmk.kv_read_int8(self.batch, self.heads, tokens, self.dim, self.length, self.block, self.keys.data_ptr(), self.values.data_ptr(),
                          self.key_absmax.data_ptr(), self.value_absmax.data_ptr(), from_each, first, k.data_ptr(), v.data_ptr(), *k.stride(),
                          cur_stream())
        return k, v

    def attention(self, q: torch.Tensor, lens, scale: float = None, causal: bool = True, pos=None, mask: torch.Tensor = None,
                  bias: torch.Tensor = None, mapping: torch.Tensor = None, bidirectional: bool = False) -> torch.Tensor:
        """softmax(scale q k^T + position bias) v over the first lens keys of every sequence (an int, or an int32 tensor with one for each).

        q (batch, query heads, queries, dim), query heads a multiple of the cache's (neighbouring ones share a head of the cache); scale: dim ** -0.5.
        pos: the first query's position (int, int32 tensor, or None: the queries are the last of the keys); causal: keys behind a query's position do not count.
        mask: bool (batch, length) or (batch, 1 or queries, length), True where a key counts.  A query without keys gives zeros.
        bias, mapping, bidirectional: PositionEmbedding's weight (query heads, num_buckets) and the table of position_embedding_init.
        The result has the shape of q, and its layout where q is dense."""
        device = self._here()
        _check_tokens(q, device)
        assert q.ndim == 4
        batch, heads, queries, dim = q.shape
        assert batch == self.batch and dim == self.dim and ((heads % self.heads == 0) if self.heads else heads == 0)
        lens_each, keys = _each(lens, self.batch, device)
        assert lens_each is not None or 0 <= keys <= self.length, "more keys than the cache has"
        pos_each, first = _each(-1 if pos is None else pos, self.batch, device)
        assert pos is None or pos_each is not None or 0 <= first < 2 ** 30
        mask_ptr, mask_batch, mask_token = None, 0, 0
        if mask is not None:
            assert mask.dtype == torch.bool and mask.device == device
            if mask.ndim == 2:
                mask = mask[:, None]
            assert mask.ndim == 3 and mask.shape[::2] == (self.batch, self.length) and mask.size(1) in (1, queries)
            assert mask.stride(2) == 1 or self.length <= 1
            mask_ptr, mask_batch, mask_token = mask.data_ptr(), mask.stride(0), mask.stride(1) if mask.size(1) > 1 else 0
        bias_ptr, mapping_ptr, buckets, distances = None, None, 0, 0
        if bias is not None:
            assert bias.dtype == torch.float16 and bias.ndim == 2 and bias.size(0) == heads and bias.is_contiguous() and bias.device == device
            assert mapping is not None and mapping.dtype == torch.int32 and mapping.ndim == 1 and mapping.is_contiguous() and mapping.device == device
            _check_gradients(bias)
            bias_ptr, mapping_ptr, buckets, distances = bias.data_ptr(), mapping.data_ptr(), bias.size(1), mapping.size(0)
        out = torch.empty_like(q)
        size = _workspace(device.index, batch, heads, self.heads, queries, dim, self.length)
        space = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        cpmk.kv_attention_int8(batch, heads, self.heads, queries, dim, self.length, self.block, q.data_ptr(), *q.stride(), self.keys.data_ptr(),
                          self.values.data_ptr(), self.key_absmax.data_ptr(), self.value_absmax.data_ptr(), lens_each, keys, pos_each, first, int(bool(causal)),
                          max(dim, 1) ** -0.5 if scale is None else scale, bias_ptr, mapping_ptr, buckets, distances, int(bool(bidirectional)), mask_ptr, mask_batch,
                          mask_token, out.data_ptr(), *out.stride(), None if space is None else space.data_ptr(), cur_stream())
        return out
