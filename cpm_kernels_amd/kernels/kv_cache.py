"""The key/value cache in 8 bits: tokens in, tokens out, and the attention over it.  Beside ``copy_data_to_kv`` and the fp16 products,
bias, mask and softmax of a decode step; the reference has no counterpart."""
from typing import Tuple

from ..library import cpmk
from .base import DevicePointer, CUDAStream

Strides = Tuple[int, int, int, int]      # of (batch, heads, tokens, dim), in elements

BLOCKS = (16, 32, 64, 128)


def _check(dim, length, block):
    assert block in BLOCKS and length % block == 0
    assert dim % 16 == 0 and dim <= 256


def kv_write_int8(batch: int, heads: int, tokens: int, dim: int, length: int, block: int,
                  k: DevicePointer, k_strides: Strides,      # (batch, heads, tokens, dim)  fp16
                  v: DevicePointer, v_strides: Strides,      # (batch, heads, tokens, dim)  fp16
                  pos_each: DevicePointer, pos: int,         # (batch)  int32, position of each sequence's first token; None: all at pos
                  count_each: DevicePointer,                 # (batch)  int32, tokens of each sequence; None: all
                  keys: DevicePointer,                       # (batch, heads, length, dim)  int8
                  values: DevicePointer,                     # (batch, heads, length / 16, dim, 16)  int8
                  key_absmax: DevicePointer,                 # (batch, heads, length / block)  fp16
                  value_absmax: DevicePointer,               # (batch, heads, length / block)  fp16
                  stream: CUDAStream):
    """Tokens into the cache: q = round(127 x / absmax of its block), older tokens of a block that grows rounded again."""
    _check(dim, length, block)
    cpmk.kv_write_int8(batch, heads, tokens, dim, length, block, k, *k_strides, v, *v_strides, pos_each, pos, count_each, keys, values,
                       key_absmax, value_absmax, stream)


def kv_read_int8(batch: int, heads: int, tokens: int, dim: int, length: int, block: int,
                 keys: DevicePointer, values: DevicePointer, key_absmax: DevicePointer, value_absmax: DevicePointer,
                 from_each: DevicePointer, first: int,       # (batch)  int32, first position of each sequence; None: all from `first`
                 k: DevicePointer, v: DevicePointer,         # (batch, heads, tokens, dim)  fp16
                 out_strides: Strides, stream: CUDAStream):
    """Positions of the cache as fp16, zeros outside of it."""
    _check(dim, length, block)
    cpmk.kv_read_int8(batch, heads, tokens, dim, length, block, keys, values, key_absmax, value_absmax, from_each, first, k, v, *out_strides, stream)


def kv_attention_int8_workspace(batch: int, heads: int, kv_heads: int, tokens: int, dim: int, length: int) -> int:
    """Bytes of device memory that kv_attention_int8 of these sizes works in."""
    return cpmk.kv_attention_int8_workspace(batch, heads, kv_heads, tokens, dim, length)


def kv_attention_int8(batch: int, heads: int, kv_heads: int, tokens: int, dim: int, length: int, block: int,
                      q: DevicePointer, q_strides: Strides,          # (batch, heads, tokens, dim)  fp16
                      keys: DevicePointer, values: DevicePointer, key_absmax: DevicePointer, value_absmax: DevicePointer,
                      lens_each: DevicePointer, len: int,            # (batch)  int32, keys of each sequence; None: all have len
                      pos_each: DevicePointer, pos: int,             # (batch)  int32, position of each first query; None: pos; pos < 0: the last keys
                      causal: bool, scale: float,
                      bias: DevicePointer,                           # (heads, num_buckets)  fp16, or None
                      mapping: DevicePointer,                        # (max_distance)  int32
                      num_buckets: int, max_distance: int, bidirectional: bool,
                      mask: DevicePointer, mask_batch: int, mask_token: int,      # rows of length bools, strides in bytes; or None
                      out: DevicePointer, out_strides: Strides,      # (batch, heads, tokens, dim)  fp16
                      workspace: DevicePointer,                      # kv_attention_int8_workspace() bytes
                      stream: CUDAStream):
    """softmax(scale q k^T + position bias) v over the cache; queries without a key give zeros."""
    _check(dim, length, block)
    assert heads == 0 or (kv_heads > 0 and heads % kv_heads == 0)
    cpmk.kv_attention_int8(batch, heads, kv_heads, tokens, dim, length, block, q, *q_strides, keys, values, key_absmax, value_absmax, lens_each, len,
                           pos_each, pos, int(bool(causal)), scale, bias, mapping, num_buckets, max_distance, int(bool(bidirectional)), mask,
                           mask_batch, mask_token, out, *out_strides, workspace, stream)
