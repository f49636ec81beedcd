"""Attention over fp16 keys and values, its gradients, and rotary positions.  Beside ``gemm_fp16``, ``mask``, ``softmax_forward`` and the position bias, which keep
the scores in memory; the reference has no counterpart."""
from typing import Tuple

from ..library import cpmk
from .base import DevicePointer, CUDAStream

Strides = Tuple[int, int, int, int]      # of (batch, heads, tokens, dim), in elements


def _check(heads, kv_heads, dim):
    assert dim <= 256
    assert heads == 0 or (kv_heads > 0 and heads % kv_heads == 0)


def attention_forward_workspace(batch: int, heads: int, kv_heads: int, tokens: int, dim: int, length: int) -> int:
    """Bytes of device memory that attention_forward of these sizes works in."""
    return cpmk.attention_forward_workspace(batch, heads, kv_heads, tokens, dim, length)


def attention_backward_workspace(batch: int, heads: int, kv_heads: int, tokens: int, length: int, max_distance: int, bidirectional: bool) -> int:
    """Bytes of device memory that attention_backward of these sizes works in (max_distance: 0 without the gradient of biases)."""
    return cpmk.attention_backward_workspace(batch, heads, kv_heads, tokens, length, max_distance, int(bool(bidirectional)))


def attention_forward(batch: int, heads: int, kv_heads: int, tokens: int, dim: int, length: int,
                      q: DevicePointer, q_strides: Strides,          # (batch, heads, tokens, dim)  fp16
                      k: DevicePointer, k_strides: Strides,          # (batch, kv_heads, length, dim)  fp16
                      v: DevicePointer, v_strides: Strides,          # (batch, kv_heads, length, dim)  fp16
                      lens_each: DevicePointer, len: int,            # (batch)  int32, keys of each sequence; None: all have len
                      pos_each: DevicePointer, pos: int,             # (batch)  int32, position of each first query; None: pos; pos < 0: the last keys
                      causal: bool, scale: float,
                      bias: DevicePointer,                           # (heads, num_buckets)  fp16, or None
                      mapping: DevicePointer,                        # (max_distance)  int32
                      num_buckets: int, max_distance: int, bidirectional: bool,
                      mask: DevicePointer, mask_batch: int, mask_token: int,      # rows of length bools, strides in bytes; or None
                      out: DevicePointer, out_strides: Strides,      # (batch, heads, tokens, dim)  fp16
                      lse: DevicePointer,                            # (batch, heads, tokens)  fp32, or None
                      rest: DevicePointer,                           # fp16 under out's strides, or None: with lse, for attention_backward
                      workspace: DevicePointer,                      # attention_forward_workspace() bytes
                      stream: CUDAStream):
    """softmax(scale q k^T + position bias) v; queries without a key give zeros."""
    _check(heads, kv_heads, dim)
    cpmk.attention_forward(batch, heads, kv_heads, tokens, dim, length, q, *q_strides, k, *k_strides, v, *v_strides, lens_each, len, pos_each, pos,
                           int(bool(causal)), scale, bias, mapping, num_buckets, max_distance, int(bool(bidirectional)), mask, mask_batch, mask_token,
                           out, *out_strides, lse, rest, workspace, stream)


def attention_backward(batch: int, heads: int, kv_heads: int, tokens: int, dim: int, length: int,
                       q: DevicePointer, q_strides: Strides, k: DevicePointer, k_strides: Strides, v: DevicePointer, v_strides: Strides,
                       lens_each: DevicePointer, len: int, pos_each: DevicePointer, pos: int, causal: bool, scale: float,
                       bias: DevicePointer, mapping: DevicePointer, num_buckets: int, max_distance: int, bidirectional: bool,
                       mask: DevicePointer, mask_batch: int, mask_token: int,
                       out: DevicePointer, out_strides: Strides,      # (batch, heads, tokens, dim)  fp16, of attention_forward
                       lse: DevicePointer, rest: DevicePointer,       # (batch, heads, tokens)  fp32; fp16 under out's strides; of attention_forward
                       dout: DevicePointer, dout_strides: Strides,    # (batch, heads, tokens, dim)  fp16
                       dq: DevicePointer, dq_strides: Strides,        # (batch, heads, tokens, dim)  fp16
                       dk: DevicePointer, dk_strides: Strides,        # (batch, kv_heads, length, dim)  fp16
                       dv: DevicePointer, dv_strides: Strides,        # (batch, kv_heads, length, dim)  fp16
                       dbias: DevicePointer,                          # (heads, num_buckets)  fp16, or None
                       workspace: DevicePointer,                      # attention_backward_workspace() bytes
                       stream: CUDAStream):
    """Gradients of q, k, v and the biases."""
    _check(heads, kv_heads, dim)
    cpmk.attention_backward(batch, heads, kv_heads, tokens, dim, length, q, *q_strides, k, *k_strides, v, *v_strides, lens_each, len, pos_each, pos,
                            int(bool(causal)), scale, bias, mapping, num_buckets, max_distance, int(bool(bidirectional)), mask, mask_batch, mask_token,
                            out, *out_strides, lse, rest, dout, *dout_strides, dq, *dq_strides, dk, *dk_strides, dv, *dv_strides, dbias, workspace, stream)


def rotary_forward(batch: int, tokens: int, dim: int, part: int, interleaved: bool,
                   heads_q: int, q: DevicePointer, q_strides: Strides, q_out: DevicePointer, q_out_strides: Strides,      # (batch, heads_q, tokens, dim)  fp16
                   heads_k: int, k: DevicePointer, k_strides: Strides, k_out: DevicePointer, k_out_strides: Strides,      # (batch, heads_k, tokens, dim)  fp16
                   turns: DevicePointer,                             # (part / 2)  fp64, turns a token
                   positions: DevicePointer, pos_batch: int, pos_token: int,     # int32 and its strides (pos_token 0: first positions), or None
                   pos: int, magnitude: float, stream: CUDAStream):
    """Pairs of the first `part` units turned by their positions' angles, the others copied."""
    assert part % 2 == 0 and part <= dim
    cpmk.rotary(batch, tokens, dim, part, int(bool(interleaved)), heads_q, q, *q_strides, q_out, *q_out_strides, heads_k, k, *k_strides, k_out, *k_out_strides,
                turns, positions, pos_batch, pos_token, pos, magnitude, 0, stream)


def rotary_backward(batch: int, tokens: int, dim: int, part: int, interleaved: bool,
                    heads_q: int, dq_out: DevicePointer, dq_out_strides: Strides, dq: DevicePointer, dq_strides: Strides,
                    heads_k: int, dk_out: DevicePointer, dk_out_strides: Strides, dk: DevicePointer, dk_strides: Strides,
                    turns: DevicePointer, positions: DevicePointer, pos_batch: int, pos_token: int, pos: int, magnitude: float, stream: CUDAStream):
    """The gradient of rotary_forward: turned back."""
    assert part % 2 == 0 and part <= dim
    cpmk.rotary(batch, tokens, dim, part, int(bool(interleaved)), heads_q, dq_out, *dq_out_strides, dq, *dq_strides, heads_k, dk_out, *dk_out_strides, dk, *dk_strides,
                turns, positions, pos_batch, pos_token, pos, magnitude, 1, stream)
