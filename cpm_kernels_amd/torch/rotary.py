"""Rotary positions: pairs of a head's units turned by angles that grow with the token's position, for queries and keys together.  Beside ``PositionEmbedding``, which adds
a bias to the scores; the reference has no counterpart.

    rotary = RotaryEmbedding(dim_head)
    q, k = rotary(q, k)                     # (batch, heads, tokens, dim_head), any strides; positions 0, 1, ...
    q, k = rotary(q, k, pos)                # first positions (int, int32 (batch,)) or all of them (int32 (batch, tokens))
    rotary.inplace(q, k, pos)               # a decode step: q and k themselves, no gradients
"""
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version
from ..library import cpmk
from ._common import cur_stream, current_device


def _arguments(x, y):
    return (0, None, 0, 0, 0, 0, None, 0, 0, 0, 0) if x is None else (x.size(1), x.data_ptr(), *x.stride(), y.data_ptr(), *y.stride())


def _launch(rotary, x, y, pos, inverse):
    """x and y: queries and keys (either may be None), what they become."""
    some = x[0] if x[0] is not None else x[1]
    batch, _, tokens, dim = some.shape
    positions = (None, 0, 0, pos)
    if isinstance(pos, torch.Tensor):
        positions = (pos.data_ptr(), pos.stride(0), pos.stride(1) if pos.ndim == 2 else 0, 0)
    cpmk.rotary(batch, tokens, dim, rotary.rotary_dim, int(rotary.interleaved), *_arguments(x[0], y[0]), *_arguments(x[1], y[1]), rotary.turns_on(some.device).data_ptr(), *positions,
                rotary.magnitude, int(inverse), cur_stream())


class OpRotary(torch.autograd.Function):
    """The gradient is turned back."""

    @staticmethod
    def forward(ctx, rotary, pos, q, k):
        ctx.set_materialize_grads(False)
        ctx.rotary = rotary
        ctx.number = None if isinstance(pos, torch.Tensor) else pos
        ctx.save_for_backward(pos if isinstance(pos, torch.Tensor) else None)
        y = torch.empty_like(q), None if k is None else torch.empty_like(k)
        _launch(rotary, (q, k), y, pos, False)
        return y

    @staticmethod
    def backward(ctx, dq, dk):
        assert not torch.is_grad_enabled(), "the gradients have no gradients"       # (create_graph; a wrapper that refuses it costs 10 us)
        grads = [x if x is not None and x.numel() > 0 else None for x in (dq, dk)]
        out = [None if x is None else torch.empty_like(x) for x in (dq, dk)]
        if any(x is not None for x in grads):
            current_device(next(x for x in grads if x is not None).device)
            pos, = ctx.saved_tensors
            _launch(ctx.rotary, grads, out, ctx.number if pos is None else pos, True)
        return None, None, out[0], out[1]


def frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = None, factor: float = 1.0, original_length: int = None):
    """(turns a token of every pair, fp64; what turned units are multiplied by).  scaling stretches positions `factor` times as far:
    "linear": all frequencies divided by the factor;
    "ntk": the base times factor ** (r / (r - 2)): the highest frequency stays, the lowest is divided by the factor;
    "parts": by the turns n that a pair makes over original_length: below 1 divided by the factor, from 32 on as they are, in between in proportion to n, and
    units multiplied by 1 + 0.1 ln(factor)."""
    r = rotary_dim
    assert scaling in (None, "linear", "ntk", "parts") and factor >= 1.0 and base > 0.0
    if scaling == "ntk" and r > 2:
        base = base * factor ** (r / (r - 2))
    turns = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / max(r, 1)) / (2 * math.pi)
    if scaling == "linear":
        return turns / factor, 1.0
    if scaling == "parts":
        assert original_length is not None and original_length > 0, "parts: the length that the frequencies were made for"
        kept = ((original_length * turns - 1) / 31).clamp(0, 1)
        return turns * (kept + (1 - kept) / factor), 1.0 + 0.1 * math.log(factor)
    return turns, 1.0


class RotaryEmbedding(torch.nn.Module):
    """dim: units of a head; rotary_dim of them are turned (even; None: all).  Pairs are units i and i + rotary_dim / 2, or, interleaved, 2 i and 2 i + 1.
    base, scaling, factor, original_length: see frequencies().  Has no parameters; angles are exact to 2^-22 of a turn at any int32 position."""

    def __init__(self, dim: int, rotary_dim: int = None, base: float = 10000.0, interleaved: bool = False, scaling: str = None, factor: float = 1.0, original_length: int = None):
        super().__init__()
        rotary_dim = dim if rotary_dim is None else rotary_dim
        assert 0 <= rotary_dim <= dim and rotary_dim % 2 == 0
        self.dim, self.rotary_dim, self.interleaved = dim, rotary_dim, bool(interleaved)
        self.turns, self.magnitude = frequencies(rotary_dim, base, scaling, factor, original_length)
        self._on = {}       # (no buffer of the module: .half() would round it)

    def turns_on(self, device) -> torch.Tensor:
        """The frequencies on a device; copied there by the first call, which may therefore not be a captured one."""
        turns = self._on.get(device)
        if turns is None:
            turns = self._on[device] = self.turns.to(device)
        return turns

    def __getstate__(self):
        return {**self.__dict__, "_on": {}}

    def _check(self, q, k, pos):
        device = current_device(q.device)
        for x in (q, k):
            assert x is None or (x.ndim == 4 and x.dtype == torch.float16 and x.device == device and x.size(3) == self.dim)
        assert k is None or (k.size(0) == q.size(0) and k.size(2) == q.size(2))
        if isinstance(pos, torch.Tensor):
            assert pos.dtype == torch.int32 and pos.device == device and pos.shape in ((q.size(0),), (q.size(0), q.size(2)))
            return pos
        number = int(pos)
        assert number == pos, "positions are integers"
        assert -2 ** 31 <= number < 2 ** 31
        return number

    def forward(self, q: torch.Tensor, k: torch.Tensor = None, pos=0):
        """q (batch, heads, tokens, dim), k (batch, any heads, tokens, dim) or None: turned copies of them, in their layouts where they are dense."""
        pos = self._check(q, k, pos)
        # (an autograd function costs 5 us of the host's time, as much as a step's kernel; one with forward-mode tangents goes through it all the same, and is refused there)
        if getattr(forward_ad, "_current_level", 0) < 0 and not (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
            out = torch.empty_like(q), None if k is None else torch.empty_like(k)
            _launch(self, (q, k), out, pos, False)
        else:
            out = OpRotary.apply(self, pos, q, k)
        return out[0] if k is None else out

    @torch.no_grad()
    def inplace(self, q: torch.Tensor, k: torch.Tensor = None, pos=0) -> None:
        """q and k themselves turned; no gradients."""
        pos = self._check(q, k, pos)
        for x in (q, k):
            assert x is None or not x.requires_grad, "in place there are no gradients"
            assert x is None or all(s != 0 or n <= 1 for s, n in zip(x.stride(), x.shape)), "elements that share memory"
        assert k is None or k.numel() == 0 or k.data_ptr() != q.data_ptr(), "one tensor turned twice at once"
        _launch(self, (q, k), (q, k), pos, False)
        for x in (q, k):
            if x is not None and not x.is_inference():
                increment_version(x)        # (a backward pass that has kept it must not run on what it has become)


class RotaryEmbeddingTH(torch.nn.Module):
    """Plain-torch formulation of the same, angles in fp64, products in fp32 (fp64 for fp64 tensors)."""

    def __init__(self, dim: int, rotary_dim: int = None, base: float = 10000.0, interleaved: bool = False, scaling: str = None, factor: float = 1.0, original_length: int = None):
        super().__init__()
        self.rotary_dim, self.interleaved = dim if rotary_dim is None else rotary_dim, interleaved
        self.turns, self.magnitude = frequencies(self.rotary_dim, base, scaling, factor, original_length)

    def forward(self, q: torch.Tensor, k: torch.Tensor = None, pos=0):
        at = torch.as_tensor(pos, device=q.device).double()
        if at.ndim < 2:
            at = at.reshape(-1, 1) + torch.arange(q.size(2), device=q.device)
        angle = 2 * math.pi * torch.frac(at[:, None, :, None] * self.turns.to(q.device))
        out = [self._turn(x, angle) for x in (q, k) if x is not None]
        return out[0] if k is None else tuple(out)

    def _turn(self, x, angle):
        r, wide = self.rotary_dim, torch.promote_types(x.dtype, torch.float32)
        cos, sin = (torch.cos(angle) * self.magnitude).to(wide), (torch.sin(angle) * self.magnitude).to(wide)
        y = x[..., :r].to(wide)
        a, b = (y[..., ::2], y[..., 1::2]) if self.interleaved else (y[..., :r // 2], y[..., r // 2:])
        parts = a * cos - b * sin, a * sin + b * cos
        y = torch.stack(parts, -1).flatten(-2) if self.interleaved else torch.cat(parts, -1)
        return torch.cat((y.to(x.dtype), x[..., r:]), -1)
