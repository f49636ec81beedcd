"""Rotary positions against float64, each result within the bound that the oracle derives from the roundings on the way."""
import copy

import numpy as np
import pytest
import torch

import cpm_kernels_amd.torch as ct
from oracle import attention as oa

pytestmark = pytest.mark.gpu


def _laid_out(x, layout):
    t = torch.from_numpy(x).cuda()
    if layout == "columns":
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    if layout == "rows":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    b, h, n, d = x.shape
    wide = torch.zeros((b, h, n, 2 * d + 1), dtype=torch.half, device="cuda")
    wide[..., 1::2] = t
    return wide[..., 1::2]


def _positions(rng, kind, b, n):
    """(what goes into the call, (b, n) integers)"""
    if kind == "start":
        return 12345, 12345 + np.tile(np.arange(n), (b, 1))
    if kind == "each":
        first = rng.integers(-1000, 2 ** 20, b)
        return torch.tensor(first, dtype=torch.int32, device="cuda"), first[:, None] + np.arange(n)
    every = rng.integers(-2 ** 31, 2 ** 31, (b, n))
    return torch.tensor(every, dtype=torch.int32, device="cuda"), every


def _check(got, want, bound):
    got = got.detach().cpu().numpy().astype(np.float64)
    off = np.abs(got - want) / np.maximum(bound, 1e-300)
    assert (off[bound > 0] <= 1).all(), off[bound > 0].max()
    assert np.array_equal(got[bound == 0], want[bound == 0])


@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["start", "each", "token"])
@pytest.mark.parametrize("b,h,held,n,d,part", [(1, 1, 1, 1, 2, 2), (2, 3, 1, 1, 64, 64), (1, 16, 16, 7, 64, 32), (2, 5, 2, 33, 80, 20), (1, 4, 4, 9, 128, 96), (3, 2, 1, 100, 72, 16),
                                               (1, 2, 2, 8, 31, 30), (1, 64, 8, 20, 128, 128), (2, 1, 1, 15, 256, 0)])
def test_forward_and_gradient(gpu, b, h, held, n, d, part, kind, interleaved, layout):
    print("rotary", b, h, held, n, d, part, kind, interleaved, layout, flush=True)
    rng = np.random.default_rng(n + d + part)
    q, k, gq, gk = (rng.standard_normal((b, x, n, d)).astype(np.float16) for x in (h, held, h, held))
    rotary = ct.RotaryEmbedding(d, rotary_dim=part, interleaved=interleaved, scaling="parts", factor=4.0, original_length=2048)
    pos, at = _positions(rng, kind, b, n)
    tq, tk, tgq, tgk = (_laid_out(x, layout) for x in (q, k, gq, gk))
    tq.requires_grad_(), tk.requires_grad_()
    out = rotary(tq, tk, pos)
    grads = torch.autograd.grad(out, (tq, tk), (tgq, tgk))
    turns = rotary.turns.numpy()
    for got, x in zip(out, (q, k)):
        _check(got, *oa.rotary(x, at, turns, rotary.magnitude, interleaved))
    for got, x in zip(grads, (gq, gk)):
        _check(got, *oa.rotary(x, at, turns, rotary.magnitude, interleaved, inverse=True))
    with torch.no_grad():
        alone = rotary(tq, pos=pos)
        assert torch.equal(alone, out[0])
        yq, yk = tq.clone(memory_format=torch.preserve_format), tk.clone(memory_format=torch.preserve_format)
        rotary.inplace(yq, yk, pos)
        assert torch.equal(yq, out[0]) and torch.equal(yk, out[1])
