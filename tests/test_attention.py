"""Attention over fp16 keys and values and rotary positions without a GPU: the argument checks of the C ABI, the plain-torch forms and the oracle against each other, and the oracle's
gradients against differences."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

from oracle import attention as oa

N, P = None, 16
S = (64, 64, 64, 1)


def _forward(b=1, h=2, kv=1, n=40, d=64, length=64, q=P, k=P, out=P, lens_each=N, len=8, pos_each=N, pos=-1, scale=0.125, bias=N, mapping=N, buckets=32, distances=128, both=0, mask=N,
             lse=N, rest=N, space=P):
    from cpm_kernels_amd.library import cpmk
    cpmk.attention_forward(b, h, kv, n, d, length, q, *S, k, *S, k, *S, lens_each, len, pos_each, pos, 1, scale, bias, mapping, buckets, distances, both, mask, 0, 0, out, *S, lse, rest,
                           space, N)


def _backward(b=1, h=2, kv=1, n=40, d=64, length=64, q=P, k=P, out=P, lens_each=N, len=8, pos_each=N, pos=-1, scale=0.125, bias=N, mapping=N, buckets=32, distances=128, both=0, mask=N,
              lse=P, rest=P, dout=P, dq=P, dk=P, dbias=N, space=P):
    from cpm_kernels_amd.library import cpmk
    cpmk.attention_backward(b, h, kv, n, d, length, q, *S, k, *S, k, *S, lens_each, len, pos_each, pos, 1, scale, bias, mapping, buckets, distances, both, mask, 0, 0, out, *S, lse, rest,
                            dout, *S, dq, *S, dk, *S, dk, *S, dbias, space, N)


def test_refusals_of_the_c_abi():
    for call in (_forward, _backward):
        for bad in (dict(b=-1), dict(h=-2), dict(kv=-1), dict(n=-1), dict(d=-8), dict(length=-1), dict(len=-1), dict(len=65), dict(kv=0), dict(h=3, kv=2), dict(q=N), dict(k=N), dict(out=N), dict(scale=float("nan")), dict(scale=float("-inf")),
                    dict(bias=P), dict(bias=P, mapping=P, buckets=0), dict(bias=P, mapping=P, distances=0), dict(bias=P, mapping=P, distances=-1)):
            with pytest.raises(RuntimeError, match="invalid argument"):
                call(**bad)
        for bad in (dict(d=257), dict(n=2 ** 30), dict(length=2 ** 30), dict(b=2 ** 16, h=2 ** 16), dict(b=2 ** 30, h=2 ** 30), dict(bias=P, mapping=P, distances=1025),
                    dict(bias=P, mapping=P, distances=513, both=1), dict(b=2 ** 10, h=2 ** 10, n=2 ** 22)):
            with pytest.raises(RuntimeError, match="limit"):
                call(**bad)
        for empty in (dict(b=0, q=N, k=N, out=N), dict(h=0, kv=0, q=N, k=N, out=N), dict(d=0, q=N, k=N, out=N)):
            call(**empty)
    _forward(n=0, q=N, out=N)
    for bad in (dict(lse=P), dict(space=N, n=1, length=2 ** 20, len=2 ** 20)):
        with pytest.raises(RuntimeError, match="invalid argument"):
            _forward(**bad)
    for bad in (dict(lse=N), dict(rest=N), dict(dout=N), dict(dq=N), dict(dk=N), dict(space=N), dict(dbias=P)):
        with pytest.raises(RuntimeError, match="invalid argument"):
            _backward(**bad)
    with pytest.raises(RuntimeError, match="limit"):
        _backward(b=2 ** 15, h=2 ** 15, kv=2 ** 15, n=1, length=2 ** 20)


def test_workspaces():
    from cpm_kernels_amd.library import cpmk
    assert cpmk.attention_forward_workspace(1, 16, 16, 4096, 64, 64) == 0           # (enough queries to fill any device)
    # parts of one query and all heads of a long cache: at least one of 16 rows with 64 units and two statistics for each of two parts
    assert cpmk.attention_forward_workspace(1, 1, 1, 1, 64, 2 ** 20) >= 2 * 16 * 66 * 4
    for bad in ((0, 4, 4, 1, 64, 64), (1, 4, 3, 1, 64, 64), (1, 4, 0, 1, 64, 64), (1, 4, 4, 1, 257, 64), (1, 4, 4, 1, 64, 2 ** 30), (2 ** 30, 2 ** 30, 1, 1, 64, 64), (-1, 1, 1, 1, 64, 64)):
        assert cpmk.attention_forward_workspace(*bad) == 0
    # D of every query, and the largest gradient of every 128
    assert cpmk.attention_backward_workspace(2, 3, 3, 200, 64, 0, 0) == (2 * 3 * 200 + 2 * 3 * 2) * 4
    assert cpmk.attention_backward_workspace(2, 3, 3, 200, 64, 128, 1) > cpmk.attention_backward_workspace(2, 3, 3, 200, 64, 128, 0) > (2 * 3 * 200 + 2 * 3 * 2 + 2 * 3 * 2 * 128) * 4
    for bad in ((0, 4, 4, 1, 64, 0, 0), (1, 4, 3, 1, 64, 0, 0), (1, 4, 4, 1, 64, -1, 0), (1, 4, 4, 1, 64, 1025, 0), (1, 4, 4, 1, 64, 513, 1)):
        assert cpmk.attention_backward_workspace(*bad) == 0


def test_refusals_of_rotary():
    from cpm_kernels_amd.library import cpmk

    def call(b=1, n=4, d=64, part=64, h=1, q=P, y=P, held=0, k=N, turns=P, pos_each=N, pos=0):
        cpmk.rotary(b, n, d, part, 0, h, q, *S, y, *S, held, k, *S[:3], 1, k, *S, turns, pos_each, 0, 0, pos, 1.0, 0, N)
    call(b=0, q=N, y=N, turns=N)
    call(n=0, q=N, y=N, turns=N)
    call(h=0, q=N, y=N)
    for bad in (dict(b=-1), dict(n=-1), dict(d=-2), dict(part=63), dict(part=66), dict(part=-2), dict(h=-1), dict(held=-1), dict(q=N), dict(y=N), dict(turns=N), dict(held=1, k=N)):
        with pytest.raises(RuntimeError, match="invalid argument|divisibility"):
            call(**bad)


def test_calls_without_a_device():
    import cpm_kernels_amd.torch as ct
    x = torch.zeros((1, 2, 3, 8), dtype=torch.half)
    with pytest.raises(Exception):
        ct.attention(x, x, x)
    with pytest.raises(Exception):
        ct.RotaryEmbedding(8)(x)


def _normal(rng, *shape):
    return rng.standard_normal(shape)


def _inputs(rng, b=2, h=4, held=2, n=5, length=9, d=6, count=8, distance=4, both=True):
    mapping = np.minimum(np.arange(distance), count // 2 - 1)
    return _normal(rng, b, h, n, d), _normal(rng, b, held, length, d), _normal(rng, b, held, length, d), _normal(rng, h, count), mapping


CASES = [(causal, kind, lens, pos) for causal in (False, True) for kind in (None, "key", "query") for lens, pos in ((None, None), ([9, 4], None), ([9, 0], [2, -3]), ([7, 9], [0, 40]))]


def _mask(rng, kind, b=2, n=5, length=9):
    if kind is None:
        return None
    mask = rng.random((b, 1 if kind == "key" else n, length)) < 0.6
    mask[-1, -1] = False
    return mask


@pytest.mark.parametrize("causal,kind,lens,pos", CASES)
def test_plain_form_and_oracle(causal, kind, lens, pos):
    """attentionTH in fp64 and its gradients by autograd are the oracle's, to rounding in fp64."""
    import cpm_kernels_amd.torch as ct
    rng = np.random.default_rng(1)
    q, k, v, table, mapping = _inputs(rng)
    mask, g = _mask(rng, kind), _normal(rng, 2, 4, 5, 6)
    every = [9, 9] if lens is None else lens
    first = [x - 5 for x in every] if pos is None else pos
    want, _ = oa.attention(q, k, v, every, first, 0.3, causal, mask, table, mapping, True, g)
    leaves = [torch.tensor(x, requires_grad=True) for x in (q, k, v, table)]
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32)         # noqa: E731
    out = ct.attentionTH(leaves[0], leaves[1], leaves[2], lens=ints(lens), scale=0.3, causal=causal, pos=ints(pos), mask=None if mask is None else torch.tensor(mask), bias=leaves[3],
                         mapping=torch.tensor(mapping, dtype=torch.int32), bidirectional=True)
    got = [out, *torch.autograd.grad(out, leaves, torch.tensor(g))]
    for x, y in zip(got, want):
        assert np.abs(x.detach().numpy() - y).max() < 1e-12


def test_oracle_against_differences():
    """A gradient of the oracle times a direction is what the result grows by along it: central differences of 2^-13, whose own error is their square."""
    rng = np.random.default_rng(2)
    q, k, v, table, mapping = _inputs(rng)
    mask, g = _mask(rng, "query"), _normal(rng, 2, 4, 5, 6)
    args = ([9, 7], [4, 2], 0.5, True, mask)
    grads, _ = oa.attention(q, k, v, *args, table, mapping, True, g)
    point = [q, k, v, table]
    for i in range(4):
        way = _normal(rng, *point[i].shape)

        def at(h):
            moved = [x + h * way if j == i else x for j, x in enumerate(point)]
            return (oa.attention(*moved[:3], *args, moved[3], mapping, True)[0] * g).sum()
        h = 2.0 ** -13
        want, size = (grads[1 + i] * way).sum(), (np.abs(grads[1 + i]) * np.abs(way)).sum()
        assert abs((at(h) - at(-h)) / (2 * h) - want) < 1e-6 * max(size, 1)


def test_oracle_of_the_bound():
    """fp16 arithmetic as the kernels round (scores fp32, probabilities and results fp16) stays within the oracle's bound; a key too many does not."""
    rng = np.random.default_rng(3)
    q, k, v = (_normal(rng, 1, 2, n, 32).astype(np.float16) for n in (7, 50, 50))
    want, bound = oa.attention(q, k, v, [50], [43], 32 ** -0.5, True)
    off, _ = oa.attention(q, k, v, [50], [44], 32 ** -0.5, True)
    s = (q.astype(np.float32) @ k.astype(np.float32).transpose(0, 1, 3, 2)) * np.float32(32 ** -0.5)
    s[..., np.arange(50)[None] > np.arange(7)[:, None] + 43] = -np.inf
    p = np.exp(s - s.max(-1, keepdims=True)).astype(np.float32)
    got = (np.float16(p * 128).astype(np.float32) @ v.astype(np.float32) / (128 * p.sum(-1, keepdims=True))).astype(np.float16)
    assert (np.abs(got - want) <= bound).all()
    assert (np.abs(off - want) > bound).any()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("part", [0, 6, 8])
def test_plain_form_of_rotary_and_oracle(part, interleaved):
    import cpm_kernels_amd.torch as ct
    rng = np.random.default_rng(4)
    x, at = _normal(rng, 2, 3, 5, 8), np.array([[0, 1, -5, 2 ** 30, 7], [9, 9, 100000, -2 ** 31, 3]])
    rotary = ct.RotaryEmbeddingTH(8, part, interleaved=interleaved, scaling="parts", factor=4.0, original_length=128)
    y = rotary(torch.tensor(x), pos=torch.tensor(at)).numpy()
    want, _ = oa.rotary(x, at, rotary.turns.numpy(), rotary.magnitude, interleaved)
    assert np.abs(y - want).max() < 2.0 ** 31 * 2.0 ** -51 * 16         # (angles of 2^31 radians in fp64)
    back, _ = oa.rotary(want, at, rotary.turns.numpy(), 1 / rotary.magnitude, interleaved, inverse=True)
    assert np.abs(back - x).max() < 1e-12


def test_frequencies():
    from cpm_kernels_amd.torch.rotary import frequencies
    plain, one = frequencies(64)
    assert one == 1.0 and plain.dtype == torch.float64 and plain.shape == (32,) and abs(plain[0].item() * 2 * math.pi - 1) < 1e-15
    assert torch.equal(frequencies(64, scaling="linear", factor=4.0)[0], plain / 4)
    ntk = frequencies(64, scaling="ntk", factor=4.0)[0]
    assert abs(ntk[0] / plain[0] - 1) < 1e-15 and abs(ntk[-1] * 4 / plain[-1] - 1) < 1e-13
    parts, magnitude = frequencies(64, scaling="parts", factor=4.0, original_length=2048)
    turns = 2048 * plain
    assert torch.equal(parts[turns >= 32], plain[turns >= 32]) and (parts[turns <= 1] * 4 / plain[turns <= 1] - 1).abs().max() < 1e-15
    assert ((parts < plain) & (parts > plain / 4))[(turns > 1) & (turns < 32)].all() and abs(magnitude - 1 - 0.1 * math.log(4)) < 1e-15
    assert frequencies(0)[0].numel() == 0 and frequencies(2, scaling="ntk", factor=2.0)[0].numel() == 1
    for bad in (dict(scaling="other"), dict(scaling="linear", factor=0.5), dict(scaling="parts", factor=2.0), dict(base=0.0)):
        with pytest.raises(AssertionError):
            frequencies(64, **bad)


def test_the_module_of_rotary():
    import cpm_kernels_amd.torch as ct
    rotary = ct.RotaryEmbedding(64, 32, base=5000.0, interleaved=True)
    for other in (copy.deepcopy(rotary), pickle.loads(pickle.dumps(rotary)), copy.deepcopy(rotary).half()):
        assert torch.equal(other.turns, rotary.turns) and other.turns.dtype == torch.float64 and other.interleaved and other.rotary_dim == 32
    assert not list(rotary.parameters()) and not rotary.state_dict()
    for bad in ((64, 66), (64, 31), (64, -2)):
        with pytest.raises(AssertionError):
            ct.RotaryEmbedding(*bad)
