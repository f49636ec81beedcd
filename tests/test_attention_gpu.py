"""Attention over fp16 keys and values and its gradients against float64, each result within the bound that the oracle derives from the roundings on the way."""
import numpy as np
import pytest
import torch

import cpm_kernels_amd.kernels as ck
import cpm_kernels_amd.torch as ct
from oracle import attention as oa

pytestmark = pytest.mark.gpu


def _laid_out(x, layout):
    """fp16 numpy (b, h, n, d) on the GPU under the strides of `layout`."""
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    if layout == "columns":
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    if layout == "rows":            # (b, n, h, d)
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "strided":         # neither axis contiguous, nor any start of a row aligned
        b, h, n, d = x.shape
        wide = torch.zeros((b, h, n, 2 * d + 1), dtype=torch.half, device="cuda")
        wide[..., 1::2] = t
        return wide[..., 1::2]
    return t


def _normal(rng, shape, std=1.0, sized=True):
    x = rng.standard_normal(shape) * std
    return (x * np.exp(0.5 * rng.standard_normal((1, shape[1], 1, shape[3]))) if sized else x).astype(np.float16)


def _mapping(both, count=32, distance=128):
    mapping = torch.empty(distance, dtype=torch.int32, device="cuda")
    ck.position_embedding_init(count, distance, mapping.data_ptr(), both, torch.cuda.current_stream().cuda_stream)
    return mapping


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class _Case:
    """Inputs of one call, in numpy and on the GPU."""

    def __init__(self, b, h, held, n, length, d, layout="rows", causal=True, bias=None, mask=None, lens=None, pos=None, scale=None, seed=0, std=1.0, gstd=0.02, layouts=None,
                 count=32, distance=128, mapping=None):
        rng = np.random.default_rng(seed + n * 7 + length * 3 + d)
        self.rng = rng
        lay = layouts or [layout] * 4
        self.q, self.k, self.v = _normal(rng, (b, h, n, d), std), _normal(rng, (b, held, length, d), std), _normal(rng, (b, held, length, d), sized=False)
        self.g = _normal(rng, (b, h, n, d), gstd, sized=False)
        self.lay = lay
        self.causal, self.both = causal, bias == "both"
        self.table = None if bias is None else (rng.standard_normal((h, count)) * 0.5).astype(np.float16)
        self.mapping = None if bias is None else (_mapping(self.both, count, distance) if mapping is None else _ints(mapping))
        if isinstance(mask, np.ndarray) or mask is None:
            self.mask = mask
        else:
            self.mask = rng.random((b, {"key": 1, "query": n}[mask], length)) < 0.7
        self.lens, self.pos, self.scale = lens, pos, scale
        self.b, self.n, self.length, self.d = b, n, length, d

    def tensors(self):
        return [_laid_out(x, lay) for x, lay in zip((self.q, self.k, self.v, self.g), self.lay)]

    def arguments(self):
        each = lambda x: _ints(x) if isinstance(x, (list, np.ndarray)) else x       # noqa: E731
        return dict(lens=each(self.lens), pos=each(self.pos), scale=self.scale, causal=self.causal, mask=None if self.mask is None else torch.from_numpy(self.mask).cuda(),
                    mapping=self.mapping, bidirectional=self.both)

    def oracle(self, train):
        lens = np.full(self.b, self.length if self.lens is None else self.lens) if not isinstance(self.lens, (list, np.ndarray)) else np.asarray(self.lens)
        lens = np.clip(lens, 0, self.length)
        first = lens - self.n if self.pos is None else np.broadcast_to(np.asarray(self.pos), (self.b,))
        return oa.attention(self.q, self.k, self.v, lens, first, self.d ** -0.5 if self.scale is None else self.scale, self.causal, self.mask, self.table,
                            None if self.mapping is None else self.mapping.cpu().numpy(), self.both, self.g if train else None)

    def run(self, train):
        q, k, v, g = self.tensors()
        table = None if self.table is None else torch.from_numpy(self.table).cuda()
        if not train:
            with torch.no_grad():
                return [ct.attention(q, k, v, bias=table, **self.arguments())]
        leaves = [x.requires_grad_() for x in (q, k, v, table) if x is not None]
        out = ct.attention(q, k, v, bias=table, **self.arguments())
        grads = torch.autograd.grad(out, leaves, g)
        for x, y in zip(leaves[:3], grads):
            assert y.shape == x.shape and (self.lay[0] == "strided" or y.stride() == x.stride())
        return [out.detach(), *grads]

    def check(self, train):
        got = self.run(train)
        want, bound = self.oracle(train)
        if not train:
            want, bound = [want], [bound]
        assert len(got) == len(want)
        for name, x, y, e in zip(("out", "dq", "dk", "dv", "dtable"), got, want, bound):
            x = x.cpu().numpy().astype(np.float64)
            assert np.isfinite(x).all(), name
            off = np.abs(x - y) / e
            assert off.max(initial=0) <= 1, (name, off.max(), np.unravel_index(off.argmax(), off.shape))


SHAPES = [  # b, h, held, n, length, d: edges of tiles, of waves and of workgroups, heads that share keys, odd sizes of everything
    (1, 1, 1, 1, 1, 64), (1, 2, 1, 1, 63, 64), (2, 3, 3, 2, 65, 64), (1, 4, 2, 31, 64, 64), (1, 2, 2, 33, 33, 64), (2, 2, 1, 100, 100, 64), (1, 1, 1, 128, 128, 64), (1, 2, 1, 129, 200, 64),
    (1, 2, 2, 64, 300, 128), (1, 4, 1, 97, 161, 128), (1, 1, 1, 257, 257, 128), (1, 3, 1, 50, 130, 80), (2, 2, 2, 70, 70, 96), (1, 2, 1, 66, 190, 256), (1, 1, 1, 40, 70, 160),
    (1, 2, 2, 45, 77, 16), (1, 1, 1, 20, 30, 8), (1, 2, 1, 17, 90, 1), (1, 1, 1, 35, 80, 33), (1, 2, 2, 30, 70, 100), (2, 1, 1, 5, 600, 72),
]


@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(gpu, shape, layout):
    print("forward", shape, layout, flush=True)
    _Case(*shape, layout=layout).check(False)


@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(gpu, shape, layout):
    print("gradients", shape, layout, flush=True)
    _Case(*shape, layout=layout, causal=shape[3] % 2 == 0, seed=1).check(True)


@pytest.mark.parametrize("bias", [None, "one", "both"])
@pytest.mark.parametrize("mask", [None, "key", "query"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 150, 64), (1, 2, 1, 200, 330, 128), (1, 2, 2, 40, 90, 256), (2, 2, 1, 1, 260, 80)], ids=str)
def test_biases_and_masks(gpu, shape, causal, mask, bias):
    print("biases and masks", shape, causal, mask, bias, flush=True)
    _Case(*shape, layout="columns" if shape[3] == 70 else "rows", causal=causal, mask=mask, bias=bias).check(True)
