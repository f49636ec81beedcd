"""Attention over fp16 keys and values and rotary positions where they can go wrong: rows without keys, numbers that are none in places that do not count, lengths and positions of any
value, unusual strides, streams, captured graphs, and a layer of all of them together."""
import copy

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

import cpm_kernels_amd.kernels as ck
import cpm_kernels_amd.torch as ct
from oracle import attention as oa
from test_attention_gpu import _Case, _ints, _mapping, _normal

pytestmark = pytest.mark.gpu

HALF = dict(dtype=torch.half, device="cuda")


def _np(x):
    return x.detach().cpu().numpy().astype(np.float64)


def _within(got, want, bound, name):
    got = _np(got)
    assert np.isfinite(got).all(), name
    off = np.abs(got - want) / bound
    assert off.max(initial=0) <= 1, (name, off.max(), np.unravel_index(off.argmax(), off.shape))


NAMES = ("out", "dq", "dk", "dv", "dtable")


# ---- lengths, positions, scales, biases ----

@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("b,h,held,n,length,d", [(4, 2, 1, 40, 100, 64), (4, 4, 1, 3, 300, 128), (4, 2, 2, 130, 72, 80)])
def test_unequal_sequences(gpu, b, h, held, n, length, d, train, layout):
    """Lengths and positions on the device: none, one, all, beyond both ends."""
    for i, (lens, pos) in enumerate((([0, 1, length, length - 7], None), ([-5, 2 ** 31 - 1, 33, 64], [0, 5, -20, 3]), ([length, length, 7, 0], [2 ** 31 - 1, -2 ** 31, -n, 0]))):
        print("unequal", b, h, held, n, length, d, train, layout, i, flush=True)
        case = _Case(b, h, held, n, length, d, layout=layout, lens=lens, pos=pos, causal=True, seed=i)
        if pos is not None:
            case.pos = np.clip(np.asarray(pos, np.int64), -2 ** 30, 2 ** 30 - 1).tolist()
        case.check(train)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0, 2.0 ** -10])
@pytest.mark.parametrize("n,d", [(3, 64), (70, 64), (70, 128), (40, 256)])
def test_scales(gpu, n, d, scale, train):
    print("scales", n, d, scale, train, flush=True)
    _Case(1, 2, 1, n, 90, d, scale=scale, bias="one", std=0.7, seed=2).check(train)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("count,distance,bias", [(1, 1, "one"), (2, 1, "both"), (2, 2, "both"), (7, 1024, "one"), (64, 512, "both"), (300, 40, "one")])
@pytest.mark.parametrize("n", [2, 80])
def test_tables_of_any_size(gpu, n, count, distance, bias, train):
    print("tables", n, count, distance, bias, train, flush=True)
    rng = np.random.default_rng(distance)
    mapping = rng.integers(0, max(1, count // 2 if bias == "both" else count), distance).astype(np.int32)
    _Case(2, 4, 2, n, 700, 64, causal=bias == "one", bias=bias, count=count, distance=distance, mapping=mapping, seed=3).check(train)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("n", [2, 80])
def test_biases_of_minus_infinity(gpu, n, train):
    """A bucket that nothing looks at: its keys count no more than masked ones, and have no gradients."""
    print("minus infinity", n, train, flush=True)
    mapping = (np.arange(64) // 8).astype(np.int32)
    case = _Case(1, 2, 1, n, 150, 64, causal=True, bias="one", count=8, distance=64, mapping=mapping, seed=4)
    case.table[:, 2] = -np.inf
    got = case.run(train)
    rel = 150 - n + np.arange(n)[:, None] - np.arange(150)
    case.mask = np.broadcast_to((mapping[np.clip(rel, 0, 63)] != 2)[None], (1, n, 150)).copy()
    case.table = case.table.copy()
    case.table[:, 2] = 0
    want, bound = case.oracle(train)
    for name, x, y, e in zip(NAMES, got, want if train else [want], bound if train else [bound]):
        _within(x, y, e, name)


@pytest.mark.parametrize("n", [2, 80])
def test_bucket_numbers_outside_of_the_table(gpu, n):
    """They are taken for its ends, by either pass."""
    print("buckets", n, flush=True)
    mapping = np.array([0, 1, 2, 99, 3, -4, 2 ** 31 - 1, -2 ** 31] * 4, np.int32)
    case = _Case(1, 2, 1, n, 100, 64, causal=True, bias="one", count=5, distance=32, mapping=mapping, seed=5)
    got = case.run(True)
    case.mapping = _ints(np.clip(mapping, 0, 4))
    for name, x, y, e in zip(NAMES, got, *case.oracle(True)):
        _within(x, y, e, name)


@pytest.mark.parametrize("n,d,mask", [(70, 256, "query"), (40, 256, "key"), (70, 64, None), (3, 128, "key"), (3, 256, None)])
@pytest.mark.parametrize("bias", ["one", "both"])
def test_largest_tables_and_far_positions(gpu, n, d, mask, bias):
    """As many distances as there may be beside the largest heads, and positions at either end of what is told apart."""
    print("largest tables", n, d, mask, bias, flush=True)
    distance = 1024 if bias == "one" else 512
    mapping = np.random.default_rng(d).integers(0, 16, distance).astype(np.int32)
    for pos in ([0, 900], [2 ** 30 - 1, -2 ** 30]):
        _Case(2, 2, 1, n, 330, d, causal=False, bias=bias, count=32, distance=distance, mapping=mapping, mask=mask, pos=pos, seed=31).check(True)


@pytest.mark.parametrize("train", [False, True])
def test_a_scale_of_nothing(gpu, train):
    print("scale of nothing", train, flush=True)
    _Case(1, 2, 1, 70, 90, 64, scale=2.0 ** -120, bias="one", seed=32).check(train)


# ---- places that do not count ----

BAD = [np.nan, np.inf, -np.inf, 65504.0]


@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
@pytest.mark.parametrize("d", [40, 64, 128, 256])
@pytest.mark.parametrize("n", [2, 90])
@pytest.mark.parametrize("kind", ["length", "key", "query"])
def test_keys_that_do_not_count(gpu, kind, n, d, layout):
    """Keys behind a sequence, and keys that a mask leaves out for all, may hold anything: results and gradients are those of zeros in their places, and they have none."""
    print("keys that do not count", kind, n, d, layout, flush=True)
    for length in (104, 203):
        case = _Case(2, 2, 1, n, length, d, layout=layout, causal=False, seed=6)
        rng = np.random.default_rng(7)
        out = np.zeros((2, length), bool)
        if kind == "length":
            case.lens, case.pos = [length - 30, 9], 0
            out[0, -30:], out[1, 9:] = True, True
        else:
            out = rng.random((2, length)) < 0.3
            out[1, 64:128] = True
            seen = ~out[:, None]
            case.mask = seen if kind == "key" else seen & (rng.random((2, n, length)) < 0.8)
        filler = np.array(BAD, np.float16)[rng.integers(0, len(BAD), case.k.shape)]
        clean = copy.copy(case)
        clean.k = np.where(out[:, None, :, None], np.float16(0), case.k)
        case.k, case.v = (np.where(out[:, None, :, None], filler, x) for x in (case.k, case.v))
        clean.v = case.v            # (whose largest finite one is in the bound)
        want, bound = clean.oracle(True)
        got = case.run(True)
        for name, x, y, e in zip(NAMES, got, want, bound):
            _within(x, y, e, name)
        for x in got[2:4]:
            assert (_np(x)[np.broadcast_to(out[:, None, :, None], x.shape)] == 0).all()
        _within(case.run(False)[0], want[0], clean.oracle(False)[1], "inference")


@pytest.mark.parametrize("layout", ["rows", "columns"])
@pytest.mark.parametrize("which", ["k", "v", "q", "g"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_numbers_that_are_none_stay_with_those_that_see_them(gpu, d, bad, which, layout):
    """Two halves of queries and keys that do not see each other, by a mask or by causality: what is wrong in one half leaves the other as it is, in both passes."""
    print("stay", d, bad, which, layout, flush=True)
    n = 168
    half = np.arange(n) >= 100
    for causal in (False, True):
        case = _Case(1, 2, 1, n, n, d, layout=layout, causal=causal, seed=8)
        if not causal:
            case.mask = (half[:, None] == half[None])[None].copy()
        want, bound = case.oracle(True)
        x = {"k": case.k, "v": case.v, "q": case.q, "g": case.g}[which]
        x[0, 0, 130, 3] = bad
        got = case.run(True)
        for i, (name, y, w, e) in enumerate(zip(NAMES, got, want, bound)):
            # (causal: the first half's keys are seen by the second half's queries, and their gradients with it)
            if causal and i >= 2:
                continue
            _within(y[:, :, :100], w[:, :, :100], e[:, :, :100], name)
        infers = case.run(False)[0]
        _within(infers[:, :, :100], want[0][:, :, :100], bound[0][:, :, :100], "inference")
        if which in ("k", "v") and np.isnan(bad):
            sees = 130 if causal else 100
            # (a key is looked at in all its units, a value in its own)
            seen = got[0][0, :, sees:] if which == "k" else got[0][0, :, sees:, 3]
            assert bool(torch.isnan(seen).all()) and bool(torch.isnan(infers[0, :, sees:, 3]).all())
        if which == "g" and np.isnan(bad):
            assert bool(torch.isnan(got[1][0, 0, 130]).all())


@pytest.mark.parametrize("n", [3, 100])
@pytest.mark.parametrize("kind", ["mask", "length", "position"])
def test_queries_without_keys(gpu, kind, n):
    """Zeros, and zeros for gradients, whatever their results' gradients are."""
    print("without keys", kind, n, flush=True)
    case = _Case(2, 2, 2, n, 120, 64, causal=kind == "position", seed=9)
    none = np.zeros((2, n), bool)
    if kind == "mask":
        case.mask = np.random.default_rng(1).random((2, n, 120)) < 0.5
        case.mask[0, n // 2:] = False
        none[0, n // 2:] = True
    elif kind == "length":
        case.lens, case.pos = [0, 50], 0
        none[0] = True
    else:
        case.pos = [-2, 5]
        none[0, :2] = True
    want, bound = case.oracle(True)
    case.g = np.where(none[:, None, :, None], np.float16(np.nan), case.g)
    got = case.run(True)
    for name, x, y, e in zip(NAMES, got, want, bound):
        _within(x, y, e, name)
    for x in (*got[:2], case.run(False)[0]):
        assert (_np(x).transpose(0, 2, 1, 3)[none] == 0).all()


def test_empty_calls(gpu):
    for b, h, held, n, length, d in ((0, 2, 1, 5, 5, 64), (1, 0, 0, 5, 5, 64), (1, 2, 1, 0, 5, 64), (1, 2, 1, 5, 0, 64), (1, 2, 1, 5, 5, 0), (2, 2, 2, 0, 0, 8)):
        print("empty", b, h, held, n, length, d, flush=True)
        for mask in (None, torch.ones((b, length), dtype=torch.bool, device="cuda"), torch.ones((b, n, length), dtype=torch.bool, device="cuda")):
            q, k, v = torch.ones((b, h, n, d), **HALF), torch.ones((b, held, length, d), **HALF), torch.ones((b, held, length, d), **HALF)
            table = torch.ones((h, 4), **HALF)
            with torch.no_grad():
                assert ct.attention(q, k, v, mask=mask).shape == q.shape
            leaves = [x.requires_grad_() for x in (q, k, v, table)]
            out = ct.attention(q, k, v, mask=mask, bias=table, mapping=_ints([0, 1, 2]), causal=False)
            assert not out.any()
            for x, g in zip(leaves, torch.autograd.grad(out, leaves, torch.ones_like(out))):
                assert g.shape == x.shape and not g.any()
    rotary = ct.RotaryEmbedding(8)
    for shape in ((0, 2, 3, 8), (1, 0, 3, 8), (1, 2, 0, 8)):
        x = torch.ones(shape, **HALF)
        assert rotary(x).shape == x.shape
        rotary.inplace(x, x.clone())
    torch.cuda.synchronize()


# ---- magnitudes ----

@pytest.mark.parametrize("gstd", [2.0 ** -20, 1.0, 2000.0])
@pytest.mark.parametrize("d", [64, 128])
def test_magnitudes_of_gradients(gpu, d, gstd):
    """From fp16's smallest numbers to a loss scale."""
    print("magnitudes", d, gstd, flush=True)
    case = _Case(1, 4, 2, 70, 150, d, gstd=gstd, seed=10)
    case.v = (case.v.astype(np.float32) * 2.0 ** -4).astype(np.float16)
    case.check(True)


@pytest.mark.parametrize("std", [4.0, 12.0])
def test_sharp_probabilities(gpu, std):
    """Rows that look at one key, almost: dp and D nearly cancel."""
    print("sharp", std, flush=True)
    _Case(1, 2, 1, 90, 200, 64, std=std ** 0.5, scale=1.0, seed=11).check(True)
    _Case(1, 2, 1, 20, 200, 64, std=std ** 0.5, scale=1.0, seed=11).check(False)


# ---- strides ----

LAYOUTS = [("rows", "columns", "rows", "strided"), ("columns", "rows", "strided", "rows"), ("strided", "rows", "columns", "columns"), ("columns", "columns", "rows", "rows")]


@pytest.mark.parametrize("layouts", LAYOUTS, ids=str)
@pytest.mark.parametrize("n,d", [(5, 64), (72, 64), (88, 128)])
def test_unlike_layouts(gpu, n, d, layouts):
    print("unlike layouts", n, d, layouts, flush=True)
    case = _Case(2, 4, 2, n, 160, d, layouts=layouts, mask="query", bias="one", seed=12)
    want, bound = case.oracle(True)
    q, k, v, g = case.tensors()
    table = torch.from_numpy(case.table).cuda()
    leaves = [x.requires_grad_() for x in (q, k, v, table)]
    out = ct.attention(q, k, v, bias=table, **case.arguments())
    for name, x, y, e in zip(NAMES, (out, *torch.autograd.grad(out, leaves, g)), want, bound):
        _within(x, y, e, name)
    _within(case.run(False)[0], want[0], case.oracle(False)[1], "inference")


@pytest.mark.parametrize("shift", [1, 4, 8])
@pytest.mark.parametrize("n", [2, 70])
def test_rows_off_their_boundaries(gpu, n, shift):
    """Units are neighbours, but rows begin anywhere."""
    print("off boundaries", n, shift, flush=True)
    case = _Case(1, 2, 2, n, 130, 64, seed=13)

    def moved(x):
        wide = torch.full((*x.shape[:3], x.shape[3] + shift), float("nan"), **HALF)
        wide[..., shift:] = torch.from_numpy(x).cuda()
        return wide[..., shift:]
    q, k, v, g = (moved(x) for x in (case.q, case.k, case.v, case.g))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = ct.attention(q, k, v)
    for name, x, y, e in zip(NAMES, (out, *torch.autograd.grad(out, leaves, g)), *case.oracle(True)):
        _within(x, y, e, name)
    _within(case.run(False)[0], case.oracle(False)[0], case.oracle(False)[1], "inference")


def test_broadcast_inputs(gpu):
    """Keys and values of one sequence for a batch, one query for all heads, one gradient for everything."""
    print("broadcast", flush=True)
    case = _Case(3, 4, 2, 40, 90, 64, causal=False, seed=14)
    case.k[:], case.v[:], case.q[:] = case.k[:1], case.v[:1], case.q[:, :1]
    case.g[:] = np.float16(0.01)
    q, k, v = (torch.from_numpy(np.ascontiguousarray(x)).cuda().requires_grad_() for x in (case.q[:, :1], case.k[:1], case.v[:1]))
    out = ct.attention(q.expand(-1, 4, -1, -1), k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), causal=False)
    grads = torch.autograd.grad(out, (q, k, v), torch.full((), 0.01, **HALF).expand(out.shape))
    want, bound = case.oracle(True)
    _within(out, want[0], bound[0], "out")
    for i, (axis, x) in enumerate(((1, grads[0]), (0, grads[1]), (0, grads[2]))):
        # (each part's bound, and the roundings of the sum of 3 or 4 fp16 numbers: half a step of each partial sum, at most the sum of magnitudes)
        total, off = want[1 + i].sum(axis, keepdims=True), bound[1 + i].sum(axis, keepdims=True) + 3 * np.abs(want[1 + i]).sum(axis, keepdims=True) * 2.0 ** -11 + 2.0 ** -24
        _within(x, total, off, NAMES[1 + i])


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("n", [1, 60])
def test_beyond_32_bit_offsets(gpu, n, columns):
    """Keys whose last ones lie further than 2^32 bytes from the first."""
    print("offsets", n, columns, flush=True)
    length, far = 72, 2 ** 25
    space = torch.zeros((71 if columns else length - 1) * far + 2 ** 20, **HALF)
    rng = np.random.default_rng(15)
    case = _Case(1, 1, 1, n, length, 64, causal=False, seed=16)

    def spread(x, offset):
        if columns:
            view = torch.as_strided(space, (1, 1, length, 64), (0, 0, 1, far), offset)
        else:
            view = torch.as_strided(space, (1, 1, length, 64), (0, 0, far, 1), offset)
        view.copy_(torch.from_numpy(x).cuda())
        return view
    q, g = (torch.from_numpy(x).cuda() for x in (case.q, case.g))
    k, v = spread(case.k, 0), spread(case.v, 128)
    want, bound = case.oracle(True)
    with torch.no_grad():
        _within(ct.attention(q, k, v, causal=False), want[0], case.oracle(False)[1], "inference")
    leaves = [x.requires_grad_() for x in (q, k.detach(), v.detach())]
    out = ct.attention(*leaves, causal=False)
    for name, x, y, e in zip(NAMES, (out, *torch.autograd.grad(out, leaves, g)), want, bound):
        _within(x, y, e, name)
    assert rng is not None


def test_masks_of_any_stride(gpu):
    """A part of a larger mask, one mask for the batch, and one of 31 keys."""
    print("masks", flush=True)
    for n, length in ((50, 150), (3, 150), (50, 31), (2, 3), (2, 31)):
        case = _Case(2, 2, 1, n, length, 64, causal=False, mask="query", seed=17)
        wide = torch.zeros((2, n + 3, length + 13), dtype=torch.bool, device="cuda")
        wide[:, 3:, 5:5 + length] = torch.from_numpy(case.mask).cuda()
        q, k, v, g = case.tensors()
        leaves = [x.requires_grad_() for x in (q, k, v)]
        for mask, every in ((wide[:, 3:, 5:5 + length], case.mask), (wide[:1, 3:, 5:5 + length].expand(2, -1, -1), np.broadcast_to(case.mask[:1], case.mask.shape)),
                            (wide[:, 4, 5:5 + length], case.mask[:, 1:2])):
            case.mask = np.ascontiguousarray(every)
            out = ct.attention(q, k, v, causal=False, mask=mask)
            for name, x, y, e in zip(NAMES, (out, *torch.autograd.grad(out, leaves, g)), *case.oracle(True)):
                _within(x, y, e, name)
            with torch.no_grad():
                _within(ct.attention(q, k, v, causal=False, mask=mask), *case.oracle(False), "inference")


# ---- long keys in parts ----

@pytest.mark.parametrize("n,h,held,d", [(1, 2, 2, 64), (1, 16, 2, 128), (4, 8, 1, 64), (7, 4, 1, 128), (40, 2, 1, 64), (100, 1, 1, 128), (1, 2, 1, 256), (3, 12, 1, 96)])
@pytest.mark.parametrize("layout", ["rows", "columns"])
def test_long_keys(gpu, n, h, held, d, layout):
    """Parts of the keys, joined: sequences of unlike lengths among them, some without a key in most parts."""
    print("long keys", n, h, held, d, layout, flush=True)
    for lens in (None, [5000, 37], [4097, 0]):
        case = _Case(2, h, held, n, 5000, d, layout=layout, lens=lens, pos=None, seed=18)
        case.check(False)
    _Case(2, h, held, n, 3000, d, layout=layout, lens=[3000, 70], pos=None, seed=19).check(True)


@pytest.mark.parametrize("n,h,held,d", [(9, 8, 2, 64), (32, 12, 2, 128), (1, 100, 1, 64), (5, 40, 1, 96), (32, 8, 2, 40), (33, 8, 2, 64), (48, 4, 1, 128), (2, 130, 1, 64)])
@pytest.mark.parametrize("bias,mask", [(None, None), ("both", "query"), ("one", "key")])
def test_rows_of_many_heads(gpu, n, h, held, d, bias, mask):
    """Heads that share keys, from a few rows to more than the kernel of few rows takes."""
    print("many heads", n, h, held, d, bias, mask, flush=True)
    _Case(2, h, held, n, 700, d, causal=bias != "both", bias=bias, mask=mask, lens=[700, 131], pos=None if mask else [660, 100], seed=30).check(False)


# ---- order, streams, graphs ----

def test_the_same_bits_again(gpu):
    """No sum depends on an order that a run decides."""
    print("same bits", flush=True)
    for d in (64, 128):
        case = _Case(2, 8, 2, 300, 300, d, bias="both", causal=False, mask="query", seed=20)
        first = case.run(True)
        for _ in range(4):
            assert all(torch.equal(x, y) for x, y in zip(case.run(True), first))


def test_two_streams(gpu):
    """Calls on streams of their own, at once, and on one that is not the tensors' own."""
    print("streams", flush=True)
    cases = [_Case(1, 4, 2, 260, 260, 64, seed=21), _Case(2, 4, 4, 130, 400, 128, layout="columns", seed=22)]
    want = [c.run(True) for c in cases]
    inputs = [c.tensors() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (q, k, v, g), stream in zip(inputs, streams):
            with torch.cuda.stream(stream):
                leaves = [x.detach().requires_grad_() for x in (q, k, v)]
                out = ct.attention(*leaves)
                got.append([out, *torch.autograd.grad(out, leaves, g)])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def _captured(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


@pytest.mark.parametrize("n,h,held,length,d", [(1, 8, 2, 3000, 64), (5, 4, 1, 2000, 128), (50, 2, 2, 2000, 64), (200, 4, 2, 200, 128)])
def test_captured_calls(gpu, n, h, held, length, d):
    """Two graphs of the same call, replayed in turn with eager work between: every replay is the eager result."""
    print("captured", n, h, held, length, d, flush=True)
    q, k, v = (torch.randn((2, x, y, d), device="cuda").half() for x, y in ((h, n), (held, length), (held, length)))
    lens, rotary = _ints([length, length // 2]), ct.RotaryEmbedding(d)

    @torch.no_grad()
    def step():
        return ct.attention(rotary(q, pos=lens), k, v, lens)
    graphs = [_captured(step) for _ in range(2)]
    for i in range(6):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda") * (1 + 0.2 * i))
        lens -= 1
        graph, out = graphs[i % 2]
        graph.replay()
        other = ct.attention(torch.randn((1, 2, 300, 64), device="cuda").half(), k[:1, :1].contiguous()[..., :64], v[:1, :1].contiguous()[..., :64])
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool(torch.isfinite(other).all())


def test_a_captured_training_step(gpu):
    print("captured training", flush=True)
    q, k, v, g = (torch.randn((2, x, 150, 64), device="cuda").half() for x in (4, 2, 2, 4))
    table, mapping, rotary = torch.randn((4, 32), device="cuda").half(), _mapping(False), ct.RotaryEmbedding(64, 32)
    leaves = [x.requires_grad_() for x in (q, k, v, table)]

    def step():
        out = ct.attention(*rotary(q, k, 7), v, bias=table, mapping=mapping)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]
    graph, got = _captured(step)
    for i in range(4):
        with torch.no_grad():
            for x in (*leaves, g):
                x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_saved_tensors_that_move(gpu):
    """What the backward pass needs, packed to host memory and unpacked elsewhere, or computed again: the same gradients."""
    print("saved tensors", flush=True)
    from torch.utils.checkpoint import checkpoint
    for layout in ("rows", "columns"):
        case = _Case(2, 4, 2, 70, 150, 64, layout=layout, bias="both", causal=False, mask="query", lens=[150, 99], pos=[80, 3], seed=29)
        want = case.run(True)
        q, k, v, g = case.tensors()
        table = torch.from_numpy(case.table).cuda()
        leaves = [x.requires_grad_() for x in (q, k, v, table)]
        with torch.autograd.graph.save_on_cpu():
            out = ct.attention(q, k, v, bias=table, **case.arguments())
        spoil = [torch.full((2, 70, 150), 77, dtype=torch.uint8, device="cuda") for _ in range(8)]         # (where the mask was, perhaps)
        got = [out, *torch.autograd.grad(out, leaves, g)]
        assert len(spoil) == 8
        for name, x, y, e in zip(NAMES, got, *case.oracle(True)):           # (unpacked they are rows: products of columns are added up in another order)
            _within(x, y, e, name)
        if layout == "rows":
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        again = checkpoint(lambda *x: ct.attention(*x[:3], bias=x[3], **case.arguments()), *leaves, use_reentrant=False)
        assert all(torch.equal(x, y) for x, y in zip((again, *torch.autograd.grad(again, leaves, g)), want))


# ---- refusals ----

def test_refusals(gpu):
    q, k = torch.zeros((2, 4, 5, 64), **HALF), torch.zeros((2, 2, 9, 64), **HALF)
    table, mapping = torch.zeros((4, 8), **HALF), _ints([0, 1])
    ones = lambda *s: torch.ones(s, dtype=torch.bool, device="cuda")           # noqa: E731
    for bad in (lambda: ct.attention(q.float(), k, k), lambda: ct.attention(q, k.float(), k), lambda: ct.attention(q, k, k[:, :, :4]), lambda: ct.attention(q, k[:1], k[:1]),
                lambda: ct.attention(q, k[..., :32], k[..., :32]), lambda: ct.attention(q[:, :3], k, k), lambda: ct.attention(q, k.cpu(), k), lambda: ct.attention(q, k, k.cpu()),
                lambda: ct.attention(q, k, k, 10), lambda: ct.attention(q, k, k, -1), lambda: ct.attention(q, k, k, 2.5), lambda: ct.attention(q, k, k, _ints([1])),
                lambda: ct.attention(q, k, k, _ints([1, 1]).long()), lambda: ct.attention(q, k, k, _ints([1, 1]).cpu()), lambda: ct.attention(q, k, k, pos=-1),
                lambda: ct.attention(q, k, k, pos=2 ** 30), lambda: ct.attention(q, k, k, scale=float("nan")), lambda: ct.attention(q, k, k, scale=float("inf")),
                lambda: ct.attention(q, k, k, mask=ones(2, 8)), lambda: ct.attention(q, k, k, mask=ones(2, 4, 9)), lambda: ct.attention(q, k, k, mask=ones(2, 9).byte()),
                lambda: ct.attention(q, k, k, mask=ones(2, 9).cpu()), lambda: ct.attention(q, k, k, mask=ones(2, 18)[:, ::2]), lambda: ct.attention(q, k, k, bias=table),
                lambda: ct.attention(q, k, k, bias=table[:2], mapping=mapping), lambda: ct.attention(q, k, k, bias=table.float(), mapping=mapping),
                lambda: ct.attention(q, k, k, bias=table, mapping=mapping.long()), lambda: ct.attention(q, k, k, bias=table[:, :0], mapping=mapping),
                lambda: ct.attention(q, k, k, bias=table, mapping=mapping[:0]), lambda: ct.attention(q, k, k, bias=table, mapping=torch.zeros(1025, dtype=torch.int32, device="cuda")),
                lambda: ct.attention(torch.zeros((1, 1, 1, 257), **HALF), torch.zeros((1, 1, 1, 257), **HALF), torch.zeros((1, 1, 1, 257), **HALF))):
        with pytest.raises(AssertionError):
            bad()
    rotary = ct.RotaryEmbedding(64)
    for bad in (lambda: rotary(q.float()), lambda: rotary(q[..., :32]), lambda: rotary(q, k), lambda: rotary(q, pos=1.5), lambda: rotary(q, pos=2 ** 31), lambda: rotary(q, pos=_ints([1])),
                lambda: rotary(q, pos=_ints([1, 1]).long()), lambda: rotary(q, pos=_ints([1, 1]).cpu()), lambda: rotary.inplace(q.clone().requires_grad_()),
                lambda: rotary.inplace(q[:, :1].expand(-1, 4, -1, -1)), lambda: rotary(q[0])):
        with pytest.raises(AssertionError):
            bad()


def test_gradients_of_gradients_and_tangents_are_refused(gpu):
    """They would be lost silently."""
    q = torch.randn((1, 2, 5, 64), device="cuda").half().requires_grad_()
    rotary = ct.RotaryEmbedding(64)
    for out in (ct.attention(q, q, q), rotary(q)):
        with pytest.raises(AssertionError, match="gradients"):
            torch.autograd.grad(out.float().sum(), q, create_graph=True)
    x = q.detach()
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: ct.attention(dual, x, x), lambda: ct.attention(x, x, dual), lambda: rotary(dual)):
            with pytest.raises(Exception):
                call()


def test_results_written_over(gpu):
    """What the backward pass needs may not be changed before it."""
    x, w = torch.randn((1, 2, 5, 64), device="cuda").half(), torch.randn(64, device="cuda").half().requires_grad_()
    kept = (w * x).float().sum()
    ct.RotaryEmbedding(64).inplace(x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(kept, w)
    with pytest.raises(AssertionError, match="twice"):
        ct.RotaryEmbedding(64).inplace(x, x)
    with torch.inference_mode():
        ct.RotaryEmbedding(64).inplace(torch.ones((1, 2, 5, 64), **HALF))
    q = torch.randn((1, 2, 5, 64), device="cuda").half().requires_grad_()
    out = ct.attention(q, q, q)
    out.detach().add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.float().sum(), q)


# ---- calls on addresses ----

@pytest.mark.parametrize("guard", [4096, 4100])
@pytest.mark.parametrize("n,d", [(2, 64), (70, 64), (70, 128)])
def test_calls_on_addresses(gpu, n, d, guard):
    """The kernels layer gives the module's results, and leaves what lies before and behind its outputs and workspaces alone, which begin anywhere on 4 bytes."""
    print("addresses", n, d, guard, flush=True)
    b, h, held, length = 2, 4, 2, 1200
    case = _Case(b, h, held, n, length, d, bias="one", mask="key", seed=23)
    want, infers = case.run(True), case.run(False)[0]
    st = torch.cuda.current_stream().cuda_stream
    q, k, v, g = (x.contiguous() for x in case.tensors())
    table, mask = torch.from_numpy(case.table).cuda(), torch.from_numpy(case.mask).cuda()

    def room(count, dtype):
        raw = torch.full((count * dtype.itemsize + 2 * guard,), 77, dtype=torch.uint8, device="cuda")
        rooms.append(raw)
        return raw[guard:raw.numel() - guard].view(dtype)
    rooms = []
    head = (b, h, held, n, d, length, q.data_ptr(), q.stride(), k.data_ptr(), k.stride(), v.data_ptr(), v.stride(), None, length, None, -1, True, d ** -0.5, table.data_ptr(),
            case.mapping.data_ptr(), 32, 128, False, mask.data_ptr(), mask.stride(0), 0)
    size = ck.attention_forward_workspace(b, h, held, n, d, length)
    out, rest = room(q.numel(), torch.half), room(q.numel(), torch.half)
    lse = room(b * (h * n + held * (length // 256 + 1)), torch.float)
    space = room(size, torch.uint8)
    ck.attention_forward(*head, out.data_ptr(), q.stride(), None, None, space.data_ptr() if size else None, st)
    assert torch.equal(out.view(q.shape), infers)
    ck.attention_forward(*head, out.data_ptr(), q.stride(), lse.data_ptr(), rest.data_ptr(), space.data_ptr() if size else None, st)
    dq, dk, dv, dtable = room(q.numel(), torch.half), room(k.numel(), torch.half), room(v.numel(), torch.half), room(table.numel(), torch.half)
    work = room(ck.attention_backward_workspace(b, h, held, n, length, 128, False), torch.uint8)
    ck.attention_backward(*head, out.data_ptr(), q.stride(), lse.data_ptr(), rest.data_ptr(), g.data_ptr(), g.stride(), dq.data_ptr(), q.stride(), dk.data_ptr(), k.stride(),
                          dv.data_ptr(), v.stride(), dtable.data_ptr(), work.data_ptr(), st)
    torch.cuda.synchronize()
    for name, x, y in zip(NAMES, (out, dq, dk, dv, dtable), want):
        assert torch.equal(x.view(y.shape), y), name
    for raw in rooms:
        assert bool((raw[:guard] == 77).all()) and bool((raw[raw.numel() - guard:] == 77).all())


# ---- against differences, and all of it together ----

@pytest.mark.parametrize("d", [64, 128])
def test_gradients_against_differences(gpu, d):
    """What the kernels' gradients say the result grows by along a direction, and by how much the formula's does (in fp64, differences of 2^-12)."""
    print("differences", d, flush=True)
    case = _Case(1, 4, 2, 60, 90, d, bias="both", causal=False, mask="query", seed=24)
    got = case.run(True)[1:]
    _, bound = case.oracle(True)
    rng = np.random.default_rng(25)
    point = [x.astype(np.float64) for x in (case.q, case.k, case.v, case.table)]
    for i in range(4):
        way = rng.standard_normal(point[i].shape)

        def at(step):
            q, k, v, table = (x + step * way if j == i else x for j, x in enumerate(point))
            return (oa.attention(q, k, v, [90], [30], d ** -0.5, False, case.mask, table, case.mapping.cpu().numpy(), True)[0] * case.g).sum()
        h = 2.0 ** -12
        slope, twice = (at(h) - at(-h)) / (2 * h), (at(2 * h) - at(-2 * h)) / (4 * h)
        # (the differences' own error is a third of what doubling the step changes; rounding: 2^-52 of the sum's size over the step)
        own = abs(twice - slope) + 2.0 ** -40
        assert abs((_np(got[i]) * way).sum() - slope) <= (bound[1 + i] * np.abs(way)).sum() + own


def test_a_layer(gpu):
    """Rotary positions, attention with shared heads, and both backward passes, against the plain forms in fp64: each step's bound carried through the next."""
    print("layer", flush=True)
    rng = np.random.default_rng(26)
    b, h, held, n, d = 2, 6, 2, 75, 64
    q, k, v, g = _normal(rng, (b, h, n, d)), _normal(rng, (b, held, n, d)), _normal(rng, (b, held, n, d)), _normal(rng, (b, h, n, d), 0.02)
    rotary = ct.RotaryEmbedding(d, 32)
    tq, tk, tv, tg = (torch.from_numpy(x).cuda().requires_grad_() for x in (q, k, v, g))
    rq, rk = rotary(tq, tk, 100)
    out = ct.attention(rq, rk, tv)
    got = torch.autograd.grad(out, (rq, rk, tv, tq, tk), tg.detach())
    # the attention on what the rotation really gave, then the rotation back of what the attention really gave
    want, bound = oa.attention(_np(rq), _np(rk), v, [n] * b, [0] * b, d ** -0.5, True, dout=g)
    for name, x, y, e in zip(NAMES, (out, *got[:3]), want, bound):
        _within(x, y, e, name)
    at, turns = np.tile(100 + np.arange(n), (b, 1)), rotary.turns.numpy()
    for x, y, dx, dy in ((q, rq, got[3], got[0]), (k, rk, got[4], got[1])):
        _within(y, *(z + (i > 0) * 1e-300 for i, z in enumerate(oa.rotary(x, at, turns, 1.0, False))), "turned")
        _within(dx, *(z + (i > 0) * 1e-300 for i, z in enumerate(oa.rotary(_np(dy), at, turns, 1.0, False, inverse=True))), "turned back")


def test_a_prompt_and_the_steps_behind_it(gpu):
    """A prompt through the fp16 attention, then steps with the rotated keys in a cache of this attention's and in one of 8 bits: the steps' rows are the prompt's, to rounding."""
    print("steps", flush=True)
    rng = np.random.default_rng(27)
    b, h, held, n, d, length = 2, 8, 2, 40, 64, 64
    q, k, v = (torch.from_numpy(_normal(rng, (b, x, n, d), sized=False)).cuda() for x in (h, held, held))
    rotary = ct.RotaryEmbedding(d)
    with torch.no_grad():
        rq, rk = rotary(q, k)
        every = ct.attention(rq, rk, v)
        keys, values = (torch.full((b, held, length, d), float("nan"), **HALF) for _ in range(2))
        cache = ct.QuantizedKV.empty(b, held, length, d)
        first = n - 6
        keys[:, :, :first], values[:, :, :first] = rk[:, :, :first], v[:, :, :first]
        cache.write(rk[:, :, :first], v[:, :, :first], 0)
        want, bound = oa.attention(_np(rq), _np(rk), _np(v), [n] * b, [0] * b, d ** -0.5, True)
        for t in range(first, n):
            sq, sk = q[:, :, t:t + 1].clone(), k[:, :, t:t + 1].clone()
            rotary.inplace(sq, sk, _ints([t, t]))
            assert torch.equal(sq, rq[:, :, t:t + 1]) and torch.equal(sk, rk[:, :, t:t + 1])
            keys[:, :, t:t + 1], values[:, :, t:t + 1] = sk, v[:, :, t:t + 1]
            cache.write(sk, v[:, :, t:t + 1], t)
            step = ct.attention(sq, keys, values, t + 1)
            _within(step, want[:, :, t:t + 1], bound[:, :, t:t + 1], "step")
            # (8 bits: a value is off by 1 / 254 of the largest at most, a score by 1 / 254 of the keys' largest times the query's sum, and a result by 2 of that times the values')
            eighth = cache.attention(sq, t + 1)
            ktop, vtop = float(rk.abs().max()), float(v.abs().max())
            score = ktop / 254 * float(sq.float().abs().sum(3).max()) * d ** -0.5
            assert float((eighth.float() - step.float()).abs().max()) <= vtop / 254 + (np.exp(2 * score) - 1) * vtop + 0.01 * vtop
        _within(every, want, bound, "prompt")


def test_rotary_of_any_tensors(gpu):
    """In place under any strides without overlap, positions on another stride, the same tensor for both, and a module taken to half precision."""
    print("rotary", flush=True)
    rng = np.random.default_rng(28)
    x = rng.standard_normal((2, 3, 20, 64)).astype(np.float16)
    rotary = ct.RotaryEmbedding(64, 48, interleaved=True)
    at = torch.from_numpy(rng.integers(-100, 5000, (20, 2)).astype(np.int32)).cuda().t()
    want, bound = oa.rotary(x, at.cpu().numpy(), rotary.turns.numpy(), 1.0, True)
    t = torch.from_numpy(x).cuda()
    ways = {"rows": t.clone(), "columns": t.transpose(2, 3).contiguous().transpose(2, 3), "heads": t.transpose(1, 2).contiguous().transpose(1, 2),
            "part": torch.zeros((2, 3, 20, 65), **HALF)[..., 1:].copy_(t)}
    results = []
    for way, y in ways.items():
        copied = rotary(y, pos=at)
        rotary.inplace(y, pos=at)
        assert torch.equal(y, copied), way
        results.append(y)
        _within(y, want, bound + 1e-300, way)
    assert all(torch.equal(y, results[0]) for y in results)
    twice = rotary(t, t, at)
    assert torch.equal(twice[0], results[0]) and torch.equal(twice[1], results[0]) and torch.equal(copy.deepcopy(rotary).half()(t, pos=at), results[0])
