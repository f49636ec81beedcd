"""The key/value cache in 8 bits against float64: what is stored bit for bit, what is read to one rounding, the attention within the bound that the oracle
derives from the roundings on the way.  Its rounding of integers is checked for every pair of a value and a magnitude by tests/native/kv_round_check.c."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

import cpm_kernels_amd.kernels as ck
import cpm_kernels_amd.torch as ct
from oracle import kv_cache as ok

pytestmark = pytest.mark.gpu


def _tokens(rng, b, h, n, d, layout, std=1.0):
    """fp16 (b, h, n, d) as numpy, and on the GPU under the strides of `layout`."""
    x = (rng.standard_normal((b, h, n, d)) * std * np.exp(0.5 * rng.standard_normal((1, h, 1, d)))).astype(np.float16)
    t = torch.from_numpy(x).cuda()
    if layout == "columns":
        t = t.transpose(2, 3).contiguous().transpose(2, 3)
    elif layout == "rows":          # (b, n, h, d)
        t = t.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "strided":       # neither axis contiguous, nor any start of a row aligned
        wide = torch.zeros((b, h, n, 2 * d + 1), dtype=torch.half, device="cuda")
        wide[..., 1::2] = t
        t = wide[..., 1::2]
    return x, t


class _Both:
    """A cache on the GPU and in numpy, of the same random content."""

    def __init__(self, rng, b, h, length, d, block, fill=True):
        self.length, self.block = length, block
        self.k = np.zeros((b, h, length, d), np.int8)
        self.v = self.k.copy()
        self.ka = np.zeros((b, h, length // block), np.float16)
        self.va = self.ka.copy()
        if fill:
            full, none = np.full(b, length), np.zeros(b, int)
            for ints, top in ((self.k, self.ka), (self.v, self.va)):
                ok.write(ints, top, (rng.standard_normal((b, h, length, d)) * np.exp(0.5 * rng.standard_normal((1, h, 1, d)))).astype(np.float16), none, full)
        self.cache = ct.QuantizedKV(*(torch.from_numpy(x).cuda() for x in (self.k, ok.by_sixteen(self.v), self.ka, self.va)))

    def write(self, k, v, pos, count=None):
        b, n = k[0].shape[0], k[0].shape[2]
        each = pos.cpu().numpy() if isinstance(pos, torch.Tensor) else np.full(b, pos)
        real = count.cpu().numpy() if count is not None else np.full(b, n)
        self.cache.write(k[1], v[1], pos, count)
        ok.write(self.k, self.ka, k[0], each, real)
        ok.write(self.v, self.va, v[0], each, real)

    def check(self):
        c = self.cache
        for got, want in ((c.key_absmax.cpu().numpy(), self.ka), (c.value_absmax.cpu().numpy(), self.va)):
            assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
        assert np.array_equal(c.keys.cpu().numpy(), self.k)
        assert np.array_equal(ok.by_token(c.values.cpu().numpy()), self.v)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


WRITES = [  # b, h, tokens, dim, length, block, pos
    (1, 1, 1, 16, 16, 16, 0), (2, 3, 1, 64, 128, 64, 100), (1, 2, 1, 80, 96, 32, 95), (1, 1, 64, 64, 64, 64, 0), (2, 2, 37, 64, 256, 64, 0),
    (2, 2, 37, 128, 256, 64, 61), (1, 2, 200, 80, 256, 16, 7), (1, 1, 300, 256, 384, 128, 70), (1, 3, 129, 240, 256, 128, 127), (3, 1, 500, 48, 512, 32, 12),
    (1, 1, 1000, 16, 1024, 16, 24), (2, 1, 5, 64, 64, 64, 59), (2, 2, 1, 256, 256, 128, 131), (1, 3, 1, 208, 64, 16, 47),
]


@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
@pytest.mark.parametrize("b,h,n,d,length,block,pos", WRITES)
def test_write(gpu, b, h, n, d, length, block, pos, layout):
    print("write", b, h, n, d, length, block, pos, layout, flush=True)
    rng = np.random.default_rng(n * d + pos)
    both = _Both(rng, b, h, length, d, block)
    both.write(_tokens(rng, b, h, n, d, layout), _tokens(rng, b, h, n, d, layout, 3.0), pos)
    both.check()


def test_write_unlike_strides(gpu):
    rng = np.random.default_rng(5)
    both = _Both(rng, 2, 2, 128, 64, 32)
    both.write(_tokens(rng, 2, 2, 70, 64, "rows"), _tokens(rng, 2, 2, 70, 64, "columns"), 9)
    both.check()


@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_write_where_each_sequence_stands(gpu, n, block):
    """Positions and numbers on the device: negative ones, ones behind the cache, ranges across its end, none and more tokens than there are."""
    print("write each", n, block, flush=True)
    rng = np.random.default_rng(n + block)
    b, h, d, length = 9, 2, 64, 256
    both = _Both(rng, b, h, length, d, block)
    k, v = _tokens(rng, b, h, n, d, "rows"), _tokens(rng, b, h, n, d, "columns")
    pos = _ints([0, 1, 17, 128, -1, 250, 255, 256, -2 ** 31])
    both.write(k, v, pos)
    both.check()
    both.write(k, v, _ints([3, 200, 40, 2 ** 31 - 1, 12, 64, 100, 255, 0]), _ints([n, 0, n // 2, n, 2 * n, -3, 1, n, 2 ** 31 - 1]))
    both.check()


@pytest.mark.parametrize("block,d", [(16, 80), (64, 64), (128, 128)])
def test_write_token_by_token(gpu, block, d):
    """Each token larger than those before it, then smaller: every write of a block changes its magnitude and rounds its older integers again, then none does."""
    print("token by token", block, d, flush=True)
    rng = np.random.default_rng(block)
    both = _Both(rng, 2, 2, 2 * block, d, block, fill=False)
    for i in range(block + 3):
        size = 1.15 ** i if i < block // 2 else 0.5
        both.write(_tokens(rng, 2, 2, 1, d, "rows", size), _tokens(rng, 2, 2, 1, d, "rows", size), i)
    both.check()


@pytest.mark.parametrize("block,d", [(16, 80), (64, 64), (128, 32)])
def test_tokens_one_by_one_stay_near_themselves(gpu, block, d):
    """Half a step of a block's magnitude for the rounding when a token comes in, and half a step of the new one each time that its block grows."""
    print("near themselves", block, d, flush=True)
    rng = np.random.default_rng(block)
    cache = ct.QuantizedKV.empty(2, 3, 2 * block, d, block)
    k, v = (_tokens(rng, 2, 3, 2 * block, d, "rows") for _ in range(2))
    off = [np.zeros((2, 3, 2 * block)) for _ in range(2)]
    grown = 0
    for i in range(2 * block):
        before = [x[:, :, i // block].clone() for x in (cache.key_absmax, cache.value_absmax)]
        cache.write(k[1][:, :, i:i + 1], v[1][:, :, i:i + 1], i)
        first = i // block * block
        for bound, old, new in zip(off, before, (cache.key_absmax, cache.value_absmax)):
            new = new[:, :, i // block].cpu().numpy().astype(np.float64)
            grows = (new > old.cpu().numpy()) & (i > first)
            grown += grows.sum()
            bound[:, :, first:i] += (grows * new / 254)[..., None]
            bound[:, :, i] = new / 254
    assert grown > 2 * 2 * 3 * 2
    for x, bound, ints, top in zip((k, v), off, (cache.keys.cpu().numpy(), ok.by_token(cache.values.cpu().numpy())), (cache.key_absmax, cache.value_absmax)):
        err = np.abs(ok.values_of(ints, top.cpu().numpy()) - x[0].astype(np.float64))
        assert (err <= bound[..., None] * (1 + 1e-12)).all(), (err / bound[..., None]).max()


@pytest.mark.parametrize("n,pos", [(40, 0), (1, 5), (23, 9)])
def test_write_of_extreme_values(gpu, n, pos):
    """Infinities count as the largest finite numbers, NaN as nothing; zeros, subnormal magnitudes, halves between two integers."""
    print("write extremes", n, pos, flush=True)
    rng = np.random.default_rng(n)
    b, h, d, length = 8, 1, 32, 64
    both = _Both(rng, b, h, length, d, 16)
    x = rng.standard_normal((b, h, n, d)).astype(np.float16)
    x[0, 0, 0, 3], x[0, 0, -1, 4] = np.inf, -np.inf
    x[1, 0, 0, 5] = np.nan
    x[2] = 0
    x[3] *= np.float16(2.0 ** -20)
    x[4] = (rng.integers(-254, 255, x[4].shape) / 2 * (2.0 ** -24)).astype(np.float16) * 2          # multiples of the smallest number
    x[5] = (rng.integers(-254, 255, x[5].shape) / 2).astype(np.float16)                             # halves beside a magnitude of 127
    x[5, 0, :, 0] = 127
    x[6] = np.nan
    x[7] = np.float16(65504) * np.sign(x[7])
    t = torch.from_numpy(x).cuda()
    both.write((x, t), (-x, -t), pos)
    both.check()


@pytest.mark.parametrize("n", [1, 3])
def test_write_of_zeros_over_other_tokens(gpu, n):
    """Zeros (and what counts as zero) at a block's start leave the block the magnitude 0, whatever it held: the tokens behind them are rounded by their own."""
    print("write zeros", n, flush=True)
    rng = np.random.default_rng(n)
    both = _Both(rng, 2, 2, 64, 32, 16)
    x = np.zeros((2, 2, n, 32), np.float16)
    x[1] = np.nan
    t = torch.from_numpy(x).cuda()
    for pos in (16, 48):
        both.write((x, t), (x, t), pos)
    both.check()
    for i in range(2):
        both.write(_tokens(rng, 2, 2, 1, 32, "rows", 1e-3), _tokens(rng, 2, 2, 1, 32, "rows", 1e-3), 16 + n + i)
    both.check()


READS = [(1, 1, 1, 16, 16, 16, 0), (2, 3, 101, 80, 256, 32, 13), (1, 2, 256, 64, 256, 64, 0), (2, 1, 300, 128, 256, 64, -20), (1, 1, 64, 256, 128, 128, 31),
         (1, 1, 5, 64, 64, 16, 70), (1, 1, 5, 64, 64, 16, -9), (2, 2, 33, 240, 96, 32, 16)]


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("b,h,n,d,length,block,start", READS)
def test_read(gpu, b, h, n, d, length, block, start, columns):
    print("read", b, h, n, d, length, block, start, columns, flush=True)
    rng = np.random.default_rng(n + d)
    both = _Both(rng, b, h, length, d, block)
    each = start + 7 * np.arange(b)
    for at in [start] * (b == 1) + [_ints(each.tolist())]:
        got = both.cache.read(at, n, columns=columns)
        for x, ints, top in zip(got, (both.k, both.v), (both.ka, both.va)):
            assert x.shape == (b, h, n, d) and x.stride(2 if columns else 3) == 1
            want = ok.read(ints, top, each, n)
            # one rounding of a product that is off by 2^-22 of itself at most
            assert (np.abs(x.cpu().numpy().astype(np.float64) - want) <= np.abs(want) * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25).all()


def test_read_to_any_strides(gpu):
    rng = np.random.default_rng(3)
    both = _Both(rng, 2, 2, 64, 48, 16)
    c = both.cache
    wide = torch.full((2, 2, 2, 40, 97), 7.0, dtype=torch.half, device="cuda")
    k, v = wide[0, ..., 1::2], wide[1, ..., 1::2]
    ck.kv_read_int8(2, 2, 40, 48, 64, 16, c.keys.data_ptr(), c.values.data_ptr(), c.key_absmax.data_ptr(), c.value_absmax.data_ptr(), None, 3,
                    k.data_ptr(), v.data_ptr(), k.stride(), torch.cuda.current_stream().cuda_stream)
    k2, v2 = c.read(3, 40)
    assert torch.equal(k, k2) and torch.equal(v, v2) and bool((wide[..., 0::2] == 7).all())


def _attend(rng, b, h, group, n, d, length, block, lens, layout="rows", **kw):
    both = _Both(rng, b, h // group, length, d, block)
    q = _tokens(rng, b, h, n, d, layout)
    each = lens.cpu().numpy() if isinstance(lens, torch.Tensor) else np.full(b, lens)
    pos = kw.get("pos")
    on_host = dict(kw)
    if pos is not None:
        on_host["pos"] = pos.cpu().numpy() if isinstance(pos, torch.Tensor) else np.full(b, pos)
    for name in ("mask", "bias", "mapping"):
        if kw.get(name) is not None:
            on_host[name] = kw[name].cpu().numpy()
    if "mask" in on_host and on_host["mask"].ndim == 2:
        on_host["mask"] = on_host["mask"][:, None]
    on_host["table"] = on_host.pop("bias", None)
    causal = on_host.pop("causal", True)
    want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, each, d ** -0.5, causal, **on_host)
    got = both.cache.attention(q[1], lens, **kw)
    assert got.shape == q[1].shape
    err = np.abs(got.cpu().numpy().astype(np.float64) - want)
    assert np.isfinite(err).all() and (err <= bound).all(), (err / bound).max()
    both.check()            # (read only)
    return both, q, got


def _bias(rng, heads, bidirectional, buckets=32, distances=128):
    mapping = torch.empty(distances, dtype=torch.int32, device="cuda")
    ck.position_embedding_init(buckets, distances, mapping.data_ptr(), bidirectional, torch.cuda.current_stream().cuda_stream)
    return dict(bias=torch.from_numpy(rng.standard_normal((heads, buckets)).astype(np.float16)).cuda(), mapping=mapping, bidirectional=bidirectional)


SHAPES = [  # b, h, group, n, d, length, block, lens
    (1, 1, 1, 1, 16, 16, 16, 1), (1, 4, 1, 1, 64, 128, 64, 101), (2, 4, 2, 1, 80, 256, 32, 255), (1, 8, 8, 1, 128, 512, 64, 511), (2, 2, 2, 3, 64, 64, 16, 64),
    (1, 3, 3, 7, 64, 192, 64, 130), (1, 20, 20, 2, 48, 96, 32, 90), (1, 2, 1, 40, 64, 128, 128, 100), (1, 2, 2, 70, 128, 256, 64, 200), (1, 1, 1, 33, 256, 256, 16, 255),
    (1, 2, 1, 17, 208, 64, 32, 64), (2, 2, 1, 150, 64, 320, 64, 300), (1, 1, 1, 1, 64, 4096, 64, 4090), (1, 2, 2, 2, 192, 2048, 128, 1999),
    (1, 1, 1, 300, 80, 512, 16, 500), (1, 2, 1, 129, 112, 256, 64, 129),
]


@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
@pytest.mark.parametrize("b,h,group,n,d,length,block,lens", SHAPES)
def test_attention(gpu, b, h, group, n, d, length, block, lens, layout):
    print("attention", b, h, group, n, d, length, block, lens, layout, flush=True)
    _attend(np.random.default_rng(d + n), b, h, group, n, d, length, block, lens, layout)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bidirectional", [True, False])
@pytest.mark.parametrize("b,h,group,n,d,length,block,lens", [SHAPES[i] for i in (0, 1, 3, 5, 6, 8, 11, 12)])
def test_attention_with_position_bias(gpu, b, h, group, n, d, length, block, lens, bidirectional, causal):
    print("attention bias", b, h, group, n, d, length, block, lens, bidirectional, causal, flush=True)
    rng = np.random.default_rng(d + n)
    _attend(rng, b, h, group, n, d, length, block, lens, causal=causal, **_bias(rng, h, bidirectional))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind", ["key", "row", "query", "broadcast"])
@pytest.mark.parametrize("b,h,group,n,d,length,block,lens", [SHAPES[i] for i in (1, 4, 5, 8, 9, 11, 14)])
def test_attention_with_mask(gpu, b, h, group, n, d, length, block, lens, kind, causal):
    """Queries whose mask leaves nothing give zeros; a stride of 0 over the batch; masks that end nowhere near 16 bytes."""
    print("attention mask", b, h, group, n, d, length, block, lens, kind, causal, flush=True)
    rng = np.random.default_rng(d + n)
    rows = n if kind in ("query", "broadcast") else 1
    mask = torch.from_numpy(rng.random((b, rows, length + 3)) < 0.3).cuda()[..., 3:]
    mask[-1, -1] = False
    mask[0, 0, :lens // 2] = False
    if kind == "key":
        mask = mask[:, 0]
    if kind == "broadcast":
        mask = mask[:1].expand(b, rows, length)
    both, _, got = _attend(rng, b, h, group, n, d, length, block, lens, causal=causal, mask=mask)
    if kind != "broadcast":
        assert bool((got[-1, :, -1] == 0).all())


@pytest.mark.parametrize("n", [1, 5, 40])
def test_attention_of_unequal_sequences(gpu, n):
    """Lengths and positions on the device: none, one, more than the cache has, queries before the first and behind the last key; what lies behind
    a sequence's keys, magnitudes that are no numbers among it, is not looked at."""
    print("attention each", n, flush=True)
    rng = np.random.default_rng(n)
    b, h, d, length, block = 8, 2, 64, 256, 32
    lens = _ints([0, 1, 33, 64, 200, 256, 1000, -5])
    _attend(rng, b, h, 1, n, d, length, block, lens)
    _attend(rng, b, h, 2, n, d, length, block, lens, causal=False)
    pos = _ints([0, 0, 40, -3, 100, 300, -2 ** 31, 2 ** 31 - 1])
    _attend(rng, b, h, 1, n, d, length, block, lens, pos=pos, **_bias(rng, h, True))
    _attend(rng, b, h, 1, n, d, length, block, 200, pos=150)
    both, q, got = _attend(rng, b, h, 1, n, d, length, block, lens)
    c = both.cache
    for i, keys in enumerate([0, 1, 33, 64, 200, 256, 256, 0]):
        behind = (keys + block - 1) // block
        c.key_absmax[i, :, behind:], c.value_absmax[i, :, behind:] = float("nan"), float("inf")
        c.keys[i, :, keys:] = 77
        c.values[i, :, (keys + 15) // 16:] = -99
    assert torch.equal(c.attention(q[1], lens), got)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 40, 70, 200])
def test_attention_in_parts(gpu, n, d):
    """Caches so long that their keys are divided among workgroups, for sequences that fill all parts, one, some of the last and none."""
    print("attention parts", n, d, flush=True)
    rng = np.random.default_rng(n + d)
    lens = _ints([0, 1, 64, 65, 1000, 2111, 2999, 3008])
    both, q, got = _attend(rng, 8, 1, 1, n, d, 3008, 32, lens)
    assert not bool(got[0].any())
    pos = _ints([5, 0, 2000, -40, 3000, 1, 2700, 100])
    _attend(rng, 8, 2, 2, n, d, 3008, 16, lens, layout="columns", pos=pos, **_bias(rng, 2, True))
    mask = torch.from_numpy(rng.random((8, n, 3008)) < 0.01).cuda()
    mask[4] = False
    _, _, got = _attend(rng, 8, 2, 1, n, d, 3008, 64, lens, causal=False, mask=mask)
    assert not bool(got[4].any())


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("n", [5, 256])
def test_attention_of_long_parts(gpu, n, d):
    """So many heads that a workgroup has dozens of tiles one after the other; two heads of one sequence are looked at."""
    print("attention long parts", n, d, flush=True)
    rng = np.random.default_rng(n + d)
    b, h, length = 2, 128, 2688
    cache = ct.QuantizedKV.empty(b, h, length, d, block=16)
    k, v, q = (torch.randn((b, h, rows, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(i + d)).half() for i, rows in enumerate((length, length, n)))
    cache.write(k, v, 0)
    bias = _bias(rng, h, False)
    got = cache.attention(q, 2650, **bias)
    some = [0, 77]
    want, bound = ok.attention(q[1:, some].cpu().numpy(), cache.keys[1:, some].cpu().numpy(), ok.by_token(cache.values[1:, some].cpu().numpy()),
                               cache.key_absmax[1:, some].cpu().numpy(), cache.value_absmax[1:, some].cpu().numpy(), [2650], d ** -0.5, True,
                               table=bias["bias"][some].cpu().numpy(), mapping=bias["mapping"].cpu().numpy())
    err = np.abs(got[1:, some].cpu().numpy().astype(np.float64) - want)
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("n", [1, 20, 100])
def test_attention_of_other_scales(gpu, n):
    """A negative factor turns the order of the scores around, 0 makes the mean of the values; a large one leaves one key."""
    print("attention scales", n, flush=True)
    rng = np.random.default_rng(n)
    for scale in (-0.125, 0.0, 4.0, -4.0):
        both = _Both(rng, 2, 2, 256, 64, 64)
        q = _tokens(rng, 2, 2, n, 64, "rows")
        want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, np.full(2, 250), scale, True)
        err = np.abs(both.cache.attention(q[1], 250, scale=scale).cpu().numpy().astype(np.float64) - want)
        assert (err <= bound).all(), (scale, (err / np.maximum(bound, 1e-30)).max())


@pytest.mark.parametrize("buckets,distances,bidirectional", [(32, 128, True), (8, 20, False), (64, 1024, False), (64, 512, True), (4, 3, True), (1, 1, False)])
@pytest.mark.parametrize("n,group", [(1, 1), (1, 20), (9, 4), (150, 1)])
def test_attention_with_bias_tables_of_any_size(gpu, n, group, buckets, distances, bidirectional):
    print("attention bias tables", n, group, buckets, distances, bidirectional, flush=True)
    rng = np.random.default_rng(n + buckets)
    mapping = torch.from_numpy(np.sort(rng.integers(0, max(buckets // (2 if bidirectional else 1), 1), distances)).astype(np.int32)).cuda()
    bias = dict(bias=torch.from_numpy(rng.standard_normal((group, buckets)).astype(np.float16)).cuda(), mapping=mapping, bidirectional=bidirectional)
    _attend(rng, 1, group, group, n, 64, 1472, 64, 1450, causal=False, pos=700, **bias)
    _attend(rng, 1, group, group, n, 64, 1472, 64, 1450, **bias)


@pytest.mark.parametrize("buckets,distances", [(4, 1), (2, 1), (1, 1), (4, 2)])
@pytest.mark.parametrize("n,group,d", [(1, 1, 64), (1, 20, 64), (9, 4, 128), (33, 2, 64), (5, 1, 256), (70, 1, 64), (150, 2, 128), (100, 1, 256)])
def test_attention_with_two_sided_bias_tables_of_few_distances(gpu, n, group, d, buckets, distances):
    """One bias for all keys up to a query's position and one for all behind it (or three): queries before the first key, among the keys, in the last of them."""
    print("attention two-sided tables", n, group, d, buckets, distances, flush=True)
    rng = np.random.default_rng(n + buckets)
    mapping = torch.from_numpy(np.arange(distances).astype(np.int32) % max(buckets // 2, 1)).cuda()
    bias = dict(bias=torch.from_numpy(rng.standard_normal((group, buckets)).astype(np.float16)).cuda(), mapping=mapping, bidirectional=True)
    for pos in (-n // 2, 700, 1440 - n):
        _attend(rng, 1, group, group, n, d, 1472, 64, 1450, causal=False, pos=_ints([pos]), **bias)
    _attend(rng, 1, group, group, n, d, 1472, 64, 1450, **bias)
    _attend(rng, 1, group, group, n, d, 192, 32, 131, causal=False, pos=60, **bias)


@pytest.mark.parametrize("n,d,group", [(1, 64, 1), (1, 128, 1), (1, 192, 1), (1, 256, 2), (3, 128, 8), (20, 64, 1), (20, 112, 1), (70, 64, 1)])
def test_attention_of_many_heads(gpu, n, d, group):
    """More heads than compute units, a position bias and a mask: what few heads share among more waves or workgroups, each here does by itself."""
    print("attention many heads", n, d, group, flush=True)
    rng = np.random.default_rng(n + d)
    b, h = 8 * group, 72
    lens = _ints(([0, 1, 130, 64, 190, 77, 192, 100] * group)[:b])
    _attend(rng, b, h, group, n, d, 192, 32, lens)
    mask = torch.from_numpy(rng.random((b, n, 192)) < 0.6).cuda()
    mask[4] = False
    _, _, got = _attend(rng, b, h, group, n, d, 192, 64, lens, mask=mask, **_bias(rng, h, True))
    assert not bool(got[4].any())


@pytest.mark.parametrize("n,d", [(1, 64), (5, 256), (40, 128), (100, 64)])
def test_attention_with_biases_of_minus_infinity(gpu, n, d):
    """Keys at distances whose bias is -inf do not count: single ones, whole tiles, all keys behind the table's end."""
    print("attention biases of -inf", n, d, flush=True)
    rng = np.random.default_rng(n + d)
    mapping = (np.arange(128) // 4).astype(np.int32)
    table = rng.standard_normal((2, 32)).astype(np.float16)
    both = _Both(rng, 2, 2, 640, d, 64)
    q = _tokens(rng, 2, 2, n, d, "rows")
    lens = np.array([600, 95])
    for without in ([5], [31], list(range(8, 32)), [0, 31]):
        bias = table.copy()
        bias[:, without] = -np.inf
        distance = np.clip((lens[:, None] - n + np.arange(n))[:, :, None] - np.arange(640), 0, 127)
        want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, lens, d ** -0.5, True, mask=~np.isin(mapping[distance], without), table=table, mapping=mapping)
        got = both.cache.attention(q[1], _ints(lens), bias=torch.from_numpy(bias).cuda(), mapping=torch.from_numpy(mapping).cuda())
        err = np.abs(got.cpu().numpy().astype(np.float64) - want)
        assert (err <= bound).all(), (without, (err / np.maximum(bound, 1e-30)).max())


@pytest.mark.parametrize("n,d", [(2, 64), (18, 128), (4, 256), (100, 64), (130, 128)])
def test_attention_of_queries_that_are_no_numbers(gpu, n, d):
    """A query with a NaN or an infinity gives NaN for itself; those beside it are as they were."""
    print("attention no numbers", n, d, flush=True)
    rng = np.random.default_rng(n + d)
    both = _Both(rng, 2, 4, 384, d, 64)
    q = _tokens(rng, 2, 8, n, d, "rows")
    want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, [380, 131], d ** -0.5, True)
    q[1][0, 3, n // 2, 7] = float("nan")
    q[1][1, 0, 0, 0] = float("inf")
    got = both.cache.attention(q[1], _ints([380, 131])).cpu().numpy().astype(np.float64)
    assert np.isnan(got[0, 3, n // 2]).all() and np.isnan(got[1, 0, 0]).any()
    got[0, 3, n // 2], got[1, 0, 0] = want[0, 3, n // 2], want[1, 0, 0]
    assert (np.abs(got - want) <= bound).all()


def test_attention_beside_magnitudes_far_apart(gpu):
    """Blocks of values 2^20 times as large as others, in and out of sight, and blocks of zeros: probabilities keep their bits."""
    print("attention magnitudes", flush=True)
    rng = np.random.default_rng(11)
    b, h, d, length, block = 3, 2, 64, 256, 16
    both = _Both(rng, b, h, length, d, block, fill=False)
    k, v = _tokens(rng, b, h, 250, d, "rows"), _tokens(rng, b, h, 250, d, "rows")
    size = np.exp2(rng.integers(-16, 5, (b, 1, 250, 1))).astype(np.float16)
    size[0, :, 32:80] = 0
    size[1, :, :] = 2.0 ** -14
    v = (v[0] * size, v[1] * torch.from_numpy(size).cuda())
    both.write(k, v, 0)
    both.check()
    for n in (1, 40):
        q = _tokens(rng, b, h, n, d, "rows", 3.0)
        want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, np.full(b, 250), d ** -0.5, True)
        err = np.abs(both.cache.attention(q[1], 250).cpu().numpy().astype(np.float64) - want)
        assert (err <= bound).all(), (err / bound).max()


def test_a_prompt_and_the_steps_behind_it(gpu):
    """Prompts of unequal length, then token by token, in the package's own layout: every step against float64 on the cache as the oracle keeps it."""
    print("prompt and steps", flush=True)
    rng = np.random.default_rng(21)
    b, h, d, block = 3, 4, 64, 16
    both = _Both(rng, b, h, 96, d, block, fill=False)
    n = 40
    real = np.array([40, 3, 17])
    bias = _bias(rng, h, False)
    k, v, q = (_tokens(rng, b, h, n, d, "columns") for _ in range(3))
    both.write(k, v, 0, _ints(real.tolist()))
    both.check()

    def check(q, lens, **kw):
        want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, lens, d ** -0.5, True, table=bias["bias"].cpu().numpy(),
                                   mapping=bias["mapping"].cpu().numpy(), **kw)
        got = both.cache.attention(q[1], _ints(lens.tolist()), pos=None if "pos" not in kw else _ints(kw["pos"].tolist()), **bias)
        assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= bound).all()
        return got
    out = check(q, real, pos=np.zeros(b, int))
    assert out.transpose(2, 3).is_contiguous()
    lens = real.copy()
    for _ in range(20):
        k, v, q = (_tokens(rng, b, h, 1, d, "rows", 1 + rng.random()) for _ in range(3))
        both.write(k, v, _ints(lens.tolist()))
        lens += 1
        check(q, lens)
    both.check()
    # three drafted tokens, of which one stays: the next write begins inside of them
    k, v, q = (_tokens(rng, b, h, 3, d, "rows") for _ in range(3))
    both.write(k, v, _ints(lens.tolist()))
    check(q, lens + 3)
    k, v, q = (_tokens(rng, b, h, 1, d, "rows", 2.0) for _ in range(3))
    both.write(k, v, _ints((lens + 1).tolist()))
    check(q, lens + 2)
    both.check()


def test_beside_a_position_embedding(gpu):
    """A module's own weight and the table of its distances, as a model has them: its biases are the module's, for a prompt and for the steps behind it."""
    print("beside a position embedding", flush=True)
    b, h, d, n, length = 2, 4, 64, 90, 192
    for bidirectional in (True, False):
        rng = np.random.default_rng(61)
        pe = ct.PositionEmbedding(h, 32, 64, bidirectional).cuda().half()
        both = _Both(rng, b, h, length, d, 32, fill=False)
        k, v, q = (_tokens(rng, b, h, n, d, "columns") for _ in range(3))
        both.write(k, v, 0)
        mapping = torch.empty(pe.max_distance, dtype=torch.int32, device="cuda")
        ck.position_embedding_init(pe.num_buckets, pe.max_distance, mapping.data_ptr(), pe.bidirectional, torch.cuda.current_stream().cuda_stream)
        table = dict(table=pe.weight.detach().cpu().numpy(), mapping=mapping.cpu().numpy(), bidirectional=bidirectional)
        distance = np.arange(n)[None, :] - np.arange(n)[:, None]
        module = pe(n, n).detach().cpu().numpy().astype(np.float64)          # (heads, keys, queries)
        assert all(np.array_equal(module[i], ok.bucket_bias(table["table"][i], table["mapping"], distance, bidirectional)) for i in range(h))
        with pytest.raises(AssertionError, match="gradients"):
            both.cache.attention(q[1], n, bias=pe.weight, mapping=mapping, bidirectional=pe.bidirectional)
        with torch.no_grad():
            for causal in (True, False):
                want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, np.full(b, n), d ** -0.5, causal, **table)
                got = both.cache.attention(q[1], n, causal=causal, bias=pe.weight, mapping=mapping, bidirectional=pe.bidirectional)
                assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= bound).all()
            lens = np.full(b, n)
            for _ in range(3):
                k, v, q = (_tokens(rng, b, h, 1, d, "rows") for _ in range(3))
                both.write(k, v, _ints(lens.tolist()))
                lens += 1
                want, bound = ok.attention(q[0], both.k, both.v, both.ka, both.va, lens, d ** -0.5, True, **table)
                got = both.cache.attention(q[1], _ints(lens.tolist()), bias=pe.weight, mapping=mapping, bidirectional=pe.bidirectional)
                assert (np.abs(got.cpu().numpy().astype(np.float64) - want) <= bound).all()
        both.check()


@pytest.mark.parametrize("n", [2, 90])
def test_bucket_numbers_outside_of_the_table(gpu, n):
    """They count as the nearest in it."""
    print("buckets outside", n, flush=True)
    rng = np.random.default_rng(n)
    both = _Both(rng, 1, 2, 192, 64, 32)
    q = _tokens(rng, 1, 2, n, 64, "rows")[1]
    bias = torch.from_numpy(rng.standard_normal((2, 8)).astype(np.float16)).cuda()
    for bidirectional in (False, True):
        outside, inside = _ints([0, 7, 8, -1, 2 ** 31 - 1, -2 ** 31, 3]), _ints([0, 7, 7, 0, 7, 0, 3])
        if bidirectional:
            # (of keys behind the query 4 is added first: 3 + 4 is the last one)
            outside, inside = _ints([0, 1, 4, -9, 2 ** 31 - 1, 2, 2 ** 31 - 2]), _ints([0, 1, 3, -4, 3, 2, 3])
        for pos in (-n, 1 - n):
            kw = dict(causal=not bidirectional, bias=bias, bidirectional=bidirectional)
            if bidirectional:
                kw["pos"] = _ints([pos])
            got = both.cache.attention(q, 180, mapping=outside, **kw)
            assert torch.equal(got, both.cache.attention(q, 180, mapping=inside, **kw))


def test_captured_steps(gpu):
    """A step with positions on the device, captured and replayed with eager calls of other sizes between the replays; two graphs beside each other."""
    print("captured steps", flush=True)
    rng = np.random.default_rng(31)
    b, h, d, length = 2, 4, 64, 2048
    both = _Both(rng, b, h, length, d, 64)
    twin, spare = (ct.QuantizedKV(*(x.clone() for x in (both.cache.keys, both.cache.values, both.cache.key_absmax, both.cache.value_absmax))) for _ in range(2))
    pos, lens = _ints([100, 1990]), _ints([101, 1991])
    k, v, q = (torch.from_numpy(_tokens(rng, b, h, 1, d, "rows")[0]).cuda() for _ in range(3))

    def step(cache):
        cache.write(k, v, pos)
        return cache.attention(q, lens)
    step(spare)         # (a first call outside of a capture; the two caches compared take the same writes)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(both.cache)
        graphs.append((graph, out))
    for i in range(6):
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, device="cuda") * (i + 1))
        graph, out = graphs[i % 2]
        graph.replay()
        other = both.cache.attention(torch.randn((b, h, 70, d), device="cuda").half(), 1000)
        want = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and bool(torch.isfinite(other).all())
        assert all(torch.equal(x, y) for x, y in zip((both.cache.keys, both.cache.values, both.cache.key_absmax), (twin.keys, twin.values, twin.key_absmax)))
        pos += 1
        lens += 1


@pytest.mark.parametrize("n", [1, 3, 40, 100])
def test_calls_on_addresses(gpu, n):
    """The kernels layer: every argument of the three calls, all strides unlike, keys in parts, against the same calls of QuantizedKV, bit for bit."""
    print("calls on addresses", n, flush=True)
    rng = np.random.default_rng(n)
    b, held, heads, d, length, block = 3, 2, 4, 80, 2112, 32
    both = _Both(rng, b, held, length, d, block)
    c = both.cache
    mine = [x.clone() for x in (c.keys, c.values, c.key_absmax, c.value_absmax)]
    at = [x.data_ptr() for x in mine]
    stream = torch.cuda.current_stream().cuda_stream
    k, v, q = _tokens(rng, b, held, n, d, "rows")[1], _tokens(rng, b, held, n, d, "columns", 2.0)[1], _tokens(rng, b, heads, n, d, "strided")[1]
    for pos_each, pos, count in ((None, 37, None), (_ints([0, 1990, -1]), 0, _ints([n, (n + 1) // 2, 1]))):
        c.write(k, v, pos if pos_each is None else pos_each, count)
        ck.kv_write_int8(b, held, n, d, length, block, k.data_ptr(), k.stride(), v.data_ptr(), v.stride(), None if pos_each is None else pos_each.data_ptr(), pos,
                         None if count is None else count.data_ptr(), *at, stream)
        assert all(torch.equal(x, y) for x, y in zip(mine, (c.keys, c.values, c.key_absmax, c.value_absmax)))
    for start in (5, _ints([-3, 100, 2100])):
        got = torch.empty((2, b, held, d, n), dtype=torch.half, device="cuda").transpose(3, 4)
        each = isinstance(start, torch.Tensor)
        ck.kv_read_int8(b, held, n, d, length, block, *at, start.data_ptr() if each else None, 0 if each else start, got[0].data_ptr(), got[1].data_ptr(), got[0].stride(), stream)
        assert all(torch.equal(x, y) for x, y in zip(got, c.read(start, n)))
    size = ck.kv_attention_int8_workspace(b, heads, held, n, d, length)
    assert size > 0
    bias = _bias(rng, heads, True)
    mask = torch.from_numpy(rng.random((b, n, length + 5)) < 0.8).cuda()[..., 5:]
    lens, pos = _ints([2112, 700, 65]), _ints([2000, 650, 3])
    calls = [dict(lens=2100), dict(lens=lens, causal=False, scale=0.2), dict(lens=lens, pos=pos, mask=mask, **bias), dict(lens=2000, pos=1500, causal=False, mask=mask[:, 0])]
    for call in calls:
        where = {name: (call[name].data_ptr(), 0) if isinstance(call.get(name), torch.Tensor) else (None, call.get(name, -1)) for name in ("lens", "pos")}
        m = call.get("mask")
        masks = (None, 0, 0) if m is None else (m.data_ptr(), m.stride(0), m.stride(1) if m.ndim == 3 else 0)
        table = (bias["bias"].data_ptr(), bias["mapping"].data_ptr(), 32, 128, True) if "bias" in call else (None, None, 0, 0, False)
        out = torch.full((b, heads, n, 2 * d), 7.0, dtype=torch.half, device="cuda")
        space = torch.empty(size, dtype=torch.uint8, device="cuda")
        ck.kv_attention_int8(b, heads, held, n, d, length, block, q.data_ptr(), q.stride(), *at, *where["lens"], *where["pos"], call.get("causal", True),
                             call.get("scale", d ** -0.5), *table, *masks, out.data_ptr(), out[..., ::2].stride(), space.data_ptr(), stream)
        rest = dict(call)
        assert torch.equal(out[..., ::2], c.attention(q, rest.pop("lens"), **rest)) and bool((out[..., 1::2] == 7).all())


@pytest.mark.parametrize("n,d", [(3, 64), (40, 128), (100, 64), (100, 128), (100, 256)])
def test_workspaces_off_16_byte_boundaries(gpu, n, d):
    """A workspace starts at any multiple of 4 bytes; what lies around it stays as it is."""
    print("workspaces", n, d, flush=True)
    rng = np.random.default_rng(n + d)
    b, h, length, block = 2, 2, 2048, 64
    both = _Both(rng, b, h, length, d, block)
    c, q = both.cache, _tokens(rng, b, h, n, d, "rows")[1]
    want = c.attention(q, 2000)
    size = ck.kv_attention_int8_workspace(b, h, h, n, d, length) // 4
    assert size > 0
    for first in (0, 1, 2, 3):
        space = torch.full((size + 8,), 7.0, dtype=torch.float32, device="cuda")
        assert space.data_ptr() % 16 == 0
        out = torch.empty_like(q)
        ck.kv_attention_int8(b, h, h, n, d, length, block, q.data_ptr(), q.stride(), c.keys.data_ptr(), c.values.data_ptr(), c.key_absmax.data_ptr(), c.value_absmax.data_ptr(),
                             None, 2000, None, -1, True, d ** -0.5, None, None, 0, 0, False, None, 0, 0, out.data_ptr(), out.stride(), space.data_ptr() + 4 * first,
                             torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out, want) and bool((space[:first] == 7).all()) and bool((space[first + size:] == 7).all())


def test_calls_on_two_streams(gpu):
    """Results do not depend on what runs beside them, and come out the same every time."""
    print("two streams", flush=True)
    rng = np.random.default_rng(41)
    both = _Both(rng, 2, 4, 4096, 64, 64)
    q = [torch.from_numpy(_tokens(rng, 2, 4, n, 64, "rows")[0]).cuda() for n in (1, 30)]
    want = [both.cache.attention(x, 4000) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(10):
        got = []
        for x, stream in zip(q, streams):
            with torch.cuda.stream(stream):
                got.append(both.cache.attention(x, 4000))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_cache_beyond_32_bit_offsets(gpu):
    """4.3 GB of keys and as much of values: the last heads hold what they are given, the first ones stay as they are."""
    print("large cache", flush=True)
    b, h, length, d = 33, 32, 65536, 64
    cache = ct.QuantizedKV.empty(b, h, length, d)
    assert cache.keys.numel() > 2 ** 32
    rng = np.random.default_rng(51)
    x = torch.zeros((b, h, 200, d), dtype=torch.half, device="cuda")
    some, t = _tokens(rng, 1, h, 200, d, "rows")
    x[-1] = t[0]
    start = length - 200
    cache.write(x, 2 * x, start)
    k, v = cache.read(start, 200)
    ints, top = np.zeros((1, h, 256, d), np.int8), np.zeros((1, h, 4), np.float16)
    ok.write(ints, top, some, [56], [200])
    want = ok.values_of(ints, top)[:, :, 56:]
    assert (np.abs(k[-1].cpu().numpy().astype(np.float64) - want[0]) <= np.abs(want[0]) * (2.0 ** -11 + 2.0 ** -21) + 2.0 ** -25).all()
    assert torch.equal(v[-1], 2 * k[-1]) and not bool(k[:-1].any()) and not bool(cache.key_absmax[:-1].any())
    # the other keys are zeros: their scores are 0 and their values nothing
    q = x[:, :, -1:].contiguous()
    got = cache.attention(q, length)[-1].double().cpu().numpy()
    score = np.einsum("hd,htd->ht", some[0, :, -1].astype(np.float64), want[0]) * d ** -0.5
    p = np.exp(score - np.maximum(score.max(1), 0)[:, None])
    rest = (length - 200) * np.exp(-np.maximum(score.max(1), 0))
    exact = np.einsum("ht,htd->hd", p, 2 * want[0]) / (p.sum(1) + rest)[:, None]
    size = np.einsum("ht,htd->hd", p, 2 * np.abs(want[0])) / (p.sum(1) + rest)[:, None]
    # probabilities and result rounded to fp16 (2^-11 each), fp32 sums of 65536 / 64 values a lane
    assert (np.abs(got[:, 0] - exact) <= size * 2.0 ** -10 + np.abs(exact) * 2.0 ** -11 + 2.0 ** -20 * size.max()).all()


def test_empty_calls(gpu):
    cache = ct.QuantizedKV.empty(0, 4, 64, 64)
    x = torch.empty((0, 4, 3, 64), dtype=torch.half, device="cuda")
    cache.write(x, x, 0)
    assert cache.read(0, 5)[0].shape == (0, 4, 5, 64) and cache.attention(x, 3).shape == x.shape
    cache = ct.QuantizedKV.empty(2, 4, 64, 64)
    x = torch.empty((2, 4, 0, 64), dtype=torch.half, device="cuda")
    cache.write(x, x, 64)
    assert cache.attention(x, 3).shape == x.shape and cache.read(64)[0].shape == x.shape
    assert not bool(cache.attention(torch.ones((2, 8, 3, 64), dtype=torch.half, device="cuda"), 0).any())


def test_heads_without_units(gpu):
    """A cache of heads without units takes and gives empty tensors."""
    cache = ct.QuantizedKV.empty(2, 3, 64, 0)
    x = torch.empty((2, 3, 5, 0), dtype=torch.half, device="cuda")
    cache.write(x, x, 7)
    assert cache.read(0, 9)[1].shape == (2, 3, 9, 0)
    for kw in ({}, dict(scale=1.0), dict(lens=_ints([3, 9]))):
        assert cache.attention(x, kw.pop("lens", 12), **kw).shape == x.shape


def test_tangents_are_refused(gpu):
    """Forward-mode tangents would be lost as silently as gradients."""
    half = dict(dtype=torch.half, device="cuda")
    cache = ct.QuantizedKV.empty(2, 2, 64, 64)
    x, bias = torch.ones((2, 2, 5, 64), **half), torch.ones((2, 32), **half)
    mapping = torch.zeros(128, dtype=torch.int32, device="cuda")
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: cache.write(dual, x, 0), lambda: cache.write(x, dual, 0), lambda: cache.attention(dual, 5),
                     lambda: cache.attention(x, 5, bias=fw.make_dual(bias, bias), mapping=mapping)):
            with pytest.raises(AssertionError, match="gradients"):
                call()
        cache.write(x, x, 0)
        assert bool((cache.attention(x, 5, bias=bias, mapping=mapping) == 1).all())
    assert cache.attention(dual, 5).shape == x.shape


def test_refusals(gpu):
    half = dict(dtype=torch.half, device="cuda")
    cache = ct.QuantizedKV.empty(2, 2, 100, 64, block=32)
    assert cache.length == 128 and cache.block == 32
    k = torch.zeros((2, 2, 5, 64), **half)
    for bad in (lambda: cache.write(k, k, 124), lambda: cache.write(k, k, -1), lambda: cache.write(k.float(), k, 0), lambda: cache.write(k, k[:, :, :4], 0),
                lambda: cache.write(k[:1], k[:1], 0), lambda: cache.write(k[..., :32], k[..., :32], 0), lambda: cache.write(k, k, _ints([0])),
                lambda: cache.write(k, k, _ints([0, 0]).long()), lambda: cache.write(k, k, _ints([0, 0]).cpu()), lambda: cache.write(k.cpu(), k, 0),
                lambda: cache.write(k, k, 0, 3), lambda: cache.write(k.clone().requires_grad_(), k, 0), lambda: cache.read(_ints([0, 0])),
                lambda: cache.attention(k, 129), lambda: cache.attention(k, -1), lambda: cache.attention(k[:, :1], 5), lambda: cache.attention(k.clone().requires_grad_(), 5),
                lambda: cache.attention(k, 5, pos=-1), lambda: cache.attention(k, 5, mask=torch.ones((2, 127), dtype=torch.bool, device="cuda")),
                lambda: cache.attention(k, 5, mask=torch.ones((2, 4, 128), dtype=torch.bool, device="cuda")),
                lambda: cache.attention(k, 5, mask=torch.ones((2, 128), dtype=torch.uint8, device="cuda")),
                lambda: cache.attention(k, 5, bias=torch.zeros((2, 32), **half)), lambda: cache.attention(k, 5, bias=torch.zeros((1, 32), **half), mapping=_ints([0])),
                lambda: ct.QuantizedKV.empty(1, 1, 64, 72), lambda: ct.QuantizedKV.empty(1, 1, 64, 272), lambda: ct.QuantizedKV.empty(1, 1, 64, 64, block=48),
                lambda: ct.QuantizedKV(cache.keys, cache.values, cache.key_absmax[..., :3].contiguous(), cache.value_absmax[..., :3].contiguous()),
                lambda: ct.QuantizedKV(cache.keys[:, :, :64], cache.values[:, :, :4], cache.key_absmax[..., :2], cache.value_absmax[..., :2])):
        with pytest.raises(AssertionError):
            bad()
    with torch.no_grad():
        cache.attention(k.clone().requires_grad_(), 5)
    with pytest.raises(RuntimeError, match="limit"):
        cache.attention(k, 5, bias=torch.zeros((2, 32), **half), mapping=torch.zeros(600, dtype=torch.int32, device="cuda"), bidirectional=True)
    torch.cuda.synchronize()
