"""The key/value cache held in 8 bits: its operators as they are measured.

A cache keeps the keys and values of every sequence and head as int8, with the largest magnitude of each block of tokens beside them: a stored
integer q of a block with the magnitude a stands for q * a / 127.  Three operators work on it:

    write   tokens enter at a position of their sequence; a block that holds older tokens already grows to the larger magnitude, and the older
            integers are rounded again to it:  q = round(127 x / a),  q' = round(q a / a'), both to the nearest integer, halves away from zero
    read    a range of tokens comes back as fp16
    attend  softmax(scale q k^T + position bias, over the keys that length, causality and mask leave) v, straight from the integers: the decode
            step's single query, a few drafted tokens, whole chunks of a prompt

Storage: keys int8 (batch, heads, length, dim); values int8 (batch, heads, length / 16, dim, 16), sixteen tokens of one unit of a head side by side;
magnitudes fp16 (batch, heads, length / block), one set each.  Heads of 64 units, 16 to 64 heads, 1 to 32 sequences, up to 1024 tokens, 32 position
buckets over 128 tokens are the sizes of bench.py and the tests; 80 and 128 units, heads of keys that several heads of queries share and long caches
are generic.
"""
import math

import torch

own = False         # whether `run` calls the framework (set from outside)

HALF = torch.float16
BUCKETS, MAX_DISTANCE = 32, 128


def listed():
    return [
        # one sequence of a small model takes one token in: nothing but latency
        dict(name="write_step_1x16", kind="write", batch=1, heads=16, dim=64, length=128, block=64, tokens=1, pos=100, ragged=False, layout="rows"),
        # a serving batch in the middle of its sequences, every one somewhere else in its block
        dict(name="write_step_32x64", kind="write", batch=32, heads=64, dim=64, length=1024, block=64, tokens=1, pos=700, ragged=True, layout="rows"),
        # prompts of a full batch, as the projections leave them: (batch, hidden, tokens)
        dict(name="write_8x512", kind="write", batch=8, heads=64, dim=64, length=1024, block=64, tokens=512, pos=0, ragged=False, layout="columns"),
        # continued prompts of unequal length behind what the sequences hold, (batch, tokens, hidden)
        dict(name="write_ragged_16x500", kind="write", batch=16, heads=8, dim=128, length=1536, block=32, tokens=500, pos=1000, ragged=True, layout="rows"),
        # a whole cache back in fp16, for a program that goes on without it
        dict(name="read_16x1024", kind="read", batch=16, heads=64, dim=64, length=1024, block=64, tokens=1024, pos=0, ragged=False, layout="columns"),
        # a short piece out of the middle, heads of 80
        dict(name="read_1x101", kind="read", batch=1, heads=16, dim=80, length=256, block=32, tokens=101, pos=13, ragged=False, layout="rows"),
        # decode step of one sequence of a small model
        dict(name="attend_step_1x16", kind="attend", batch=1, heads=16, group=1, dim=64, length=128, block=64, tokens=1, keys=101, ragged=False,
             causal=True, bias=True, mask="", layout="rows"),
        # decode step of a serving batch
        dict(name="attend_step_32x64", kind="attend", batch=32, heads=64, group=1, dim=64, length=1024, block=64, tokens=1, keys=1024, ragged=True,
             causal=True, bias=True, mask="", layout="rows"),
        # decode step over long sequences, eight heads of queries to one of keys
        dict(name="attend_step_long", kind="attend", batch=4, heads=64, group=8, dim=128, length=32768, block=64, tokens=1, keys=32768, ragged=True,
             causal=True, bias=False, mask="", layout="rows"),
        # five drafted tokens looked over at once, each under a mask of its own
        dict(name="attend_draft_8x5", kind="attend", batch=8, heads=32, group=4, dim=128, length=4096, block=16, tokens=5, keys=3500, ragged=True,
             causal=False, bias=False, mask="query", layout="rows"),
        # the second half of a prompt, as the projections leave it
        dict(name="attend_chunk_8x512", kind="attend", batch=8, heads=64, group=1, dim=64, length=1024, block=64, tokens=512, keys=1024, ragged=False,
             causal=True, bias=True, mask="", layout="columns"),
        # the last chunk of a long prompt, no size a whole tile
        dict(name="attend_chunk_2000", kind="attend", batch=1, heads=32, group=4, dim=128, length=8192, block=64, tokens=2000, keys=8011, ragged=False,
             causal=True, bias=False, mask="", layout="rows"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _drawn(rng):
    kind = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend"])
    block = rng.choice([16, 32, 64, 64, 128])
    dim = rng.choice([64, 64, 80, 128, 128, 256])
    c = dict(kind=kind, batch=_log(rng, 1, 32), dim=dim, block=block, layout=rng.choice(["rows", "rows", "columns"]), ragged=rng.random() < 0.5)
    if kind != "attend":
        c["heads"] = _log(rng, 1, 64)
        c["tokens"] = rng.choice([1, _log(rng, 2, 2048)])
        c["pos"] = rng.choice([0, _log(rng, 1, 4096)])
        c["length"] = -(-(c["pos"] + c["tokens"] + rng.randrange(64)) // block) * block
        return c
    c["group"] = rng.choice([1, 1, 2, 4, 8])
    c["heads"] = _log(rng, 1, 64 // c["group"]) * c["group"]
    c["tokens"] = rng.choice([1, 1, rng.randrange(2, 9), _log(rng, 9, 2048), _log(rng, 64, 2048)])
    c["keys"] = c["tokens"] + _log(rng, 1, 32768) - 1
    c["length"] = -(-(c["keys"] + rng.randrange(64)) // block) * block
    c["causal"] = rng.random() < 0.7
    c["bias"] = rng.random() < 0.4
    c["mask"] = rng.choice(["", "", "key", "query"])
    return c


def draw(rng):
    most = max(_cost(c) for c in listed() if c["kind"] == "attend"), max(_cost(c) for c in listed() if c["kind"] != "attend")
    while True:
        c = _drawn(rng)
        if _cost(c) <= most[c["kind"] != "attend"] and _held(c) <= 2 ** 31:
            return c


def _cost(c):
    w = work(c)
    return w["bytes"] / 6e12 + w["flops"] / 6e14


def _held(c):
    """Bytes of the largest thing of a case: its cache, the scores of the plain form."""
    scores = 4 * c["batch"] * c["heads"] * c["tokens"] * c["length"] if c["kind"] == "attend" else 0
    return max(scores, 8 * c["batch"] * c["heads"] // c.get("group", 1) * c["length"] * c["dim"])


def _span(c):
    """Tokens that come back: of a write every block that it touches."""
    if c["kind"] == "read":
        return c["tokens"]
    return -(-(c["block"] - 1 + c["tokens"]) // c["block"]) * c["block"] if c["ragged"] else c["pos"] % c["block"] + c["tokens"]


# ---- inputs ---------------------------------------------------------------------------------------

class _Source:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32).mul_(std).half()

    def integers(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda", dtype=torch.int32)

    def tokens(self, batch, heads, tokens, dim, layout):
        """(batch, heads, tokens, dim) as a projection leaves it: units of very different size, as keys have them."""
        x = self.normal(batch, heads * dim, tokens) if layout == "columns" else self.normal(batch, tokens, heads * dim)
        size = torch.exp(0.5 * torch.randn((heads * dim, 1), generator=self.gen, device="cuda")).half()
        x *= size if layout == "columns" else size[:, 0]
        return x.view(batch, heads, dim, tokens).transpose(2, 3) if layout == "columns" else x.view(batch, tokens, heads, dim).transpose(1, 2)


def _nearest(x):
    """The nearest integer, halves away from zero."""
    return torch.sign(x) * torch.floor(x.abs() + 0.5)


def _cache(src, batch, heads, length, dim, block):
    """Keys or values (batch, heads, length, dim) as integers, and the blocks' magnitudes."""
    x = src.normal(batch, heads, length, dim)
    x *= torch.exp(0.5 * torch.randn((heads, 1, dim), generator=src.gen, device="cuda")).half()
    blocks = x.view(batch, heads, length // block, block, dim)
    top = blocks.abs().amax((3, 4))
    ints = _nearest(127 * blocks.float() / top[..., None, None].float().clamp(min=1e-30)).to(torch.int8)
    return ints.view(batch, heads, length, dim), top


def _by_sixteen(ints):
    """(batch, heads, length, dim) -> (batch, heads, length / 16, dim, 16)"""
    b, h, n, d = ints.shape
    return ints.view(b, h, n // 16, 16, d).transpose(3, 4).contiguous()


def _by_token(values):
    """The other way round."""
    b, h, n, d, _ = values.shape
    return values.transpose(3, 4).reshape(b, h, n * 16, d)


def _mapping():
    """Distance -> bucket of a one-sided bias: exact up to half of the buckets, logarithmic from there on."""
    exact = BUCKETS // 2
    far = [exact + int(math.log(i / exact) / math.log(MAX_DISTANCE / exact) * (BUCKETS - exact)) for i in range(exact, MAX_DISTANCE)]
    return torch.tensor(list(range(exact)) + [min(b, BUCKETS - 1) for b in far], dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    c, src = case, _Source(seed)
    b, held = c["batch"], c["heads"] // c.get("group", 1)
    s = {"case": c}
    keys, s["key_absmax"] = _cache(src, b, held, c["length"], c["dim"], c["block"])
    values, s["value_absmax"] = _cache(src, b, held, c["length"], c["dim"], c["block"])
    s["keys"], s["values"] = keys, _by_sixteen(values)
    if c["kind"] in ("write", "read"):
        # ragged: every sequence at a position of its own, in writes of several tokens with a number of its own too
        lo, hi = (c["pos"] + 1) // 2, c["pos"]
        s["pos"] = src.integers(lo, hi + 1, b) if c["ragged"] else c["pos"]
        s["count"] = src.integers((c["tokens"] + 1) // 2, c["tokens"] + 1, b) if c["ragged"] and c["tokens"] > 1 else None
        s["from"], s["span"] = s["pos"], _span(c)
        if c["kind"] == "write":        # what comes back of a write begins with its first block, whose older tokens may have changed
            s["from"] = s["pos"] // c["block"] * c["block"]
            s["k"], s["v"] = (src.tokens(b, c["heads"], c["tokens"], c["dim"], c["layout"]) for _ in range(2))
        return s
    s["q"] = src.tokens(b, c["heads"], c["tokens"], c["dim"], c["layout"])
    s["scale"] = c["dim"] ** -0.5
    # ragged: sequences of half to all of the keys, the queries always the last of them
    s["lens"] = src.integers(max((c["keys"] + 1) // 2, c["tokens"]), c["keys"] + 1, b) if c["ragged"] else c["keys"]
    s["table"], s["mapping"] = (src.normal(c["heads"], BUCKETS, std=0.5), _mapping()) if c["bias"] else (None, None)
    s["mask"] = None
    if c["mask"]:       # True where a key may be looked at; a batch of masks per query is padded with a query that sees nothing
        rows = c["tokens"] if c["mask"] == "query" else 1
        s["mask"] = torch.rand((b, rows, c["length"]), generator=src.gen, device="cuda") < 0.8
        if rows > 1:
            s["mask"][-1, -1] = False
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        import cpm_kernels_amd.torch as ct
        s["cache"] = ct.QuantizedKV(s["keys"], s["values"], s["key_absmax"], s["value_absmax"])
    return s


# ---- one pass -------------------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    if own:
        with torch.no_grad():
            cache = s["cache"]
            if c["kind"] == "attend":
                return cache.attention(s["q"], s["lens"], scale=s["scale"], causal=c["causal"], mask=s["mask"], bias=s["table"], mapping=s["mapping"],
                                       bidirectional=False)
            if c["kind"] == "write":
                cache.write(s["k"], s["v"], s["pos"], s["count"])
            k, v = cache.read(s["from"], s["span"], columns=c["layout"] == "columns")
            return (k, v, cache.key_absmax, cache.value_absmax) if c["kind"] == "write" else (k, v)
    if c["kind"] == "attend":
        return _attend(s)
    if c["kind"] == "write":
        _write(s, s["keys"], s["key_absmax"], s["k"], False)
        _write(s, s["values"], s["value_absmax"], s["v"], True)
    out = _read(s, s["keys"], s["key_absmax"], False), _read(s, s["values"], s["value_absmax"], True)
    return out + (s["key_absmax"], s["value_absmax"]) if c["kind"] == "write" else out


def _per_sequence(x, batch):
    return x.long() if isinstance(x, torch.Tensor) else torch.full((batch,), x, dtype=torch.long, device="cuda")


def _write(s, ints, top, x, values):
    c = s["case"]
    b, h, n, d, block = c["batch"], c["heads"], c["tokens"], c["dim"], c["block"]
    pos = _per_sequence(s["pos"], b)
    count = _per_sequence(s["count"] if s["count"] is not None else n, b)
    first = pos // block
    blocks = min((block - 1 + n + block - 1) // block, top.size(2))
    first = torch.minimum(first, torch.full_like(first, top.size(2) - blocks))       # a window of whole blocks, inside the cache
    at = first[:, None] * block + torch.arange(blocks * block, device="cuda")         # (batch, window): positions
    batches = torch.arange(b, device="cuda")[:, None]
    new = (at >= pos[:, None]) & (at < (pos + count)[:, None])
    old = (at < pos[:, None]) & (at >= (pos // block * block)[:, None])
    picked = x.transpose(1, 2)[batches, (at - pos[:, None]).clamp(0, n - 1)].float().clamp(-65504, 65504)        # (batch, window, heads, dim)
    picked = torch.where(new[:, :, None, None], picked, torch.zeros_like(picked))
    at_block = first[:, None] + torch.arange(blocks, device="cuda")
    before = top.transpose(1, 2)[batches, at_block].float()                           # (batch, blocks, heads)
    kept = old.view(b, blocks, block).any(2)[:, :, None]
    touched = new.view(b, blocks, block).any(2)[:, :, None]
    after = picked.view(b, blocks, block, h, d).abs().amax((2, 4))
    after = torch.where(kept, torch.maximum(after, before), after)
    after = torch.where(touched, after, before)
    where = (batches, at // 16) if values else (batches, at)
    if values:
        held = ints.permute(0, 2, 4, 1, 3)[batches, at // 16, at % 16].float()
    else:
        held = ints.transpose(1, 2)[batches, at].float()
    div = torch.where(after > 0, after, torch.ones_like(after)).repeat_interleave(block, 1)[..., None]
    again = _nearest(held * before.repeat_interleave(block, 1)[..., None] / div)
    fresh = _nearest(127 * picked / div)
    moved = old & touched.view(b, blocks).repeat_interleave(block, 1)
    result = torch.where(new[:, :, None, None], fresh, torch.where(moved[:, :, None, None], again, held)).to(torch.int8)
    if values:
        ints.permute(0, 2, 4, 1, 3)[where[0], where[1], at % 16] = result
    else:
        ints.transpose(1, 2)[where] = result
    top.transpose(1, 2)[batches, at_block] = after.half()


def _read(s, ints, top, values):
    c = s["case"]
    b, n, block = c["batch"], s["span"], c["block"]
    at = _per_sequence(s["from"], b)[:, None] + torch.arange(n, device="cuda")
    inside = (at >= 0) & (at < c["length"])
    at = at.clamp(0, c["length"] - 1)
    batches = torch.arange(b, device="cuda")[:, None]
    picked = ints.permute(0, 2, 4, 1, 3)[batches, at // 16, at % 16] if values else ints.transpose(1, 2)[batches, at]        # (batch, tokens, heads, dim)
    out = picked.float() * top.transpose(1, 2)[batches, at // block].float()[..., None] / 127
    out = torch.where(inside[:, :, None, None], out, torch.zeros_like(out)).half()
    if c["layout"] == "columns":
        return out.permute(0, 2, 3, 1).contiguous().transpose(2, 3)
    return out.transpose(1, 2).contiguous()


def _attend(s):
    c = s["case"]
    b, h, g, n, d, length, block = c["batch"], c["heads"], c["group"], c["tokens"], c["dim"], c["length"], c["block"]
    lens = _per_sequence(s["lens"], b)
    key = s["keys"].float() * s["key_absmax"].float().repeat_interleave(block, 2)[..., None] / 127
    value = _by_token(s["values"]).float() * s["value_absmax"].float().repeat_interleave(block, 2)[..., None] / 127
    q = s["q"].float().reshape(b, h // g, g * n, d)
    scores = (torch.matmul(q, key.transpose(2, 3).contiguous()) * s["scale"]).view(b, h, n, length)
    at = torch.arange(length, device="cuda")
    where = (lens - n)[:, None] + torch.arange(n, device="cuda")                      # (batch, tokens): positions of the queries
    if c["bias"]:
        far = (where[:, :, None] - at).clamp(0, MAX_DISTANCE - 1)
        scores += s["table"].float()[:, s["mapping"].long()[far]].transpose(0, 1)
    seen = (at < lens[:, None])[:, None].expand(b, n, length)
    if c["causal"]:
        seen = seen & (at <= where[:, :, None])
    if s["mask"] is not None:
        seen = seen & s["mask"]
    scores.masked_fill_(~seen[:, None], float("-inf"))
    p = torch.exp(scores - scores.amax(3, keepdim=True).clamp(min=-1e30))
    total = p.sum(3, keepdim=True)
    out = torch.matmul(p.view(b, h // g, g * n, length), value).view(b, h, n, d) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.half()
    if c["layout"] == "columns":
        return out.transpose(2, 3).contiguous().transpose(2, 3)
    return out.transpose(1, 2).contiguous().transpose(1, 2)


# ---- the definition in 64 bits, sequence by sequence ----------------------------------------------

def _exact_write(ints, top, x, pos, count, block):
    """One sequence: ints (heads, length, dim) and top (heads, blocks) in float64, brought up to date."""
    length = ints.size(1)
    t = pos
    while t < min(pos + count, length):
        blk = t // block
        end = min((blk + 1) * block, pos + count, length)
        fresh = x[:, t - pos:end - pos].double().clamp(-65504, 65504)
        a = fresh.abs().amax((1, 2))
        if t > blk * block:
            a = torch.maximum(a, top[:, blk])
            again = ints[:, blk * block:t] * top[:, blk, None, None] / a.clamp(min=1e-300)[:, None, None]
            ints[:, blk * block:t] = torch.where(again < 0, torch.ceil(again - 0.5), torch.floor(again + 0.5))
        parts = 127 * fresh / a.clamp(min=1e-300)[:, None, None]
        ints[:, t:end] = torch.where(parts < 0, torch.ceil(parts - 0.5), torch.floor(parts + 0.5))
        top[:, blk] = a
        t = end


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    b, n, block, length = c["batch"], c["tokens"], c["block"], c["length"]
    number = lambda x, i: int(x[i]) if isinstance(x, torch.Tensor) else x         # noqa: E731
    outs = []
    for i in range(b):
        seq = {"keys": s["keys"][i].double(), "values": s["values"][i].transpose(2, 3).reshape(-1, length, c["dim"]).double()}
        tops = {"keys": s["key_absmax"][i].double(), "values": s["value_absmax"][i].double()}
        if c["kind"] == "attend":
            outs.append(_exact_attend(c, s, i, number(s["lens"], i), seq, tops))
            continue
        pos = number(s["pos"], i)
        row = []
        for name, x in (("keys", s.get("k")), ("values", s.get("v"))):
            if x is not None:
                _exact_write(seq[name], tops[name], x[i], pos, n if s["count"] is None else number(s["count"], i), block)
            whole = seq[name] * tops[name].repeat_interleave(block, 1)[..., None] / 127
            piece = torch.zeros((c["heads"], s["span"], c["dim"]), dtype=torch.float64, device="cuda")
            begin = number(s["from"], i)
            end = min(begin + s["span"], length)
            piece[:, :end - begin] = whole[:, begin:end]
            row.append(piece)
        outs.append(row + ([tops["keys"], tops["values"]] if c["kind"] == "write" else []))
    if c["kind"] == "attend":
        return torch.stack(outs)
    return tuple(torch.stack(parts) for parts in zip(*outs))


def _exact_attend(c, s, i, keys, seq, tops):
    """One sequence, head by head of the cache: (heads, tokens, dim)."""
    g, n, d, block = c["group"], c["tokens"], c["dim"], c["block"]
    out = torch.zeros((c["heads"], n, d), dtype=torch.float64, device="cuda")
    index = torch.arange(keys, device="cuda")
    place = keys - n + torch.arange(n, device="cuda")
    hidden = torch.zeros((n, keys), dtype=torch.bool, device="cuda")
    if c["causal"]:
        hidden |= index[None] > place[:, None]
    if s["mask"] is not None:
        hidden |= ~s["mask"][i, :, :keys]
    times = torch.arange(keys, device="cuda") // block
    for head in range(c["heads"]):
        kv = head // g
        key = seq["keys"][kv, :keys] * (tops["keys"][kv][times] / 127)[:, None]
        value = seq["values"][kv, :keys] * (tops["values"][kv][times] / 127)[:, None]
        score = s["q"][i, head].double() @ key.t().contiguous() * s["scale"]
        if c["bias"]:
            score = score + s["table"][head].double()[s["mapping"].long()[(place[:, None] - index).clamp(0, MAX_DISTANCE - 1)]]
        weight = torch.where(hidden, torch.zeros_like(score), torch.exp(score - score.masked_fill(hidden, -math.inf).amax(1, keepdim=True).clamp(min=-1e300)))
        total = weight.sum(1, keepdim=True)
        out[head] = weight @ value / torch.where(total > 0, total, torch.ones_like(total))
    return out


# ---- what a pass cannot do without ------------------------------------------------------------------
# Each call's inputs read once and its outputs written once: a write takes fp16 tokens in and leaves integers, a read the other way round.  Ragged
# batches count by the means of their positions and lengths.

def work(case):
    c = case
    b, h, n, d, block = c["batch"], c["heads"], c["tokens"], c["dim"], c["block"]
    if c["kind"] != "attend":
        written = n * 0.75 if c["ragged"] and n > 1 else n
        cells = 2 * b * h * _span(c) * d
        tops = 2 * 2 * b * h * (-(-_span(c) // block))
        nbytes = 3 * cells + tops                                  # integers in, fp16 out
        flops = 2 * cells
        if c["kind"] == "write":
            nbytes += 3 * 2 * b * h * written * d + tops           # fp16 in, integers out
            flops += 3 * 2 * b * h * written * d
        return {"bytes": int(nbytes), "flops": int(flops)}
    keys = c["keys"] * (0.75 if c["ragged"] else 1)
    kept = 2 * b * (h // c["group"]) * keys * d * (1 + 2 / (block * d))
    nbytes = kept + 2 * 2 * b * h * n * d + (b * (n if c["mask"] == "query" else 1) * keys if c["mask"] else 0) + (2 * h * BUCKETS if c["bias"] else 0)
    pairs = n * keys - (n * (n - 1) / 2 if c["causal"] else 0)
    return {"bytes": int(nbytes), "flops": int(4 * b * h * pairs * d)}
