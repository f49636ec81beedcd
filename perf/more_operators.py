"""Rotary positions, attention over fp16 keys and values, and its gradients: the operators as they are measured.

    rotate  queries and keys turned by the angles of their positions: pairs of units side by side or half a head apart, all of a head or a part of it,
            frequencies as they are or stretched for long contexts; with "train" the gradients, which are turned back
    attend  softmax(scale q k^T + position bias, over the keys that length, causality and mask leave) v: a decode step's single query, a few drafted
            tokens, chunks of a prompt
    train   the same and its gradients to queries, keys, values and the table of position biases, the probabilities computed again

Tensors are (batch, heads, tokens, dim) fp16, laid out as a projection leaves them: (batch, tokens, heads, dim) in memory ("rows") or
(batch, heads, dim, tokens) ("columns", the layout of this package's activations).  Heads of 64 units, 12 to 64 heads, up to 1024 tokens and 32 position
buckets over 128 tokens are the sizes of bench.py and the tests; 80 to 256 units, heads of keys that several heads of queries share and long sequences are
generic.
"""
import math

import torch

own = False         # whether `run` calls the framework (set from outside)

BUCKETS, MAX_DISTANCE = 32, 128


def listed():
    return [
        # one new token of a small model: nothing but latency
        dict(name="rotate_step_1x16", kind="rotate", train=False, batch=1, heads=16, group=1, tokens=1, dim=64, part=64, interleaved=False, layout="rows",
             start=1000, pos="start", scaling=""),
        # a batch of prompts in this package's own layout
        dict(name="rotate_prompt_8x512", kind="rotate", train=False, batch=8, heads=64, group=1, tokens=512, dim=64, part=64, interleaved=True, layout="columns",
             start=0, pos="start", scaling=""),
        # a training step on long sequences packed to rows: positions token by token, half of the head turned, frequencies stretched by parts
        dict(name="rotate_train_2x8191", kind="rotate", train=True, batch=2, heads=32, group=4, tokens=8191, dim=128, part=64, interleaved=False, layout="rows",
             start=100000, pos="token", scaling="parts"),
        # a decode step of one sequence, with a position bias
        dict(name="attend_step_1x16_bias", kind="attend", batch=1, heads=16, group=1, tokens=1, keys=101, spare=27, dim=64, layout="rows", causal=True,
             bias="one", mask="", ragged=False),
        # a decode step of a serving batch, every sequence of its own length
        dict(name="attend_step_32x64", kind="attend", batch=32, heads=64, group=1, tokens=1, keys=1024, spare=0, dim=64, layout="rows", causal=True,
             bias="", mask="", ragged=True),
        # a decode step over long contexts, eight heads of queries on each head of keys
        dict(name="attend_step_4x64_shared_long", kind="attend", batch=4, heads=64, group=8, tokens=1, keys=32768, spare=0, dim=128, layout="rows", causal=True,
             bias="", mask="", ragged=True),
        # five drafted tokens of each sequence, a tree among them: a mask for each
        dict(name="attend_draft_8x32_shared", kind="attend", batch=8, heads=32, group=4, tokens=5, keys=3500, spare=12, dim=128, layout="rows", causal=False,
             bias="", mask="query", ragged=True),
        # a chunk at the end of a long prompt
        dict(name="attend_prompt_2000_of_8011", kind="attend", batch=1, heads=32, group=4, tokens=2000, keys=8011, spare=0, dim=128, layout="rows", causal=True,
             bias="", mask="", ragged=False),
        # an encoder's layer on padded sequences: biases for both directions, a mask of keys
        dict(name="attend_encoder_8x64_bias", kind="attend", batch=8, heads=64, group=1, tokens=512, keys=512, spare=0, dim=64, layout="columns", causal=False,
             bias="both", mask="key", ragged=False),
        # a training step of a small model
        dict(name="train_2x12x100_bias", kind="train", batch=2, heads=12, group=1, tokens=100, keys=100, spare=0, dim=64, layout="columns", causal=True,
             bias="one", mask="", ragged=False),
        # a training step on sequences padded to 512 tokens
        dict(name="train_8x64x512_bias", kind="train", batch=8, heads=64, group=1, tokens=512, keys=512, spare=0, dim=64, layout="columns", causal=True,
             bias="one", mask="", ragged=True),
        # a training step on one long sequence, four heads of queries on each head of keys
        dict(name="train_1x32_shared_8192", kind="train", batch=1, heads=32, group=4, tokens=8192, keys=8192, spare=0, dim=128, layout="rows", causal=True,
             bias="", mask="", ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _drawn(rng):
    kind = rng.choice(["rotate", "rotate", "attend", "attend", "attend", "train", "train", "train"])
    group = rng.choice([1, 1, 2, 4, 8])
    c = dict(kind=kind, batch=_log(rng, 1, 32), group=group, heads=_log(rng, 1, 64 // group) * group, dim=rng.choice([64, 64, 80, 96, 128, 128, 256]),
             layout=rng.choice(["rows", "rows", "columns"]))
    if kind == "rotate":
        c["train"] = rng.random() < 0.5
        c["tokens"] = _log(rng, 2, 8192) if c["train"] else rng.choice([1, 1, _log(rng, 2, 8192), _log(rng, 2, 8192)])
        c["part"] = c["dim"] // rng.choice([1, 1, 2, 4]) // 2 * 2
        c["interleaved"] = rng.random() < 0.5
        c["start"] = rng.choice([0, 0, _log(rng, 1, 1000000)])
        c["pos"] = rng.choice(["start", "each", "token"])
        c["scaling"] = rng.choice(["", "linear", "ntk", "parts"])
        return c
    c["bias"] = rng.choice(["", "", "one", "both"])
    c["mask"] = rng.choice(["", "", "key", "query"])
    c["ragged"] = rng.random() < 0.5
    c["causal"] = rng.random() < 0.7
    if kind == "attend":
        c["tokens"] = rng.choice([1, 1, rng.randrange(2, 9), _log(rng, 9, 2048), _log(rng, 64, 2048)])
        c["keys"] = c["tokens"] + _log(rng, 1, 32768) - 1
        c["spare"] = rng.choice([0, rng.randrange(64)])
    else:
        c["tokens"] = _log(rng, 2, 8192)
        c["keys"] = rng.choice([c["tokens"], c["tokens"], _log(rng, c["tokens"], 8192)])
        c["spare"] = 0
    return c


def draw(rng):
    most = {kind: max(_cost(c) for c in listed() if c["kind"] == kind) for kind in ("rotate", "attend", "train")}
    while True:
        c = _drawn(rng)
        if _cost(c) <= most[c["kind"]] and _held(c) <= 2 ** (33 if c["kind"] == "train" else 32):
            return c


def _cost(c):
    w = work(c)
    return w["bytes"] / 6e12 + w["flops"] / 6e14


def _held(c):
    """Bytes of the largest thing of a case: a tensor in fp32, the scores of the plain form (once more for a bias and for a mask of every query)."""
    n = c["tokens"] if c["kind"] == "rotate" else c["keys"] + c["spare"]
    scores = 0 if c["kind"] == "rotate" else 4 * c["batch"] * c["heads"] * c["tokens"] * n * (1 + bool(c["bias"]))
    return max(scores, 4 * c["batch"] * c["heads"] * max(n, c["tokens"]) * c["dim"])


# ---- inputs ---------------------------------------------------------------------------------------

class _Source:
    """Seeded values on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32).mul_(std).half()

    def integers(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.gen, device="cuda", dtype=torch.int32)

    def tokens(self, batch, heads, tokens, dim, layout, std=1.0, sized=True):
        """(batch, heads, tokens, dim) as a projection leaves it: with `sized` units of very different size, as queries and keys have them."""
        columns = layout == "columns"
        x = self.normal(batch, heads * dim, tokens, std=std) if columns else self.normal(batch, tokens, heads * dim, std=std)
        if sized:
            size = torch.exp(0.5 * torch.randn((heads * dim, 1), generator=self.gen, device="cuda")).half()
            x *= size if columns else size[:, 0]
        return x.view(batch, heads, dim, tokens).transpose(2, 3) if columns else x.view(batch, tokens, heads, dim).transpose(1, 2)


def _mapping(both):
    """Distance -> bucket: exact up to half of the buckets (of a sign), logarithmic from there on."""
    count = BUCKETS // 2 if both else BUCKETS
    exact = count // 2
    far = [exact + int(math.log(i / exact) / math.log(MAX_DISTANCE / exact) * (count - exact)) for i in range(exact, MAX_DISTANCE)]
    return torch.tensor(list(range(exact)) + [min(b, count - 1) for b in far], dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    c, src = case, _Source(seed)
    b, h, n, d, held = c["batch"], c["heads"], c["tokens"], c["dim"], c["heads"] // c["group"]
    s = {"case": c}
    if c["kind"] == "rotate":
        s["q"], s["k"] = (src.tokens(b, x, n, d, c["layout"]) for x in (h, held))
        if c["train"]:
            s["dq"], s["dk"] = (src.tokens(b, x, n, d, c["layout"], std=0.02) for x in (h, held))
        each = src.integers(c["start"], c["start"] + 1000, b)
        if c["pos"] == "start":
            s["pos"] = c["start"]
        elif c["pos"] == "each":
            s["pos"] = each
        else:       # packed: the positions begin again with every document
            at, length = torch.arange(n, device="cuda", dtype=torch.int32), max(n // 3, 1)
            s["pos"] = each[:, None] + (at % length)[None]
        return s
    length = c["keys"] + c["spare"]
    s["q"] = src.tokens(b, h, n, d, c["layout"])
    s["k"] = src.tokens(b, held, length, d, c["layout"])
    s["v"] = src.tokens(b, held, length, d, c["layout"], sized=False)
    s["scale"] = d ** -0.5
    # ragged: sequences of half to all of the keys.  Their queries are the last of the keys where a cache is read, and begin with them where they are padded
    s["lens"], s["first"] = (c["keys"], c["keys"] - n) if c["ragged"] is False else (src.integers((c["keys"] + 1) // 2, c["keys"] + 1, b), None)
    if c["ragged"] and c["kind"] == "attend":
        s["lens"] = torch.clamp(s["lens"], min=n)
        s["first"] = s["lens"] - n
    elif c["ragged"]:
        s["first"] = c["keys"] - n
    s["table"] = s["mapping"] = s["mask"] = None
    if c["bias"]:
        s["table"], s["mapping"] = src.normal(h, BUCKETS, std=0.5), _mapping(c["bias"] == "both")
    if c["mask"]:       # True where a key may be looked at; masks per query leave the last query nothing
        rows = n if c["mask"] == "query" else 1
        s["mask"] = torch.rand((b, rows, length), generator=src.gen, device="cuda") < 0.8
        if rows > 1:
            s["mask"][-1, -1] = False
    if c["kind"] == "train":
        s["dout"] = src.tokens(b, h, n, d, c["layout"], std=0.02, sized=False)
    return s


def _stretch(c):
    return dict(scaling=c["scaling"], factor=8.0, original_length=4096) if c["scaling"] else {}


def prepare(case, seed):
    s, c = _inputs(case, seed), case
    if own:
        import cpm_kernels_amd.torch as ct
        if c["kind"] == "rotate":
            s["rotary"] = ct.RotaryEmbedding(c["dim"], rotary_dim=c["part"], interleaved=c["interleaved"], **_stretch(c)).cuda()
        else:
            s["attention"] = ct.attention
        wanted = {"rotate": ("q", "k") if c.get("train") else (), "attend": (), "train": ("q", "k", "v", "table")}[c["kind"]]
        s["leaves"] = [s[x].requires_grad_() for x in wanted if s[x] is not None]
    return s


# ---- one pass -------------------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rotate": _rotate, "attend": _attend, "train": _train}[c["kind"]](s)
    if c["kind"] == "rotate":
        outs = s["rotary"](s["q"], s["k"], s["pos"])
        return tuple(x.detach() for x in outs) + torch.autograd.grad(outs, s["leaves"], (s["dq"], s["dk"])) if c["train"] else outs
    out = s["attention"](s["q"], s["k"], s["v"], lens=s["lens"], scale=s["scale"], causal=c["causal"], pos=s["first"], mask=s["mask"], bias=s["table"],
                         mapping=s["mapping"], bidirectional=c["bias"] == "both")
    return (out.detach(),) + torch.autograd.grad(out, s["leaves"], s["dout"]) if c["kind"] == "train" else out


def _frequencies(c):
    """Turns a token of every pair, in 64 bits, and what the result is multiplied by."""
    r, stretch = c["part"], _stretch(c)
    base, factor = 10000.0, stretch.get("factor", 1.0)
    if c["scaling"] == "ntk":
        base *= factor ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r) / (2 * math.pi)
    if c["scaling"] == "linear":
        f = f / factor
    if c["scaling"] == "parts":
        kept = ((stretch["original_length"] * f - 1) / 31).clamp(0, 1)
        return f * (kept + (1 - kept) / factor), 1 + 0.1 * math.log(factor)
    return f, 1.0


def _positions(s):
    c = s["case"]
    if c["pos"] == "token":
        return s["pos"].double()
    first = s["pos"].double()[:, None] if c["pos"] == "each" else torch.full((c["batch"], 1), float(s["pos"]), dtype=torch.float64, device="cuda")
    return first + torch.arange(c["tokens"], dtype=torch.float64, device="cuda")


def _as_laid_out(x, layout):
    return x.transpose(2, 3).contiguous().transpose(2, 3) if layout == "columns" else x.transpose(1, 2).contiguous().transpose(1, 2)


def _turn(x, cos, sin, c):
    r = c["part"]
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if c["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
    first, second = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((first, second), -1).flatten(-2) if c["interleaved"] else torch.cat((first, second), -1)
    return _as_laid_out(torch.cat((turned, y[..., r:]), -1).half(), c["layout"])


def _rotate(s):
    c = s["case"]
    f, size = _frequencies(c)
    turns = _positions(s)[:, None, :, None] * f
    angle = (turns - turns.round()) * (2 * math.pi)
    cos, sin = (torch.cos(angle) * size).float(), (torch.sin(angle) * size).float()
    outs = _turn(s["q"], cos, sin, c), _turn(s["k"], cos, sin, c)
    return outs + (_turn(s["dq"], cos, -sin, c), _turn(s["dk"], cos, -sin, c)) if c["train"] else outs


def _per_sequence(x, batch):
    return x.long() if isinstance(x, torch.Tensor) else torch.full((batch,), x, dtype=torch.long, device="cuda")


def _buckets(c, mapping, rel):
    """Of distances query - key."""
    if c["bias"] == "one":
        return mapping.long()[rel.clamp(0, MAX_DISTANCE - 1)]
    return mapping.long()[rel.abs().clamp(max=MAX_DISTANCE - 1)] + torch.where(rel < 0, BUCKETS // 2, 0)


def _forward(s):
    """(probabilities (batch, kv heads, group * tokens, keys), result, and what a gradient needs besides), in 32 bits."""
    c = s["case"]
    b, h, g, n, d = c["batch"], c["heads"], c["group"], c["tokens"], c["dim"]
    length = s["k"].size(2)
    lens = _per_sequence(s["lens"], b)
    key, value = s["k"].detach().float(), s["v"].detach().float()
    q = s["q"].detach().float().reshape(b, h // g, g * n, d)
    scores = torch.matmul(q, key.transpose(2, 3).contiguous()).mul_(s["scale"]).view(b, h, n, length)
    at = torch.arange(length, device="cuda")
    where = _per_sequence(s["first"], b)[:, None] + torch.arange(n, device="cuda")       # (batch, tokens): positions of the queries
    bucket = None
    if c["bias"]:
        bucket = _buckets(c, s["mapping"], where[:, :, None] - at)
        scores += s["table"].detach().float()[:, bucket].transpose(0, 1)
    seen = (at < lens[:, None])[:, None].expand(b, n, length)
    if c["causal"]:
        seen = seen & (at <= where[:, :, None])
    if s["mask"] is not None:
        seen = seen & s["mask"]
    scores.masked_fill_(~seen[:, None], float("-inf"))
    scores.sub_(scores.amax(3, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(3, keepdim=True)
    p = scores.div_(torch.where(total > 0, total, torch.ones_like(total))).view(b, h // g, g * n, length)
    return p, torch.matmul(p, value), q, key, value, bucket


def _attend(s):
    c = s["case"]
    out = _forward(s)[1].view(c["batch"], c["heads"], c["tokens"], c["dim"])
    return _as_laid_out(out.half(), c["layout"])


def _train(s):
    c = s["case"]
    b, h, g, n, d = c["batch"], c["heads"], c["group"], c["tokens"], c["dim"]
    p, out, q, key, value, bucket = _forward(s)
    dout = s["dout"].float().reshape(b, h // g, g * n, d)
    dvalue = torch.matmul(p.transpose(2, 3).contiguous(), dout)
    ds = torch.matmul(dout, value.transpose(2, 3).contiguous())
    ds.sub_((dout * out).sum(3, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, key).mul_(s["scale"])
    dkey = torch.matmul(ds.transpose(2, 3).contiguous(), q).mul_(s["scale"])
    results = [_as_laid_out(x.view(b, -1, x.size(2) // (g if i in (0, 1) else 1), d).half(), c["layout"]) for i, x in enumerate((out, dq, dkey, dvalue))]
    if c["bias"]:       # long sums: in 64 bits
        by_head = ds.view(b, h, n, -1)
        results.append(torch.stack([torch.where((bucket == i)[:, None], by_head, 0.0).sum((0, 2, 3), dtype=torch.float64) for i in range(BUCKETS)], 1).half())
    return tuple(results)


# ---- the definition in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_rotation(case, s) if case["kind"] == "rotate" else _exact_attention(case, s)


def _exact_rotation(c, s):
    """Units as complex numbers, sequence by sequence."""
    r = c["part"]
    freq, size = [], 1.0
    for i in range(r // 2):
        base = 10000.0 * (8.0 ** (r / (r - 2.0)) if c["scaling"] == "ntk" else 1.0)
        w = base ** (-2.0 * i / r)
        if c["scaling"] == "linear":
            w /= 8.0
        elif c["scaling"] == "parts":
            rounds = 4096 * w / (2 * math.pi)
            share = min(max((rounds - 1) / 31, 0.0), 1.0)
            w, size = share * w + (1 - share) * w / 8.0, 0.1 * math.log(8.0) + 1
        freq.append(w)
    freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
    one = [2 * i for i in range(r // 2)] if c["interleaved"] else list(range(r // 2))
    other = [i + 1 for i in one] if c["interleaved"] else [i + r // 2 for i in one]

    def turned(x, back):
        out = x.double()
        for b in range(c["batch"]):
            at = s["pos"] if c["pos"] == "start" else s["pos"][b].double()
            if c["pos"] != "token":
                at = at + torch.arange(c["tokens"], dtype=torch.float64, device="cuda")
            spin = torch.polar(torch.full((c["tokens"], r // 2), size, dtype=torch.float64, device="cuda"), at[:, None] * freq * (-1 if back else 1))
            z = torch.complex(out[b][..., one], out[b][..., other]) * spin
            out[b][..., one], out[b][..., other] = z.real, z.imag
        return out
    outs = turned(s["q"], False), turned(s["k"], False)
    return outs + (turned(s["dq"], True), turned(s["dk"], True)) if c["train"] else outs


def _exact_attention(c, s):
    """Sequence by sequence and head by head; only the keys of a sequence's length are looked at."""
    b, h, g, n, d = c["batch"], c["heads"], c["group"], c["tokens"], c["dim"]
    train = c["kind"] == "train"
    number = lambda x, i: int(x[i]) if isinstance(x, torch.Tensor) else x         # noqa: E731
    zeros = lambda x: torch.zeros(x.shape, dtype=torch.float64, device="cuda")    # noqa: E731
    out, dq, dk, dv = zeros(s["q"]), zeros(s["q"]), zeros(s["k"]), zeros(s["v"])
    dtable = zeros(s["table"]) if c["bias"] else None
    for i in range(b):
        keys = number(s["lens"], i)
        index = torch.arange(keys, device="cuda")
        rel = (number(s["first"], i) + torch.arange(n, device="cuda"))[:, None] - index
        hidden = rel < 0 if c["causal"] else torch.zeros((n, keys), dtype=torch.bool, device="cuda")
        if s["mask"] is not None:
            hidden = hidden | ~s["mask"][i, :, :keys]
        if c["bias"]:
            near = rel.abs() if c["bias"] == "both" else rel.clamp(min=0)
            which = s["mapping"].long()[near.clamp(max=MAX_DISTANCE - 1)]
            if c["bias"] == "both":
                which = which + BUCKETS // 2 * (rel < 0)
        for head in range(h):
            query, key, value = s["q"][i, head].double(), s["k"][i, head // g, :keys].double(), s["v"][i, head // g, :keys].double()
            score = query @ key.t().contiguous() * s["scale"]
            if c["bias"]:
                score += s["table"][head].double()[which]
            score.masked_fill_(hidden, -math.inf)
            top = score.amax(1, keepdim=True)
            weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
            total = weight.sum(1, keepdim=True)
            weight /= torch.where(total == 0, 1.0, total)
            out[i, head] = weight @ value
            if not train:
                continue
            grad = s["dout"][i, head].double()
            dv[i, head // g, :keys] += weight.t().contiguous() @ grad
            back = grad @ value.t().contiguous()
            back = weight * (back - (weight * back).sum(1, keepdim=True))
            dq[i, head] = back @ key * s["scale"]
            dk[i, head // g, :keys] += back.t().contiguous() @ query * s["scale"]
            if c["bias"]:
                dtable[head] += torch.bincount(which.reshape(-1), back.reshape(-1), minlength=BUCKETS)
    if not train:
        return out
    return (out, dq, dk, dv, dtable) if c["bias"] else (out, dq, dk, dv)


# ---- what a pass cannot do without ------------------------------------------------------------------
# Each input read once, each output written once; two operations a multiply-add, of a training step seven products of queries and keys.  Ragged batches
# count by the means of their lengths.

def work(case):
    c = case
    b, h, n, d, held = c["batch"], c["heads"], c["tokens"], c["dim"], c["heads"] // c["group"]
    if c["kind"] == "rotate":
        cells = b * (h + held) * n * d * (2 if c["train"] else 1)
        return {"bytes": 4 * cells + (4 * b * n if c["pos"] == "token" else 0), "flops": 3 * cells * c["part"] // d}
    keys = c["keys"] * (0.75 if c["ragged"] else 1)
    masks = b * (n if c["mask"] == "query" else 1) * keys if c["mask"] else 0
    table = 2 * h * BUCKETS if c["bias"] else 0
    pairs = n * keys
    if c["causal"]:     # query i sees first + i + 1 keys, up to the length; of a cache the queries are the last keys
        first = (c["keys"] if c["kind"] == "train" else keys) - n
        some = min(max(keys - first, 0), n)         # queries that see fewer keys than there are
        pairs = some * first + some * (some + 1) / 2 + (n - some) * keys
    train = c["kind"] == "train"
    nbytes = 2 * b * d * (n * h * (4 if train else 2) + 2 * held * keys + (2 * held * c["keys"] if train else 0)) + masks + table * (2 if train else 1)
    return {"bytes": int(nbytes), "flops": int((14 if train else 4) * b * h * pairs * d)}
