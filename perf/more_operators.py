"""The operators of caches in 4 bits, and of what a model's answers are judged by:

  decode   a layer's decode attention for a batch of sequences whose caches are
           held in 4 bits (the new tokens' keys and values appended on the way)
  chunk    a layer's causal attention for a prompt chunk over such a cache
  stage    a context's keys and values written into the cache, and read back
  logprob  log probabilities of given tokens, the entropy of their distributions
           and the likeliest alternatives, from rows of logits

A cache keeps blocks of 32 tokens. x16 are the values rounded to f16. A group is
32 tokens of one key channel, or 64 dims of one token's value; with lo and hi its
smallest and largest x16, s = (hi - lo) / 15 (the difference and its product with
1/15 in f32) cut off to f16, so that no value leaves lo .. hi; a code is (x16 - lo)
* (1 / s) in f32, rounded to the nearest whole number (ties to even) and clamped to
0 .. 15 (0 where s is 0), and it stands for code * s + lo, rounded to f16. A block that is not whole is kept in f16, keys
[token][dim] and values [dim][token]. Attention sees the cache as it is after the
call's own tokens are in it. Keys are normalised and rotated in 64 bits and
rounded to f32, then to f16.

Log probabilities are natural logarithms; a logit of -inf or NaN has probability
0; alternatives come by falling logit, the lowest token first among equals.

Where `own` is false, `run` computes this in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
HEAD = 128
BLOCK = 32
GROUP = 64
EPS = 1e-6
BASE = 1.0e6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One sequence at the start of its answer: all launch and latency.
        dict(name="decode_1x57", kind="decode", q_heads=32, kv_heads=8, members=1, context=57, scaling="none"),
        # Eight sequences of different lengths, an ordinary serving step.
        dict(name="decode_8x4001", kind="decode", q_heads=32, kv_heads=8, members=8, context=4001, scaling="none"),
        # A wide batch of medium contexts, eight query heads to a KV head.
        dict(name="decode_31x1203", kind="decode", q_heads=64, kv_heads=8, members=31, context=1203, scaling="none"),
        # One sequence at the end of the scaled range of positions.
        dict(name="decode_1x131071", kind="decode", q_heads=32, kv_heads=8, members=1, context=131071, scaling="yarn"),
        # A short question put after a cached document.
        dict(name="chunk_29", kind="chunk", q_heads=32, kv_heads=8, tokens=29, position=3040, scaling="none"),
        # A whole prompt chunk from the start.
        dict(name="chunk_2047", kind="chunk", q_heads=32, kv_heads=8, tokens=2047, position=0, scaling="none"),
        # A later chunk of a long prompt, at an odd size.
        dict(name="chunk_1801", kind="chunk", q_heads=32, kv_heads=8, tokens=1801, position=8192, scaling="yarn"),
        # A short shared prefix put into a new sequence's cache and taken out again.
        dict(name="stage_77", kind="stage", kv_heads=8, tokens=77, dtype="f32"),
        # A long document's keys and values moved into the cache and out.
        dict(name="stage_32768", kind="stage", kv_heads=8, tokens=32768, dtype="f16"),
        # A decode step's one row, with the alternatives that an API shows.
        dict(name="logprob_1", kind="logprob", rows=1, vocab=151936, pad=0, dtype="f32", top=5),
        # A serving batch's rows out of a wider buffer, an odd vocabulary.
        dict(name="logprob_33", kind="logprob", rows=33, vocab=32001, pad=63, dtype="bf16", top=20),
        # A prompt chunk scored token by token.
        dict(name="logprob_2047", kind="logprob", rows=2047, vocab=151936, pad=0, dtype="f32", top=1),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "chunk", "chunk", "stage", "logprob", "logprob"))
    heads = rng.choice(((8, 8), (16, 8), (32, 8), (32, 8), (64, 8), (32, 4), (4, 2)))
    scaling = rng.choice(("none", "none", "yarn", "linear"))
    if kind == "decode":
        members = _log_int(rng, 1, 31)
        return dict(kind="decode", q_heads=heads[0], kv_heads=heads[1], members=members,
                    context=_log_int(rng, 1, 131071 // members), scaling=scaling)
    if kind == "chunk":
        tokens = _log_int(rng, 1, 2047)
        room = int(min(12000, 15.0e6 / tokens * 32 / max(32, heads[0]) - tokens / 2)) // BLOCK
        # (a chunk begins where a block of the cache does, as chunks of whole blocks put one after another do: only then
        # can it be computed again, since a block taken back into is rounded to 4 bits once more)
        position = 0 if rng.random() < 0.4 or room < 1 else BLOCK * _log_int(rng, 1, room)
        return dict(kind="chunk", q_heads=heads[0], kv_heads=heads[1], tokens=tokens, position=position, scaling=scaling)
    if kind == "stage":
        return dict(kind="stage", kv_heads=heads[1], tokens=_log_int(rng, 1, 32000), dtype=rng.choice(("f16", "f32")))
    rows = _log_int(rng, 1, 2047)
    vocab = _log_int(rng, 300, min(151936, 2047 * 151936 // rows))
    return dict(kind="logprob", rows=rows, vocab=vocab, pad=rng.choice((0, 0, 1, 8, 63)), dtype=rng.choice(tuple(DTYPES)),
                top=rng.choice((0, 1, 5, 20, 32)))


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * seed + 31)
    return g


def _gamma(g):
    return torch.randn(HEAD, device=DEV, generator=g).mul_(0.1).add_(1.0)


def _scaling(name):
    """factor, original context of a scaling."""
    return {"none": (1.0, 0), "linear": (4.0, 0), "yarn": (4.0, 32768)}[name]


def _contexts(case):
    """Cached tokens of each member: the longest has `context`, the others 40-100% of it."""
    rng = np.random.default_rng(case["context"])
    m = case["members"]
    return [case["context"]] + [max(1, int(case["context"] * v)) for v in rng.uniform(0.4, 1.0, m - 1)]


def _context_values(g, kv_heads, tokens):
    """Keys as a cache holds them (a few channels of each head much larger than
    the rest, some with a mean of their own), and values: f16 [tokens][kv_heads][128]."""
    wide = torch.rand((1, kv_heads, HEAD), device=DEV, generator=g)
    gain = torch.where(wide > 0.97, 6.0, 0.5 + wide)
    mean = torch.randn((1, kv_heads, HEAD), device=DEV, generator=g) * (wide < 0.25)
    keys = torch.randn((tokens, kv_heads, HEAD), device=DEV, generator=g).mul_(gain).add_(mean).half()
    values = torch.randn((tokens, kv_heads, HEAD), device=DEV, generator=g).mul_(0.5).half()
    return keys, values


class _State:
    pass


class _DeviceArray:
    """An f16 device range of the library's, for torch.as_tensor."""

    def __init__(self, ptr, shape, strides, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "strides": strides, "typestr": "<f2", "version": 2}


def _tails(cache, kv_heads):
    """The f16 block a cache's sequence stands in: keys [kv_heads][32][128], values [kv_heads][128][32]."""
    keys, values, stride = cache.tail(0)
    return [torch.as_tensor(_DeviceArray(p, (kv_heads, *shape), (2 * stride, 2 * shape[1], 2), cache), device=DEV)
            for p, shape in ((keys, (BLOCK, HEAD)), (values, (HEAD, BLOCK)))]


def _logits(case, g):
    """Rows as a model leaves them: a bell of unlikely tokens, and one raised by so much that the model is anything from
    at a loss to certain; in one row of eight most tokens are masked, as a grammar does it. -> (logits, given tokens)"""
    rows, vocab = case["rows"], case["vocab"]
    wide = torch.empty((rows, vocab + case["pad"]), dtype=DTYPES[case["dtype"]], device=DEV)
    likely = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    other = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    lift = torch.rand(rows, device=DEV, generator=g) * 24.0
    for lo in range(0, rows, 256):  # (a piece at a time: the noise is f32 whatever the type)
        hi = min(rows, lo + 256)
        x = torch.randn((hi - lo, vocab + case["pad"]), device=DEV, generator=g).mul_(2.0)
        x[torch.arange(hi - lo, device=DEV), likely[lo:hi]] += lift[lo:hi]
        masked = torch.rand((1, vocab + case["pad"]), device=DEV, generator=g) > 0.1
        x[7::8] = x[7::8].masked_fill(masked, -math.inf)
        wide[lo:hi] = x
    given = torch.where(torch.rand(rows, device=DEV, generator=g) < 0.7, likely, other)
    return wide[:, :vocab], given.int()


def _inputs(case, seed):
    """What the calls work on, and the contexts that are to be in the caches."""
    s = _State()
    s.case = case
    kind = case["kind"]
    g = _generator(seed)
    if kind == "logprob":
        s.logits, s.given = _logits(case, g)
        return s
    kv = case["kv_heads"]
    if kind == "stage":
        s.keys, s.values = (v.to(DTYPES[case["dtype"]]) for v in _context_values(g, kv, case["tokens"]))
        s.lengths, s.contexts = [case["tokens"]], []
        return s
    s.lengths = _contexts(case) if kind == "decode" else [case["position"]]
    rows = case["members"] if kind == "decode" else case["tokens"]
    s.q = torch.randn((rows, case["q_heads"] * HEAD), device=DEV, generator=g)
    s.k, s.v = (torch.randn((rows, kv * HEAD), device=DEV, generator=g) for _ in range(2))
    s.q_norm, s.k_norm = _gamma(g), _gamma(g)
    s.positions = torch.tensor(s.lengths, dtype=torch.int32, device=DEV)
    s.contexts = [_context_values(g, kv, n) for n in s.lengths]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "logprob":
        n, top = case["rows"], case["top"]
        s.logprobs, s.entropy = (torch.zeros(n, device=DEV) for _ in range(2))
        s.tokens = torch.zeros((n, top), dtype=torch.int32, device=DEV)
        s.alternatives = torch.zeros((n, top), device=DEV)
    elif kind == "stage":
        s.back = [torch.empty(s.keys.shape, dtype=torch.float16, device=DEV) for _ in range(2)]
    else:
        s.y = torch.zeros(s.q.numel(), device=DEV)
    if own:
        _prepare_own(s, case)
    elif kind in ("decode", "chunk"):
        s.freq, s.gain = _frequencies(case["scaling"])
        _prepare_plain(s, case["kv_heads"], max(s.lengths) + (1 if kind == "decode" else case["tokens"]))
    s.contexts = None  # the caches hold them now
    return s


def _prepare_own(s, case):
    import engine_amd as E

    kind = case["kind"]
    s.ctx = E.AmdContext(0)
    if kind == "logprob":
        s.ops = E.AmdQwenOps(s.ctx)
        return
    factor, original = _scaling(case.get("scaling", "none"))
    s.cfg = E.AmdQwen3Config(layers=1, hidden=4096, q_heads=case.get("q_heads", case["kv_heads"]), kv_heads=case["kv_heads"],
                             head_dim=HEAD, ffn=12288, vocab=1024, rope_base=BASE, epsilon=EPS)
    rope = None
    if factor != 1.0:
        rope = E.AmdRopeSpec(head_dim=HEAD, base=BASE, scaling=case["scaling"], factor=factor, original_context=original)
    extra = {"decode": 1, "chunk": case.get("tokens", 0), "stage": 0}[kind]
    s.caches = [E.AmdKvCache(s.ctx, s.cfg, n + extra, format=E.KV_I4, rope=rope) for n in s.lengths]
    for cache, (keys, values) in zip(s.caches, s.contexts):
        if len(keys):
            cache.write(0, keys, values, 0)
    if kind != "stage":
        rows = [(n + extra - 1) % BLOCK + 1 for n in s.lengths]
        s.tails = [(k[:, :n], v[:, :, :n]) for (k, v), n in zip((_tails(c, case["kv_heads"]) for c in s.caches), rows)]


def _prepare_plain(s, kv, room):
    """Codes, scales and lows of the whole blocks, padded to the longest sequence, and each sequence's f16 block."""
    blocks = -(-room // BLOCK)
    m = len(s.contexts)
    s.held = []
    for part in range(2):
        groups = (1, HEAD, 1) if part == 0 else (BLOCK, HEAD // GROUP, 1)
        s.held.append([torch.zeros((m, kv, blocks, BLOCK, HEAD), dtype=torch.uint8, device=DEV),
                       *(torch.zeros((m, kv, blocks, *groups), dtype=torch.float16, device=DEV) for _ in range(2))])
    s.tail = [torch.zeros((m, kv, BLOCK, HEAD), dtype=torch.float16, device=DEV), torch.zeros((m, kv, HEAD, BLOCK), dtype=torch.float16, device=DEV)]
    for i, pair in enumerate(s.contexts):
        n = len(pair[0])
        whole, last = n // BLOCK, max(0, (n - 1) // BLOCK * BLOCK)
        for part, x in enumerate(pair):
            x = x.transpose(0, 1)
            for held, new in zip(s.held[part], _quantise(x[:, :whole * BLOCK].reshape(kv, whole, BLOCK, HEAD), part)):
                held[i, :, :whole] = new
            rows = s.tail[0][i] if part == 0 else s.tail[1][i].transpose(1, 2)
            rows[:, :n - last] = x[:, last:]


# -------------------------------------------------------------------- plain form

def _frequencies(scaling):
    """Turns a position adds to each pair's angle, in 64 bits, and the gain of cosine and sine."""
    i = torch.arange(HEAD // 2, dtype=torch.float64, device=DEV)
    f = BASE ** (-2.0 * i / HEAD)
    factor, original = _scaling(scaling)
    gain = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        # pairs that turn often within the trained length stay, slow ones stretch
        low, high = (HEAD * math.log(original / (2.0 * math.pi * beta)) / (2.0 * math.log(BASE)) for beta in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), HEAD - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        f = f / factor * ramp + f * (1.0 - ramp)
        gain = 0.1 * math.log(factor) + 1.0
    return f / (2.0 * math.pi), gain


def _angles(s, positions):
    """Cosine and sine [tokens][pairs] in 64 bits: far positions need them."""
    turns = positions.double()[:, None] * s.freq
    turns = (turns - torch.floor(turns)) * (2.0 * math.pi)
    return turns.cos() * s.gain, turns.sin() * s.gain


def _rotate(x, c, s):
    """x [tokens][heads][128]; c, s [tokens][64]."""
    c, s = c[:, None], s[:, None]
    a, b = x[..., :HEAD // 2], x[..., HEAD // 2:]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def _groups(x, part):
    """Blocks [..., 32, 128] so that a group lies along one axis, and that axis."""
    return (x[..., None], -3) if part == 0 else (x.unflatten(-1, (HEAD // GROUP, GROUP)), -1)


def _quantise(x, part):
    """Codes, scales and lows of whole blocks [..., 32, 128] of f16 keys (part 0) or values (1)."""
    grouped, axis = _groups(x, part)
    low, high = grouped.amin(axis, keepdim=True), grouped.amax(axis, keepdim=True)
    wide = (high.float() - low.float()) * (1.0 / 15.0)
    scale = wide.half()
    scale = torch.where(scale.float() > wide, (scale.view(torch.int16) - 1).view(torch.float16), scale)
    inverse = torch.where(scale > 0, 1.0 / scale.float(), 0.0)
    codes = ((grouped.float() - low.float()) * inverse).round().clamp(0, 15).to(torch.uint8)
    return codes.reshape(x.shape), scale, low


def _values(codes, scale, low, part):
    grouped, _ = _groups(codes, part)
    return (grouped.float() * scale.float() + low.float()).half().float().reshape(codes.shape)


def _heads(x, n, gamma):
    """[rows][n * 128] normalised per head, [rows][n][128], in x's type."""
    x = x.view(len(x), n, HEAD)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma


def _new_rows(s, positions):
    """Queries in 32 bits; keys (64 bits, rounded to f32 and f16) and values in f16: [rows][heads][128]."""
    kv = s.case["kv_heads"]
    c, sn = _angles(s, positions)
    q = _rotate(_heads(s.q, s.case["q_heads"], s.q_norm), c.float(), sn.float())
    k = _rotate(_heads(s.k.double(), kv, s.k_norm.double()), c, sn).float().half()
    return q, k, s.v.view(-1, kv, HEAD).half()


def _attend(q, keys, values, seen):
    """q [..., rows, 128], keys and values [..., tokens, 128], seen [..., rows, tokens]."""
    sc = torch.matmul(q, keys.transpose(-1, -2)) * (1.0 / math.sqrt(HEAD))
    sc = sc.masked_fill(~seen, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    return torch.matmul(p, values) / p.sum(-1, keepdim=True)


def _plain_decode(s):
    kv, m, per = s.case["kv_heads"], s.case["members"], s.case["q_heads"] // s.case["kv_heads"]
    pos = s.positions.long()
    q, k, v = _new_rows(s, s.positions)
    row, at, every = pos % BLOCK, pos // BLOCK, torch.arange(m, device=DEV)
    whole = (row == BLOCK - 1)[:, None, None, None]
    s.tail[0][every, :, row] = k
    s.tail[1][every, :, :, row] = v
    cached = []
    for part, rows in enumerate((s.tail[0], s.tail[1].transpose(2, 3))):
        new = _quantise(rows, part)
        for held, x in zip(s.held[part], new):
            pick = whole if x.dim() == 4 else whole[..., None]
            held[every, :, at] = torch.where(pick, x, held[every, :, at])
        x = _values(*s.held[part], part)
        x[every, :, at] = torch.where(whole, _values(*new, part), rows.float())
        cached.append(x.flatten(2, 3))
    seen = (torch.arange(cached[0].shape[2], device=DEV)[None] <= pos[:, None])[:, None, None]
    s.y.view(m, kv, per, HEAD)[:] = _attend(q.view(m, kv, per, HEAD), *cached, seen)


def _plain_chunk(s):
    kv, n, p0, per = s.case["kv_heads"], s.case["tokens"], s.case["position"], s.case["q_heads"] // s.case["kv_heads"]
    q, k, v = _new_rows(s, p0 + torch.arange(n, device=DEV))
    first, end = p0 // BLOCK, p0 + n  # (p0 is a whole number of blocks)
    whole = end // BLOCK
    last = (end - 1) // BLOCK * BLOCK - p0
    cached = []
    for part, (new, rows) in enumerate(zip((k, v), (s.tail[0][0], s.tail[1][0].transpose(1, 2)))):
        x = new.transpose(0, 1)
        done = (whole - first) * BLOCK
        for held, y in zip(s.held[part], _quantise(x[:, :done].reshape(kv, -1, BLOCK, HEAD), part)):
            held[0, :, first:whole] = y
        cached.append(torch.cat((_values(*(h[0, :, :whole] for h in s.held[part]), part).flatten(1, 2), x[:, done:].float()), 1))
        rows[:, :n - last] = x[:, last:]
    seen = torch.arange(end, device=DEV)[None] <= p0 + torch.arange(n, device=DEV)[:, None]
    q = q.view(n, kv, per, HEAD).permute(1, 2, 0, 3).reshape(kv, per * n, HEAD)
    out = _attend(q, *cached, seen.repeat(per, 1)[None])
    s.y.view(n, kv, per, HEAD)[:] = out.view(kv, per, n, HEAD).permute(2, 0, 1, 3)


def _plain_stage(s):
    whole = s.case["tokens"] // BLOCK * BLOCK
    for part, (x, y) in enumerate(zip((s.keys, s.values), s.back)):
        x = x.half()
        blocks = x[:whole].unflatten(0, (-1, BLOCK)).transpose(1, 2)
        y[:whole] = _values(*_quantise(blocks, part), part).half().transpose(1, 2).flatten(0, 1)
        y[whole:] = x[whole:]


def _plain_logprob(s):
    top, vocab = s.case["top"], s.case["vocab"]
    x = s.logits.float() + 0.0  # (no negative zeros)
    x = torch.where(torch.isnan(x), -math.inf, x)
    least = x.amax(-1, keepdim=True)
    t = x - least
    e = torch.exp(t)
    total = e.sum(-1, dtype=torch.float64)  # 64 bits: 1e-9 beside the largest token's 1 is a certain model's log probability
    weighted = torch.where(e > 0, e * t, 0.0).sum(-1, dtype=torch.float64)
    log_total = torch.log(total)
    s.entropy.copy_(log_total - weighted / total)
    s.logprobs.copy_(t.gather(1, s.given.long()[:, None])[:, 0].double() - log_total)
    if top:
        # one whole number a token that orders as (logit, lower token first)
        bits = x.view(torch.int32)
        key = (torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32) + (vocab - 1 - torch.arange(vocab, device=DEV))
        tokens = vocab - 1 - (torch.topk(key, top, -1)[0] & 0xffffffff)
        s.tokens.copy_(tokens)
        s.alternatives.copy_(t.gather(1, tokens).double() - log_total[:, None])


# -------------------------------------------------------------------- a pass

def run(s):
    kind = s.case["kind"]
    if own:
        import engine_amd as E

        if kind == "decode":
            E.attention_decode(s.ctx, s.cfg, s.caches, 0, s.q, s.k, s.v, s.q_norm, s.k_norm, s.positions, s.y)
        elif kind == "chunk":
            E.attention_prefill(s.ctx, s.cfg, s.caches[0], 0, s.q, s.k, s.v, s.q_norm, s.k_norm, s.case["tokens"],
                                s.case["position"], s.y)
        elif kind == "stage":
            s.caches[0].write(0, s.keys, s.values, 0)
            s.caches[0].read(0, 0, *s.back)
        elif s.case["top"]:
            s.ops.logprobs_into(s.logits, s.given, s.logprobs, s.entropy, s.tokens, s.alternatives)
        else:
            s.ops.logprobs_into(s.logits, s.given, s.logprobs, s.entropy)
        if kind in ("decode", "chunk"):
            return {"y": s.y, "tail": s.tails}
    else:
        {"decode": _plain_decode, "chunk": _plain_chunk, "stage": _plain_stage, "logprob": _plain_logprob}[kind](s)
    if kind == "stage":
        return s.back
    if kind == "logprob":
        return {"logprobs": s.logprobs, "entropy": s.entropy, "tokens": s.tokens, "alternatives": s.alternatives}
    # the output, and the f16 block each sequence stands in, as far as it is filled
    if kind == "decode":
        rows = [n % BLOCK + 1 for n in s.lengths]
    else:
        rows = [(s.case["position"] + s.case["tokens"] - 1) % BLOCK + 1]
    tails = s.tails if own else list(zip(*s.tail))
    return {"y": s.y, "tail": [(k[:, :n], v[:, :, :n]) for (k, v), n in zip(tails, rows)]}


# ------------------------------------------------------ what a pass must move

def work(case):
    kind = case["kind"]
    if kind == "logprob":
        n = case["rows"] * case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 1.0 * n * size + case["rows"] * (12.0 + 8.0 * case["top"]), "flops": 5.0 * n}
    kv = case["kv_heads"]
    # codes of key and value, and their share of the block's scales and lows
    token = kv * (HEAD + 4.0 * HEAD / BLOCK + 4.0 * HEAD / GROUP)
    if kind == "stage":
        n = case["tokens"]
        size = 2 if case["dtype"] == "f16" else 4
        return {"bytes": n * (2.0 * kv * HEAD * (size + 2) + 2.0 * token), "flops": 10.0 * n * kv * HEAD}
    q = case["q_heads"]
    if kind == "decode":
        cached, new = sum(_contexts(case)), case["members"]
        pairs = cached + new
    else:
        cached, new = case["position"], case["tokens"]
        pairs = new * cached + new * (new + 1) / 2
    return {"bytes": cached * token + new * (HEAD * (8.0 * q + 8.0 * kv) + token), "flops": 4.0 * HEAD * q * pairs}


# ------------------------------------------------------------ 64-bit results

def _turned(x, positions, scaling):
    """x [tokens][heads][128] in 64 bits, its pairs as complex numbers turned by their angle."""
    pairs = np.arange(HEAD // 2, dtype=np.float64)
    theta = np.exp(-2.0 * pairs / HEAD * np.log(BASE))
    factor, original = _scaling(scaling)
    gain = 1.0
    if scaling == "linear":
        theta = theta / factor
    if scaling == "yarn":
        bound = [HEAD * np.log(original / (2 * np.pi * b)) / (2 * np.log(BASE)) for b in (32.0, 1.0)]
        low, high = max(np.floor(bound[0]), 0), min(np.ceil(bound[1]), HEAD - 1)
        stretched = np.clip((pairs - low) / max(high - low, 0.001), 0, 1)
        theta = theta * (1 - stretched + stretched / factor)
        gain = 1.0 + 0.1 * np.log(factor)
    angle = positions.double().cpu()[:, None] * torch.from_numpy(theta)
    turn = torch.polar(torch.full_like(angle, gain), torch.remainder(angle, 2 * math.pi)).to(DEV)[:, None]
    z = torch.complex(x[..., :HEAD // 2].contiguous(), x[..., HEAD // 2:].contiguous()) * turn
    return torch.cat((z.real, z.imag), -1)


def _stored(x, keys):
    """What whole blocks [n, 32, 128] of a head's f16 keys (or values) are held as, in 64 bits. (The scale's and the
    quotient's f32 roundings are the format's: a 64-bit result rounded to f32.)"""
    x = x.double()
    if keys:
        x = x.transpose(1, 2)  # [n][128][32]: a group is a row
    rows = x.reshape(-1, BLOCK if keys else GROUP)
    if not len(rows):
        return x
    ordered = rows.sort(-1)[0]
    low, spread = ordered[:, :1], (ordered[:, -1:] - ordered[:, :1]).float().double()
    scale = (spread * np.float64(np.float32(1 / 15))).float().double()
    unit = torch.clamp(2.0 ** (torch.frexp(scale)[1].double() - 11.0), min=2.0 ** -24)  # a step of f16 there
    scale = torch.floor(scale / unit) * unit
    per = torch.where(scale == 0, 0.0, (1 / scale.clamp(min=2.0 ** -24)).float().double())
    codes = torch.round(((rows - low).float().double() * per).float().double())
    held = (torch.clamp(codes, max=15) * scale + low).float().half().double().reshape(x.shape)
    return held.transpose(1, 2) if keys else held


def _sequence(old, new, keys):
    """A head's tokens as the cache holds them: whole blocks by their codes, the rest in f16. -> f64 [tokens][128], f16 rows of the last block."""
    x = torch.cat((old, new))
    n = len(x) // BLOCK * BLOCK
    last = (len(x) - 1) // BLOCK * BLOCK
    return torch.cat((_stored(x[:n].view(-1, BLOCK, HEAD), keys).reshape(n, HEAD), x[n:].double())), x[last:]


def _exact_logprob(s):
    out = {"logprobs": [], "entropy": [], "tokens": [], "alternatives": []}
    top = s.case["top"]
    for lo in range(0, s.case["rows"], 64):
        x = torch.nan_to_num(s.logits[lo:lo + 64].double(), nan=-math.inf, neginf=-math.inf, posinf=math.inf)
        # the logarithm of 1 and what the others have beside the likeliest's 1: near a certain model's 0 too
        best, at = x.max(-1, keepdim=True)
        others = torch.exp(x - best).scatter(1, at, 0.0).sum(-1, keepdim=True)
        p = x - best - torch.log1p(others)
        out["logprobs"].append(p.gather(1, s.given[lo:lo + 64].long()[:, None])[:, 0])
        out["entropy"].append(torch.special.entr(torch.exp(p)).sum(-1))
        ranked = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top]
        out["tokens"].append(ranked.int())
        out["alternatives"].append(p.gather(1, ranked))
    return {k: torch.cat(v) for k, v in out.items()}


def exact(case, seed):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind == "logprob":
        return _exact_logprob(s)
    if kind == "stage":
        kv = case["kv_heads"]
        out = []
        for i, x in enumerate((s.keys.half(), s.values.half())):
            out.append(torch.stack([_sequence(x[:0, h], x[:, h], i == 0)[0] for h in range(kv)], 1))
        return out
    kv, per = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    unit = [x.double().view(len(x), -1, HEAD) for x in (s.q, s.k)]
    rows = s.positions if kind == "decode" else case["position"] + torch.arange(case["tokens"], device=DEV)
    q, k = (_turned(x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double(), rows, case["scaling"])
            for x, w in zip(unit, (s.q_norm, s.k_norm)))
    k, v = k.float().half(), s.v.view(-1, kv, HEAD).half()
    outs, tails = [], []
    for i, (old_k, old_v) in enumerate(s.contexts):
        mine = slice(i, i + 1) if kind == "decode" else slice(None)
        p0, heads, tail = len(old_k), [], ([], [])
        for h in range(kv):
            keys, tk = _sequence(old_k[:, h], k[mine, h], True)
            values, tv = _sequence(old_v[:, h], v[mine, h], False)
            tail[0].append(tk)
            tail[1].append(tv.t())
            unseen = torch.arange(len(keys), device=DEV)[None] > p0 + torch.arange(len(k[mine]), device=DEV)[:, None]
            for j in range(per):
                sc = (q[mine, h * per + j] @ keys.t()) / math.sqrt(HEAD)
                heads.append(torch.softmax(sc.masked_fill(unseen, -math.inf), -1) @ values)
        outs.append(torch.stack(heads, 1))
        tails.append(tuple(torch.stack(t).double() for t in tail))
    return {"y": torch.cat(outs).flatten(), "tail": tails}
