"""The operators of long contexts: what a user's program has the library do.

  decode  a layer's decode attention for a batch of sequences whose caches are
          held in 8 bits (the new tokens' keys and values appended on the way)
  chunk   a layer's causal attention for a prompt chunk over such a cache
  stage   a context's keys and values written into the cache, and read back
  rope    rotary positions of queries and keys, in both layouts, on part of the
          head or all of it, unscaled or scaled for long contexts

A cache keeps blocks of 32 tokens, one power-of-two scale per block and KV head
for the keys and one for the values: with x16 the values rounded to f16 and a
their largest magnitude in the block, e = max(floor(log2 a) - 6, -24), a code
is x16 * 2^-e rounded to the nearest whole number (ties to even) and clamped to
+-127, and it stands for code * 2^e. A block that is not whole is kept in f16,
keys [token][dim] and values [dim][token]. Attention sees the cache as it is
after the call's own tokens are in it. Keys are normalised and rotated in 64
bits and rounded to f32, then to f16.

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
EPS = 1e-6
BASE = 1.0e6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One sequence at the start of its answer: all launch and latency.
        dict(name="decode_1x40", kind="decode", q_heads=32, kv_heads=8, members=1, context=40, scaling="none"),
        # Eight sequences of different lengths, an ordinary serving step.
        dict(name="decode_8x3000", kind="decode", q_heads=32, kv_heads=8, members=8, context=3000, scaling="none"),
        # A wide batch of medium contexts, eight query heads to a KV head.
        dict(name="decode_24x1501", kind="decode", q_heads=64, kv_heads=8, members=24, context=1501, scaling="none"),
        # One sequence at the end of the scaled range of positions.
        dict(name="decode_1x131071", kind="decode", q_heads=32, kv_heads=8, members=1, context=131071, scaling="yarn"),
        # A short question put after a cached document.
        dict(name="chunk_37", kind="chunk", q_heads=32, kv_heads=8, tokens=37, position=2011, scaling="none"),
        # A whole prompt chunk from the start.
        dict(name="chunk_2047", kind="chunk", q_heads=32, kv_heads=8, tokens=2047, position=0, scaling="none"),
        # A later chunk of a long prompt, at odd sizes.
        dict(name="chunk_1999", kind="chunk", q_heads=32, kv_heads=8, tokens=1999, position=6203, scaling="yarn"),
        # A short shared prefix put into a new sequence's cache and taken out again.
        dict(name="stage_100", kind="stage", kv_heads=8, tokens=100, dtype="f16"),
        # A long document's keys and values moved into the cache and out.
        dict(name="stage_32768", kind="stage", kv_heads=8, tokens=32768, dtype="f16"),
        # One token's queries and keys, out of a fused projection's row.
        dict(name="rope_1", kind="rope", tokens=1, q_heads=32, kv_heads=8, head=128, rotary=128, layout="half", dtype="f32",
             scaling="none", fused=True),
        # A serving batch's prompt chunk, interleaved pairs on half of each head.
        dict(name="rope_2047", kind="rope", tokens=2047, q_heads=16, kv_heads=16, head=128, rotary=64, layout="interleaved",
             dtype="bf16", scaling="linear", fused=True),
        # A long document at once, scaled positions.
        dict(name="rope_32768", kind="rope", tokens=32768, q_heads=32, kv_heads=8, head=128, rotary=128, layout="half",
             dtype="f32", scaling="yarn", fused=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "chunk", "chunk", "stage", "rope", "rope"))
    heads = rng.choice(((8, 8), (16, 8), (32, 8), (32, 8), (64, 8), (32, 4), (4, 2)))
    scaling = rng.choice(("none", "none", "yarn", "linear"))
    if kind == "decode":
        members = _log_int(rng, 1, 31)
        return dict(kind="decode", q_heads=heads[0], kv_heads=heads[1], members=members,
                    context=_log_int(rng, 1, 131071 // members), scaling=scaling)
    if kind == "chunk":
        tokens = _log_int(rng, 1, 2047)
        room = int(min(12000, 13.0e6 / tokens * 32 / max(32, heads[0]) - tokens / 2))
        position = 0 if rng.random() < 0.4 or room < 2 else _log_int(rng, 1, room)
        return dict(kind="chunk", q_heads=heads[0], kv_heads=heads[1], tokens=tokens, position=position, scaling=scaling)
    if kind == "stage":
        return dict(kind="stage", kv_heads=heads[1], tokens=_log_int(rng, 1, 32000), dtype=rng.choice(("f16", "f32")))
    head = rng.choice((64, 80, 96, 128, 128, 192, 256))
    rotary = head if rng.random() < 0.6 else 2 * rng.randint(1, head // 2)
    kv = rng.choice((1, 2, 4, 8))
    q = kv * rng.choice((1, 2, 4, 8))
    most = int(32768 * 40 * 128 / ((q + kv) * head))
    return dict(kind="rope", tokens=_log_int(rng, 1, min(most, 32768)), q_heads=q, kv_heads=kv, head=head, rotary=rotary,
                layout=rng.choice(("half", "interleaved")), dtype=rng.choice(tuple(DTYPES)), scaling=scaling,
                fused=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * seed + 29)
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
    the rest), and values: f16 [tokens][kv_heads][128]."""
    wide = torch.rand((1, kv_heads, HEAD), device=DEV, generator=g)
    gain = torch.where(wide > 0.97, 6.0, 0.5 + wide)
    keys = torch.randn((tokens, kv_heads, HEAD), device=DEV, generator=g).mul_(gain).half()
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


def _inputs(case, seed):
    """What the calls work on, and the contexts that are to be in the caches."""
    s = _State()
    s.case = case
    kind = case["kind"]
    g = _generator(seed)
    if kind == "rope":
        tokens, head, dtype = case["tokens"], case["head"], DTYPES[case["dtype"]]
        q, kv = case["q_heads"], case["kv_heads"]
        if case["fused"]:  # queries, keys and values of a token in one row, as a fused projection leaves them
            row = torch.randn((tokens, q + 2 * kv, head), device=DEV, generator=g).to(dtype)
            s.x = [row[:, :q], row[:, q:q + kv]]
        else:
            s.x = [torch.randn((tokens, n, head), device=DEV, generator=g).to(dtype) for n in (q, kv)]
        far = 131072 if case["scaling"] == "yarn" else 32768
        first = int(torch.randint(0, max(1, far - tokens + 1), (1,), device=DEV, generator=g).item())
        s.positions = torch.arange(first, first + tokens, dtype=torch.int32, device=DEV)
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
    if kind == "rope":
        s.y = [torch.empty(x.shape, dtype=x.dtype, device=DEV) for x in s.x]
    elif kind == "stage":
        s.back = [torch.empty(s.keys.shape, dtype=torch.float16, device=DEV) for _ in range(2)]
    else:
        s.y = torch.zeros(s.q.numel(), device=DEV)
    if own:
        _prepare_own(s, case)
    elif kind == "rope":
        s.freq, s.gain = _frequencies(case["rotary"], case["scaling"])
    elif kind != "stage":
        s.freq, s.gain = _frequencies(HEAD, case["scaling"])
        _prepare_plain(s, case["kv_heads"], max(s.lengths) + (1 if kind == "decode" else case["tokens"]))
    s.contexts = None  # the caches hold them now
    return s


def _prepare_own(s, case):
    import engine_amd as E

    kind = case["kind"]
    s.ctx = E.AmdContext(0)
    factor, original = _scaling(case.get("scaling", "none"))
    if kind == "rope":
        s.rope = E.AmdRope(s.ctx, E.AmdRopeSpec(head_dim=case["head"], rotary_dim=case["rotary"], layout=case["layout"],
                                                base=BASE, scaling=case["scaling"], factor=factor, original_context=original))
        return
    s.cfg = E.AmdQwen3Config(layers=1, hidden=4096, q_heads=case.get("q_heads", case["kv_heads"]), kv_heads=case["kv_heads"],
                             head_dim=HEAD, ffn=12288, vocab=1024, rope_base=BASE, epsilon=EPS)
    rope = None
    if factor != 1.0:
        rope = E.AmdRopeSpec(head_dim=HEAD, base=BASE, scaling=case["scaling"], factor=factor, original_context=original)
    extra = {"decode": 1, "chunk": case.get("tokens", 0), "stage": 0}[kind]
    s.caches = [E.AmdKvCache(s.ctx, s.cfg, n + extra, format=E.KV_I8, rope=rope) for n in s.lengths]
    for cache, (keys, values) in zip(s.caches, s.contexts):
        if len(keys):
            cache.write(0, keys, values, 0)
    if kind != "stage":
        rows = [(n + extra - 1) % BLOCK + 1 for n in s.lengths]
        s.tails = [(k[:, :n], v[:, :, :n]) for (k, v), n in zip((_tails(c, case["kv_heads"]) for c in s.caches), rows)]


def _prepare_plain(s, kv, room):
    """Codes and exponents of the whole blocks, padded to the longest sequence, and each sequence's f16 block."""
    blocks = -(-room // BLOCK)
    m = len(s.contexts)
    s.codes = [torch.zeros((m, kv, blocks, BLOCK, HEAD), dtype=torch.int8, device=DEV) for _ in range(2)]
    s.exps = [torch.full((m, kv, blocks, 1, 1), -24, dtype=torch.int32, device=DEV) for _ in range(2)]
    s.tail = [torch.zeros((m, kv, BLOCK, HEAD), dtype=torch.float16, device=DEV), torch.zeros((m, kv, HEAD, BLOCK), dtype=torch.float16, device=DEV)]
    s.end = list(s.lengths)
    for i, pair in enumerate(s.contexts):
        n = len(pair[0])
        whole, last = n // BLOCK, max(0, (n - 1) // BLOCK * BLOCK)
        for part, x in enumerate(pair):
            x = x.transpose(0, 1)
            s.codes[part][i, :, :whole], s.exps[part][i, :, :whole] = _quantise(x[:, :whole * BLOCK].reshape(kv, whole, BLOCK, HEAD))
            rows = s.tail[0][i] if part == 0 else s.tail[1][i].transpose(1, 2)
            rows[:, :n - last] = x[:, last:]


# -------------------------------------------------------------------- plain form

def _frequencies(rotary, scaling):
    """Turns a position adds to each pair's angle, in 64 bits, and the gain of cosine and sine."""
    i = torch.arange(rotary // 2, dtype=torch.float64, device=DEV)
    f = BASE ** (-2.0 * i / rotary)
    factor, original = _scaling(scaling)
    gain = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        # pairs that turn often within the trained length stay, slow ones stretch
        low, high = (rotary * math.log(original / (2.0 * math.pi * beta)) / (2.0 * math.log(BASE)) for beta in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rotary - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        f = f / factor * ramp + f * (1.0 - ramp)
        gain = 0.1 * math.log(factor) + 1.0
    return f / (2.0 * math.pi), gain


def _angles(s, positions):
    """Cosine and sine [tokens][pairs] in 64 bits: far positions need them."""
    turns = positions.double()[:, None] * s.freq
    turns = (turns - torch.floor(turns)) * (2.0 * math.pi)
    return turns.cos() * s.gain, turns.sin() * s.gain


def _rotate(x, c, s, layout, rotary):
    """x [tokens][heads][head]; c, s [tokens][pairs]."""
    c, s = c[:, None], s[:, None]
    if layout == "half":
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        return torch.cat((a * c - b * s, a * s + b * c, x[..., rotary:]), -1)
    a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    return torch.cat((torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2), x[..., rotary:]), -1)


def _power(e):
    """2^e in f32, from its bits: a device's pow() need not be exact, and codes lie on ties."""
    return ((e + 127) << 23).view(torch.float32)


def _quantise(x):
    """Codes and exponents of whole blocks [..., 32, 128]."""
    x = x.float()
    e = (torch.frexp(x.abs().amax((-2, -1), keepdim=True))[1] - 7).clamp(min=-24)
    return (x * _power(-e)).round().clamp(-127, 127).to(torch.int8), e


def _values(codes, exps):
    return codes.float() * _power(exps)


def _heads(x, n, gamma):
    """[rows][n * 128] normalised per head, [rows][n][128], in x's type."""
    x = x.view(len(x), n, HEAD)
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma


def _new_rows(s, positions):
    """Queries in 32 bits; keys (64 bits, rounded to f32 and f16) and values in f16: [rows][heads][128]."""
    kv = s.case["kv_heads"]
    c, sn = _angles(s, positions)
    q = _rotate(_heads(s.q, s.case["q_heads"], s.q_norm), c.float(), sn.float(), "half", HEAD)
    k = _rotate(_heads(s.k.double(), kv, s.k_norm.double()), c, sn, "half", HEAD).float().half()
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
        codes, exps = _quantise(rows)
        s.codes[part][every, :, at] = torch.where(whole, codes, s.codes[part][every, :, at])
        s.exps[part][every, :, at] = torch.where(whole, exps, s.exps[part][every, :, at])
        x = _values(s.codes[part], s.exps[part])
        x[every, :, at] = torch.where(whole, _values(codes, exps), rows.float())
        cached.append(x.flatten(2, 3))
    seen = (torch.arange(cached[0].shape[2], device=DEV)[None] <= pos[:, None])[:, None, None]
    s.y.view(m, kv, per, HEAD)[:] = _attend(q.view(m, kv, per, HEAD), *cached, seen)


def _plain_chunk(s):
    kv, n, p0, per = s.case["kv_heads"], s.case["tokens"], s.case["position"], s.case["q_heads"] // s.case["kv_heads"]
    q, k, v = _new_rows(s, p0 + torch.arange(n, device=DEV))
    first, before, end = p0 // BLOCK, p0 % BLOCK, p0 + n
    whole = end // BLOCK
    held = s.end[0] > 0 and (s.end[0] - 1) // BLOCK == first  # else the block's earlier rows are its codes' values
    cached = []
    for part, (new, rows) in enumerate(zip((k, v), (s.tail[0][0], s.tail[1][0].transpose(1, 2)))):
        codes, exps = s.codes[part][0], s.exps[part][0]
        old = rows[:, :before] if held else _values(codes[:, first], exps[:, first])[:, :before].half()
        x = torch.cat((old, new.transpose(0, 1)), 1)
        done = (whole - first) * BLOCK
        codes[:, first:whole], exps[:, first:whole] = _quantise(x[:, :done].reshape(kv, -1, BLOCK, HEAD))
        cached.append(torch.cat((_values(codes[:, :whole], exps[:, :whole]).flatten(1, 2), x[:, done:].float()), 1))
        last = (end - 1) // BLOCK * BLOCK - first * BLOCK
        rows[:, :x.shape[1] - last] = x[:, last:]
    s.end[0] = end
    seen = torch.arange(end, device=DEV)[None] <= p0 + torch.arange(n, device=DEV)[:, None]
    q = q.view(n, kv, per, HEAD).permute(1, 2, 0, 3).reshape(kv, per * n, HEAD)
    out = _attend(q, *cached, seen.repeat(per, 1)[None])
    s.y.view(n, kv, per, HEAD)[:] = out.view(kv, per, n, HEAD).permute(2, 0, 1, 3)


def _plain_stage(s):
    whole = s.case["tokens"] // BLOCK * BLOCK
    for x, y in zip((s.keys, s.values), s.back):
        x = x.half()
        blocks = x[:whole].unflatten(0, (-1, BLOCK)).transpose(1, 2)
        y[:whole] = _values(*_quantise(blocks)).transpose(1, 2).flatten(0, 1).half()
        y[whole:] = x[whole:]


def _plain_rope(s):
    c, sn = _angles(s, s.positions)
    c, sn = c.float(), sn.float()
    s.y = [_rotate(x.float(), c, sn, s.case["layout"], s.case["rotary"]).to(x.dtype) for x in s.x]


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
        else:
            s.rope.execute_group(s.x, s.positions, s.y)
        if kind in ("decode", "chunk"):
            return {"y": s.y, "tail": s.tails}
    else:
        {"decode": _plain_decode, "chunk": _plain_chunk, "stage": _plain_stage, "rope": _plain_rope}[kind](s)
    if kind == "stage":
        return s.back
    if kind == "rope":
        return s.y
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
    if kind == "rope":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        size = 2 if case["dtype"] != "f32" else 4
        return {"bytes": 2.0 * n * case["head"] * size + 4.0 * case["tokens"], "flops": 3.0 * n * case["rotary"]}
    kv = case["kv_heads"]
    token = kv * (2.0 * HEAD + 8.0 / BLOCK)  # codes of key and value, and their share of the block's scales
    if kind == "stage":
        n = case["tokens"]
        size = 2 if case["dtype"] == "f16" else 4
        return {"bytes": n * (2.0 * kv * HEAD * (size + 2) + 2.0 * token), "flops": 4.0 * n * kv * HEAD}
    q = case["q_heads"]
    if kind == "decode":
        cached, new = sum(_contexts(case)), case["members"]
        pairs = cached + new
    else:
        cached, new = case["position"], case["tokens"]
        pairs = new * cached + new * (new + 1) / 2
    return {"bytes": cached * token + new * (HEAD * (8.0 * q + 8.0 * kv) + token), "flops": 4.0 * HEAD * q * pairs}


# ------------------------------------------------------------ 64-bit results

def _turned(x, positions, rotary, layout, scaling):
    """x [tokens][heads][head] in 64 bits, its pairs as complex numbers turned by their angle."""
    pairs = np.arange(rotary // 2, dtype=np.float64)
    theta = np.exp(-2.0 * pairs / rotary * np.log(BASE))
    factor, original = _scaling(scaling)
    gain = 1.0
    if scaling == "linear":
        theta = theta / factor
    if scaling == "yarn":
        bound = [rotary * np.log(original / (2 * np.pi * b)) / (2 * np.log(BASE)) for b in (32.0, 1.0)]
        low, high = max(np.floor(bound[0]), 0), min(np.ceil(bound[1]), rotary - 1)
        stretched = np.clip((pairs - low) / max(high - low, 0.001), 0, 1)
        theta = theta * (1 - stretched + stretched / factor)
        gain = 1.0 + 0.1 * np.log(factor)
    angle = positions.double().cpu()[:, None] * torch.from_numpy(theta)
    turn = torch.polar(torch.full_like(angle, gain), torch.remainder(angle, 2 * math.pi)).to(DEV)[:, None]
    y = x.clone()
    if layout == "half":
        z = torch.complex(x[..., :rotary // 2].contiguous(), x[..., rotary // 2:rotary].contiguous()) * turn
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = z.real, z.imag
    else:
        z = torch.view_as_complex(x[..., :rotary].reshape(*x.shape[:-1], rotary // 2, 2).contiguous()) * turn
        y[..., :rotary] = torch.view_as_real(z).flatten(-2)
    return y


def _stored(x):
    """What whole blocks [..., 32, 128] of f16 values are held as, in 64 bits."""
    x = x.double()
    most = x.abs().amax((-2, -1), keepdim=True)
    powers = torch.tensor([2.0 ** k for k in range(-18, 17)], dtype=torch.float64, device=x.device)
    at = (most[..., None] >= powers).sum(-1) - 1  # the largest power of two up to `most`
    unit = powers[at.clamp(min=0)] / 64.0         # 2^(floor(log2 most) - 6), 2^-24 at least
    return (x / unit).round().clamp(-127, 127) * unit


def _sequence(old, new):
    """A head's tokens as the cache holds them: whole blocks by their codes, the rest in f16. -> f64 [tokens][128], f16 rows of the last block."""
    x = torch.cat((old, new))
    n = len(x) // BLOCK * BLOCK
    last = (len(x) - 1) // BLOCK * BLOCK
    return torch.cat((_stored(x[:n].view(-1, BLOCK, HEAD)).reshape(n, HEAD), x[n:].double())), x[last:]


def exact(case, seed):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind == "rope":
        return [_turned(x.double(), s.positions, case["rotary"], case["layout"], case["scaling"]) for x in s.x]
    if kind == "stage":
        kv = case["kv_heads"]
        out = []
        for x in (s.keys.half(), s.values.half()):
            out.append(torch.stack([_sequence(x[:0, h], x[:, h])[0] for h in range(kv)], 1))
        return out
    kv, per = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    unit = [x.double().view(len(x), -1, HEAD) for x in (s.q, s.k)]
    rows = s.positions if kind == "decode" else case["position"] + torch.arange(case["tokens"], device=DEV)
    q, k = (_turned(x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w.double(), rows, HEAD, "half", case["scaling"])
            for x, w in zip(unit, (s.q_norm, s.k_norm)))
    k, v = k.float().half(), s.v.view(-1, kv, HEAD).half()
    outs, tails = [], []
    for i, (old_k, old_v) in enumerate(s.contexts):
        mine = slice(i, i + 1) if kind == "decode" else slice(None)
        p0, heads, tail = len(old_k), [], ([], [])
        for h in range(kv):
            keys, tk = _sequence(old_k[:, h], k[mine, h])
            values, tv = _sequence(old_v[:, h], v[mine, h])
            tail[0].append(tk)
            tail[1].append(tv.t())
            unseen = torch.arange(len(keys), device=DEV)[None] > p0 + torch.arange(len(k[mine]), device=DEV)[:, None]
            for j in range(per):
                sc = (q[mine, h * per + j] @ keys.t()) / math.sqrt(HEAD)
                heads.append(torch.softmax(sc.masked_fill(unseen, -math.inf), -1) @ values)
        outs.append(torch.stack(heads, 1))
        tails.append(tuple(torch.stack(t).double() for t in tail))
    return {"y": torch.cat(outs).flatten(), "tail": tails}
