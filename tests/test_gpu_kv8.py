"""GPU tests of the KV cache in 8 bits, through the public entry points, against
oracle/longctx_oracle.py (64 bits, numpy).

  * what a cache holds is compared for equality: keys are formed in 64 bits on
    both sides and rounded f32, f16, code; values are rounded as they come;
  * attention within ATTN_TOL normwise. q is formed in f32 (about six roundings
    of 2^-24) and carried as two f16 pieces (2^-23), a score is a sum of 128 f32
    products (rounding 2^-24 of a partial sum each, about sqrt(128) of them
    adding up): with sum |q_i k_i| / sqrt(128) up to 25 for these inputs, scores are
    off by up to 25 * 12 * 2^-24 = 1.8e-5, probabilities by as much relatively,
    and an output, a mean of values with these weights, by less of the largest value.
    The cache itself adds nothing: its values are the oracle's.
"""
import ctypes

import numpy as np
import pytest

from oracle import longctx_oracle as L
from .gpu_helpers import max_rel_err

pytestmark = pytest.mark.gpu

ATTN_TOL = 2e-5
BASE, EPS = 1.0e6, 1.0e-6
YARN = dict(scaling="yarn", factor=4.0, original_context=32768)


def case(**kw):
    print("CASE", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


@pytest.fixture(scope="module")
def env():
    import torch
    import engine_amd as E
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return {"E": E, "ctx": E.AmdContext(0), "torch": torch}


def config(env, q_heads, kv_heads, layers=1, **kw):
    return env["E"].AmdQwen3Config(layers=layers, hidden=4096, q_heads=q_heads, kv_heads=kv_heads, head_dim=128, ffn=768,
                                   vocab=1024, rope_base=BASE, epsilon=EPS, **kw)


def dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")
    return t if dtype is None else t.to(dtype)


def read(env, cache, cfg, layer, position, tokens, dtype=None):
    """[2][kv_heads][tokens][128] as numpy."""
    torch = env["torch"]
    out = [torch.full((tokens, cfg.kv_heads, 128), 7.0, dtype=dtype or torch.float32, device="cuda:0") for _ in range(2)]
    cache.read(layer, position, *out)
    torch.cuda.synchronize()
    return np.stack([o.float().cpu().numpy().transpose(1, 0, 2) for o in out])


def rows(rng, tokens, heads):
    """Keys with a few large channels, values: f32 [tokens][heads][128]."""
    gain = np.where(rng.random((1, heads, 128)) > 0.97, 6.0, 0.5 + rng.random((1, heads, 128)))
    return (rng.standard_normal((tokens, heads, 128)) * gain).astype(np.float32), \
        (0.5 * rng.standard_normal((tokens, heads, 128))).astype(np.float32)


class Seq:
    """One sequence: the library's cache and the oracle's, layer 0 .. layers - 1."""

    def __init__(self, env, cfg, capacity, rope=None):
        self.env, self.cfg, self.capacity = env, cfg, capacity
        self.cache = env["E"].AmdKvCache(env["ctx"], cfg, capacity, format=env["E"].KV_I8, rope=rope)
        self.model = [L.Kv8(cfg.kv_heads, capacity) for _ in range(cfg.layers)]

    def fill(self, rng, tokens, layer=0):
        k, v = rows(rng, tokens, self.cfg.kv_heads)
        self.cache.write(layer, dev(k), dev(v), self.model[layer].end)
        self.model[layer].append(self.model[layer].end, k, v)

    def check(self, layer=0):
        m = self.model[layer]
        np.testing.assert_array_equal(read(self.env, self.cache, self.cfg, layer, 0, m.end), m.rows())


def table(rope):
    return L.rope_turns(128, BASE, **(dict(scaling=rope["scaling"], factor=rope["factor"], original=rope.get("original_context", 0))
                                      if rope else {}))


class Step:
    """Random inputs of a decode step or a prompt chunk (`n` rows)."""

    def __init__(self, rng, cfg, n, gain=1.0):
        self.q = (gain * rng.standard_normal((n, cfg.q_heads, 128))).astype(np.float32)
        self.k, self.v = (rng.standard_normal((n, cfg.kv_heads, 128)).astype(np.float32) for _ in range(2))
        self.qn, self.kn = ((1 + 0.1 * rng.standard_normal(128)).astype(np.float32) for _ in range(2))

    def device(self):
        return [dev(x) for x in (self.q.reshape(-1), self.k.reshape(-1), self.v.reshape(-1), self.qn, self.kn)]

    def turned(self, positions, tab):
        q = L.rope(L.rms_norm(self.q, self.qn, EPS), positions, *tab)
        k = L.rope(L.rms_norm(self.k, self.kn, EPS), positions, *tab)
        return q, k


def decode(env, seqs, step, positions, layer=0, ctx=None):
    cfg = seqs[0].cfg
    out = dev(np.full(len(seqs) * cfg.q_heads * 128, np.nan, np.float32))
    env["E"].attention_decode(ctx or env["ctx"], cfg, [s.cache for s in seqs], layer, *step.device(),
                              dev(np.array(positions, np.int32)), out)
    env["torch"].cuda.synchronize()
    return out.cpu().numpy().reshape(len(seqs), cfg.q_heads, 128)


def check_decode(env, seqs, step, positions, tab, layer=0):
    got = decode(env, seqs, step, positions, layer)
    q, k = step.turned(positions, tab)
    for i, (s, p) in enumerate(zip(seqs, positions)):
        s.model[layer].append(p, k[i:i + 1], step.v[i:i + 1])
        want = L.attend(q[i], *s.model[layer].rows())
        err = max_rel_err(got[i], want)
        assert err <= ATTN_TOL, (i, p, err)
    return got


def prefill(env, seq, step, tokens, position, layer=0):
    out = dev(np.full(tokens * seq.cfg.q_heads * 128, np.nan, np.float32))
    env["E"].attention_prefill(env["ctx"], seq.cfg, seq.cache, layer, *step.device(), tokens, position, out)
    env["torch"].cuda.synchronize()
    return out.cpu().numpy().reshape(tokens, seq.cfg.q_heads, 128)


def check_prefill(env, seq, step, tokens, position, tab, layer=0, every=1):
    got = prefill(env, seq, step, tokens, position, layer)
    q, k = step.turned(position + np.arange(tokens), tab)
    m = seq.model[layer]
    m.append(position, k, step.v)
    held = m.rows()
    for t in sorted({*range(0, tokens, every), 0, tokens - 1}):
        want = L.attend(q[t], *held[:, :, :position + t + 1])
        err = max_rel_err(got[t], want)
        assert err <= ATTN_TOL, (t, err)
    assert np.isfinite(got).all()
    seq.check(layer)


# ------------------------------------------------------------- write and read

@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_write_read(env, tokens, dtype):
    case(test="write_read", tokens=tokens, dtype=dtype)
    torch = env["torch"]
    cfg = config(env, 4, 2, layers=2)
    s = Seq(env, cfg, tokens + 5)
    rng = np.random.default_rng(tokens)
    k, v = rows(rng, tokens, 2)
    kd, vd = dev(k, getattr(torch, dtype)), dev(v, getattr(torch, dtype))
    s.cache.write(1, kd, vd, 0)
    s.model[1].append(0, kd.float().cpu().numpy(), vd.float().cpu().numpy())
    s.check(1)
    got = read(env, s.cache, cfg, 1, 0, tokens + 5, getattr(torch, dtype))
    np.testing.assert_array_equal(got[:, :, :tokens], s.model[1].rows())
    assert not got[:, :, tokens:].any()                                # past the end: zeros
    assert not read(env, s.cache, cfg, 0, 0, tokens + 5).any()         # the other layer: untouched
    for lo, n in ((0, 1), (tokens - 1, 1), (tokens // 2, tokens - tokens // 2), (max(0, tokens - 34), min(tokens, 34))):
        np.testing.assert_array_equal(read(env, s.cache, cfg, 1, lo, n), s.model[1].rows()[:, :, lo:lo + n])


@pytest.mark.parametrize("pieces", [(1, 1, 1), (31, 1, 32), (5, 27), (32, 32, 7), (33, 31, 40), (20, 90, 3, 200), (64, 1, 63, 1)])
def test_writes_in_pieces_are_one_write(env, pieces):
    case(test="pieces", pieces=pieces)
    cfg = config(env, 2, 2)
    rng = np.random.default_rng(sum(pieces))
    s, one = Seq(env, cfg, sum(pieces)), Seq(env, cfg, sum(pieces))
    k, v = rows(rng, sum(pieces), 2)
    at = 0
    for n in pieces:
        s.cache.write(0, dev(k[at:at + n]), dev(v[at:at + n]), at)
        s.model[0].append(at, k[at:at + n], v[at:at + n])
        s.check()
        at += n
    one.cache.write(0, dev(k), dev(v), 0)
    np.testing.assert_array_equal(read(env, one.cache, cfg, 0, 0, at), read(env, s.cache, cfg, 0, 0, at))


def test_values_at_the_edges(env):
    """Infinities, NaN, the largest and smallest f16, ties, zeros, one large value among small ones."""
    case(test="edges")
    cfg = config(env, 2, 1)
    rng = np.random.default_rng(3)
    x = np.zeros((9, 32, 1, 128), np.float32)
    x[1, 0, 0, :4] = (np.inf, -np.inf, np.nan, 1.0)
    x[2] = 65504.0 * np.sign(rng.standard_normal((32, 1, 128)))
    x[3] = 2.0 ** -24 * rng.integers(-3, 4, (32, 1, 128))
    x[4] = (rng.integers(-127, 128, (32, 1, 128)) + 0.5) * 2.0 ** -3
    x[5] = rng.standard_normal((32, 1, 128)) * 1e-3
    x[5, 7, 0, 9] = 1000.0
    x[6, 31, 0, 127] = -127.75
    x[7] = -0.0
    x[8] = 1e30
    s = Seq(env, cfg, 9 * 32)
    k, v = x.reshape(-1, 1, 128), x[::-1].reshape(-1, 1, 128)
    for n in (9 * 32 - 5, 9 * 32):  # the last block in f16, then in 8 bits
        s.cache.write(0, dev(k[:n]), dev(v[:n]), 0)
        s.model[0].append(0, k[:n], v[:n])
        s.check()
    # attention over such a cache is finite
    step = Step(rng, cfg, 1)
    big = Seq(env, cfg, 9 * 32 + 1)
    big.cache.write(0, dev(k), dev(v), 0)
    assert np.isfinite(decode(env, [big], step, [9 * 32])).all()


def test_f16_caches_take_and_give_rows(env):
    case(test="f16_rows")
    torch, E = env["torch"], env["E"]
    cfg = config(env, 4, 2, layers=2)
    rng = np.random.default_rng(9)
    k, v = rows(rng, 70, 2)
    cache = E.AmdKvCache(env["ctx"], cfg, 90)
    cache.write(1, dev(k[:50]), dev(v[:50]), 3)
    cache.write(1, dev(k[50:], torch.float16), dev(v[50:], torch.float16), 53)
    want = np.stack([k, v]).transpose(0, 2, 1, 3).astype(np.float16).astype(np.float32)
    np.testing.assert_array_equal(read(env, cache, cfg, 1, 3, 70), want)
    np.testing.assert_array_equal(read(env, cache, cfg, 1, 20, 11, torch.float16), want[:, :, 17:28])
    view = np.zeros((2, 90, 128), np.uint16)
    lib = env["ctx"]._lib
    assert lib.ribn_amd_memcpy_dtoh(env["ctx"].handle, view.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(cache.layer(1)[1]), view.nbytes) == 0
    np.testing.assert_array_equal(view.view(np.float16)[:, 3:73].astype(np.float32), want[1])


# ---------------------------------------------------------------- decode attention

@pytest.mark.parametrize("position", [0, 1, 14, 15, 16, 30, 31, 32, 33, 62, 63, 64, 95, 96, 127, 128, 129, 255, 256, 511, 700, 1023, 1500])
def test_decode_positions(env, position):
    case(test="decode_positions", position=position)
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(position)
    s = Seq(env, cfg, position + 3)
    if position:
        s.fill(rng, position)
    check_decode(env, [s], Step(rng, cfg, 1), [position], table(None))
    s.check()
    check_decode(env, [s], Step(rng, cfg, 1), [position + 1], table(None))
    s.check()


@pytest.mark.parametrize("heads", [(1, 1), (2, 1), (4, 1), (8, 1), (8, 8), (16, 8), (32, 8), (64, 8), (6, 3), (40, 5)])
@pytest.mark.parametrize("rope", [None, YARN, dict(scaling="linear", factor=2.0)], ids=("plain", "yarn", "linear"))
def test_decode_heads(env, heads, rope):
    case(test="decode_heads", heads=heads, rope=rope)
    if (heads[0] * 128) % 256:
        heads = (2 * heads[0], 2 * heads[1])
    E = env["E"]
    cfg = config(env, *heads)
    spec = E.AmdRopeSpec(base=BASE, **rope) if rope else None
    rng = np.random.default_rng(sum(heads))
    lengths = [1, 95, 330]
    seqs = [Seq(env, cfg, n + 40 * i + 1, spec) for i, n in enumerate(lengths)]
    for s, n in zip(seqs, lengths):
        s.fill(rng, n)
    check_decode(env, seqs, Step(rng, cfg, 3), lengths, table(rope))


@pytest.mark.parametrize("members", [1, 2, 8, 9, 17, 64])
def test_decode_members(env, members):
    """Every batch size; up to 8 members a member's bits are its own call's, from 9
    on those of any other batch of that range."""
    case(test="decode_members", members=members)
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(members)
    lengths = [int(n) for n in rng.integers(1, 600, members)]
    seqs = [Seq(env, cfg, 640) for _ in range(members)]
    for s, n in zip(seqs, lengths):
        s.fill(rng, n)
    step = Step(rng, cfg, members)
    got = check_decode(env, seqs, step, lengths, table(None))
    order = list(range(members))[::-1][:9] if members > 8 else [members - 1]
    part = Step(rng, cfg, len(order))
    for a in ("q", "k", "v"):
        setattr(part, a, getattr(step, a)[order])
    part.qn, part.kn = step.qn, step.kn
    again = decode(env, [seqs[i] for i in order], part, [lengths[i] for i in order])
    np.testing.assert_array_equal(again, got[order])


def test_bits_do_not_depend_on_the_other_members_caches(env):
    """Capacities of one chunk, a few and many in one launch, each member as on its own."""
    case(test="capacities")
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(77)
    shape = [(130, 140), (130, 5000), (250, 256), (250, 20000), (700, 701), (700, 12000), (8400, 8500), (8400, 40000)]
    seqs = []
    for n, cap in shape:
        seqs.append(Seq(env, cfg, cap))
        seqs[-1].fill(np.random.default_rng(n), n)  # the same context for equal lengths
    step = Step(rng, cfg, len(shape))
    for i in range(1, len(shape), 2):
        for a in ("q", "k", "v"):
            getattr(step, a)[i] = getattr(step, a)[i - 1]
    lengths = [n for n, _ in shape]
    got = decode(env, seqs, step, lengths)
    for i in range(0, len(shape), 2):
        np.testing.assert_array_equal(got[i], got[i + 1])
    for i, (n, cap) in enumerate(shape):
        one = Step(rng, cfg, 1)
        for a in ("q", "k", "v"):
            setattr(one, a, getattr(step, a)[i:i + 1])
        one.qn, one.kn = step.qn, step.kn
        np.testing.assert_array_equal(decode(env, [seqs[i]], one, [n])[0], got[i])


def test_a_sequence_from_its_start(env):
    """Seventy steps from an empty cache, then back into the latest block, into an
    earlier one, onto a block's first position, and on from there."""
    case(test="sequence")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(1)
    s = Seq(env, cfg, 128)
    path = [*range(70), 66, 67, 68, 69, 70, 70, 40, 41, 42, 63, 64, 32, 33, 31, 32, 0, 1]
    for p in path:
        if p == 63:  # the tokens up to it, so that no position is skipped
            for x in range(43, 63):
                check_decode(env, [s], Step(rng, cfg, 1), [x], table(None))
        check_decode(env, [s], Step(rng, cfg, 1), [p], table(None))
        s.check()


def test_decode_far_positions(env):
    """A context of 131,071 tokens under scaled rope: angles, offsets and the
    merge of the chunks at the far end, and cache offsets past 2^25 bytes a head."""
    case(test="far")
    E = env["E"]
    cfg = config(env, 2, 1)
    rng = np.random.default_rng(4)
    s = Seq(env, cfg, 131072, E.AmdRopeSpec(base=BASE, **YARN))
    # the oracle's cache in whole blocks at once
    k, v = rows(rng, 131071, 1)
    s.cache.write(0, dev(k), dev(v), 0)
    m = s.model[0]
    x = L.half(np.stack([k, v]).transpose(0, 2, 1, 3))
    whole = 131071 // 32
    codes, scale = L.quantise(x[:, :, :whole * 32].reshape(2, 1, whole, 32, 128))
    m.held[:, :, :whole] = codes * scale
    m.tail[:, :, :31] = x[:, :, whole * 32:]
    m.end = 131071
    check_decode(env, [s], Step(rng, cfg, 1), [131071], table(YARN))
    np.testing.assert_array_equal(read(env, s.cache, cfg, 0, 131000, 72), m.rows()[:, :, 131000:])


def test_positions_out_of_range_write_nothing(env):
    """Device positions past the capacity or below 0: the append is dropped, the
    other members are served, a member without tokens gets zeros."""
    case(test="out_of_range")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(8)
    seqs = [Seq(env, cfg, 64) for _ in range(4)]
    for s in seqs[:3]:
        s.fill(rng, 64)
    step = Step(rng, cfg, 4)
    got = decode(env, seqs, step, [64, -1, 10, -5])
    q, k = step.turned([64, -1, 10, -5], table(None))
    for s in seqs[:2]:
        s.check()
    assert max_rel_err(got[0], L.attend(q[0], *seqs[0].model[0].rows())) <= ATTN_TOL
    assert not got[1].any() and not got[3].any()
    seqs[2].model[0].append(10, k[2:3], step.v[2:3])
    assert max_rel_err(got[2], L.attend(q[2], *seqs[2].model[0].rows())) <= ATTN_TOL
    assert not read(env, seqs[3].cache, cfg, 0, 0, 64).any()


def test_the_largest_and_smallest_positions(env):
    """Any int32 may be a position: the largest reads what the cache holds, the smallest is no token."""
    case(test="extreme_positions")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(18)
    seqs = [Seq(env, cfg, 64) for _ in range(2)]
    for s in seqs:
        s.fill(rng, 50)
    step = Step(rng, cfg, 2)
    positions = [2 ** 31 - 1, -2 ** 31]
    got = decode(env, seqs, step, positions)
    for s in seqs:
        s.check()
    # (the query's f32 cosines at 2^31 - 1 are those of 64-bit angles: 2^31 * 2^-53 turns)
    q, _ = step.turned(positions, table(None))
    assert max_rel_err(got[0], L.attend(q[0], *seqs[0].model[0].rows())) <= ATTN_TOL
    assert not got[1].any()


@pytest.mark.parametrize("gain", [1e-18, 1e18])
def test_queries_of_any_size(env, gain):
    """The norm brings q to size; its weight may be anything (here 1e4 times the usual: a softmax of one key)."""
    case(test="q_size", gain=gain)
    cfg = config(env, 4, 1)
    rng = np.random.default_rng(2)
    s = Seq(env, cfg, 200)
    s.fill(rng, 150)
    step = Step(rng, cfg, 1, gain)
    if gain > 1:
        step.qn *= np.float32(1e4)
    q, k = step.turned([150], table(None))
    got = decode(env, [s], step, [150])
    s.model[0].append(150, k, step.v)
    want = L.attend(q[0], *s.model[0].rows())
    if gain > 1:  # scores of 1e5: f32 ones are off by 1e-2, the key they pick is the same
        assert max_rel_err(got[0], want) <= 5e-2
    else:         # the norm's epsilon dominates: q is tiny, the mean of the values
        assert max_rel_err(got[0], want) <= ATTN_TOL


def test_a_query_that_is_not_a_number_stays_alone(env):
    case(test="nan_query")
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(6)
    seqs = [Seq(env, cfg, 100) for _ in range(2)]
    for s in seqs:
        s.fill(rng, 80)
    step = Step(rng, cfg, 2)
    step.q[0, 3, 5] = np.nan
    step.q[1, 6, 0] = np.inf
    step.k[0, 0, 3] = np.nan   # enters the cache as zeros
    step.v[0, 1, 7] = np.inf   # held at 65504
    got = decode(env, seqs, step, [80, 80])
    bad = {(0, 3), (1, 6)}
    for i in range(2):
        for h in range(8):
            assert np.isfinite(got[i, h]).all() == ((i, h) not in bad), (i, h)
    held = read(env, seqs[0].cache, cfg, 0, 0, 81)
    assert np.isfinite(held).all() and not held[0, 0, 80].any() and held[1, 1, 80, 7] == 65504


# --------------------------------------------------------------------- prompt chunks

@pytest.mark.parametrize("tokens,position", [(1, 0), (1, 31), (1, 32), (2, 63), (16, 0), (17, 0), (31, 0), (32, 0), (33, 0), (64, 0),
                                             (100, 0), (37, 20), (12, 20), (11, 20), (130, 95), (200, 33), (96, 32), (5, 500)])
def test_chunks(env, tokens, position):
    case(test="chunks", tokens=tokens, position=position)
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(tokens + 1000 * position)
    s = Seq(env, cfg, position + tokens + 2)
    if position:
        s.fill(rng, position)
    check_prefill(env, s, Step(rng, cfg, tokens), tokens, position, table(None))
    check_decode(env, [s], Step(rng, cfg, 1), [position + tokens], table(None))


@pytest.mark.parametrize("heads", [(2, 2), (4, 2), (8, 2), (16, 2)])
@pytest.mark.parametrize("rope", [None, YARN], ids=("plain", "yarn"))
def test_chunk_heads(env, heads, rope):
    case(test="chunk_heads", heads=heads, rope=rope)
    E = env["E"]
    cfg = config(env, *heads)
    rng = np.random.default_rng(sum(heads))
    s = Seq(env, cfg, 400, E.AmdRopeSpec(base=BASE, **rope) if rope else None)
    s.fill(rng, 77)
    check_prefill(env, s, Step(rng, cfg, 150), 150, 77, table(rope), every=3)
    check_prefill(env, s, Step(rng, cfg, 90), 90, 227, table(rope), every=3)


@pytest.mark.parametrize("heads", [(8, 8), (16, 8), (32, 8), (64, 8)])
def test_chunk_wide_form(env, heads):
    """Enough tokens for the many-token form of every group size, at ragged sizes."""
    case(test="chunk_wide", heads=heads)
    cfg = config(env, *heads)
    rng = np.random.default_rng(sum(heads))
    n = {8: 1100, 16: 1500, 32: 801, 64: 1101}[heads[0]]
    s = Seq(env, cfg, n + 45)
    s.fill(rng, 45)
    check_prefill(env, s, Step(rng, cfg, n), n, 45, table(None), every=97)


def test_chunk_taken_back(env):
    case(test="chunk_back")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(12)
    s = Seq(env, cfg, 300)
    for tokens, position in ((200, 0), (50, 77), (3, 125), (60, 100), (40, 160), (33, 160), (1, 0), (64, 1)):
        check_prefill(env, s, Step(rng, cfg, tokens), tokens, position, table(None), every=7)


# ----------------------------------------------------------------- f16 caches with a rope

@pytest.mark.parametrize("seed", range(6))
def test_a_walk_of_all_calls(env, seed):
    """Steps, chunks and rows in, at the end or somewhere before it, in any order over two sequences and two layers:
    each answer and each cache as the formulas have them."""
    rng = np.random.default_rng(100 + seed)
    q_heads, kv_heads = [(4, 2), (2, 2), (8, 1)][seed % 3]
    cfg = config(env, q_heads, kv_heads, layers=2)
    seqs = [Seq(env, cfg, 260) for _ in range(2)]
    tab = table(None)
    for turn in range(30):
        layer, s = int(rng.integers(2)), seqs[int(rng.integers(2))]
        end = s.model[layer].end
        position = end if end == 0 or rng.random() < 0.6 else int(rng.integers(end))
        room = s.capacity - position
        kind = rng.choice(["step", "both", "chunk", "rows"]) if room else "past"
        n = min(room, int(rng.choice([1, 3, 31, 32, 33, 70])))
        case(test="walk", seed=seed, turn=turn, kind=str(kind), layer=layer, position=position, n=n)
        if kind == "step":
            check_decode(env, [s], Step(rng, cfg, 1), [position], tab, layer)
        elif kind == "both":
            positions = [min(x.model[layer].end, x.capacity - 1) for x in seqs]
            check_decode(env, seqs, Step(rng, cfg, 2), positions, tab, layer)
        elif kind == "chunk":
            check_prefill(env, s, Step(rng, cfg, n), n, position, tab, layer)
        elif kind == "rows":
            k, v = rows(rng, n, kv_heads)
            half = rng.random() < 0.5
            if half:
                k, v = k.astype(np.float16), v.astype(np.float16)
            s.cache.write(layer, dev(k), dev(v), position)
            s.model[layer].append(position, k.astype(np.float32), v.astype(np.float32))
        else:
            got = decode(env, [s], step := Step(rng, cfg, 1), [s.capacity + turn], layer)
            q, _ = step.turned([s.capacity + turn], tab)
            assert max_rel_err(got[0], L.attend(q[0], *s.model[layer].rows())) <= ATTN_TOL
        for x in seqs:
            for i in range(2):
                if x.model[i].end:
                    x.check(i)


@pytest.mark.parametrize("rope", [dict(), YARN], ids=("plain", "yarn"))
def test_f16_cache_with_a_rope(env, rope):
    """Decode, many-member and prompt attention over f16 caches whose angles come
    from a table, far out too. (Their keys are formed in f32: a value next to a
    border may round the other way, 2^-11 of it at most.)"""
    case(test="f16_rope", rope=rope)
    E, torch = env["E"], env["torch"]
    cfg = config(env, 8, 2)
    spec = E.AmdRopeSpec(base=BASE, **rope)
    tab = table(rope or None)
    rng = np.random.default_rng(21)
    far = 30000 if not rope else 120000
    cache = E.AmdKvCache(env["ctx"], cfg, far + 300, rope=spec)
    ctx_k, ctx_v = rows(rng, far, 2)
    ctx_k, ctx_v = ctx_k.astype(np.float16), ctx_v.astype(np.float16)
    cache.write(0, dev(ctx_k), dev(ctx_v), 0)
    held = np.stack([ctx_k, ctx_v]).transpose(0, 2, 1, 3).astype(np.float64)
    for tokens, call in ((1, "decode"), (40, "prefill")):
        step = Step(rng, cfg, tokens)
        pos = held.shape[2] + np.arange(tokens)
        q, k = step.turned(pos, tab)
        out = dev(np.zeros(tokens * 8 * 128, np.float32))
        if call == "decode":
            E.attention_decode(env["ctx"], cfg, [cache], 0, *step.device(), dev(pos.astype(np.int32)), out)
        else:
            E.attention_prefill(env["ctx"], cfg, cache, 0, *step.device(), tokens, int(pos[0]), out)
        torch.cuda.synchronize()
        new = read(env, cache, cfg, 0, int(pos[0]), tokens).astype(np.float64)
        # f32 norm and rotation (8 roundings of 2^-24 of the pair) and one f16 rounding
        assert np.abs(new[0] - k.transpose(1, 0, 2)).max() <= np.abs(k).max() * (2.0 ** -11 + 16 * 2.0 ** -24)
        np.testing.assert_array_equal(new[1], step.v.astype(np.float16).transpose(1, 0, 2).astype(np.float64))
        held = np.concatenate([held, new], 2)
        got = out.cpu().numpy().reshape(tokens, 8, 128)
        for t in {0, tokens // 2, tokens - 1}:
            assert max_rel_err(got[t], L.attend(q[t], *held[:, :, :pos[t] + 1])) <= ATTN_TOL


def test_default_f16_cache_is_what_it_was(env):
    """No options, and F16 without rope: the same bits as ribn_amd_kv_cache_create."""
    case(test="default")
    E = env["E"]
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(31)
    step = Step(rng, cfg, 1)
    outs = []
    for make in range(2):
        cache = E.AmdKvCache(env["ctx"], cfg, 40)
        if make == 0:
            cache.close()
            c = cfg.to_c()
            lib = env["ctx"]._lib
            assert lib.ribn_amd_kv_cache_create(env["ctx"].handle, ctypes.byref(c), 40, ctypes.byref(cache.handle)) == 0
        outs.append(decode(env, [type("S", (), {"cfg": cfg, "cache": cache})()], step, [0]))
    np.testing.assert_array_equal(outs[0], outs[1])


# ------------------------------------------------- streams, graphs, several at once

def test_captured_attention_replays(env):
    """Decode and prompt attention, and the rows' write and read, captured into a
    graph and replayed between eager work: every replay gives the eager call's bits."""
    case(test="capture")
    E, torch = env["E"], env["torch"]
    stream = torch.cuda.Stream()
    ctx = E.AmdContext(0, stream=stream)
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(41)
    k, v = rows(rng, 90, 2)
    step, chunk = Step(rng, cfg, 2), Step(rng, cfg, 37)
    with torch.cuda.stream(stream):
        caches = [E.AmdKvCache(ctx, cfg, 160, format=E.KV_I8) for _ in range(2)]
        kd, vd = dev(k), dev(v)
        back = [torch.zeros_like(kd) for _ in range(2)]
        sd, cd = step.device(), chunk.device()
        pos = dev(np.array([127, 127], np.int32))
        out, cout = dev(np.zeros(2 * 8 * 128, np.float32)), dev(np.zeros(37 * 8 * 128, np.float32))

        def work():
            for c in caches:
                c.write(0, kd, vd, 0)
            for c in caches:
                E.attention_prefill(ctx, cfg, c, 0, *cd, 37, 90, cout)
            E.attention_decode(ctx, cfg, caches, 0, *sd, pos, out)
            caches[1].read(0, 0, *back)

        work()
        stream.synchronize()
        want = [t.clone() for t in (out, cout, *back)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            work()
        for i in range(4):
            for t in (out, cout, *back):
                t.zero_()
            graph.replay()
            stream.synchronize()
            for a, b in zip((out, cout, *back), want):
                assert torch.equal(a, b), i
            work()  # eager work between replays
            stream.synchronize()
            assert torch.equal(out, want[0])
    ctx.synchronize()


def test_two_contexts_at_once(env):
    """Calls on two streams with caches of their own do not touch each other."""
    case(test="two_contexts")
    E, torch = env["E"], env["torch"]
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(43)
    lanes = []
    for i in range(2):
        stream = torch.cuda.Stream()
        ctx = E.AmdContext(0, stream=stream)
        k, v = rows(rng, 500, 2)
        step = Step(rng, cfg, 1)
        cache = E.AmdKvCache(ctx, cfg, 600, format=E.KV_I8)
        lanes.append((stream, ctx, k, v, step, cache, dev(k), dev(v), step.device(), dev(np.array([500], np.int32)),
                      dev(np.zeros(8 * 128, np.float32))))
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, ctx, k, v, step, cache, kd, vd, sd, pos, out in lanes:
            cache.write(0, kd, vd, 0)
            E.attention_decode(ctx, cfg, [cache], 0, *sd, pos, out)
    torch.cuda.synchronize()
    for stream, ctx, k, v, step, cache, kd, vd, sd, pos, out in lanes:
        q, key = step.turned([500], table(None))
        m = L.Kv8(2, 600)
        m.append(0, k, v)
        m.append(500, key, step.v)
        assert max_rel_err(out.cpu().numpy().reshape(8, 128), L.attend(q[0], *m.rows())) <= ATTN_TOL


# ----------------------------------------------------------------------- refusals

def test_refusals(env):
    case(test="refusals")
    E, torch, ctx = env["E"], env["torch"], env["ctx"]
    cfg = config(env, 4, 2)
    i8, f16 = E.AmdKvCache(ctx, cfg, 64, format=E.KV_I8), E.AmdKvCache(ctx, cfg, 64)
    roped = E.AmdKvCache(ctx, cfg, 64, rope=E.AmdRopeSpec(base=BASE))
    assert (i8.format(), f16.format(), roped.format(), i8.capacity()) == (E.KV_I8, E.KV_F16, E.KV_F16, 64)

    def refused(kind, call):
        with pytest.raises(E.AmdModelKernelError) as e:
            call()
        assert e.value.kind == kind, str(e.value)

    refused("Unsupported", lambda: i8.layer(0))
    refused("Unsupported", lambda: f16.tail(0))
    refused("InvalidPlan", lambda: i8.tail(1))
    refused("InvalidArgument", lambda: E.AmdKvCache(ctx, cfg, 64, format=2))
    refused("InvalidPlan", lambda: E.AmdKvCache(ctx, cfg, 0, format=E.KV_I8))
    refused("InvalidPlan", lambda: E.AmdKvCache(ctx, cfg, (1 << 20) + 1, format=E.KV_I8))
    for bad in (dict(layout="interleaved"), dict(rotary_dim=64), dict(head_dim=64), dict(base=0.5)):
        refused("InvalidPlan", lambda: E.AmdKvCache(ctx, cfg, 64, rope=E.AmdRopeSpec(**bad)))

    rng = np.random.default_rng(1)
    step = Step(rng, cfg, 2)
    out, pos = dev(np.zeros(2 * 4 * 128, np.float32)), dev(np.zeros(2, np.int32))

    def attend(caches, config=cfg, o=out):
        E.attention_decode(ctx, config, caches, 0, *step.device(), pos, o)

    refused("InvalidPlan", lambda: attend([i8, f16]))
    refused("InvalidPlan", lambda: attend([f16, roped]))
    refused("InvalidPlan", lambda: attend([i8, i8]))
    refused("OutputLength", lambda: attend([i8]))
    other = E.AmdQwen3Config(**{**cfg.__dict__, "rope_base": 5.0e5})
    one = dev(np.zeros(4 * 128, np.float32))
    refused("InvalidPlan", lambda: attend([i8], other, one))
    refused("InvalidPlan", lambda: attend([roped], other, one))
    refused("InvalidPlan", lambda: E.attention_prefill(ctx, other, i8, 0, *step.device(), 2, 0, out))
    refused("PositionOverflow", lambda: E.attention_prefill(ctx, cfg, i8, 0, *step.device(), 2, 63, out))
    attend([f16], other, one)  # a cache without a rope of its own goes by the call's base, as before

    k = torch.zeros((3, 2, 128), device="cuda:0")
    for call in (i8.write, f16.write):
        refused("PositionOverflow", lambda: call(0, k, k, 62))
        refused("PositionOverflow", lambda: call(0, k, k, 0xffffffff))
        refused("InvalidPlan", lambda: call(1, k, k, 0))
        with pytest.raises(TypeError):
            call(0, k.double(), k.double(), 0)
        with pytest.raises(TypeError):
            call(0, k, k.half(), 0)
        with pytest.raises(ValueError):
            call(0, k, k[:2], 0)
        with pytest.raises(ValueError):
            call(0, k.transpose(0, 1), k.transpose(0, 1), 0)
    lib = ctx._lib
    kp = ctypes.c_void_p(k.data_ptr())
    name = lambda st: E._lib.STATUS_NAMES[st]  # noqa: E731
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i8.handle, 0, 0, 0, kp, kp, 0, 0)) == "InputLength"
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i8.handle, 0, 0, 3, kp, kp, 767, 0)) == "InputLength"
    assert name(lib.ribn_amd_kv_cache_read(ctx.handle, i8.handle, 0, 0, 3, kp, kp, 767, 0)) == "OutputLength"
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i8.handle, 0, 0, 3, kp, kp, 768, 1)) == "InvalidArgument"
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i8.handle, 0, 0, 3, None, kp, 768, 0)) == "InvalidArgument"
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i8.handle, 0, 0, 3, ctypes.c_void_p(k.data_ptr() + 2), kp, 768, 0)) == "InvalidArgument"
    host = np.zeros(768, np.float32)
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i8.handle, 0, 0, 3, host.ctypes.data_as(ctypes.c_void_p), kp, 768, 0)) == "InvalidArgument"


@pytest.mark.parametrize("fmt", ["KV_I8", "KV_F16"])
def test_a_rope_of_another_base_is_refused(env, fmt):
    """The base of a cache's rope is its config's: a spec whose base was left at the default, on a
    model with another one, would turn by angles that no call asks for."""
    case(test="rope_base", fmt=fmt)
    E, ctx = env["E"], env["ctx"]
    cfg = E.AmdQwen3Config(**{**config(env, 4, 2).__dict__, "rope_base": 5.0e5})
    for given in (cfg, E.AmdQwen3Config(**{**cfg.__dict__, "rope": E.AmdRopeSpec(**YARN)})):
        with pytest.raises(E.AmdModelKernelError) as e:
            E.AmdKvCache(ctx, given, 64, format=getattr(E, fmt), rope=None if given.rope else E.AmdRopeSpec(**YARN))
        assert e.value.kind == "InvalidPlan" and "base 1e+06" in str(e.value) and "500000" in str(e.value), str(e.value)
    cache = E.AmdKvCache(ctx, cfg, 64, format=getattr(E, fmt), rope=E.AmdRopeSpec(base=5.0e5, **YARN))
    step = Step(np.random.default_rng(3), cfg, 1)
    out = dev(np.full(4 * 128, np.nan, np.float32))
    E.attention_decode(ctx, cfg, [cache], 0, *step.device(), dev(np.zeros(1, np.int32)), out)
    env["torch"].cuda.synchronize()
    # one key: its value
    assert max_rel_err(out.cpu().numpy().reshape(4, 128), L.half(step.v[0]).astype(np.float64).repeat(2, 0)) <= ATTN_TOL


@pytest.mark.parametrize("fmt", ["KV_I8", "KV_F16"])
def test_rows_of_another_shape_are_refused(env, fmt):
    """[kv_heads][tokens][128], an f16 cache's own layout, has as many values: it is no [tokens][kv_heads][128]."""
    case(test="row_shapes", fmt=fmt)
    E, torch = env["E"], env["torch"]
    cfg = config(env, 4, 2)
    cache = E.AmdKvCache(env["ctx"], cfg, 64, format=getattr(E, fmt))
    for shape in ((2, 6, 128), (6, 256), (6 * 256,), (1, 6, 2, 128), (12, 1, 128), (6, 4, 64)):
        x = torch.ones(shape, device="cuda:0")
        for call in (lambda: cache.write(0, x, x, 0), lambda: cache.read(0, 0, x, x)):
            with pytest.raises(ValueError, match="cache rows are"):
                call()
    x = torch.ones((6, 2, 128), device="cuda:0")
    cache.write(0, x, x, 0)
    y = [torch.zeros_like(x) for _ in range(2)]
    cache.read(0, 0, *y)
    assert all(torch.equal(v, x) for v in y)
