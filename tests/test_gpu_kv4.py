"""GPU tests of the KV cache in 4 bits, through the public entry points, against
oracle/longctx_oracle.py (64 bits, numpy). As for the 8-bit cache (test_gpu_kv8.py, whose helpers and whose derivation of
ATTN_TOL these are): what a cache holds is compared for equality, attention within ATTN_TOL
normwise, since the attention's own arithmetic is the same and the cache's values are the oracle's."""
import ctypes

import numpy as np
import pytest

from oracle import longctx_oracle as L
from . import test_gpu_kv8 as K8
from .gpu_helpers import max_rel_err
from .test_gpu_kv8 import ATTN_TOL, BASE, EPS, YARN, Step, case, check_decode, check_prefill, config, decode, dev, read, rows, table

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import engine_amd as E
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return {"E": E, "ctx": E.AmdContext(0), "torch": torch}


class Seq(K8.Seq):
    def __init__(self, env, cfg, capacity, rope=None):
        self.env, self.cfg, self.capacity = env, cfg, capacity
        self.cache = env["E"].AmdKvCache(env["ctx"], cfg, capacity, format=env["E"].KV_I4, rope=rope)
        self.model = [L.Kv4(cfg.kv_heads, capacity) for _ in range(cfg.layers)]


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
    """Infinities, NaN, the largest and smallest f16, the whole of its range in a group, constant groups, ties, zeros, one
    large value among small ones."""
    case(test="edges")
    cfg = config(env, 2, 1)
    rng = np.random.default_rng(3)
    x = np.zeros((10, 32, 1, 128), np.float32)
    x[1, 0, 0, :4] = (np.inf, -np.inf, np.nan, 1.0)
    x[2] = 65504.0 * np.sign(rng.standard_normal((32, 1, 128)))
    x[3] = 2.0 ** -24 * rng.integers(-20, 21, (32, 1, 128))
    x[4] = rng.integers(0, 31, (32, 1, 128)) * 0.5   # halves of a step where a group has 0 and 15
    x[5] = rng.standard_normal((32, 1, 128)) * 1e-3
    x[5, 7, 0, 9] = 1000.0
    x[6] = 1000.0 + 0.5 * rng.integers(0, 2, (32, 1, 128))
    x[7] = -0.0
    x[8] = 1e30
    x[9] = 65504.0 * rng.integers(0, 2, (32, 1, 128))
    s = Seq(env, cfg, 10 * 32)
    k, v = x.reshape(-1, 1, 128), x[::-1].reshape(-1, 1, 128)
    for n in (10 * 32 - 5, 10 * 32):  # the last block in f16, then in 4 bits
        s.cache.write(0, dev(k[:n]), dev(v[:n]), 0)
        s.model[0].append(0, k[:n], v[:n])
        s.check()
    # attention over such a cache is finite
    step = Step(rng, cfg, 1)
    big = Seq(env, cfg, 10 * 32 + 1)
    big.cache.write(0, dev(k), dev(v), 0)
    assert np.isfinite(decode(env, [big], step, [10 * 32])).all()


def test_steps_and_writes_quantise_alike(env):
    """A block's 32nd row by a step of decode attention: the codes of a write."""
    case(test="alike")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(30)
    s = Seq(env, cfg, 64)
    k, v = rows(rng, 31, 2)
    s.cache.write(0, dev(k), dev(v), 0)
    s.model[0].append(0, k, v)
    step = Step(rng, cfg, 1)
    step.v *= np.float32(1000)
    check_decode(env, [s], step, [31], table(None))
    s.check()


def test_skipped_tokens_are_finite(env):
    """A call past the end: what the tokens skipped read is undefined, and finite."""
    case(test="skipped")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(31)
    junk = [env["torch"].full((1 << 20,), float("nan"), device="cuda:0") for _ in range(8)]
    del junk
    s = Seq(env, cfg, 4000)
    assert np.isfinite(decode(env, [s], Step(rng, cfg, 1), [3700])).all()
    out = K8.prefill(env, s, Step(rng, cfg, 40), 40, 3900)
    assert np.isfinite(out).all()


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


@pytest.mark.parametrize("heads", [(2, 2), (4, 2), (4, 1), (8, 1), (8, 8), (16, 8), (32, 8), (64, 8), (6, 3), (40, 5)])
@pytest.mark.parametrize("rope", [None, YARN, dict(scaling="linear", factor=2.0)], ids=("plain", "yarn", "linear"))
def test_decode_heads(env, heads, rope):
    case(test="decode_heads", heads=heads, rope=rope)
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


@pytest.mark.parametrize("heads", [(2, 2), (4, 2), (8, 2), (16, 2)])
def test_steps_that_fill_blocks(env, heads):
    """Members whose new token is a block's last, among others, in caches with room for just that and for more; the codes
    they leave, and the next steps over these."""
    case(test="fill", heads=heads)
    cfg = config(env, *heads)
    rng = np.random.default_rng(heads[0])
    lengths = [31, 63, 30, 511, 255, 1023, 31]
    seqs = [Seq(env, cfg, n + room) for n, room in zip(lengths, (4, 200, 3, 4, 900, 4, 2000))]
    for s, n in zip(seqs, lengths):
        s.fill(rng, n)
    for step in range(3):
        check_decode(env, seqs, Step(rng, cfg, len(seqs)), [n + step for n in lengths], table(None))
        for s in seqs:
            s.check()
    full = Seq(env, cfg, 32)
    full.fill(rng, 31)
    check_decode(env, [full], Step(rng, cfg, 1), [31], table(None))
    full.check()


def test_a_cache_of_one_token(env):
    case(test="one")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(8)
    s = Seq(env, cfg, 1)
    check_decode(env, [s], Step(rng, cfg, 1), [0], table(None))
    s.check()
    t = Seq(env, cfg, 1)
    check_prefill(env, t, Step(rng, cfg, 1), 1, 0, table(None))
    t.check()


def test_a_sequence_from_its_start(env):
    """Seventy steps from an empty cache, then back into the latest block, into an
    earlier one, onto a block's first position, and on from there."""
    case(test="sequence")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(1)
    s = Seq(env, cfg, 128)
    path = [*range(70), 66, 67, 68, 69, 70, 70, 40, 41, 42, *range(43, 65), 32, 33, 31, 32, 0, 1]
    for p in path:
        check_decode(env, [s], Step(rng, cfg, 1), [p], table(None))
        s.check()


def test_decode_far_positions(env):
    """A context of 131,071 tokens under scaled rope: angles, offsets and the merge of the chunks at the far end."""
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
    m.held[:, :, :whole] = L.Kv4.stored(x[:, :, :whole * 32].reshape(2, 1, whole, 32, 128))
    m.tail[:, :, :31] = x[:, :, whole * 32:]
    m.end = 131071
    check_decode(env, [s], Step(rng, cfg, 1), [131071], table(YARN))
    np.testing.assert_array_equal(read(env, s.cache, cfg, 0, 131000, 72), m.rows()[:, :, 131000:])


def test_the_largest_cache(env):
    """The largest capacity: a region's blocks lie past 2^27 bytes, its last block's tokens where a position says."""
    case(test="largest")
    cfg = config(env, 2, 1)
    rng = np.random.default_rng(5)
    cap = 1 << 20
    s = Seq(env, cfg, cap)
    k, v = rows(rng, 70, 1)
    s.cache.write(0, dev(k), dev(v), cap - 70)
    got = read(env, s.cache, cfg, 0, cap - 70, 70)
    m = L.Kv4(1, 96)  # the last three blocks
    pad = np.zeros((26, 1, 128), np.float32)
    m.append(0, np.concatenate([pad, k]), np.concatenate([pad, v]))
    np.testing.assert_array_equal(got, m.rows()[:, :, 26:])


def test_positions_out_of_range_write_nothing(env):
    """Device positions past the capacity or below 0: the append is dropped, the
    other members are served, a member without tokens gets zeros. Any int32 is a position."""
    case(test="out_of_range")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(8)
    seqs = [Seq(env, cfg, 64) for _ in range(6)]
    for i in (0, 1, 2, 4):
        seqs[i].fill(rng, 64)
    step = Step(rng, cfg, 6)
    positions = [64, -1, 10, -5, 2 ** 31 - 1, -2 ** 31]
    got = decode(env, seqs, step, positions)
    q, k = step.turned(positions, table(None))
    for i in (0, 1, 4):
        seqs[i].check()
    for i in (0, 4):
        assert max_rel_err(got[i], L.attend(q[i], *seqs[i].model[0].rows())) <= ATTN_TOL
    assert not got[1].any() and not got[3].any() and not got[5].any()
    seqs[2].model[0].append(10, k[2:3], step.v[2:3])
    assert max_rel_err(got[2], L.attend(q[2], *seqs[2].model[0].rows())) <= ATTN_TOL
    assert not read(env, seqs[3].cache, cfg, 0, 0, 64).any()


def test_what_is_not_a_number_stays_out(env):
    case(test="nan")
    cfg = config(env, 8, 2)
    rng = np.random.default_rng(6)
    seqs = [Seq(env, cfg, 100) for _ in range(2)]
    for s in seqs:
        s.fill(rng, 95)
    step = Step(rng, cfg, 2)
    step.q[0, 3, 5] = np.nan
    step.q[1, 6, 0] = np.inf
    step.k[0, 0, 3] = np.nan   # enters the cache as zeros
    step.v[0, 1, 7] = np.inf   # held at 65504
    got = decode(env, seqs, step, [95, 95])  # (the block is whole then)
    bad = {(0, 3), (1, 6)}
    for i in range(2):
        for h in range(8):
            assert np.isfinite(got[i, h]).all() == ((i, h) not in bad), (i, h)
    q, k = step.turned([95, 95], table(None))
    seqs[0].model[0].append(95, k[:1], step.v[:1])
    seqs[0].check()
    assert np.isfinite(read(env, seqs[0].cache, cfg, 0, 0, 96)).all()


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


@pytest.mark.parametrize("tokens,position", [(700, 0), (650, 3), (641, 31), (672, 32), (690, 100)])
def test_chunk_wide_ends(env, tokens, position):
    """The many-token form where the prompt's last block ends at every place of a pair of blocks."""
    case(test="chunk_wide_ends", tokens=tokens, position=position)
    cfg = config(env, 16, 8)
    rng = np.random.default_rng(tokens)
    s = Seq(env, cfg, position + tokens + 1)
    if position:
        s.fill(rng, position)
    check_prefill(env, s, Step(rng, cfg, tokens), tokens, position, table(None), every=53)


def test_chunk_taken_back(env):
    case(test="chunk_back")
    cfg = config(env, 4, 2)
    rng = np.random.default_rng(12)
    s = Seq(env, cfg, 300)
    for tokens, position in ((200, 0), (50, 77), (3, 125), (60, 100), (40, 160), (33, 160), (1, 0), (64, 1)):
        check_prefill(env, s, Step(rng, cfg, tokens), tokens, position, table(None), every=7)


@pytest.mark.parametrize("seed", range(6))
def test_a_walk_of_all_calls(env, seed):
    """Steps, chunks and rows in, at the end or somewhere before it, in any order over two sequences and two layers:
    each answer and each cache as the formulas have them."""
    rng = np.random.default_rng(200 + seed)
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
        caches = [E.AmdKvCache(ctx, cfg, 160, format=E.KV_I4) for _ in range(2)]
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
        cache = E.AmdKvCache(ctx, cfg, 600, format=E.KV_I4)
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
        m = L.Kv4(2, 600)
        m.append(0, k, v)
        m.append(500, key, step.v)
        assert max_rel_err(out.cpu().numpy().reshape(8, 128), L.attend(q[0], *m.rows())) <= ATTN_TOL


# ----------------------------------------------------------------------- refusals

def test_refusals(env):
    case(test="refusals")
    E, torch, ctx = env["E"], env["torch"], env["ctx"]
    cfg = config(env, 4, 2)
    i4, i8, f16 = (E.AmdKvCache(ctx, cfg, 64, format=f) for f in (E.KV_I4, E.KV_I8, E.KV_F16))
    assert (i4.format(), i8.format(), f16.format(), i4.capacity()) == (E.KV_I4, E.KV_I8, E.KV_F16, 64)

    def refused(kind, call):
        with pytest.raises(E.AmdModelKernelError) as e:
            call()
        assert e.value.kind == kind, str(e.value)

    refused("Unsupported", lambda: i4.layer(0))
    refused("InvalidPlan", lambda: i4.tail(1))
    refused("InvalidPlan", lambda: i4.layer(1))
    for unknown in (2, 3, 5, 1000):
        refused("InvalidArgument", lambda: E.AmdKvCache(ctx, cfg, 64, format=unknown))
    refused("InvalidPlan", lambda: E.AmdKvCache(ctx, cfg, 0, format=E.KV_I4))
    refused("InvalidPlan", lambda: E.AmdKvCache(ctx, cfg, (1 << 20) + 1, format=E.KV_I4))
    for bad in (dict(layout="interleaved"), dict(rotary_dim=64), dict(head_dim=64), dict(base=0.5)):
        refused("InvalidPlan", lambda: E.AmdKvCache(ctx, cfg, 64, format=E.KV_I4, rope=E.AmdRopeSpec(**bad)))

    rng = np.random.default_rng(1)
    step = Step(rng, cfg, 2)
    out, pos = dev(np.zeros(2 * 4 * 128, np.float32)), dev(np.zeros(2, np.int32))

    def attend(caches, config=cfg, o=out):
        E.attention_decode(ctx, config, caches, 0, *step.device(), pos, o)

    refused("InvalidPlan", lambda: attend([i4, i8]))
    refused("InvalidPlan", lambda: attend([f16, i4]))
    refused("InvalidPlan", lambda: attend([i4, i4]))
    refused("OutputLength", lambda: attend([i4]))
    other = E.AmdQwen3Config(**{**cfg.__dict__, "rope_base": 5.0e5})
    one = dev(np.zeros(4 * 128, np.float32))
    refused("InvalidPlan", lambda: attend([i4], other, one))
    refused("InvalidPlan", lambda: E.attention_prefill(ctx, other, i4, 0, *step.device(), 2, 0, out))
    refused("PositionOverflow", lambda: E.attention_prefill(ctx, cfg, i4, 0, *step.device(), 2, 63, out))

    k = torch.zeros((3, 2, 128), device="cuda:0")
    refused("PositionOverflow", lambda: i4.write(0, k, k, 62))
    refused("PositionOverflow", lambda: i4.read(0, 62, k, k))
    refused("InvalidPlan", lambda: i4.write(1, k, k, 0))
    with pytest.raises(TypeError):
        i4.write(0, k.double(), k.double(), 0)
    with pytest.raises(ValueError):
        i4.write(0, k, k[:2], 0)
    lib = ctx._lib
    kp = ctypes.c_void_p(k.data_ptr())
    name = lambda st: E._lib.STATUS_NAMES[st]  # noqa: E731
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i4.handle, 0, 0, 0, kp, kp, 0, 0)) == "InputLength"
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i4.handle, 0, 0, 3, kp, kp, 767, 0)) == "InputLength"
    assert name(lib.ribn_amd_kv_cache_read(ctx.handle, i4.handle, 0, 0, 3, kp, kp, 767, 0)) == "OutputLength"
    assert name(lib.ribn_amd_kv_cache_write(ctx.handle, i4.handle, 0, 0, 3, kp, kp, 768, 1)) == "InvalidArgument"
    assert EPS and not read(env, i4, cfg, 0, 0, 64).any()  # nothing was written
