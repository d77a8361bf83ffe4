"""4-bit caches and log probabilities as they are used: the decoder's steps, prompts and generation and the
serving dispatcher over 4-bit caches, log probabilities of its steps, and prompts scored over caches of each format,
against the oracle step with the same cache in 64 bits (oracle/longctx_oracle.py, oracle/logprob_oracle.py).

Bars. While nothing is in 4 bits yet, logits within LOGIT_TOL normwise of the oracle, as the decoder tests over
f16 caches have it. Then CODE_TOL: the GEMVs' sums come in another order than the oracle's, 1e-6 of a value or so. Codes
lie s = 4.1 .. 4.7 deviations / 15 = 0.3 deviations apart, so a value goes to the other code with 2e-6 / 0.3 = 7e-6, 0.12
of a block's 16,384 (two KV heads, keys and values); and a group's lowest or highest value rounds to another f16 with
1e-6 * 2^11 each, 4e-3 a group, 1.5 of a block's 384 groups, whose low or scale then moves by 2^-10: up to 0.015 codes
of each of its 32 or 64 values, of which up to one goes to another code. Two such values a block, then, each off by s. One moves the
outputs of its KV head's four query heads by its probability times s in one dim (a value), or a token's probability by
s |q| / sqrt(128) = 0.026 of itself (a key), 1/32 * 0.3 = 9e-3 deviations both ways; an output's norm is
sqrt(1024 / 32) = 5.7 deviations, so by 9e-3 * sqrt(4) / 5.7 = 3.2e-3 of it. With up to eight of them a layer, two layers, adding up as
squares, and the o projection's share of the residual at most all of it: 3.2e-3 * sqrt(16) = 1.3e-2, doubled for
probabilities that are not all alike.
After a prompt on the prefill matmul (f16 operands: keys and values off by 1e-3 deviations) 1e-3 * 1.5 / 0.3 = 0.5 % of the values have
the other code, a noise of sqrt(0.005) * 0.3 = 0.02 deviations in keys and in values: 0.02 of the probabilities and 0.02
of the outputs, 0.029 of an attention layer's output, of two layers 0.04 of the residual at most; with that path's
own 4e-3: PROMPT_TOL.
A log probability is off by at most twice what the logits are. Equalities (graph replays, batches, the dispatcher against
the decoder, caches after scoring, scores in pieces) are bit for bit.
"""
import numpy as np
import pytest

from engine_amd import serving as S
from oracle import kquant_oracle as O
from oracle import logprob_oracle as P
from oracle import longctx_oracle as L

from .decode_helpers import small_weights
from .gpu_helpers import max_rel_err, to_dev

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-3
CODE_TOL = 2.6e-2
MATMUL_TOL = 4e-3
PROMPT_TOL = 4.5e-2
TINY = dict(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=4608, vocab=2048, rope_base=1.0e6, epsilon=1.0e-6)
YARN = dict(scaling="yarn", factor=4.0, original_context=64)
CAP = 160
# log probabilities from given logits: sums over 2,048 tokens and the result's rounding
EPS, HALF_STEP = 6e-6, 2.0 ** -24


def case(**kw):
    print("CASE", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


@pytest.fixture(scope="module")
def env():
    import torch
    import engine_amd as E
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    ctx = E.AmdContext(0)
    w = small_weights(TINY, 778, centered=True)
    store, handles = E.AmdWeightStore(ctx), {}
    for name, val in w.items():
        if isinstance(val, tuple):
            t, k, n, enc = val
            store.materialize_quantized(name, [k, n], t, enc)
            handles[name] = store.quantized_tensor(name)
        else:
            handles[name] = to_dev(val)
    layers = [{f: handles[f"blk.{l}.{f}"] for f in
               ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down", "attn_norm",
                "attn_q_norm", "attn_k_norm", "ffn_norm")} for l in range(TINY["layers"])]

    def decoder(cfg, members=8, norm=None):
        return E.AmdQwen3Decode(ctx, cfg, handles["token_embd"], handles["output"], handles["output_norm"] if norm is None else norm, layers, members)

    return {"E": E, "ctx": ctx, "w": w, "decoder": decoder, "torch": torch}


def model(env, rope=None):
    E = env["E"]
    spec = E.AmdRopeSpec(**rope) if rope else None
    kw = dict(scaling=rope["scaling"], factor=rope["factor"], original=rope.get("original_context", 0)) if rope else {}
    return E.AmdQwen3Config(**TINY, rope=spec), L.rope_turns(128, TINY["rope_base"], **kw)


def prompt(n, seed=1):
    return [int(t) for t in np.random.default_rng(seed).integers(0, TINY["vocab"], n)]


def same(dec, orc, tol, what):
    err = max_rel_err(dec.copy_logits(0), orc.logits)
    assert err <= tol, (what, err)


def bar(orc):
    return CODE_TOL if orc.caches[0].end >= 32 else LOGIT_TOL


def held(env, cache, end):
    torch = env["torch"]
    out = []
    for l in range(TINY["layers"]):
        rows = [torch.zeros((end, TINY["kv_heads"], 128), device="cuda:0") for _ in range(2)]
        cache.read(l, 0, *rows)
        torch.cuda.synchronize()
        out.append(np.stack([r.cpu().numpy().transpose(1, 0, 2) for r in rows]))
    return np.stack(out)


def caches_agree(env, cache, orc):
    """Against the oracle's: values here and there one code off, and groups whose low or scale is the next f16."""
    for l, m in enumerate(orc.caches):
        want, whole = m.rows(), m.end // 32 * 32
        off = np.abs(held(env, cache, m.end)[l] - want)
        blocks, model_ = (x[:, :, :whole].reshape(2, TINY["kv_heads"], -1, 32, 128) for x in (off, want))
        step = (model_.max((-2, -1), keepdims=True) - model_.min((-2, -1), keepdims=True)) / 15
        assert (blocks <= 1.1 * step).all(), l
        assert 500 * (blocks > step / 16).sum() <= blocks.size, l
        # the f16 rows: an f32 difference of 1e-5 of the largest value, and two roundings, each by up to 2^-11 of a value:
        # where the two sides of a midpoint round apart, a whole step (0.25 at 406)
        assert off[:, :, whole:].size == 0 or off[:, :, whole:].max() <= np.abs(want).max() * (1e-5 + 2 * 2.0 ** -11), l


def agree(got, logits, targets, top):
    """Results against those from `logits` themselves (f32 rows, tokens equal)."""
    given, entropy, order, alternatives = P.logprobs(np.asarray(logits, np.float64), targets, top)
    for have, want in ((got.logprobs, given), (got.top_logprobs, alternatives)):
        if have is None:
            continue
        finite = np.isfinite(want)
        np.testing.assert_array_equal(np.isfinite(have), finite)
        assert (np.abs(have[finite] - want[finite]) <= EPS + HALF_STEP * np.abs(want[finite])).all()
    if got.entropy is not None:
        # (terms under 2^-126 may be none: 2,047 of them, each p (-log p) <= 2^-126 * 88)
        assert (np.abs(got.entropy - entropy) <= (2 * EPS + HALF_STEP) * entropy + 2.2e-33).all()
    if top:
        np.testing.assert_array_equal(got.top_tokens, order)


@pytest.mark.parametrize("rope", [None, YARN], ids=("plain", "yarn"))
def test_steps_follow_the_oracle(env, rope):
    case(test="steps", rope=rope)
    E = env["E"]
    cfg, table = model(env, rope)
    dec = env["decoder"](cfg)
    cache = E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I4)
    orc = L.LongContextQwen3(TINY, env["w"], CAP, table, kind=L.Kv4)
    tokens = prompt(70)
    for p, t in enumerate(tokens):  # past two whole blocks
        dec.decode_step(cache, t, p)
        orc.step(t, p)
        same(dec, orc, bar(orc), p)
    caches_agree(env, cache, orc)
    for p in (52, 53, 54):  # back into the second block, and on
        dec.decode_step(cache, tokens[0], p)
        orc.step(tokens[0], p)
        same(dec, orc, CODE_TOL, ("back", p))


def test_graphs_batches_and_generation(env):
    """Steps captured and replayed, direct ones, members alone and together, generation; and the log probabilities of each."""
    case(test="graphs")
    E = env["E"]
    cfg, _ = model(env, YARN)
    dec, direct = env["decoder"](cfg), env["decoder"](cfg)
    direct.set_graphs(False)
    prompts = [prompt(n, n) for n in (29, 5, 40)]

    def filled():
        caches = [E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I4) for _ in prompts]
        for c, toks in zip(caches, prompts):
            for p, t in enumerate(toks):
                direct.prefill_step(c, t, p)
        return caches

    a, b, alone, gen = filled(), filled(), filled(), filled()
    tokens, lengths = [7, 8, 9], [len(p) for p in prompts]
    feed, seen = list(tokens), []
    for s in range(6):  # across the first sequence's block border
        pos = [n + s for n in lengths]
        x = dec.decode_step_batch(a, feed, pos)
        logits = np.stack([dec.copy_logits(i) for i in range(3)])
        scores = dec.logprobs(3, entropy=True, top=4)
        agree(scores, logits, x, 4)
        np.testing.assert_array_equal(scores.logprobs, scores.top_logprobs[:, 0])
        assert direct.decode_step_batch(b, feed, pos) == x
        np.testing.assert_array_equal(direct.logprobs(3).logprobs, scores.logprobs)
        for i in range(3):
            np.testing.assert_array_equal(direct.copy_logits(i), logits[i])
            assert dec.decode_step(alone[i], feed[i], pos[i]) == x[i]
            np.testing.assert_array_equal(dec.copy_logits(0), logits[i])
        feed = x
        seen.append(x)
    np.testing.assert_array_equal(dec.generate(gen, tokens, lengths, 6), np.array(seen).T)
    agree(dec.logprobs(3), logits, seen[-1], 0)


@pytest.mark.parametrize("start,count", [(0, 7), (25, 7), (28, 8), (30, 5)])
def test_prefill_chunks(env, start, count):
    """A chunk's tokens as members of one step: inside a block the serial steps bit for bit."""
    case(test="prefill_chunk", start=start, count=count)
    E = env["E"]
    cfg, table = model(env)
    dec = env["decoder"](cfg)
    toks = prompt(start + count + 1, 5)
    one, other = (E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I4) for _ in range(2))
    orc = L.LongContextQwen3(TINY, env["w"], CAP, table, kind=L.Kv4)
    for p in range(start):
        dec.prefill_step(one, toks[p], p)
        dec.prefill_step(other, toks[p], p)
        orc.step(toks[p], p, head=False)
    dec.prefill_chunk(one, toks[start:start + count], start)
    orc.chunk(toks[start:start + count], start)
    for p in range(start, start + count):
        dec.prefill_step(other, toks[p], p)
    end = start + count
    if (end - 1) // 32 == start // 32 and end % 32:
        np.testing.assert_array_equal(held(env, one, end), held(env, other, end))
    dec.decode_step(one, toks[end], end)
    orc.step(toks[end], end)
    same(dec, orc, bar(orc), "after the chunk")
    caches_agree(env, one, orc)


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_I8", "KV_I4"])
@pytest.mark.parametrize("chunk", [16, 48, 2048])
@pytest.mark.parametrize("gain", [1.0, 1 / 64], ids=("sharp", "flat"))
def test_prompts_are_scored(env, fmt, chunk, gain):
    """A text's log probabilities, of logits up to some hundreds and of a few; the cache after it; a step after it."""
    case(test="score", fmt=fmt, chunk=chunk, gain=gain)
    E = env["E"]
    cfg, table = model(env, YARN)
    weights = dict(env["w"], output_norm=env["w"]["output_norm"] * np.float32(gain))
    dec = env["decoder"](cfg, norm=to_dev(weights["output_norm"]))
    toks = prompt(91, 6)
    cache, plain = (E.AmdKvCache(env["ctx"], cfg, CAP, format=getattr(E, fmt)) for _ in range(2))
    goal = np.array(toks[1:], np.uint32)
    goal[7] = TINY["vocab"]
    goal[8] = 2 ** 32 - 1
    got = dec.score_prompt(cache, toks[:90], 0, goal, entropy=True, top=5, chunk_tokens=chunk)
    dec.prefill_prompt(plain, toks[:90], 0, chunk)
    np.testing.assert_array_equal(held(env, cache, 90), held(env, plain, 90))
    orc = L.LongContextQwen3(TINY, weights, CAP, table, i8=fmt != "KV_F16", kind=L.Kv4 if fmt == "KV_I4" else L.Kv8)
    logits = []
    for c0 in range(0, 90, chunk):
        orc.chunk(toks[c0:min(c0 + chunk, 90)], c0)
        logits += [orc._gemv("output", O.rms_norm_raw(h, orc.w["output_norm"], TINY["epsilon"])) for h in orc.hiddens]
    logits = np.stack(logits).astype(np.float64)
    tol = {"KV_F16": MATMUL_TOL, "KV_I8": MATMUL_TOL + 6e-3, "KV_I4": PROMPT_TOL}[fmt]
    off = 2 * tol * np.abs(logits).max(1)
    given, entropy, _, alternatives = P.logprobs(logits, goal, 5)
    finite = np.isfinite(given)
    np.testing.assert_array_equal(np.isfinite(got.logprobs), finite)
    assert (np.abs(got.logprobs[finite] - given[finite]) <= off[finite]).all()
    assert (np.abs(got.top_logprobs - alternatives) <= off[:, None]).all()
    # the entropy's derivative by a logit is at most p |log p + H|, over all of them 2 max |log p| <= 2 log(2048 e^(2 max))
    assert (np.abs(got.entropy - entropy) <= off * (np.log(2048) + 2 * np.abs(logits).max(1))).all()
    # each alternative's log probability is its own token's
    back = np.take_along_axis(logits - logits.max(1, keepdims=True), got.top_tokens.astype(np.int64), 1)
    back -= np.log(np.exp(logits - logits.max(1, keepdims=True)).sum(1, keepdims=True))
    assert (np.abs(got.top_logprobs - back) <= off[:, None]).all()
    dec.decode_step(cache, toks[90], 90)
    logits = dec.copy_logits(0)
    dec.decode_step(plain, toks[90], 90)
    np.testing.assert_array_equal(dec.copy_logits(0), logits)
    orc.step(toks[90], 90)
    same(dec, orc, tol, "after")
    agree(dec.logprobs(targets=[5], entropy=True, top=32), logits[None], [5], 32)


@pytest.mark.parametrize("vocab", [1237, 300, 33])
def test_odd_vocabularies(env, vocab):
    """Output matrices whose rows end inside a tile of the prefill matmul, and alternatives of nearly all tokens."""
    case(test="vocab", vocab=vocab)
    E = env["E"]
    geometry = dict(TINY, vocab=vocab, layers=1)
    w = small_weights(geometry, 12, centered=True)
    store, handles = E.AmdWeightStore(env["ctx"]), {}
    for name, val in w.items():
        if isinstance(val, tuple):
            t, k, n, enc = val
            store.materialize_quantized(name, [k, n], t, enc)
            handles[name] = store.quantized_tensor(name)
        else:
            handles[name] = to_dev(val)
    layers = [{f: handles[f"blk.0.{f}"] for f in ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down", "attn_norm",
                                                  "attn_q_norm", "attn_k_norm", "ffn_norm")}]
    cfg = E.AmdQwen3Config(**geometry)
    dec = E.AmdQwen3Decode(env["ctx"], cfg, handles["token_embd"], handles["output"], handles["output_norm"], layers, 2)
    cache = E.AmdKvCache(env["ctx"], cfg, 64)
    toks = [int(t) for t in np.random.default_rng(3).integers(0, vocab, 38)]
    got = dec.score_prompt(cache, toks[:37], 0, toks[1:], entropy=True, top=32)
    orc = L.LongContextQwen3(geometry, w, 64, L.rope_turns(128, TINY["rope_base"]), i8=False)
    orc.chunk(toks[:37], 0)
    logits = np.stack([orc._gemv("output", O.rms_norm_raw(h, orc.w["output_norm"], TINY["epsilon"])) for h in orc.hiddens]).astype(np.float64)
    off = 2 * MATMUL_TOL * np.abs(logits).max(1)
    given, _, _, alternatives = P.logprobs(logits, toks[1:], 32)
    assert (np.abs(got.logprobs - given) <= off).all() and (np.abs(got.top_logprobs - alternatives) <= off[:, None]).all()
    assert (got.top_tokens < vocab).all() and all(len(set(r)) == 32 for r in got.top_tokens.tolist())
    dec.decode_step(cache, toks[37], 37)
    agree(dec.logprobs(targets=[vocab - 1], entropy=True, top=32), dec.copy_logits(0)[None], [vocab - 1], 32)


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_I4"])
def test_scores_in_pieces(env, fmt):
    """Calls that go on from one another are the chunks of one call; what is not asked for changes nothing."""
    case(test="pieces", fmt=fmt)
    E = env["E"]
    cfg, _ = model(env)
    dec = env["decoder"](cfg)
    toks = prompt(97, 4)
    caches = [E.AmdKvCache(env["ctx"], cfg, CAP, format=getattr(E, fmt)) for _ in range(4)]
    whole = dec.score_prompt(caches[0], toks[:96], 0, toks[1:], entropy=True, top=3, chunk_tokens=32)
    for c0 in range(0, 96, 32):
        part = dec.score_prompt(caches[1], toks[c0:c0 + 32], c0, toks[c0 + 1:c0 + 33], entropy=True, top=3)
        for name in ("logprobs", "entropy", "top_tokens", "top_logprobs"):
            np.testing.assert_array_equal(getattr(part, name), getattr(whole, name)[c0:c0 + 32])
    np.testing.assert_array_equal(held(env, caches[0], 96), held(env, caches[1], 96))
    only = dec.score_prompt(caches[2], toks[:96], 0, entropy=True, chunk_tokens=32)
    assert only.logprobs is None and only.top_tokens is None
    np.testing.assert_array_equal(only.entropy, whole.entropy)
    only = dec.score_prompt(caches[3], toks[:96], 0, toks[1:], chunk_tokens=32)
    assert only.entropy is None
    np.testing.assert_array_equal(only.logprobs, whole.logprobs)


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_I4"])
def test_long_prompts(env, fmt):
    """More rows than logits are held of at once; one chunk and several, and a single token."""
    case(test="long", fmt=fmt)
    E = env["E"]
    cfg, _ = model(env)
    dec = env["decoder"](cfg)
    toks = prompt(1101, 2)
    a, b = (E.AmdKvCache(env["ctx"], cfg, 1200, format=getattr(E, fmt)) for _ in range(2))
    one = dec.score_prompt(a, toks[:1100], 0, toks[1:], entropy=True, top=2)
    several = dec.score_prompt(b, toks[:1100], 0, toks[1:], entropy=True, top=2, chunk_tokens=256)
    tol = 2 * (MATMUL_TOL if fmt == "KV_F16" else PROMPT_TOL)
    last = dec.score_prompt(a, toks[1100:], 1100, [3], top=32)
    dec.decode_step(b, toks[1100], 1100)
    logits = dec.copy_logits(0)
    far = 2 * tol * np.abs(logits).max() * 2  # (logits of other rows may be twice as large)
    assert (np.abs(one.logprobs - several.logprobs) <= far).all() and (np.abs(one.top_logprobs - several.top_logprobs) <= far).all()
    # (logits lie hundreds apart: what a certain token leaves the others, e^-88 and less, is 0 in f32)
    assert np.isfinite(one.logprobs).all() and (one.logprobs <= 0).all() and (one.entropy >= 0).all()
    want = P.logprobs(logits[None].astype(np.float64), [3], 32)
    assert abs(last.logprobs[0] - want[0][0]) <= far and (np.abs(last.top_logprobs - want[3]) <= far).all()


def test_scores_between_steps(env):
    """A prompt scored on one cache while another sequence is being decoded, graphs on: the steps are what they were."""
    case(test="between")
    E = env["E"]
    cfg, _ = model(env)
    dec = env["decoder"](cfg)
    a, b, c = (E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I4) for _ in range(3))
    toks = prompt(50, 8)

    def run(cache, between):
        out, t = [], 11
        for p in range(40):
            t = dec.decode_step(cache, t, p)
            out.append((t, dec.copy_logits(0)))
            if between and p % 9 == 4:
                s = dec.score_prompt(c, toks[:40], 0, toks[1:41], top=2)
                scored.append(s)
                np.testing.assert_array_equal(dec.copy_logits(0), out[-1][1])
        return out

    scored = []
    plain, mixed = run(a, False), run(b, True)
    for (t, x), (u, y) in zip(plain, mixed):
        assert t == u
        np.testing.assert_array_equal(x, y)
    for s in scored[1:]:  # the same prompt from position 0 again
        np.testing.assert_array_equal(s.logprobs, scored[0].logprobs)


def test_the_dispatcher(env):
    """Rows over 4-bit states equal direct decoder calls; bytes and reuse count the format."""
    case(test="dispatcher")
    E = env["E"]
    cfg, _ = model(env, YARN)
    dec = env["decoder"](cfg)
    per = S.kv_bytes(cfg, CAP, E.KV_I4)
    # 4,864 bytes for 32 tokens' 16,384, and a 33rd block in f16 whatever the length: here 5 blocks
    assert 4 * (5 * 4864 + 16384) <= per <= 4 * (5 * 4864 + 16384 + 256) < S.kv_bytes(cfg, CAP, E.KV_F16)
    assert 3.3 * S.kv_bytes(cfg, 32768, E.KV_I4) < S.kv_bytes(cfg, 32768, E.KV_F16)
    disp = S.AmdServingDispatcher(dec, 4, kv_budget_bytes=2 * per).with_kv_format(E.KV_I4).with_prompt_prefill(48)
    greedy = S.SamplingParams.greedy()

    def run(state, phase, toks, pos):
        seg = S.ExecutionSegment(request=state.state_id, phase=phase, state_position=pos, token_count=len(toks), tokens=tuple(toks),
                                 sampling=greedy)
        out = disp.dispatch(None, seg, None, state)
        state.token_position = pos + len(toks)
        return out.output_token

    def direct(toks, steps):
        cache = E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I4)
        dec.prefill_prompt(cache, toks[:-1], 0, 48)
        got = [dec.decode_step(cache, toks[-1], len(toks) - 1)]
        for s in range(steps):
            got.append(dec.decode_step(cache, got[-1], len(toks) + s))
        return got

    states = [_state(i + 1) for i in range(2)]
    for st, n in zip(states, (60, 33)):
        toks = prompt(n, n)
        got = [run(st, S.Phase.PREFILL, toks, 0)]
        for s in range(4):
            got.append(run(st, S.Phase.DECODE, [got[-1]], n + s))
        assert got == direct(toks, 4)
    assert disp.state_bytes() == (2 * per, 0)
    third = _state(9)
    with pytest.raises(S.BackendError):
        run(third, S.Phase.PREFILL, prompt(20, 9), 0)   # over the budget
    disp.release_inference_state(states[0])
    assert disp.state_bytes() == (per, per)
    toks = prompt(45, 9)                                # a cache used before
    assert run(third, S.Phase.PREFILL, toks, 0) == direct(toks, 0)[0]


def _state(i):
    return S.InferenceStateSet(state_id=i, kv_tokens=CAP, token_position=None)


def test_refusals(env):
    case(test="refusals")
    E = env["E"]
    cfg, _ = model(env)
    dec = env["decoder"](cfg, 4)
    cache = E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I4)
    toks = prompt(40)
    dec.decode_step(cache, 1, 0)
    logits = dec.copy_logits(0)

    def refused(kind, call, *args, **kw):
        with pytest.raises(E.AmdKernelError) as e:
            call(*args, **kw)
        assert e.value.kind == kind, (kind, e.value.kind, str(e.value))

    score, step = dec.score_prompt, dec.logprobs
    refused("InvalidArgument", score, cache, toks, 0)                            # nothing asked for
    refused("InvalidArgument", score, cache, toks, 0, toks, top=33)
    refused("InputLength", score, cache, [], 0, [])
    refused("InvalidArgument", score, cache, toks, 0, toks, chunk_tokens=15)
    refused("InvalidArgument", score, cache, toks, 0, toks, chunk_tokens=2049)
    refused("PositionOverflow", score, cache, toks, CAP - 39, toks)
    refused("InvalidPlan", score, cache, toks[:5] + [TINY["vocab"]], 0, toks[:6])
    other = E.AmdKvCache(env["ctx"], E.AmdQwen3Config(**{**TINY, "kv_heads": 4}), CAP)
    refused("InvalidPlan", score, other, toks, 0, toks)
    refused("InvalidArgument", step, 1, logprobs=False)
    refused("InvalidArgument", step, 1, targets=[1], logprobs=False, entropy=True)
    refused("InvalidArgument", step, 1, top=33)
    refused("InvalidPlan", step, 5)
    refused("InputLength", step, 0)
    for call in (lambda: score(cache, toks, 0, toks[:3]), lambda: step(2, [1]), lambda: step(1, top=-1), lambda: score(cache, toks, 0, toks, top=4096)):
        with pytest.raises(ValueError):
            call()
    lib, n = dec.ctx._lib, None
    assert lib.ribn_amd_qwen3_logprobs(n, 1, n, n, n, n, n, 0) != 0
    assert lib.ribn_amd_qwen3_score_prompt(n, cache.handle, n, 1, 0, 0, n, n, n, n, n, 0) != 0
    np.testing.assert_array_equal(dec.copy_logits(0), logits)  # nothing ran
    agree(step(1, targets=[TINY["vocab"]], top=1), logits[None], [TINY["vocab"]], 1)


def test_rows_that_no_step_computed_are_refused(env):
    """Log probabilities are of the last step with an output head: of no more members than it had, of none before it."""
    case(test="no_step")
    E = env["E"]
    cfg, _ = model(env)
    dec = env["decoder"](cfg, 4)
    caches = [E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I4) for _ in range(4)]
    toks = prompt(40)

    def have(n):
        got = dec.logprobs(n, entropy=True, top=3) if n else None
        for m in range(n + 1, 5):
            with pytest.raises(E.AmdKernelError) as e:
                dec.logprobs(m, entropy=True, top=3)
            assert e.value.kind == "InvalidPlan", str(e.value)
        if n:
            agree(got, np.stack([dec.copy_logits(i) for i in range(n)]), got.top_tokens[:, 0], 3)

    have(0)
    dec.prefill_step(caches[0], toks[0], 0)
    dec.prefill_chunk(caches[0], toks[1:4], 1)
    dec.prefill_prompt(caches[0], toks[4:20], 4)
    dec.score_prompt(caches[0], toks[20:39], 20, toks[21:40])
    have(0)
    dec.decode_step(caches[0], toks[39], 39)
    have(1)
    dec.decode_step_batch(caches[1:], [1, 2, 3], [0, 0, 0])
    have(3)
    dec.prefill_chunk(caches[0], [4, 5, 6, 7], 40)  # (no output head)
    have(3)
    dec.set_graphs(False)
    dec.decode_step_batch(caches[1:3], [1, 2], [1, 1])
    have(2)
    with pytest.raises(E.AmdKernelError):
        dec.decode_step_batch(caches, [1, 2, 3, 4], [44, 2, 2, CAP])  # refused before anything runs
    have(2)
    dec.generate(caches, [1, 2, 3, 4], [44, 2, 2, 1], 3)
    have(4)
    dec.decode_step(caches[0], 1, 47)
    have(1)


# ------------------------------------------- scored prompts by their whole distributions

WHOLE = dict(TINY, vocab=32)  # as many tokens as there are alternatives: every token's log probability of every row
FLAT = np.float32(1 / 64)     # of the output norm: logits up to 9, entropies of 0.1 to 2.7


@pytest.fixture(scope="module")
def whole(env):
    E = env["E"]
    w = small_weights(WHOLE, 12, centered=True)
    w["output_norm"] = w["output_norm"] * FLAT
    store, handles = E.AmdWeightStore(env["ctx"]), {}
    for name, val in w.items():
        if isinstance(val, tuple):
            t, k, n, enc = val
            store.materialize_quantized(name, [k, n], t, enc)
            handles[name] = store.quantized_tensor(name)
        else:
            handles[name] = to_dev(val)
    layers = [{f: handles[f"blk.{l}.{f}"] for f in ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down", "attn_norm",
                                                    "attn_q_norm", "attn_k_norm", "ffn_norm")} for l in range(WHOLE["layers"])]
    cfg = E.AmdQwen3Config(**WHOLE)
    return cfg, w, E.AmdQwen3Decode(env["ctx"], cfg, handles["token_embd"], handles["output"], handles["output_norm"], layers, 2)


def distributions(got, targets):
    """[rows][tokens] log probabilities, all of which the alternatives are. What was given of targets is among them bit for bit;
    they add up to 1; and the entropy is theirs: each is off by eps = EPS and a rounding, p log p by p |log p + 1| eps at
    most, the entropy itself by 2 EPS and a rounding."""
    lp = np.full(got.top_tokens.shape, np.nan)
    np.put_along_axis(lp, got.top_tokens.astype(np.int64), got.top_logprobs.astype(np.float64), 1)
    assert np.isfinite(lp).all()
    np.testing.assert_array_equal(got.logprobs, lp[np.arange(len(lp)), targets].astype(np.float32))
    eps = EPS + HALF_STEP * np.abs(lp).max(1)
    p = np.exp(lp)
    assert (np.abs(p.sum(1) - 1) <= eps * (1 + eps)).all()
    h = -(p * lp).sum(1)
    assert (np.abs(got.entropy - h) <= (h + 1) * eps * (1 + eps) + (2 * EPS + HALF_STEP) * h).all()
    return lp


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_I8", "KV_I4"])
@pytest.mark.parametrize("chunk", [16, 48, 2048])
def test_scores_are_whole_distributions(env, whole, fmt, chunk):
    """Every row against the oracle's, whose neighbouring rows are further apart than the bars: with logits off by d, a log
    probability is off by 2 d, and the entropy log Z - sum p x by 2 d + (e^2d - 1) sum p |x - sum p x|, since no p changes by
    more than e^2d."""
    case(test="whole", fmt=fmt, chunk=chunk)
    E = env["E"]
    cfg, w, dec = whole
    toks = [int(t) for t in np.random.default_rng(6).integers(0, 32, 91)]
    cache = E.AmdKvCache(env["ctx"], cfg, CAP, format=getattr(E, fmt))
    got = dec.score_prompt(cache, toks[:90], 0, toks[1:], entropy=True, top=32, chunk_tokens=chunk)
    lp = distributions(got, toks[1:])
    orc = L.LongContextQwen3(WHOLE, w, CAP, L.rope_turns(128, WHOLE["rope_base"]), i8=fmt != "KV_F16", kind=L.Kv4 if fmt == "KV_I4" else L.Kv8)
    x = []
    for c0 in range(0, 90, chunk):
        orc.chunk(toks[c0:min(c0 + chunk, 90)], c0)
        x += [orc._gemv("output", O.rms_norm_raw(h, orc.w["output_norm"], WHOLE["epsilon"])) for h in orc.hiddens]
    x = np.stack(x).astype(np.float64)
    _, entropy, order, alternatives = P.logprobs(x, None, 32)
    want = np.empty_like(x)
    np.put_along_axis(want, order, alternatives, 1)
    d = {"KV_F16": MATMUL_TOL, "KV_I8": MATMUL_TOL + 6e-3, "KV_I4": PROMPT_TOL}[fmt] * np.abs(x).max(1)
    assert (np.abs(lp - want) <= 2 * d[:, None]).all()
    assert (np.abs(want[1:] - want[:-1]).max(1) > 4 * d[1:]).mean() > 0.9
    p = np.exp(want)
    bound = 2 * d + np.expm1(2 * d) * (p * np.abs(x - (p * x).sum(1, keepdims=True))).sum(1)
    assert (np.abs(got.entropy - entropy) <= bound).all()
    if fmt == "KV_F16":
        assert (np.abs(entropy[1:] - entropy[:-1]) > 2 * bound[1:]).mean() > 0.7


@pytest.mark.parametrize("fmt", ["KV_F16", "KV_I4"])
def test_rows_past_the_first_logits(env, whole, fmt):
    """1,100 rows, of which logits are held of 1,024 at once, against the same text by 256 (one group a chunk). A row's
    largest |logit| is no more than its log probabilities' span, logits of both signs being there; two calls' are
    off by 2 tol of it each. Neighbouring rows are further apart."""
    case(test="past_1024", fmt=fmt)
    E = env["E"]
    cfg, _, dec = whole
    toks = [int(t) for t in np.random.default_rng(16).integers(0, 32, 1101)]
    caches = [E.AmdKvCache(env["ctx"], cfg, 1200, format=getattr(E, fmt)) for _ in range(3)]
    one = dec.score_prompt(caches[0], toks[:1100], 0, toks[1:], entropy=True, top=32)
    several = dec.score_prompt(caches[1], toks[:1100], 0, toks[1:], entropy=True, top=32, chunk_tokens=256)
    a, b = distributions(one, toks[1:]), distributions(several, toks[1:])
    far = 4 * (MATMUL_TOL if fmt == "KV_F16" else PROMPT_TOL) * (b.max(1) - b.min(1))
    assert (np.abs(a - b).max(1) <= far).all()
    assert (np.abs(b[1:] - b[:-1]).max(1) > far[1:]).mean() > (0.9 if fmt == "KV_F16" else 0.5)
    only = dec.score_prompt(caches[2], toks[:1100], 0, entropy=True)
    np.testing.assert_array_equal(only.entropy, one.entropy)
