"""The long-context operators as they are used: the decoder, prompt prefill and the
serving dispatcher over caches in 8 bits and under scaled rope, against the oracle
step with the same cache and rope in 64 bits (oracle/longctx_oracle.py).

Bars: logits of a step within LOGIT_TOL normwise of the oracle, as the decoder tests over f16
caches have it, while nothing is in 8 bits yet. From a first whole block on,
CODE_TOL: the GEMVs' sums come in another order than the oracle's, 1e-6 of a value
or so, and a value that near to the border between two codes goes to the other one.
Borders lie 2^e >= a / 128 apart, a about 4 standard deviations of the values, so one in
1e-6 / (4 / 128) / 2 = 2e-5 .. 6e-5 does: about one of a block's 16,384 (two KV heads, keys
and values). Such a value moves the outputs of its KV head's four query heads in one dim by
its probability times 2^e <= a / 64, 1/32 * 4 / 64 = 2e-3 deviations; an output
vector's norm is sqrt(1024 / 32) = 5.7 deviations, so by 2e-3 * sqrt(4) / 5.7 = 7e-4 of it. With up
to eight of them a layer, two layers, adding up as squares, and the o projection's
share of the residual at most all of it: 7e-4 * sqrt(16) = 2.8e-3, doubled for
probabilities that are not all alike. The caches themselves are compared too: at
most one value in 500 differs from the oracle's, by one code.
After a prompt on the prefill matmul PROMPT_TOL, that path's own bar, and the
same on top (its f16 operands are 2^-11 apart: every code may move by one, a
relative 1 / 128 / sqrt(12) noise of keys and values, averaged over 90 tokens: 1e-3).
Equalities (graph replays, batches, chunks inside a block, the dispatcher
against the decoder) are bit for bit.
"""
import numpy as np
import pytest

from engine_amd import serving as S
from oracle import longctx_oracle as L

from .decode_helpers import small_weights
from .gpu_helpers import max_rel_err, to_dev

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-3
CODE_TOL = 6e-3
PROMPT_TOL = 4e-3 + CODE_TOL
TINY = dict(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, ffn=4608, vocab=2048, rope_base=1.0e6, epsilon=1.0e-6)
YARN = dict(scaling="yarn", factor=4.0, original_context=64)
CAP = 160


def case(**kw):
    print("CASE", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


@pytest.fixture(scope="module")
def env():
    import torch
    import engine_amd as E
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    ctx = E.AmdContext(0)
    w = small_weights(TINY, 777, centered=True)
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

    def decoder(cfg, members=8):
        return E.AmdQwen3Decode(ctx, cfg, handles["token_embd"], handles["output"], handles["output_norm"], layers, members)

    return {"E": E, "ctx": ctx, "w": w, "decoder": decoder, "torch": torch}


def model(env, rope=None):
    """The config under a rope, and the oracle's table of it."""
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
    return CODE_TOL if orc.i8 and orc.caches[0].end >= 32 else LOGIT_TOL


def caches_agree(env, cache, orc):
    """The 8-bit cache against the oracle's: equal but for a value here and there that is one code off."""
    torch = env["torch"]
    for l, model in enumerate(orc.caches):
        want = model.rows()
        whole = model.end // 32 * 32
        rows = [torch.zeros((model.end, TINY["kv_heads"], 128), device="cuda:0") for _ in range(2)]
        cache.read(l, 0, *rows)
        torch.cuda.synchronize()
        got = np.stack([r.cpu().numpy().transpose(1, 0, 2) for r in rows]).astype(np.float64)
        off = np.abs(got - want)
        blocks = off[:, :, :whole].reshape(2, TINY["kv_heads"], -1, 32, 128)
        step = np.abs(want[:, :, :whole]).reshape(blocks.shape).max((-2, -1), keepdims=True) / 64
        assert (blocks <= step).all() and 500 * (blocks > 0).sum() <= blocks.size, l
        # the f16 rows: an f32 difference of 1e-5 of the largest value, and a rounding of 2^-11
        assert off[:, :, whole:].size == 0 or off[:, :, whole:].max() <= np.abs(want).max() * (1e-5 + 2.0 ** -11), l


@pytest.mark.parametrize("i8", [True, False], ids=("i8", "f16"))
@pytest.mark.parametrize("rope", [None, YARN, dict(scaling="linear", factor=2.0)], ids=("plain", "yarn", "linear"))
def test_steps_follow_the_oracle(env, i8, rope):
    case(test="steps", i8=i8, rope=rope)
    E = env["E"]
    cfg, table = model(env, rope)
    dec = env["decoder"](cfg)
    cache = E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I8 if i8 else E.KV_F16)
    orc = L.LongContextQwen3(TINY, env["w"], CAP, table, i8)
    tokens = prompt(40)
    for p, t in enumerate(tokens):  # past the first whole block
        got = dec.decode_step(cache, t, p)
        want = orc.step(t, p)
        same(dec, orc, bar(orc), p)
        top = np.sort(orc.logits)[-2:]
        if top[1] - top[0] > 4 * bar(orc) * np.abs(orc.logits).max():
            assert got == want, p
    if i8:
        caches_agree(env, cache, orc)
    # back into the first block, and on
    for p in (20, 21, 22):
        dec.decode_step(cache, tokens[0], p)
        orc.step(tokens[0], p)
        same(dec, orc, CODE_TOL if i8 else LOGIT_TOL, ("back", p))


def test_graphs_batches_and_generation(env):
    case(test="graphs")
    E = env["E"]
    cfg, _ = model(env, YARN)
    dec, direct = env["decoder"](cfg), env["decoder"](cfg)
    direct.set_graphs(False)
    prompts = [prompt(n, n) for n in (29, 5, 40)]

    def filled():
        caches = [E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I8) for _ in prompts]
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
        logits = [dec.copy_logits(i) for i in range(3)]
        assert direct.decode_step_batch(b, feed, pos) == x
        for i in range(3):
            np.testing.assert_array_equal(direct.copy_logits(i), logits[i])
            assert dec.decode_step(alone[i], feed[i], pos[i]) == x[i]
            np.testing.assert_array_equal(dec.copy_logits(0), logits[i])
        feed = x
        seen.append(x)
    np.testing.assert_array_equal(dec.generate(gen, tokens, lengths, 6), np.array(seen).T)


def test_kinds_of_cache_side_by_side(env):
    """One decoder, graphs on: f16, 8-bit and roped caches in turn, each its own answers."""
    case(test="kinds")
    E = env["E"]
    plain, _ = model(env)
    spec = E.AmdRopeSpec(**YARN)
    dec = env["decoder"](plain)
    kinds = (dict(), dict(format=E.KV_I8), dict(rope=spec), dict(format=E.KV_I8, rope=spec))
    caches = [E.AmdKvCache(env["ctx"], plain, CAP, **kw) for kw in kinds]
    tables = [(model(env)[1], kw.get("format") == E.KV_I8) if "rope" not in kw else (model(env, YARN)[1], kw.get("format") == E.KV_I8) for kw in kinds]
    oracles = [L.LongContextQwen3(TINY, env["w"], CAP, t, i8) for t, i8 in tables]
    for p, t in enumerate(prompt(34, 3)):
        for c, o in zip(caches, oracles):
            dec.decode_step(c, t, p)
            if p >= 31 or p < 2:
                o.step(t, p)
                same(dec, o, bar(o), p)
            else:
                o.step(t, p, head=False)
    with pytest.raises(E.AmdKernelError) as e:
        dec.decode_step_batch(caches[:2], [1, 1], [34, 34])
    assert e.value.kind == "InvalidPlan"


@pytest.mark.parametrize("start,count", [(0, 7), (3, 8), (25, 7), (28, 8), (31, 2), (30, 5)])
def test_prefill_chunks(env, start, count):
    """A chunk's tokens as members of one step. Inside a block it is the serial
    steps bit for bit; over a border its tokens see the border's block in 8 bits."""
    case(test="prefill_chunk", start=start, count=count)
    E = env["E"]
    cfg, table = model(env)
    dec = env["decoder"](cfg)
    toks = prompt(start + count + 1, 5)
    one, other = (E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I8) for _ in range(2))
    orc = L.LongContextQwen3(TINY, env["w"], CAP, table)
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
        rows = [[env["torch"].zeros((end, 2, 128), device="cuda:0") for _ in range(2)] for _ in range(2)]
        for l in range(TINY["layers"]):
            one.read(l, 0, *rows[0])
            other.read(l, 0, *rows[1])
            env["torch"].cuda.synchronize()
            assert all(env["torch"].equal(x, y) for x, y in zip(*rows))
    dec.decode_step(one, toks[end], end)
    orc.step(toks[end], end)
    same(dec, orc, bar(orc), "after the chunk")
    caches_agree(env, one, orc)


@pytest.mark.parametrize("rope", [None, YARN], ids=("plain", "yarn"))
@pytest.mark.parametrize("chunk", [16, 48, 2048])
def test_prompts(env, rope, chunk):
    case(test="prompt", rope=rope, chunk=chunk)
    E = env["E"]
    cfg, table = model(env, rope)
    dec = env["decoder"](cfg)
    toks = prompt(91, 6)
    cache = E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I8)
    dec.prefill_prompt(cache, toks[:90], 0, chunk)
    dec.decode_step(cache, toks[90], 90)
    orc = L.LongContextQwen3(TINY, env["w"], CAP, table)
    for c0 in range(0, 90, chunk):
        orc.chunk(toks[c0:min(c0 + chunk, 90)], c0)
    orc.step(toks[90], 90)
    same(dec, orc, PROMPT_TOL, "prompt")


def test_the_dispatcher(env):
    """Eager and queued rows over 8-bit states equal direct decoder calls; bytes
    and reuse count the format; the format is fixed while states live."""
    case(test="dispatcher")
    E = env["E"]
    cfg, _ = model(env, YARN)
    dec = env["decoder"](cfg)
    per = S.kv_bytes(cfg, CAP, E.KV_I8)
    disp = S.AmdServingDispatcher(dec, 4, kv_budget_bytes=2 * per).with_kv_format(E.KV_I8).with_prompt_prefill(48)
    greedy = S.SamplingParams.greedy()

    def run(state, phase, toks, pos):
        seg = S.ExecutionSegment(request=state.state_id, phase=phase, state_position=pos, token_count=len(toks), tokens=tuple(toks),
                                 sampling=greedy)
        out = disp.dispatch(None, seg, None, state)
        state.token_position = pos + len(toks)
        return out.output_token

    def direct(toks, steps):
        cache = E.AmdKvCache(env["ctx"], cfg, CAP, format=E.KV_I8)
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
    with pytest.raises(S.BackendError):
        disp.with_kv_format(E.KV_F16)
    third = _state(9)
    with pytest.raises(S.BackendError):
        run(third, S.Phase.PREFILL, prompt(20, 9), 0)   # over the budget
    disp.release_inference_state(states[0])
    assert disp.state_bytes() == (per, per)
    toks = prompt(45, 9)                                # a cache used before
    assert run(third, S.Phase.PREFILL, toks, 0) == direct(toks, 0)[0]
    assert disp.state_bytes() == (2 * per, 0)
    for st in (states[1], third):
        disp.release_inference_state(st)
    disp.with_kv_format(E.KV_F16)
    assert disp.state_bytes() == (0, 0)
    fresh = _state(11)
    run(fresh, S.Phase.PREFILL, prompt(20, 2), 0)
    assert disp.state_bytes() == (S.kv_bytes(cfg, CAP, E.KV_F16), 0)


def test_a_config_with_a_rope_reaches_the_dispatchers_caches(env):
    case(test="config_rope")
    E = env["E"]
    cfg, _ = model(env, YARN)
    dec = env["decoder"](cfg)
    disp = S.AmdServingDispatcher(dec, 2)
    toks = prompt(70, 8)
    cache = E.AmdKvCache(env["ctx"], cfg, CAP)
    for p, t in enumerate(toks[:-1]):
        dec.prefill_step(cache, t, p)
    want = dec.decode_step(cache, toks[-1], 69)
    logits = dec.copy_logits(0)
    seg = S.ExecutionSegment(request=1, phase=S.Phase.PREFILL, state_position=0, token_count=70, tokens=tuple(toks),
                             sampling=S.SamplingParams.greedy())
    assert disp.dispatch(None, seg, None, _state(1)).output_token == want
    np.testing.assert_array_equal(dec.copy_logits(0), logits)


def test_the_dispatcher_refuses_a_rope_of_another_base(env):
    case(test="dispatcher_base")
    E = env["E"]
    dec = env["decoder"](model(env)[0])
    disp = S.AmdServingDispatcher(dec, 2)
    with pytest.raises(S.BackendError) as e:
        disp.with_kv_format(E.KV_I8, E.AmdRopeSpec(base=5.0e5, **YARN))
    assert "base 500000" in str(e.value), str(e.value)
    toks = prompt(40, 3)  # the caches are as they were: f16, unscaled
    seg = S.ExecutionSegment(request=1, phase=S.Phase.PREFILL, state_position=0, token_count=40, tokens=tuple(toks),
                             sampling=S.SamplingParams.greedy())
    disp.dispatch(None, seg, None, _state(1))
    assert disp.state_bytes() == (S.kv_bytes(dec.config, CAP, E.KV_F16), 0)


def _state(i):
    return S.InferenceStateSet(state_id=i, kv_tokens=CAP, token_position=None)
