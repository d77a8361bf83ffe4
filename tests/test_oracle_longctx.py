"""CPU checks of the long-context operators: the 64-bit oracle against itself
written another way, the host-only frequency table against the oracle, and
every refusal that needs no device."""
import ctypes
import math

import numpy as np
import pytest

import engine_amd as E
from engine_amd import _lib
from engine_amd.gguf import GgufError, GgufFile
from engine_amd import gguf_writer as W
from oracle import longctx_oracle as L

SPECS = [dict(), dict(rotary_dim=64), dict(head_dim=80, rotary_dim=22, layout="interleaved", base=1.0e4),
         dict(scaling="linear", factor=8.0), dict(scaling="linear", factor=0.5),
         dict(scaling="yarn", factor=4.0, original_context=32768),
         dict(scaling="yarn", factor=4.0, original_context=32768, attention_factor=1.25),
         dict(scaling="yarn", factor=40.0, original_context=4096, beta_fast=16.0, beta_slow=2.0, base=1.0e4, rotary_dim=96),
         dict(scaling="yarn", factor=1.0, original_context=7),
         dict(freq_factors=tuple(1.0 + 0.125 * i for i in range(64)), scaling="linear", factor=2.0)]


def oracle_table(spec):
    rotary = spec.rotary_dim or spec.head_dim
    return L.rope_turns(rotary, spec.base, spec.scaling, spec.factor, spec.original_context, spec.beta_fast, spec.beta_slow,
                        spec.attention_factor, spec.freq_factors)


@pytest.mark.parametrize("kw", SPECS, ids=str)
def test_frequencies_are_the_oracles(kw):
    spec = E.AmdRopeSpec(**kw)
    turns, gain = E.rope_frequencies(spec)
    want, want_gain = oracle_table(spec)
    assert len(turns) == len(want)
    # both sides in 64 bits: a power, a product and a quotient or two apart
    np.testing.assert_allclose(turns, want, rtol=16 * 2.0 ** -53)
    assert math.isclose(gain, want_gain, rel_tol=4 * 2.0 ** -53)


def test_yarn_keeps_fast_pairs_and_stretches_slow_ones():
    plain, _ = E.rope_frequencies(E.AmdRopeSpec())
    yarn, gain = E.rope_frequencies(E.AmdRopeSpec(scaling="yarn", factor=4.0, original_context=32768))
    ratio = np.array(plain) / np.array(yarn)
    assert ratio[0] == 1.0 and abs(ratio[-1] - 4.0) < 1e-12 and np.all(np.diff(ratio) >= -1e-12)
    turned = np.array(plain) * 32768  # turns of a pair within the trained length
    assert np.all(ratio[turned > 64] == 1.0) and np.all(np.abs(ratio[turned < 0.5] - 4.0) < 1e-12)
    assert abs(gain - (0.1 * math.log(4.0) + 1.0)) < 1e-15


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(head_dim=3, rotary_dim=2), dict(head_dim=1026), dict(rotary_dim=130),
                                dict(rotary_dim=0), dict(rotary_dim=7), dict(base=1.0), dict(base=-2.0),
                                dict(base=float("inf")), dict(base=float("nan")), dict(scaling="linear", factor=0.0),
                                dict(scaling="linear", factor=float("nan")), dict(scaling="yarn", factor=float("inf"), original_context=8),
                                dict(scaling="yarn", factor=2.0), dict(scaling="yarn", factor=2.0, original_context=8, beta_slow=0.0),
                                dict(scaling="yarn", factor=2.0, original_context=8, beta_fast=1.0),
                                dict(scaling="yarn", factor=2.0, original_context=8, beta_fast=float("inf")),
                                dict(attention_factor=-1.0), dict(attention_factor=float("nan")),
                                dict(freq_factors=(0.0,) * 64), dict(freq_factors=(1.0,) * 63 + (float("inf"),))], ids=str)
def test_bad_specs_are_invalid_plans(kw):
    with pytest.raises(E.AmdModelKernelError) as e:
        E.rope_frequencies(E.AmdRopeSpec(**kw))
    assert e.value.kind == "InvalidPlan"


def test_unknown_names_and_factor_counts():
    for kw in (dict(layout="third"), dict(scaling="other"), dict(freq_factors=(1.0,) * 63)):
        with pytest.raises(ValueError):
            E.AmdRopeSpec(**kw).to_c()
    lib = _lib.load()
    spec = E.AmdRopeSpec().to_c()
    turns, gain = (ctypes.c_double * 64)(), ctypes.c_double()
    assert _lib.STATUS_NAMES[lib.ribn_amd_rope_frequencies(None, turns, 64, ctypes.byref(gain))] == "InvalidArgument"
    assert _lib.STATUS_NAMES[lib.ribn_amd_rope_frequencies(ctypes.byref(spec), None, 64, ctypes.byref(gain))] == "InvalidArgument"
    assert _lib.STATUS_NAMES[lib.ribn_amd_rope_frequencies(ctypes.byref(spec), turns, 63, ctypes.byref(gain))] == "OutputLength"
    for field, bad in (("layout", 2), ("scaling", 3)):
        spec = E.AmdRopeSpec().to_c()
        setattr(spec, field, bad)
        assert _lib.STATUS_NAMES[lib.ribn_amd_rope_frequencies(ctypes.byref(spec), turns, 64, ctypes.byref(gain))] == "InvalidPlan"


def test_null_handles_are_refused():
    lib = _lib.load()
    cfg, p = E.QWEN3_8B.to_c(), ctypes.c_void_p()
    name = lambda st: _lib.STATUS_NAMES[st]  # noqa: E731
    spec, rows = E.AmdRopeSpec().to_c(), _lib.RopeRows()
    options = _lib.KvOptions(1, None)
    n = ctypes.c_size_t()
    assert name(lib.ribn_amd_rope_create(None, ctypes.byref(spec), ctypes.byref(p))) == "InvalidArgument"
    assert name(lib.ribn_amd_rope_execute(None, None, 1, ctypes.byref(rows), 1, 0)) == "InvalidArgument"
    assert name(lib.ribn_amd_kv_cache_create_with(None, ctypes.byref(cfg), 8, ctypes.byref(options), ctypes.byref(p))) == "InvalidArgument"
    assert name(lib.ribn_amd_kv_cache_tail(None, 0, ctypes.byref(p), ctypes.byref(p), ctypes.byref(n))) == "InvalidArgument"
    assert name(lib.ribn_amd_kv_cache_write(None, None, 0, 0, 1, None, None, 0, 0)) == "InvalidArgument"
    assert name(lib.ribn_amd_kv_cache_read(None, None, 0, 0, 1, None, None, 0, 0)) == "InvalidArgument"
    assert name(lib.ribn_amd_serving_set_kv_options(None, ctypes.byref(options))) == "InvalidArgument"
    assert lib.ribn_amd_kv_cache_format(None) == 0
    lib.ribn_amd_rope_destroy(None)


def test_cache_bytes():
    lib = _lib.load()
    cfg = E.QWEN3_8B.to_c()
    assert lib.ribn_amd_kv_bytes(ctypes.byref(cfg), 1000, 0) == lib.ribn_amd_qwen3_kv_bytes(ctypes.byref(cfg), 1000)
    for tokens in (1, 32, 33, 4096, 1 << 20):
        blocks = -(-tokens // 32)
        region = blocks * 8192 + 16384 + blocks * 8 + 4
        assert lib.ribn_amd_kv_bytes(ctypes.byref(cfg), tokens, 1) == 36 * 8 * (-(-region // 256) * 256)
    # half an f16 cache's bytes, and the scales and the block in f16 beside them
    assert lib.ribn_amd_kv_bytes(ctypes.byref(cfg), 32768, 1) < 0.51 * lib.ribn_amd_kv_bytes(ctypes.byref(cfg), 32768, 0)
    assert lib.ribn_amd_kv_bytes(ctypes.byref(cfg), 8, 2) == 0 and lib.ribn_amd_kv_bytes(None, 8, 1) == 0
    assert lib.ribn_amd_kv_bytes(ctypes.byref(cfg), (1 << 20) + 1, 1) == 0


def test_oracle_cache_taken_back_keeps_its_values():
    rng = np.random.default_rng(5)
    c = L.Kv8(1, 256)
    x = rng.standard_normal((2, 200, 1, 128))
    c.append(0, *x)
    before = c.rows()
    assert before.shape == (2, 1, 200, 128)
    # within 0.5 of a step of 2^e <= max / 64, and in f16 past the last whole block
    step = np.abs(x[0, :192, 0]).reshape(6, 32 * 128).max(1)
    assert np.all(np.abs(before[0, 0, :192].reshape(6, -1) - x[0, :192, 0].reshape(6, -1)).max(1) <= step / 64 * 0.51)
    np.testing.assert_array_equal(before[:, 0, 192:], x[:, 192:, 0].astype(np.float32).astype(np.float16))
    # the same token again: nothing moves; back into a whole block: its values stay, and go to
    # the same codes when it is whole again
    c.append(199, x[0, 199:], x[1, 199:])
    np.testing.assert_array_equal(c.rows(), before)
    c.append(40, before[0, 0, 40:64][:, None], before[1, 0, 40:64][:, None])
    np.testing.assert_array_equal(c.rows(), before[:, :, :64])


def test_codes_at_the_edges():
    x = np.zeros((7, 32, 128), np.float16)
    x[1, 0, 0] = 65504
    x[2, 3, 5] = 2.0 ** -24
    x[3, 0, :4] = (127.0, -126.5, 0.5, 1.5)          # ties go to even
    x[4, 0, :2] = (127.75, -127.75)                  # past the largest code
    x[5, 0, :2] = (128.0, 1.0)
    x[6] = L.half(np.full((32, 128), np.inf))
    codes, scale = L.quantise(x)
    values = codes * scale
    assert not values[0].any() and values[1, 0, 0] == 127 * 512.0 and values[2, 3, 5] == 2.0 ** -24
    assert list(values[3, 0, :4]) == [127, -126, 0, 2]
    assert list(values[4, 0, :2]) == [127, -127] and list(values[5, 0, :2]) == [128, 0]
    assert np.all(values == values.astype(np.float16))
    assert list(L.half(np.array([np.nan, np.inf, -1e9, 65519.9]))) == [0, 65504, -65504, 65504]


def gguf_file(tmp_path, extra, tensors=()):
    md = [("general.architecture", W.STRING, "qwen3"), ("qwen3.block_count", W.U32, 1),
          ("qwen3.embedding_length", W.U32, 512), ("qwen3.feed_forward_length", W.U32, 768),
          ("qwen3.attention.head_count", W.U32, 4), ("qwen3.attention.head_count_kv", W.U32, 2),
          ("qwen3.attention.key_length", W.U32, 128), *extra]
    path = tmp_path / "m.gguf"
    path.write_bytes(W.build(md, [("token_embd.weight", [512, 2], 12, bytes(2 * 2 * 144)), *tensors]))
    return GgufFile.open(str(path))


def test_gguf_rope_scaling(tmp_path):
    key = "qwen3.rope.scaling."
    assert E.qwen3_config_from_gguf(gguf_file(tmp_path, [])).rope is None
    assert E.qwen3_config_from_gguf(gguf_file(tmp_path, [(key + "type", W.STRING, "none")])).rope is None
    cfg = E.qwen3_config_from_gguf(gguf_file(tmp_path, [(key + "type", W.STRING, "yarn"), (key + "factor", W.F32, 4.0),
                                                        (key + "original_context_length", W.U32, 32768)]))
    assert cfg.rope == E.AmdRopeSpec(scaling="yarn", factor=4.0, original_context=32768) and cfg.to_c().rope_base == 1.0e6
    cfg = E.qwen3_config_from_gguf(gguf_file(tmp_path, [("qwen3.rope.freq_base", W.F32, 5.0e5), (key + "type", W.STRING, "linear"),
                                                        (key + "factor", W.F32, 2.0)]))
    assert cfg.rope == E.AmdRopeSpec(base=5.0e5, scaling="linear", factor=2.0)
    for extra, kind in (([(key + "type", W.STRING, "longrope")], "MetadataTypeMismatch"),
                        ([(key + "type", W.STRING, "linear")], "MissingMetadata"),
                        ([(key + "type", W.STRING, "yarn"), (key + "factor", W.F32, 4.0)], "MissingMetadata")):
        with pytest.raises(GgufError) as e:
            E.qwen3_config_from_gguf(gguf_file(tmp_path, extra))
        assert e.value.kind == kind


def test_gguf_rope_betas_and_factors(tmp_path):
    key = "qwen3.rope.scaling."
    yarn = [(key + "type", W.STRING, "yarn"), (key + "factor", W.F32, 4.0), (key + "original_context_length", W.U32, 32768)]
    cfg = E.qwen3_config_from_gguf(gguf_file(tmp_path, yarn + [(key + "yarn_beta_fast", W.F32, 16.0), (key + "yarn_beta_slow", W.F32, 2.0)]))
    assert cfg.rope == E.AmdRopeSpec(scaling="yarn", factor=4.0, original_context=32768, beta_fast=16.0, beta_slow=2.0)
    with pytest.raises(GgufError) as e:  # a key that would change the angles
        E.qwen3_config_from_gguf(gguf_file(tmp_path, yarn + [(key + "attn_factor", W.F32, 2.0)]))
    assert e.value.kind == "MetadataTypeMismatch"
    factors = tuple(float(1 + i % 8) for i in range(64))
    cfg = E.qwen3_config_from_gguf(gguf_file(tmp_path, [], [("rope_freqs.weight", [64], 0, W.f32_payload(factors))]))
    assert cfg.rope == E.AmdRopeSpec(freq_factors=factors)
    turns, gain = E.rope_frequencies(cfg.rope)
    plain, _ = E.rope_frequencies(E.AmdRopeSpec())
    np.testing.assert_allclose(turns, np.array(plain) / factors, rtol=1e-15)
    assert gain == 1.0
    with pytest.raises(GgufError):
        E.qwen3_config_from_gguf(gguf_file(tmp_path, [], [("rope_freqs.weight", [32], 0, W.f32_payload(factors[:32]))]))


def test_gguf_rope_factor_without_a_type(tmp_path):
    """A factor without a type is a linear one, under its older name too; keys that are not known are
    refused whether a type is there or not, and type none leaves the rope unscaled whatever stands beside it."""
    key = "qwen3.rope.scaling."
    factor, old = (key + "factor", W.F32, 4.0), ("qwen3.rope.scale_linear", W.F32, 2.0)
    linear = lambda f, **kw: E.AmdRopeSpec(scaling="linear", factor=f, **kw)  # noqa: E731
    rope = lambda extra, tensors=(): E.qwen3_config_from_gguf(gguf_file(tmp_path, extra, tensors)).rope  # noqa: E731
    assert rope([factor]) == linear(4.0)
    assert rope([old]) == linear(2.0)
    assert rope([factor, old]) == linear(4.0)
    assert rope([factor, (key + "original_context_length", W.U32, 32768), (key + "finetuned", W.BOOL, True)]) == linear(4.0)
    assert rope([(key + "type", W.STRING, "linear"), old]) == linear(2.0)
    assert rope([(key + "type", W.STRING, "yarn"), old, (key + "original_context_length", W.U32, 32768)]) == \
        E.AmdRopeSpec(scaling="yarn", factor=2.0, original_context=32768)
    none = (key + "type", W.STRING, "none")
    for extra in ([(key + "factor", W.F32, 1.0)], [(key + "factor", W.F32, 0.0)], [(key + "original_context_length", W.U32, 32768)],
                  [none, factor, old, (key + "attn_factor", W.F32, 2.0)]):
        assert rope(extra) is None, extra
    factors = tuple(float(1 + i % 8) for i in range(64))
    assert rope([factor], [("rope_freqs.weight", [64], 0, W.f32_payload(factors))]) == linear(4.0, freq_factors=factors)
    for extra in ([(key + "attn_factor", W.F32, 2.0)], [factor, (key + "attn_factor", W.F32, 2.0)],
                  [factor, (key + "original_context_length", W.U32, 32768), (key + "yarn_ext_factor", W.F32, 1.0)]):
        with pytest.raises(GgufError) as e:
            rope(extra)
        assert e.value.kind == "MetadataTypeMismatch"


@pytest.mark.parametrize("wide", [False, True])
def test_what_eight_bits_cost(wide):
    """Attention over what the codes stand for against the values themselves, 3,008 random tokens, without and
    with a few key channels six times as wide. A value is off by 2^e / sqrt(12) rms, independently of the others: a
    score (q of rms 1) by as much in nats, a relative error of each weight and so, where all weights are
    small, of their mean of random values; the values' own error adds in squares. (rms over 8 heads x 128 dims
    x 8 seeds: the two agree within 15%. A score's error is a mean over 190,000, within 2%.)"""
    off, base, scores, step_k, step_v = [], [], [], [], []
    for seed in range(8):
        rng = np.random.default_rng(seed)
        r = rng.random(128)
        gain = np.where(r > 0.97, 6.0, 0.5 + r) if wide else 0.5 + r
        k, v = rng.standard_normal((1, 3008, 128)) * gain, 0.5 * rng.standard_normal((1, 3008, 128))
        q = rng.standard_normal((8, 128))
        q /= np.sqrt((q * q).mean(-1, keepdims=True))
        held = []
        for x, steps in ((k, step_k), (v, step_v)):
            codes, scale = L.quantise(L.half(x).reshape(1, -1, 32, 128))
            held.append((codes * scale).reshape(1, 3008, 128))
            steps.append((scale ** 2).mean() / 12)
        want = L.attend(q, k, v)
        off.append(((L.attend(q, *held) - want) ** 2).mean())
        base.append((want ** 2).mean())
        scores.append((((held[0] - k)[0] @ q.T / np.sqrt(128.0)) ** 2).mean())
    score, output = np.sqrt(np.mean(scores)), np.sqrt(np.mean(off) / np.mean(base))
    expect = np.sqrt(np.mean(step_k))
    assert abs(score / expect - 1) <= 0.02, (score, expect)
    expect = np.sqrt(np.mean(step_k) + np.mean(step_v) / 0.25)
    assert abs(output / expect - 1) <= 0.15, (output, expect)
    assert 0.05 < output < 0.08 if wide else 0.018 < output < 0.025, output
