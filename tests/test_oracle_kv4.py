"""CPU tests of the 4-bit cache's definition (oracle/longctx_oracle.py), of what it costs, and of
the library's host-side answers about it."""
import ctypes

import numpy as np
import pytest

import engine_amd as E
from engine_amd import _lib, serving
from oracle import longctx_oracle as L


def blocks(rng, n=40):
    gain = np.where(rng.random(128) > 0.97, 6.0, 0.5 + rng.random(128))
    mean = rng.standard_normal(128) * (rng.random(128) < 0.25)
    return L.half(rng.standard_normal((n, 32, 128)) * gain + mean)


@pytest.mark.parametrize("keys", [True, False], ids=("keys", "values"))
def test_groups_scales_and_codes(keys):
    """By loops over groups, from the definition: the scale in f32 cut off to f16, codes, values in lo .. hi."""
    x = blocks(np.random.default_rng(1), 6)
    codes, s, lo = L.quantise4(x, keys)
    held = L.values4(codes, s, lo)
    for b in range(len(x)):
        groups = [x[b, :, d] for d in range(128)] if keys else [x[b, t, 64 * h:64 * h + 64] for t in range(32) for h in range(2)]
        got = [held[b, :, d] for d in range(128)] if keys else [held[b, t, 64 * h:64 * h + 64] for t in range(32) for h in range(2)]
        for g, have in zip(groups, got):
            low, high = g.min(), g.max()
            wide = np.float32(np.float32(high) - np.float32(low)) * np.float32(1 / 15)
            step = np.float16(wide)
            if np.float32(step) > wide:
                step = np.nextafter(step, np.float16(0))
            assert np.float32(step) <= wide and np.float32(np.nextafter(step, np.float16(np.inf))) > wide
            c = np.clip(np.rint((np.float32(g) - np.float32(low)) * (np.float32(1) / np.float32(step))), 0, 15)
            want = np.float16(c.astype(np.float64) * float(step) + float(low))
            np.testing.assert_array_equal(have, want.astype(np.float64))
            assert have.min() == low and have.max() <= high
            # half a step, what the cut leaves of fifteen (15 units of 2^-11 relative, for the codes at the top) and an f16 rounding
            bound = 0.5 * float(step) + 15 * float(step) * 2.0 ** -10 + np.abs(g).max() * 2.0 ** -11
            assert np.abs(have - g).max() <= bound


def test_values_at_the_edges():
    """Constant groups, the whole range of f16, its smallest values: finite, inside the group's range."""
    x = np.zeros((6, 32, 128), np.float16)
    x[1] = 3.14
    x[2, ::2], x[2, 1::2], x[2, :, 1::2] = 65504, -65504, -65504
    x[2, :, ::4] = 65504
    x[3] = 2.0 ** -24 * np.random.default_rng(2).integers(-20, 21, (32, 128))
    x[4, :, 5] = 65504
    x[5] = -0.0
    for keys in (True, False):
        codes, s, lo = L.quantise4(x, keys)
        held = L.values4(codes, s, lo)
        assert np.isfinite(held).all() and np.abs(held).max() <= 65504
        np.testing.assert_array_equal(held[[0, 1, 5]], x[[0, 1, 5]].astype(np.float64))
        axis = -2 if keys else -1
        assert (held.max(axis) <= x.astype(np.float64).max(axis)).all() and (held.min(axis) >= x.astype(np.float64).min(axis)).all()


@pytest.mark.parametrize("wide", [False, True], ids=("even", "wide"))
def test_what_four_bits_cost(wide):
    """Attention over what the codes stand for against the values themselves, 3,008 random tokens, without and with a few
    key channels six times as wide. A value is off by s / sqrt(12) rms but for the group's lowest (and nearly its highest):
    a score (q of rms 1) by as much in nats, a relative error of each weight and so of their mean of random values; the
    values' own error adds in squares. (The mean over 8 seeds: a score's error within 3%, an output's within 15%. Errors of a
    quarter of a nat are no small ones: the weights' rise as exp's, sqrt(exp(e^2) - 1) of it.)"""
    off, base, scores, step_k, step_v = [], [], [], [], []
    for seed in range(8):
        rng = np.random.default_rng(seed)
        r = rng.random(128)
        gain = np.where(r > 0.97, 6.0, 0.5 + r) if wide else 0.5 + r
        k, v = rng.standard_normal((1, 3008, 128)) * gain, 0.5 * rng.standard_normal((1, 3008, 128))
        q = rng.standard_normal((8, 128))
        q /= np.sqrt((q * q).mean(-1, keepdims=True))
        held = []
        for i, (x, steps, group) in enumerate(((k, step_k, 32), (v, step_v, 64))):
            codes, s, lo = L.quantise4(L.half(x).reshape(1, -1, 32, 128), i == 0)
            held.append(L.values4(codes, s, lo).reshape(1, 3008, 128))
            steps.append((s ** 2).mean() / 12 * (group - 2) / group)
        want = L.attend(q, k, v)
        off.append(((L.attend(q, *held) - want) ** 2).mean())
        base.append((want ** 2).mean())
        scores.append((((held[0] - k)[0] @ q.T / np.sqrt(128.0)) ** 2).mean())
    score, output = np.sqrt(np.mean(scores)), np.sqrt(np.mean(off) / np.mean(base))
    expect = np.sqrt(np.mean(step_k))
    assert abs(score / expect - 1) <= 0.03, (score, expect)
    expect = np.sqrt(np.exp(np.mean(step_k)) - 1 + np.mean(step_v) / 0.25)
    assert abs(output / expect - 1) <= 0.15, (output, expect)
    assert 0.10 < output < 0.14 if not wide else 0.12 < output < 0.20, output


def test_bytes_and_formats():
    cfg = E.AmdQwen3Config()
    for tokens, blocks_ in ((1, 1), (32, 1), (33, 2), (131072, 4096)):
        region = -(-(blocks_ * 4864 + 16384 + 4) // 256) * 256
        assert serving.kv_bytes(cfg, tokens, E.KV_I4) == 36 * 8 * region
    assert serving.kv_bytes(cfg, (1 << 20) + 1, E.KV_I4) == 0
    for unknown in (2, 3, 5, 7, 0xffffffff):
        assert serving.kv_bytes(cfg, 32, unknown) == 0
    assert len({E.KV_F16, E.KV_I8, E.KV_I4}) == 3
    lib = _lib.load()
    assert lib.ribn_amd_kv_cache_format(None) == E.KV_F16
    out = ctypes.c_void_p()
    options = _lib.KvOptions(E.KV_I4, None)
    assert lib.ribn_amd_kv_cache_create_with(None, ctypes.byref(cfg.to_c()), 32, ctypes.byref(options), ctypes.byref(out)) != 0
    assert not out
