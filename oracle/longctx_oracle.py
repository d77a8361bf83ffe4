"""Plain 64-bit forms of the long-context operators -- TEST INFRASTRUCTURE ONLY.

  rope_turns / rope     rotary positions: layouts, part of the head, scalings
  Kv8                   one layer's KV cache in 8 bits, appended token by token
  attend                softmax attention over given keys and values
  LongContextQwen3      the oracle decode step (qwen3_oracle) with such a cache,
                        or an f16 one, and any rope

numpy float64 throughout, from the definitions in include/ribn_amd.h.
"""
from __future__ import annotations

import numpy as np

from . import kquant_oracle as O
from .qwen3_oracle import OracleQwen3

BLOCK = 32
HEAD = 128


def rope_turns(rotary, base, scaling="none", factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0, attention_factor=0.0,
               freq_factors=None):
    """(turns a position adds to each pair's angle, gain). Parameters as the f32 values the C struct holds."""
    f32 = lambda v: float(np.float32(v))  # noqa: E731
    base, factor = f32(base), f32(factor)
    i = np.arange(rotary // 2, dtype=np.float64)
    f = base ** (-2.0 * i / rotary)
    gain = 1.0
    if freq_factors is not None:
        f = f / np.asarray(freq_factors, np.float32).astype(np.float64)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        lo, hi = (rotary * np.log(original / (2 * np.pi * f32(b))) / (2 * np.log(base)) for b in (beta_fast, beta_slow))
        lo, hi = max(np.floor(lo), 0.0), min(np.ceil(hi), rotary - 1.0)
        r = np.clip((i - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        f = f * (1.0 - r) + f / factor * r
        if factor > 1.0:
            gain = 1.0 + 0.1 * np.log(factor)
    return f / (2 * np.pi), f32(attention_factor) if attention_factor else gain


def rope(x, positions, turns, gain, layout="half"):
    """x [tokens][heads][dim] (f64), positions [tokens]."""
    x = np.asarray(x, np.float64)
    n = len(turns)
    # whole turns off before the product with 2 pi
    t = np.asarray(positions, np.float64)[:, None] * turns
    p = (t - np.floor(t)) * 2 * np.pi
    c, s = (gain * f(p)[:, None] for f in (np.cos, np.sin))
    y = x.copy()
    a, b = (x[..., :n], x[..., n:2 * n]) if layout == "half" else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
    lo, hi = a * c - b * s, a * s + b * c
    if layout == "half":
        y[..., :n], y[..., n:2 * n] = lo, hi
    else:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = lo, hi
    return y


def rms_norm(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * np.asarray(w, np.float64)


def half(x):
    """f16 as an 8-bit cache takes it: by way of f32, saturated, NaN as 0."""
    with np.errstate(over="ignore", invalid="ignore"):
        x = np.asarray(x, np.float32)
        return np.clip(np.where(np.isnan(x), np.float32(0), x), -65504, 65504).astype(np.float16)


def quantise(x16):
    """Codes and scale of blocks [..., 32, 128] of f16 values."""
    x = np.asarray(x16, np.float64)
    a = np.abs(x).max((-2, -1), keepdims=True)
    e = np.maximum(np.frexp(a)[1] - 7, -24)  # frexp's exponent is floor(log2 a) + 1
    e = np.where(a == 0, -24, e)
    scale = np.ldexp(1.0, e)
    return np.clip(np.rint(x / scale), -127, 127), scale


class Kv8:
    """Keys and values of one layer, [kv_heads] sequences in step."""

    def __init__(self, kv_heads, capacity):
        n = -(-capacity // BLOCK)
        self.held = np.zeros((2, kv_heads, n, BLOCK, HEAD))             # what the codes stand for
        self.tail = np.zeros((2, kv_heads, BLOCK, HEAD), np.float16)
        self.end = 0

    def append(self, position, keys, values):
        """keys, values [tokens][kv_heads][128], not yet rounded, at position, position + 1, ..."""
        pair = half(np.stack([np.asarray(keys), np.asarray(values)]))
        for t in range(pair.shape[1]):
            b, r = divmod(position + t, BLOCK)
            if r and not (self.end > 0 and (self.end - 1) // BLOCK == b):
                self.tail[:, :, :r] = self.held[:, :, b, :r]
            self.tail[:, :, r] = pair[:, t]
            if r == BLOCK - 1:
                codes, scale = quantise(self.tail)
                self.held[:, :, b] = codes * scale
            self.end = position + t + 1

    def rows(self, count=None):
        """[2][kv_heads][count][128] as attention reads them (count: up to `end`)."""
        whole = self.end // BLOCK
        x = np.concatenate([self.held[:, :, :whole].reshape(2, self.held.shape[1], -1, HEAD),
                            self.tail[:, :, :self.end % BLOCK].astype(np.float64)], 2)
        return x if count is None else x[:, :, :count]


def attend(q, keys, values):
    """q [q_heads][128], keys / values [kv_heads][tokens][128] (f64): [q_heads][128]."""
    per = q.shape[0] // keys.shape[0]
    out = []
    for h in range(q.shape[0]):
        s = keys[h // per] @ q[h] / np.sqrt(HEAD)
        p = np.exp(s - s.max())
        out.append(p @ values[h // per] / p.sum())
    return np.stack(out)


class LongContextQwen3(OracleQwen3):
    """The oracle step with attention in 64 bits over an 8-bit (`i8`) or f16 cache and the given rope (turns, gain)."""

    def __init__(self, cfg, weights, capacity, rope_table, i8=True):
        super().__init__(cfg, weights, capacity)
        self.table, self.i8 = rope_table, i8
        self.caches = [Kv8(cfg["kv_heads"], capacity) for _ in range(cfg["layers"])]
        self.f16 = [np.zeros((2, cfg["kv_heads"], capacity, HEAD)) for _ in range(cfg["layers"])]

    def _attention(self, l, q, k, v, qn, kn, pos):
        """q, k, v [tokens][...] at pos, pos + 1, ...: all of them appended, then each attends up to its own."""
        c, n = self.cfg, len(q)
        at = pos + np.arange(n)
        q = rope(rms_norm(np.reshape(q, (n, c["q_heads"], HEAD)), qn, c["epsilon"]), at, *self.table)
        k = rope(rms_norm(np.reshape(k, (n, c["kv_heads"], HEAD)), kn, c["epsilon"]), at, *self.table)
        v = np.reshape(v, (n, c["kv_heads"], HEAD))
        if self.i8:
            self.caches[l].append(pos, k, v)
            rows = self.caches[l].rows()
        else:
            self.f16[l][:, :, pos:pos + n] = half(np.stack([k, v])).transpose(0, 2, 1, 3)
            rows = self.f16[l]
        return [attend(q[t], *rows[:, :, :pos + t + 1]).reshape(-1).astype(np.float32) for t in range(n)]

    def chunk(self, tokens, pos):
        """A prompt chunk: every layer over all tokens. Returns the last token's hidden state."""
        c = self.cfg
        hs = [self.embed(t) for t in tokens]
        for l in range(c["layers"]):
            p = f"blk.{l}."
            qkv = []
            for h in hs:
                normed = O.rms_norm_raw(h, self.w[p + "attn_norm"], c["epsilon"])
                qkv.append([self._gemv(p + n, normed) for n in ("attn_q", "attn_k", "attn_v")])
            attn = self._attention(l, *zip(*qkv), self.w[p + "attn_q_norm"], self.w[p + "attn_k_norm"], pos)
            for i, h in enumerate(hs):
                h = (h + self._gemv(p + "attn_output", attn[i])).astype(np.float32)
                normed = O.rms_norm_raw(h, self.w[p + "ffn_norm"], c["epsilon"])
                act = O.swiglu(self._gemv(p + "ffn_gate", normed), self._gemv(p + "ffn_up", normed))
                hs[i] = (h + self._gemv(p + "ffn_down", act)).astype(np.float32)
        self.hidden = hs[-1]
        return self.hidden

    def step(self, token, pos, head=True):
        self.chunk([token], pos)
        if not head:
            return None
        self.logits = self._gemv("output", O.rms_norm_raw(self.hidden, self.w["output_norm"], self.cfg["epsilon"]))
        return O.argmax(self.logits)
