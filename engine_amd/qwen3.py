"""Host-side mirror of the reference's decode executor over the C ABI.

  AmdQwen3Config   <- the Qwen3 geometry (decode.rs keeps it in constants)
  AmdKvCache       <- CudaKvState, the KV part of CudaHybridState (state.rs:99-254, 529-660)
  AmdQwen3Decode   <- CudaQwen35Decode (decode.rs:236-800) and CudaQwen35BatchDecode
                      (decode.rs:1626-1960): new, prefill_step, decode_step,
                      decode_step_batch, copy_hidden, copy_logits; score_prompt and
                      logprobs (TokenLogprobs) have no counterpart
  attention_decode <- the per-layer sequence q/k norm + rope + kv_append_f16 +
                      attn_score_gqa (decode.rs:929-1034)

Every computation runs in libribn_amd.so; weights are AmdQuantizedWeight
handles and norm vectors are f32 device tensors (torch is only the allocator).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _lib
from .kquant import RANK_CACHE, RANK_DECODER, AmdModelKernelError, _check, _live, _own, _ptr
from .rope import AmdRopeSpec, _dtype

# What a KV cache holds a value in: f16; 8 bits with a power-of-two scale for
# each block of 32 tokens and KV head; or 4 bits with a scale and a low for each
# 32 tokens of a key dim, each 64 dims of a token's value.
KV_F16, KV_I8, KV_I4 = 0, 1, 4


@dataclass(frozen=True)
class AmdQwen3Config:
    layers: int = 36
    hidden: int = 4096
    q_heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 12288
    vocab: int = 151936
    rope_base: float = 1.0e6
    epsilon: float = 1.0e-6
    # Rope of the caches made for this model, None: half layout, unscaled, rope_base.
    rope: Optional[AmdRopeSpec] = None

    def to_c(self) -> _lib.Qwen3Config:
        return _lib.Qwen3Config(self.layers, self.hidden, self.q_heads, self.kv_heads, self.head_dim, self.ffn,
                                self.vocab, self.rope_base, self.epsilon)


QWEN3_8B = AmdQwen3Config()


def kv_options(config: AmdQwen3Config, format: int = KV_F16, rope: Optional[AmdRopeSpec] = None):
    """ribn_amd_kv_options for a model's caches: `rope`, or else the config's."""
    options = _lib.KvOptions(format, None)
    spec = rope if rope is not None else config.rope
    if spec is not None:
        options.rope = ctypes.pointer(spec.to_c())
    return options


class AmdKvCache:
    """One sequence's KV cache for every layer: f16 ([layer][kv_head][token][head_dim])
    or, with KV_I8 or KV_I4, 8 or 4 bits (ribn_amd_kv_cache_create_with). `rope`, or the config's, is how
    its keys (and the queries that read them) are rotated."""

    def __init__(self, ctx, config: AmdQwen3Config, capacity: int, format: int = KV_F16,
                 rope: Optional[AmdRopeSpec] = None):
        self.ctx = ctx
        self.config = config
        self._cfg = config.to_c()
        self.handle = ctypes.c_void_p()
        options = kv_options(config, format, rope)
        _check(ctx._lib.ribn_amd_kv_cache_create_with(ctx.handle, ctypes.byref(self._cfg), capacity, ctypes.byref(options),
                                                      ctypes.byref(self.handle)), AmdModelKernelError)
        _own(self, RANK_CACHE)

    def format(self) -> int:
        return int(self.ctx._lib.ribn_amd_kv_cache_format(self.handle))

    def tail(self, layer: int):
        """Of a KV_I8 or KV_I4 cache: device addresses of the f16 block its sequence stands
        in, keys [kv_heads][32][128] and values [kv_heads][128][32], and the
        elements between KV heads."""
        k, v, stride = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_size_t()
        _check(self.ctx._lib.ribn_amd_kv_cache_tail(self.handle, layer, ctypes.byref(k), ctypes.byref(v),
                                                    ctypes.byref(stride)), AmdModelKernelError)
        return k.value, v.value, int(stride.value)

    def write(self, layer: int, keys, values, position: int):
        """Puts rows [tokens][kv_heads][128] (f16 or f32; keys normalised and rotated
        already) into the cache at position, position + 1, ..."""
        self._move(self.ctx._lib.ribn_amd_kv_cache_write, layer, position, keys, values)

    def read(self, layer: int, position: int, keys, values):
        """Fills keys and values [tokens][kv_heads][128] (f16 or f32) with what the cache holds there."""
        self._move(self.ctx._lib.ribn_amd_kv_cache_read, layer, position, keys, values)

    def _move(self, call, layer, position, keys, values):
        dtype = _dtype(keys)
        if dtype not in (0, 2) or values.dtype != keys.dtype:
            raise TypeError(f"cache rows are float32 or float16, got {keys.dtype} and {values.dtype}")
        shape = keys.shape
        if shape != values.shape or not keys.is_contiguous() or not values.is_contiguous():
            raise ValueError("keys and values must be contiguous and of one shape")
        if len(shape) != 3 or shape[1] != self.config.kv_heads or shape[2] != self.config.head_dim:
            raise ValueError(f"cache rows are [tokens][{self.config.kv_heads}][{self.config.head_dim}], got {tuple(shape)}")
        _check(call(self.ctx.handle, self.handle, layer, position, shape[0], keys.data_ptr(), values.data_ptr(), keys.numel(),
                    dtype), AmdModelKernelError)

    def capacity(self) -> int:
        return int(self.ctx._lib.ribn_amd_kv_cache_capacity(self.handle))

    def layer(self, layer: int):
        """Device addresses of one layer's key and value caches."""
        k = ctypes.c_void_p()
        v = ctypes.c_void_p()
        _check(self.ctx._lib.ribn_amd_kv_cache_layer(self.handle, layer, ctypes.byref(k), ctypes.byref(v)),
               AmdModelKernelError)
        return k.value, v.value

    def close(self):
        if self.handle and _live():
            self.ctx._lib.ribn_amd_kv_cache_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _handles(caches):
    return b"".join([c.handle for c in caches])  # pointers in a row


def attention_decode(ctx, config: AmdQwen3Config, caches, layer: int, q, k, v, q_norm, k_norm, positions, output):
    """One layer's decode attention for len(caches) members (positions: device int32)."""
    _check(ctx._lib.ribn_amd_attention_decode(ctx.handle, ctypes.byref(config.to_c()), _handles(caches), len(caches), layer,
                                              q.data_ptr(), k.data_ptr(), v.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(),
                                              positions.data_ptr(), output.data_ptr(), output.numel()), AmdModelKernelError)


def attention_prefill(ctx, config: AmdQwen3Config, cache, layer: int, q, k, v, q_norm, k_norm, tokens: int,
                      position: int, output):
    """One layer's causal attention for a prompt chunk of `tokens` tokens at
    `position` (the K/V appended first)."""
    _check(ctx._lib.ribn_amd_attention_prefill(ctx.handle, ctypes.byref(config.to_c()), cache.handle, layer, q.data_ptr(),
                                               k.data_ptr(), v.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(), tokens,
                                               position, output.data_ptr(), output.numel()), AmdModelKernelError)


@dataclass
class TokenLogprobs:
    """Log probabilities of rows (tokens of a prompt, members of a step); what was not asked for is None."""

    logprobs: Optional[np.ndarray]      # [rows] of the targets
    entropy: Optional[np.ndarray]       # [rows]
    top_tokens: Optional[np.ndarray]    # [rows][top], the likeliest first
    top_logprobs: Optional[np.ndarray]  # [rows][top]

    @staticmethod
    def _room(rows: int, logprobs: bool, entropy: bool, top: int) -> "TokenLogprobs":
        def new(want, *shape, dtype=np.float32):
            return np.zeros(shape, dtype) if want else None
        return TokenLogprobs(new(logprobs, rows), new(entropy, rows), new(top > 0, rows, top, dtype=np.uint32), new(top > 0, rows, top))

    def _pointers(self):
        return [None if a is None else a.ctypes.data for a in (self.logprobs, self.entropy, self.top_tokens, self.top_logprobs)]


def _host_tokens(tokens, vocab: int) -> np.ndarray:
    """Whole numbers as the library takes tokens, those outside the vocabulary as one that 32 bits hold."""
    t = np.asarray(tokens).reshape(-1)
    if t.size and t.dtype.kind not in "iu":
        raise TypeError(f"tokens are whole numbers, got {t.dtype}")
    out = t.astype(np.uint32)
    out[(t < 0) | (t >= vocab)] = 0xffffffff
    return out


class AmdQwen3Decode:
    """Decode-step executor (CudaQwen35Decode + CudaQwen35BatchDecode).

    `layers` is a list of dicts with the weight handles attn_q, attn_k, attn_v,
    attn_output, ffn_gate, ffn_up, ffn_down and the f32 device tensors
    attn_norm, attn_q_norm, attn_k_norm, ffn_norm."""

    def __init__(self, ctx, config: AmdQwen3Config, token_embd, output, output_norm, layers, max_members: int = 1):
        self.ctx = ctx
        self.config = config
        self._cfg = config.to_c()
        # The decoder reads these every step: weight handles and norm tensors
        # stay referenced for its lifetime (the C side does not own them).
        self._keep = [output_norm, token_embd, output]
        arr = (_lib.Qwen3Layer * len(layers))()
        for i, lw in enumerate(layers):
            for name in _lib.QWEN3_LAYER_FIELDS:
                obj = lw[name]
                if hasattr(obj, "handle"):
                    setattr(arr[i], name, obj.handle.value)
                else:
                    setattr(arr[i], name, obj.data_ptr())
                self._keep.append(obj)
        self.handle = ctypes.c_void_p()
        _check(ctx._lib.ribn_amd_qwen3_decode_create(ctx.handle, ctypes.byref(self._cfg), token_embd.handle,
                                                     output.handle, _ptr(output_norm), arr, max_members,
                                                     ctypes.byref(self.handle)), AmdModelKernelError)
        _own(self, RANK_DECODER)

    def set_graphs(self, enabled: bool):
        _check(self.ctx._lib.ribn_amd_qwen3_decode_set_graphs(self.handle, 1 if enabled else 0))

    def set_gemv_mode(self, mode: int):
        """CudaQwen35Decode::set_gemv_mode (decode.rs:738-741): GEMV_WARP (f32
        activations, default) or GEMV_FIXED16 (opt-in block fixed point)."""
        _check(self.ctx._lib.ribn_amd_qwen3_decode_set_gemv_mode(self.handle, mode))

    def gemv_mode(self) -> int:
        return int(self.ctx._lib.ribn_amd_qwen3_decode_gemv_mode(self.handle))

    def prefill_step(self, cache: AmdKvCache, token: int, position: int):
        _check(self.ctx._lib.ribn_amd_qwen3_prefill_step(self.handle, cache.handle, token, position),
               AmdModelKernelError)

    def prefill_chunk(self, cache: AmdKvCache, tokens, position: int):
        """Consecutive prompt tokens of one sequence as one step's members."""
        n = len(tokens)
        tok = (ctypes.c_uint32 * n)(*[int(t) for t in tokens])
        _check(self.ctx._lib.ribn_amd_qwen3_prefill_chunk(self.handle, cache.handle, tok, n, position),
               AmdModelKernelError)

    def prefill_prompt(self, cache: AmdKvCache, tokens, position: int, chunk_tokens: int = 0):
        """A whole prompt (consecutive tokens of one sequence from `position`)
        on the prefill matmul, in chunks of `chunk_tokens` (0: 2048): the
        projections as matmuls over the chunk, causal chunk attention on the
        matrix cores, K/V written to the cache, no output head. Stands where
        the reference runs run_prefill_chunk (decode.rs:2149-2267)."""
        import numpy as np
        tok = np.ascontiguousarray(np.asarray(tokens, dtype=np.uint32).reshape(-1))
        ptr = tok.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32))
        _check(self.ctx._lib.ribn_amd_qwen3_prefill_prompt(self.handle, cache.handle, ptr, tok.size, position,
                                                           chunk_tokens), AmdModelKernelError)

    def score_prompt(self, cache: AmdKvCache, tokens, position: int, targets=None, entropy: bool = False, top: int = 0,
                     chunk_tokens: int = 0) -> TokenLogprobs:
        """prefill_prompt, and of each token's successor: the log probability of targets[i] (host tokens, one per prompt
        token; one outside the vocabulary has -inf), the distribution's entropy, and the `top` likeliest tokens with
        their log probabilities (ribn_amd_qwen3_score_prompt). Blocking."""
        tok = _host_tokens(tokens, self.config.vocab)
        goal = None if targets is None else _host_tokens(targets, self.config.vocab)
        if goal is not None and goal.size != tok.size:
            raise ValueError(f"{tok.size} tokens need as many targets, got {goal.size}")
        if not 0 <= top <= self.config.vocab:
            raise ValueError(f"{top} alternatives of {self.config.vocab} tokens")
        out = TokenLogprobs._room(tok.size, goal is not None, entropy, top)
        _check(self.ctx._lib.ribn_amd_qwen3_score_prompt(self.handle, cache.handle, tok.ctypes.data, tok.size, position, chunk_tokens,
                                                         None if goal is None else goal.ctypes.data, *out._pointers(), top),
               AmdModelKernelError)
        return out

    def logprobs(self, members: int = 1, targets=None, logprobs: bool = True, entropy: bool = False, top: int = 0) -> TokenLogprobs:
        """Log probabilities of the first `members` members of the last step with an output head (no more than it had): of
        `targets` (host tokens, by default the ones the step selected), the entropy, and the `top` likeliest tokens
        (ribn_amd_qwen3_logprobs). Blocking."""
        goal = None if targets is None else _host_tokens(targets, self.config.vocab)
        if goal is not None and goal.size != members:
            raise ValueError(f"{members} members need as many targets, got {goal.size}")
        if not 0 <= top <= self.config.vocab:
            raise ValueError(f"{top} alternatives of {self.config.vocab} tokens")
        out = TokenLogprobs._room(members, logprobs, entropy, top)
        _check(self.ctx._lib.ribn_amd_qwen3_logprobs(self.handle, members, None if goal is None else goal.ctypes.data, *out._pointers(), top),
               AmdModelKernelError)
        return out

    def reserve_prompt(self, chunk_tokens: int = 0):
        """Allocates the prompt workspace for chunks of `chunk_tokens` tokens ahead of prefill_prompt."""
        _check(self.ctx._lib.ribn_amd_qwen3_reserve_prompt(self.handle, chunk_tokens), AmdModelKernelError)

    def decode_step(self, cache: AmdKvCache, token: int, position: int) -> int:
        out = ctypes.c_uint32()
        _check(self.ctx._lib.ribn_amd_qwen3_decode_step(self.handle, cache.handle, token, position,
                                                        ctypes.byref(out)), AmdModelKernelError)
        return out.value

    def decode_step_batch(self, caches, tokens, positions) -> list[int]:
        m = len(caches)
        tok = (ctypes.c_uint32 * m)(*[int(t) for t in tokens])
        pos = (ctypes.c_uint32 * m)(*[int(p) for p in positions])
        out = (ctypes.c_uint32 * m)()
        _check(self.ctx._lib.ribn_amd_qwen3_decode_step_batch(self.handle, _handles(caches), tok, pos, m, out),
               AmdModelKernelError)
        return list(out)

    def generate(self, caches, tokens, positions, steps: int) -> np.ndarray:
        """Greedy tokens [members][steps], looping on the device."""
        m = len(caches)
        tok = (ctypes.c_uint32 * m)(*[int(t) for t in tokens])
        pos = (ctypes.c_uint32 * m)(*[int(p) for p in positions])
        out = np.zeros((m, steps), np.uint32)
        _check(self.ctx._lib.ribn_amd_qwen3_generate(self.handle, _handles(caches), tok, pos, m, steps,
                                                     out.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32))),
               AmdModelKernelError)
        return out

    def copy_hidden(self, member: int = 0) -> np.ndarray:
        out = np.zeros(self.config.hidden, np.float32)
        _check(self.ctx._lib.ribn_amd_qwen3_copy_hidden(self.handle, member, out.ctypes.data_as(ctypes.c_void_p),
                                                        out.size))
        return out

    def copy_logits(self, member: int = 0) -> np.ndarray:
        out = np.zeros(self.config.vocab, np.float32)
        _check(self.ctx._lib.ribn_amd_qwen3_copy_logits(self.handle, member, out.ctypes.data_as(ctypes.c_void_p),
                                                        out.size))
        return out

    def close(self):
        if self.handle and _live():
            self.ctx._lib.ribn_amd_qwen3_decode_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
