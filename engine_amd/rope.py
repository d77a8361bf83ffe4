"""Rotary positions over the C ABI.

  AmdRopeSpec  which dims turn together, their frequencies and how these are
               stretched for contexts past the trained length
  AmdRope      the operator on query and key rows; with the half layout, unscaled,
               CudaQwen35Ops::rope_neox (model_ops.rs:2012-2070)

A KV cache takes a spec too (AmdKvCache): its keys are cached rotated.
"""
from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass
from typing import Optional, Sequence

from . import _lib
from .kquant import RANK_RESOURCE, AmdModelKernelError, _check, _live, _own

_LAYOUTS = {"half": 0, "interleaved": 1}
_SCALINGS = {"none": 0, "linear": 1, "yarn": 2}


@dataclass(frozen=True)
class AmdRopeSpec:
    """ribn_amd_rope_spec. `rotary_dim` None: the whole head. `attention_factor` 0:
    the scaling's own (YaRN 0.1 ln(factor) + 1). `freq_factors`: one divisor per pair."""
    head_dim: int = 128
    rotary_dim: Optional[int] = None
    layout: str = "half"
    base: float = 1.0e6
    scaling: str = "none"
    factor: float = 1.0
    original_context: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float = 0.0
    freq_factors: Optional[Sequence[float]] = None

    def to_c(self) -> _lib.RopeSpec:
        """The C struct (it keeps the factors' array alive)."""
        if self.layout not in _LAYOUTS:
            raise ValueError(f"rope layout must be one of {sorted(_LAYOUTS)}, got {self.layout!r}")
        if self.scaling not in _SCALINGS:
            raise ValueError(f"rope scaling must be one of {sorted(_SCALINGS)}, got {self.scaling!r}")
        rotary = self.head_dim if self.rotary_dim is None else self.rotary_dim
        spec = _lib.RopeSpec(_LAYOUTS[self.layout], self.head_dim, rotary, _SCALINGS[self.scaling], self.base,
                             self.factor, self.original_context, self.beta_fast, self.beta_slow,
                             self.attention_factor, None)
        if self.freq_factors is not None:
            if len(self.freq_factors) != rotary // 2:
                raise ValueError(f"{rotary // 2} pairs need as many frequency factors, got {len(self.freq_factors)}")
            spec.freq_factors = (ctypes.c_float * (rotary // 2))(*self.freq_factors)
        return spec


def rope_frequencies(spec: AmdRopeSpec):
    """Host-only check of a spec; the turns a position adds to each pair's angle, and the gain."""
    lib = _lib.load()
    c = spec.to_c()
    turns = (ctypes.c_double * max(1, c.rotary_dim // 2))()
    gain = ctypes.c_double()
    _check(lib.ribn_amd_rope_frequencies(ctypes.byref(c), turns, c.rotary_dim // 2, ctypes.byref(gain)), AmdModelKernelError)
    return list(turns), gain.value


_POSITIONS = 3
_DTYPES: dict = {}
_ROWS = struct.Struct("18N")  # queries and keys


def _dtype(t):
    """The C element type of a tensor (_POSITIONS for int32), None for others."""
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.int32: _POSITIONS})
    return _DTYPES.get(t.dtype)


def _length(t) -> int:
    """Elements from the tensor's first to its storage's end."""
    return t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()


class AmdRope:
    """Rotates rows [tokens][heads][head_dim] (f32, bf16 or f16; any strides over
    tokens and heads, dims contiguous) by their tokens' positions (device int32)."""

    def __init__(self, ctx, spec: AmdRopeSpec):
        self.ctx = ctx
        self.spec = spec
        self.handle = ctypes.c_void_p()
        c = spec.to_c()
        _check(ctx._lib.ribn_amd_rope_create(ctx.handle, ctypes.byref(c), ctypes.byref(self.handle)), AmdModelKernelError)
        _own(self, RANK_RESOURCE)

    def execute(self, input, positions, output):
        """output = rope(input); `output` may be `input`."""
        self.execute_group([input], positions, [output])

    def execute_group(self, inputs, positions, outputs):
        """Up to four tensors sharing their tokens' positions (queries and keys) in one launch."""
        count = len(inputs)
        if count != len(outputs):
            raise ValueError(f"{count} inputs and {len(outputs)} outputs")
        if _dtype(positions) != _POSITIONS or positions.dim() != 1 or not positions.is_contiguous():
            raise TypeError("positions must be a contiguous vector of int32")
        tokens = positions.shape[0]
        dim = self.spec.head_dim
        kind = inputs[0].dtype if count else None
        dtype = _DTYPES.get(kind, 0 if kind is None else _POSITIONS)
        rows = []  # ribn_amd_rope_rows, nine words each
        for x, y in zip(inputs, outputs):
            if dtype == _POSITIONS or x.dtype is not kind or y.dtype is not kind:
                raise TypeError("rope takes float32, bfloat16 or float16 tensors of one type")
            shape = x.shape
            if len(shape) != 3 or shape != y.shape or shape[0] != tokens or shape[2] != dim:
                raise ValueError(f"rope rows are [{tokens}][heads][{dim}], got {tuple(shape)} and {tuple(y.shape)}")
            xt, xh, xd = x.stride()
            yt, yh, yd = y.stride()
            if xd != 1 or yd != 1:
                raise ValueError("the dims of a head must be contiguous")
            rows += (x.data_ptr(), _length(x), xt, xh, y.data_ptr(), _length(y), yt, yh, shape[1])
        status = self.ctx._lib.ribn_amd_rope_execute(self.handle, positions.data_ptr(), tokens, _ROWS.pack(*rows) if count == 2
                                                     else struct.pack(f"{9 * count}N", *rows), count, dtype)
        if status:
            _check(status, AmdModelKernelError)

    def close(self):
        if self.handle and _live():
            self.ctx._lib.ribn_amd_rope_destroy(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
