"""Rotary positions of queries and keys, before they are cached and attended to.

`make_rotary_table` builds the table of cosines and sines of a model once (64-bit angles, every common way of stretching
the context); `rotary_embedding` turns q and k of a step in one launch.  The reference leaves this to the serving engine.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from turboquant.kernels import _native


def _frequencies(rotary_dim: int, max_position: int, base: float, scaling: Optional[dict]) -> tuple[torch.Tensor, float]:
    """fp64 angular frequencies of the rotary_dim / 2 pairs, and the factor on cosines and sines."""
    spec = dict(scaling or {})
    kind = spec.get("rope_type", spec.get("type", "default"))
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freq = torch.pow(torch.tensor(float(base), dtype=torch.float64), -pair / rotary_dim)
    if kind == "default":
        return freq, 1.0
    factor = float(spec["factor"])
    if factor < 1.0:
        raise ValueError("a rope scaling factor is at least 1")
    if kind == "linear":
        return freq / factor, 1.0
    original = int(spec["original_max_position_embeddings"])
    if kind == "dynamic":
        # the base grows with the length beyond the trained one, here the table's
        length = max(max_position, original)
        grown = base * (factor * length / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
        return torch.pow(torch.tensor(grown, dtype=torch.float64), -pair / rotary_dim), 1.0
    if kind == "llama3":
        low, high = float(spec["low_freq_factor"]), float(spec["high_freq_factor"])
        turns = original * freq / (2 * math.pi)                       # of a pair over the trained length
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return freq * keep + freq / factor * (1 - keep), 1.0
    if kind == "yarn":
        fast, slow = float(spec.get("beta_fast", 32.0)), float(spec.get("beta_slow", 1.0))

        def pair_of(turns: float) -> float:
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
        stretch = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        attention = spec.get("attention_factor")
        return (freq * (1 - stretch) + freq / factor * stretch,
                0.1 * math.log(factor) + 1.0 if attention is None else float(attention))
    raise ValueError(f"rope scaling of type {kind!r} is not known (default, linear, dynamic, llama3, yarn)")


def make_rotary_table(rotary_dim: int, max_position: int, base: float = 10000.0, scaling: Optional[dict] = None,
                      device=None) -> torch.Tensor:
    """fp32 [max_position, rotary_dim]: the cosines of a position's rotary_dim / 2 angles, then their sines.

    scaling: None, or a model configuration's rope_scaling ("rope_type" default, linear, dynamic, llama3 or yarn with its
    parameters).  Angles are 64-bit, so that those of far positions are as exact as those of near ones.
    """
    if rotary_dim < 2 or rotary_dim % 2 or max_position < 1:
        raise ValueError("rotary_dim must be even and max_position positive")
    freq, factor = _frequencies(rotary_dim, max_position, base, scaling)
    freq = freq.to(device)
    table = torch.empty(max_position, rotary_dim, dtype=torch.float32, device=device)
    for a in range(0, max_position, 1 << 16):
        b = min(a + (1 << 16), max_position)
        angle = torch.arange(a, b, dtype=torch.float64, device=device)[:, None] * freq
        table[a:b, :rotary_dim // 2] = angle.cos() * factor
        table[a:b, rotary_dim // 2:] = angle.sin() * factor
    return table


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, cos_sin: torch.Tensor,
                     interleaved: bool = False, inverse: bool = False,
                     out: Optional[tuple] = None) -> tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turn q [T, Hq, D] and k [T, Hkv, D] (or None) by their tokens' positions [T]; returns the turned (q, k).

    fp16, bf16 or fp32, any strides with contiguous heads: views of a fused projection are fine.  cos_sin: the table of
    `make_rotary_table`, [P, R] with even R <= D; values of a head from R on are passed through.  Pairs are (i, i + R/2), or
    (2i, 2i + 1) when interleaved.  inverse turns back.  out: (q_out, k_out) to write to, which may be (q, k) themselves.
    Positions outside the table are clamped to it and set STATUS_BAD_POSITION.  No autograd: the gradient of a turn is the
    call with inverse=True.
    """
    if out is None and not torch.compiler.is_compiling():
        res = _native.host().rotary(q, k, positions, cos_sin, interleaved, inverse)
        if res is not None:
            return res
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if out is None:
        q_out, k_out = torch.ops.tq_b200.rotary(q, k, positions.contiguous(), cos_sin, bool(interleaved), bool(inverse))
        return q_out, (None if k is None else k_out)
    q_out, k_out = out
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_out, k_out)):
        raise RuntimeError("rotary_embedding(out=...) has no autograd")
    _native._rotary_impl(q, k, q_out, k_out, positions.contiguous(), cos_sin, bool(interleaved), bool(inverse))
    return q_out, k_out
