"""Rotary positions of queries and keys, before they are cached and attended to.

`make_rotary_table` builds the table of cosines and sines of a model once (64-bit angles, every common way of stretching
the context); `rotary_embedding` turns q and k of a step in one launch.  The reference leaves this to the serving engine.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from turboquant.kernels import _native


# Parameters of a type of scaling: those it needs and those it may have.  What is in neither is refused, as a table without it would be wrong.
_SCALINGS = {
    "default": ((), ()),
    "linear": (("factor",), ("original_max_position_embeddings",)),
    "dynamic": (("factor", "original_max_position_embeddings"), ()),
    "llama3": (("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"), ()),
    "yarn": (("factor", "original_max_position_embeddings"),
             ("beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim")),
}


def _scaling(scaling: Optional[dict], base: float) -> tuple[str, dict]:
    """Type and parameters of a rope_scaling; those that are None count as absent."""
    spec = {k: v for k, v in (scaling or {}).items() if v is not None}
    kinds = {spec.pop(k) for k in ("rope_type", "type") if k in spec} or {"default"}
    if len(kinds) > 1:
        raise ValueError("rope_type and type name different scalings")
    kind = kinds.pop()
    if kind not in _SCALINGS:
        raise ValueError(f"rope scaling of type {kind!r} is not known ({', '.join(_SCALINGS)})")
    if float(spec.pop("rope_theta", base)) != float(base):
        raise ValueError("rope_theta of the scaling differs from base")
    spec.pop("partial_rotary_factor", None)                           # the caller's rotary_dim says it
    needed, optional = _SCALINGS[kind]
    for key in needed:
        if key not in spec:
            raise ValueError(f"rope scaling of type {kind!r} needs {key!r}")
    for key in spec:
        if key not in needed and key not in optional:
            raise ValueError(f"{key!r} is not known to rope scaling of type {kind!r}")
    return kind, spec


def _frequencies(rotary_dim: int, max_position: int, base: float, scaling: Optional[dict]) -> tuple[torch.Tensor, float]:
    """fp64 angular frequencies of the rotary_dim / 2 pairs, and the factor on cosines and sines."""
    kind, spec = _scaling(scaling, base)
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freq = torch.pow(torch.tensor(float(base), dtype=torch.float64), -pair / rotary_dim)
    if kind == "default":
        return freq, 1.0
    factor = float(spec["factor"])
    if not 1.0 <= factor < math.inf:
        raise ValueError("a rope scaling factor is at least 1")
    if kind == "linear":
        return freq / factor, 1.0
    original = int(spec["original_max_position_embeddings"])
    if original < 1:
        raise ValueError("original_max_position_embeddings must be positive")
    if kind == "dynamic":
        # the base grows with the length beyond the trained one, here the table's
        if rotary_dim < 4:
            raise ValueError("dynamic scaling needs a rotary_dim above 2")
        length = max(max_position, original)
        grown = base * (factor * length / original - (factor - 1)) ** (rotary_dim / (rotary_dim - 2))
        return torch.pow(torch.tensor(grown, dtype=torch.float64), -pair / rotary_dim), 1.0
    if kind == "llama3":
        low, high = float(spec["low_freq_factor"]), float(spec["high_freq_factor"])
        if not low < high:
            raise ValueError("low_freq_factor must be below high_freq_factor")
        turns = original * freq / (2 * math.pi)                       # of a pair over the trained length
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return freq * keep + freq / factor * (1 - keep), 1.0

    fast, slow = float(spec.get("beta_fast", 32.0)), float(spec.get("beta_slow", 1.0))
    if fast <= 0 or slow <= 0 or base <= 1:
        raise ValueError("yarn scaling needs positive beta_fast and beta_slow and a base above 1")

    def pair_of(turns: float) -> float:
        return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    def size_of(mscale: float) -> float:
        return 0.1 * mscale * math.log(factor) + 1.0

    low, high = pair_of(fast), pair_of(slow)
    if spec.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, rotary_dim - 1)
    stretch = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    freq = freq * (1 - stretch) + freq / factor * stretch
    if "attention_factor" in spec:
        return freq, float(spec["attention_factor"])
    if spec.get("mscale") and spec.get("mscale_all_dim"):             # as configurations define it: one without the other changes nothing
        return freq, size_of(float(spec["mscale"])) / size_of(float(spec["mscale_all_dim"]))
    return freq, size_of(1.0)


def make_rotary_table(rotary_dim: int, max_position: int, base: float = 10000.0, scaling: Optional[dict] = None,
                      device=None) -> torch.Tensor:
    """fp32 [max_position, rotary_dim]: the cosines of a position's rotary_dim / 2 angles, then their sines.

    scaling: None, or a model configuration's rope_scaling ("rope_type" default, linear, dynamic, llama3 or yarn with its
    parameters); parameters that the type does not know, or lacks, are refused.  Configurations that leave
    original_max_position_embeddings out of a dynamic scaling mean the model's max_position_embeddings: give it there.
    Angles are 64-bit, so that those of far positions are as exact as those of near ones.
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
