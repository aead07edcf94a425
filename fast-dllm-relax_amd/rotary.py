"""Rotary positions: which dims of a head turn, in which pairs and how fast (include/fdllm.h: fdllm_rotary).

The reference's model turns whole heads in halves with one base (fast_dllm_relax/model/cuda.py:15-29), which is what the calls
that take a ``Rotary`` do without one.
"""

from __future__ import annotations

import ctypes
import math

from . import _lib

HEAD_DIM = 128


class Rotary:
    """The first ``dim`` dims of a head turn, pair j of them by position x frequencies[j] radians, and are multiplied by
    ``factor``.  Pairs are (j, j + dim / 2), or (2 j, 2 j + 1) where ``interleaved``.  Frequencies are theta^(-2 j / dim),
    changed for longer contexts by ``scaling``:

      {"type": "linear", "factor": s}   all of them divided by s (positions are interpolated)
      {"type": "ntk", "factor": s}      theta x s^(dim / (dim - 2)): the fastest pair as it was, the slowest s times slower
      {"type": "yarn", "factor": s, "original_len": n, "beta_fast": 32, "beta_slow": 1, "attention_factor": None}
                                        pairs that turn more than beta_fast times in n positions as they were, those that turn
                                        less than beta_slow times s times slower, between them (by j) a mix; turned
                                        dims are multiplied by attention_factor, by default 0.1 ln s + 1

    or given outright (``frequencies``, dim / 2 of them).  dim 0 turns nothing.  An object keeps what it was made with."""

    __slots__ = ("dim", "interleaved", "factor", "frequencies", "struct", "address", "_freq")

    def __init__(self, *, theta: float = 1e6, dim: int = HEAD_DIM, interleaved: bool = False, scaling: dict | None = None,
                 frequencies=None, factor: float = 1.0):
        if dim % 16 or not 0 <= dim <= HEAD_DIM:
            raise ValueError(f"dim must be a multiple of 16 up to {HEAD_DIM}, got {dim}")
        if frequencies is None:
            frequencies, gain = scaled_frequencies(theta, dim, scaling)
            factor = factor * gain
        elif scaling is not None:
            raise ValueError("scaling changes the frequencies of theta; these are given")
        freq = tuple(float(f) for f in frequencies)
        if len(freq) != dim // 2 or not all(abs(f) <= 1e3 for f in freq):
            raise ValueError(f"{dim // 2} frequencies of at most 1000 are wanted for {dim} dims, got {freq}")
        if not abs(factor) <= 1e6:
            raise ValueError(f"factor must be a number of at most 10^6, got {factor}")
        put = lambda name, value: object.__setattr__(self, name, value)  # noqa: E731
        put("dim", int(dim))
        put("interleaved", bool(interleaved))
        put("factor", float(factor))
        put("frequencies", freq)
        put("_freq", (ctypes.c_double * max(1, len(freq)))(*freq))
        held = _lib.FdllmRotary(ctypes.cast(self._freq, ctypes.POINTER(ctypes.c_double)), self.dim, int(self.interleaved), self.factor)
        put("struct", ctypes.byref(held))  # (which keeps it)
        put("address", ctypes.addressof(held))

    def __setattr__(self, name, value):
        raise AttributeError("a Rotary keeps what it was made with: make another")


def scaled_frequencies(theta: float, dim: int, scaling: dict | None) -> tuple[list[float], float]:
    """(radians a position of each pair, factor of the turned dims)"""
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"theta must be a positive number, got {theta}")
    base = [theta ** (-2 * j / dim) for j in range(dim // 2)]
    if scaling is None:
        return base, 1.0
    keys = {"linear": set(), "ntk": set(), "yarn": {"original_len", "beta_fast", "beta_slow", "attention_factor"}}
    kind = scaling.get("type")
    if kind not in keys or not set(scaling) <= keys[kind] | {"type", "factor"} or not {"type", "factor"} <= set(scaling):
        raise ValueError(f"scaling must be a type of {tuple(keys)} with its factor, got {scaling}")
    s = float(scaling["factor"])
    if not 1.0 <= s <= 1e6:
        raise ValueError(f"a scaling factor is at least 1, got {s}")
    if kind == "linear":
        return [f / s for f in base], 1.0
    if kind == "ntk":
        return ([(theta * s ** (dim / (dim - 2))) ** (-2 * j / dim) for j in range(dim // 2)] if dim > 2 else base), 1.0
    n, fast, slow = float(scaling.get("original_len", 0)), float(scaling.get("beta_fast", 32)), float(scaling.get("beta_slow", 1))
    if not (n >= 1 and fast > slow > 0 and theta > 1):
        raise ValueError(f"yarn needs original_len >= 1 and beta_fast > beta_slow > 0, got {scaling}")

    def pair(turns):  # the pair that turns so often in n positions
        return dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
    mix = [min(1.0, max(0.0, (j - low) / max(high - low, 0.001))) for j in range(dim // 2)]
    gain = scaling.get("attention_factor")
    return [f * (1 - m) + f / s * m for f, m in zip(base, mix)], 0.1 * math.log(s) + 1 if gain is None else float(gain)
