"""Rotary positions of query and key heads (``sacq_rotate_heads``) and the frequencies they turn with."""
from __future__ import annotations

import math

import torch

from . import _lib
from .attention import _heads, refuse_grad

_LAYOUTS = {"half": 0, "interleaved": 1}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None, device="cuda"):
    """``(inv_freq, amplitude)`` for ``rotate_heads``: float64 radians per position of the ``rotary_dim / 2`` pairs,
    ``base ** (-2 i / rotary_dim)``, on ``device``, and the factor of cosine and sine.  ``scaling`` stretches a context:

    * ``{"kind": "linear", "factor": s}``: positions divided by ``s``;
    * ``{"kind": "base", "factor": s}``: the base raised so that the slowest pair turns ``s`` times slower and the fastest as before;
    * ``{"kind": "yarn", "factor": s, "original": n}`` (optionally ``beta_fast`` 32, ``beta_slow`` 1, ``amplitude``): pairs that turn less than
      ``beta_slow`` times over the ``n`` positions of training are divided by ``s``, those above ``beta_fast`` turns kept, a ramp over the pair's
      index in between; amplitude ``0.1 ln s + 1``;
    * ``{"kind": "wavelength", "factor": s, "original": n}`` (optionally ``low`` 1, ``high`` 4): the same with a ramp over the number of turns,
      from ``low`` to ``high``, amplitude 1."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be a positive even number")
    if not 1.0 < base < math.inf:
        raise ValueError("base must be above 1")
    exponents = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    freq, amplitude = base ** -exponents, 1.0
    if scaling is not None:
        kind, s = scaling.get("kind"), float(scaling.get("factor", 0.0))
        if not 1.0 <= s < math.inf:
            raise ValueError("scaling needs a factor of at least 1")
        known = {"linear": (), "base": (), "yarn": ("original", "beta_fast", "beta_slow", "amplitude"),
                 "wavelength": ("original", "low", "high")}
        if kind not in known:
            raise ValueError(f"unknown kind of scaling {kind!r}")
        unknown = set(scaling) - {"kind", "factor", *known[kind]}
        if unknown:
            raise ValueError(f"scaling of kind {kind!r} does not take {sorted(unknown)}")
        if "original" in known[kind] and not scaling.get("original", 0) > 0:
            raise ValueError(f"scaling of kind {kind!r} needs the number of positions it was trained on as 'original'")
        if kind == "linear":
            freq = freq / s
        elif kind == "base":
            if rotary_dim == 2:
                raise ValueError("scaling of kind 'base' needs two pairs at least")
            freq = (base * s ** (rotary_dim / (rotary_dim - 2))) ** -exponents
        elif kind == "yarn":
            fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
            if not 0.0 < slow < fast:
                raise ValueError("beta_slow must lie between 0 and beta_fast")
            # index of the pair that turns `turns` times over the original positions
            at = lambda turns: rotary_dim * math.log(scaling["original"] / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
            ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            freq = freq * (1.0 - ramp) + freq / s * ramp
            amplitude = float(scaling.get("amplitude", 0.1 * math.log(s) + 1.0))
        else:
            low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
            if not 0.0 < low < high:
                raise ValueError("low must lie between 0 and high")
            turns = scaling["original"] * freq / (2 * math.pi)
            keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
            freq = freq * keep + freq / s * (1.0 - keep)
    return freq.to(device), amplitude


def rotate_heads(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 layout: str = "half", amplitude: float = 1.0, out=None):
    """Turns the pairs of every head by ``positions[t] * inv_freq[i]``, in one launch for both tensors; returns ``(q', k')``.

    ``q``, ``k`` (or ``None``): bf16 ``[tokens, heads, head_dim]``, any strides with a unit inner one.  ``positions``: int32 or int64
    ``[tokens]``; ``inv_freq``: float64 ``[rotary_dim / 2]`` (``rotary_frequencies``); ``rotary_dim`` is at most ``head_dim`` and what lies behind it
    is copied.  ``layout``: ``"half"`` pairs element ``i`` with ``i + rotary_dim / 2``, ``"interleaved"`` ``2 i`` with ``2 i + 1``.
    ``out=(q_out, k_out)`` receives the results; ``out=(q, k)`` turns in place, views of one fused buffer too.  Angles are made in double and reduced there: right to 2e-7
    radians up to 2^28 radians, to 3 x 2^-53 of the angle beyond (3e-6 at 2^33); positions above 2^53 are rounded."""
    if layout not in _LAYOUTS:
        raise ValueError(f"unknown layout {layout!r}")
    q_out, k_out = (None, None) if out is None else out
    made = _lib.native().rotate_heads(q, k, positions, inv_freq, _LAYOUTS[layout], float(amplitude), q_out, k_out)
    if made is not None:
        return made
    _heads(q, "q")
    if k is not None:
        _heads(k, "k")
        if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or k.device != q.device:
            raise ValueError("k must have q's tokens, head_dim and device")
    refuse_grad("rotate_heads", q, k, q_out, k_out)
    t, d = q.shape[0], q.shape[2]
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64) or positions.ndim != 1:
        raise TypeError("positions must be an int32 or int64 vector")
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dtype != torch.float64 or inv_freq.ndim != 1:
        raise TypeError("inv_freq must be a float64 vector")
    if positions.device != q.device or inv_freq.device != q.device:
        raise ValueError("positions and inv_freq must be on q's device")
    if positions.numel() != t:
        raise ValueError("positions must have one entry per token")
    if not 0 < 2 * inv_freq.numel() <= d:
        raise ValueError(f"{inv_freq.numel()} pairs do not fit heads of {d}")
    if k is None and k_out is not None:
        raise ValueError("there is no k for out[1]")
    for x, other, y, what in ((q, k, q_out, "out[0]"), (k, q, k_out, "out[1]")):
        if y is None:
            continue
        _heads(y, what)
        if y.shape != x.shape or y.device != x.device or (y.stride(2) != 1 and d > 1):
            raise ValueError(f"{what} must have the shape and device of its input, and a unit inner stride")
        same = y.data_ptr() == x.data_ptr() and y.stride() == x.stride()
        if any(n > 1 and s == 0 for n, s in zip(y.shape, y.stride())):
            raise ValueError(f"{what} has elements that share memory")
        if _lib.native().overlaps(y, (other,) if same else (x, other)):
            raise ValueError(f"{what} overlaps an input that it does not replace")
    if q_out is not None and k_out is not None and _lib.native().overlaps(q_out, (k_out,)):
        raise ValueError("the results overlap each other")
    q, k = (x if x is None or x.stride(2) == 1 or d == 1 else x.contiguous() for x in (q, k))
    made = _lib.native().rotate_heads(q, k, positions.contiguous(), inv_freq.contiguous(), _LAYOUTS[layout], float(amplitude),
                                      q_out, k_out)
    if made is None:
        raise ValueError("rotate_heads: unsupported arguments")
    return made
