"""Attention over packed sequences (``sacq_attention_packed``).

The reference leaves attention to its framework; here it is one call on the rows that the quantized projections
produce, for requests of different lengths without padding, and for single tokens against a long past."""
from __future__ import annotations

import ctypes
import math

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib


def refuse_grad(name: str, *tensors) -> None:
    given = [t for t in tensors if isinstance(t, torch.Tensor)]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")
    if any(forward_ad.unpack_dual(t).tangent is not None for t in given):
        raise RuntimeError(f"{name} has no forward-mode derivative: call it on the primals of dual tensors")


def _heads(t, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.ndim != 3 or t.dtype != torch.bfloat16:
        raise TypeError(f"{what} must be a bfloat16 tensor [tokens, heads, head_dim]")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor; there is no CPU path")
    return t


def block_steps_status(device=None) -> int:
    """0, or a nonzero code once a bounded wait of ``attention_packed`` or ``residual_norm_quantize_rows`` has given up on ``device`` (the
    current one by default): what that call returned is not its result.  Synchronises the device (``sacq_block_steps_status``)."""
    word = ctypes.c_int(0)
    with torch.cuda.device(device):
        _lib.check(_lib.load().sacq_block_steps_status(ctypes.byref(word)))
    return word.value


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k: torch.Tensor | None = None, *,
                     causal: bool = False, scale: float | None = None, out: torch.Tensor | None = None,
                     return_lse: bool = False):
    """Softmax attention of sequences that lie one behind the other.

    ``q`` ``[tokens_q, heads, head_dim]``, ``k`` and ``v`` ``[tokens_k, kv_heads, head_dim]``: bf16, any strides with a unit
    inner one (views of a fused projection are read where they lie); ``heads`` is a multiple of ``kv_heads``,
    ``head_dim`` at most 256 (multiples of 8 up to 128 run on the tensor cores).  ``cu_q``, ``cu_k`` (int32,
    ``[sequences + 1]``, on the device): the first row of each sequence and the end of the last; ``cu_k=None``: ``cu_q``.

    ``causal``: query ``i`` of ``n`` sees keys up to ``i + (keys - n)``, so that new tokens behind a longer past see all of it.
    ``scale`` defaults to ``head_dim ** -0.5``.  Returns ``out`` like ``q`` (and with ``return_lse`` the fp32
    ``[tokens_q, heads]`` logarithm of each row's sum of exponentials).  A query that sees no key gets zeros and ``-inf``.
    Rows outside of every sequence are not written.  Offsets may go down: such a sequence is empty.  Room behind a past in a cache is a sequence
    without queries (``cu_q = [0, 1, 1, 2, 2]``, ``cu_k = [0, 500, 4096, 4696, 8192]``).  Kernel and chunks of keys are chosen from the averages of the call: a batch
    of very unlike sequences may be faster as two calls.  The call does not read the offsets on the host and can be captured in a
    CUDA graph."""
    made = _lib.native().attention_packed(q, k, v, cu_q, cu_k, bool(causal), scale, out, bool(return_lse))
    if made is not None:
        return made
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        _heads(t, what)
    refuse_grad("attention_packed", q, k, v, out)
    if k.shape != v.shape or k.device != q.device or v.device != q.device:
        raise ValueError("k and v must have one shape, on q's device")
    h, d = q.shape[1], q.shape[2]
    if k.shape[2] != d or d == 0 or h == 0 or k.shape[1] == 0 or h % k.shape[1] != 0:
        raise ValueError(f"{h} query heads of {d} do not go with {k.shape[1]} key-value heads of {k.shape[2]}")
    if d > 256:
        raise ValueError("head_dim above 256 is not supported")
    offsets = [cu_q, cu_q if cu_k is None else cu_k]
    for cu, what in zip(offsets, ("cu_q", "cu_k")):
        if not isinstance(cu, torch.Tensor) or cu.dtype != torch.int32 or cu.ndim != 1 or cu.numel() < 1:
            raise TypeError(f"{what} must be an int32 vector of sequences + 1 offsets")
        if cu.device != q.device:
            raise ValueError(f"{what} must be on q's device")
    if offsets[0].numel() != offsets[1].numel():
        raise ValueError("cu_q and cu_k must have one number of sequences")
    if scale is not None and not (0.0 < float(scale) < math.inf):
        raise ValueError("scale must be positive and finite")
    if out is not None:
        _heads(out, "out")
        if out.shape != q.shape or out.device != q.device or (out.stride(2) != 1 and d > 1):
            raise ValueError("out must have q's shape and device, and a unit inner stride")
        if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
            raise ValueError("out has elements that share memory")
        if _lib.native().overlaps(out, (q, k, v)):
            raise ValueError("out may not overlap q, k or v")
    q, k, v = (t if t.stride(2) == 1 or d == 1 else t.contiguous() for t in (q, k, v))
    made = _lib.native().attention_packed(q, k, v, *(cu.contiguous() for cu in offsets), bool(causal),
                                          None if scale is None else float(scale), out, bool(return_lse))
    if made is None:
        raise ValueError("attention_packed: unsupported arguments")
    return made
