"""Per-token FP8 activation quantizer (fused CUDA kernel).

Same contract as the reference's ``quantize_rows(x, mode)``
(gr00t_libero/acceleration/sources/libero_pro_eval/inference_acceleration_2026_10_11/
a8_accuracy_recovery_2026_10_20_r1/perrow_a8_candidate_r3.py:17-25) for
``mode == 'fp8_e4m3fn'``: returns ``(encoded [M, K] float8_e4m3fn, scale [M, 1] float32)``
with ``scale = absmax / 448`` per row (1 for an all-zero row), and for
``mode == 'int8_symmetric'`` (the deployed recipe): ``(encoded [M, K] int8, scale)`` with
``scale = absmax / 127`` and round-half-to-even.
"""
from __future__ import annotations

import torch

from . import _lib


def quantize_rows(x: torch.Tensor, mode: str = "fp8_e4m3fn", out: torch.Tensor | None = None,
                  scale_out: torch.Tensor | None = None):
    if out is None and scale_out is None and (mode == "fp8_e4m3fn" or mode == "int8_symmetric"):
        pair = _lib.native().quantize_rows(x, mode == "int8_symmetric")
        if pair is not None:
            return pair
    if x.ndim != 2 or x.dtype != torch.bfloat16:
        raise TypeError("quantize_rows expects a 2-D bfloat16 tensor")
    if mode not in ("fp8_e4m3fn", "int8_symmetric"):
        raise ValueError(f"unsupported mode {mode!r}; this implementation provides 'fp8_e4m3fn' and 'int8_symmetric'")
    if not x.is_cuda:
        raise ValueError("quantize_rows needs a CUDA tensor; there is no CPU path")
    lib = _lib.load()
    if x.stride(1) != 1:
        x = x.contiguous()
    m, k = x.shape
    q = out if out is not None else torch.empty((m, k), dtype=torch.uint8, device=x.device)
    s = scale_out if scale_out is not None else torch.empty((m, 1), dtype=torch.float32, device=x.device)
    if m > 0 and k > 0:
        fn = lib.sacq_quant_act_fp8 if mode == "fp8_e4m3fn" else lib.sacq_quant_act_int8
        with torch.cuda.device(x.device):
            _lib.check(fn(x.data_ptr(), x.stride(0), m, k, q.data_ptr(), s.data_ptr(),
                          torch.cuda.current_stream().cuda_stream))
    if mode == "int8_symmetric":
        return (q.view(torch.int8) if q.dtype == torch.uint8 else q), s
    return (q.view(torch.float8_e4m3fn) if q.dtype == torch.uint8 else q), s


def act_quantize_rows(kind: str, a: torch.Tensor, b: torch.Tensor | None = None):
    """Activation function fused into the per-token quantizer (``sacq_act_quant_fp8``):

    * ``kind='silu_mul'``: the bytes of ``quantize_rows(F.silu(a) * b)`` (gated MLP);
    * ``kind='gelu'``:     the bytes of ``quantize_rows(F.gelu(a))`` (erf form);

    in one launch, without materialising the ``[M, K]`` intermediate."""
    kinds = {"silu_mul": 0, "gelu": 1}
    if kind not in kinds:
        raise ValueError(f"unknown activation kind {kind!r}")
    pair = _lib.native().act_quantize_rows(kinds[kind], a, b)
    if pair is not None:
        return pair
    if a.ndim != 2 or a.dtype != torch.bfloat16 or not a.is_cuda:
        raise TypeError("act_quantize_rows expects 2-D bfloat16 CUDA tensors")
    if kind == "silu_mul":
        if b is None or b.shape != a.shape or b.dtype != torch.bfloat16 or b.device != a.device:
            raise TypeError("silu_mul needs a second bfloat16 tensor of the same shape and device")
        if b.stride(1) != 1:
            b = b.contiguous()
    if a.stride(1) != 1:
        a = a.contiguous()
    lib = _lib.load()
    m, k = a.shape
    q = torch.empty((m, k), dtype=torch.uint8, device=a.device)
    s = torch.empty((m, 1), dtype=torch.float32, device=a.device)
    if m > 0 and k > 0:
        with torch.cuda.device(a.device):
            _lib.check(lib.sacq_act_quant_fp8(kinds[kind], a.data_ptr(), a.stride(0),
                                              b.data_ptr() if kind == "silu_mul" else None,
                                              b.stride(0) if kind == "silu_mul" else 0, m, k, q.data_ptr(),
                                              s.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return q.view(torch.float8_e4m3fn), s


def modulate_quantize_rows(x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor):
    """AdaLN modulation fused into the quantizer (``sacq_modulate_quant_fp8``): the bytes of
    ``quantize_rows(x * (1 + scale) + shift)`` for bf16 ``x [M, K]`` and bf16 vectors
    ``scale, shift [K]``, in one launch."""
    pair = _lib.native().modulate_quantize_rows(x, scale, shift)
    if pair is not None:
        return pair
    if x.ndim != 2 or x.dtype != torch.bfloat16 or not x.is_cuda:
        raise TypeError("modulate_quantize_rows expects a 2-D bfloat16 CUDA tensor")
    k = x.shape[1]
    for v in (scale, shift):
        if v.dtype != torch.bfloat16 or v.numel() != k or v.device != x.device:
            raise TypeError("scale and shift must be bfloat16 vectors of K elements on x's device")
    scale, shift = scale.reshape(-1).contiguous(), shift.reshape(-1).contiguous()
    if x.stride(1) != 1:
        x = x.contiguous()
    lib = _lib.load()
    m = x.shape[0]
    q = torch.empty((m, k), dtype=torch.uint8, device=x.device)
    s = torch.empty((m, 1), dtype=torch.float32, device=x.device)
    if m > 0 and k > 0:
        with torch.cuda.device(x.device):
            _lib.check(lib.sacq_modulate_quant_fp8(x.data_ptr(), x.stride(0), scale.data_ptr(), shift.data_ptr(), m, k,
                                                   q.data_ptr(), s.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return q.view(torch.float8_e4m3fn), s


def layernorm_quantize_rows(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                            eps: float = 1e-5, mod_scale: torch.Tensor | None = None,
                            mod_shift: torch.Tensor | None = None, return_normalized: bool = False):
    """LayerNorm over the last dimension, optionally the AdaLN modulation ``y * (1 + s) + t``,
    and the per-token FP8 quantizer in one launch (``sacq_layernorm_quant_fp8``).  Returns
    ``(q, scale)`` or ``(q, scale, y)`` with the bf16 normalised tensor.  ``y`` agrees with
    ``torch.nn.functional.layer_norm`` to one bf16 ulp (different reduction order); ``q`` and
    ``scale`` are exactly ``quantize_rows(y)``."""
    made = _lib.native().layernorm_quantize_rows(x, weight, bias, eps, mod_scale, mod_shift, return_normalized)
    if made is not None:
        return made
    if x.ndim != 2 or x.dtype != torch.bfloat16 or not x.is_cuda:
        raise TypeError("layernorm_quantize_rows expects a 2-D bfloat16 CUDA tensor")
    k = x.shape[1]
    vecs = []
    for v in (weight, bias, mod_scale, mod_shift):
        if v is not None:
            if v.dtype != torch.bfloat16 or v.numel() != k or v.device != x.device:
                raise TypeError("weight, bias and modulation vectors must be bfloat16 with K elements on x's device")
            v = v.reshape(-1).contiguous()
        vecs.append(v)
    if (vecs[2] is None) != (vecs[3] is None):
        raise ValueError("modulation needs both its scale and its shift vector")
    if x.stride(1) != 1:
        x = x.contiguous()
    lib = _lib.load()
    m = x.shape[0]
    q = torch.empty((m, k), dtype=torch.uint8, device=x.device)
    s = torch.empty((m, 1), dtype=torch.float32, device=x.device)
    y = torch.empty((m, k), dtype=torch.bfloat16, device=x.device) if return_normalized else None
    if m > 0 and k > 0:
        ptr = [None if v is None else v.data_ptr() for v in vecs]
        with torch.cuda.device(x.device):
            _lib.check(lib.sacq_layernorm_quant_fp8(x.data_ptr(), x.stride(0), ptr[0], ptr[1], float(eps), ptr[2], ptr[3],
                                                    m, k, None if y is None else y.data_ptr(), k, q.data_ptr(),
                                                    s.data_ptr(), torch.cuda.current_stream().cuda_stream))
    q = q.view(torch.float8_e4m3fn)
    return (q, s, y) if return_normalized else (q, s)


_NORMS = {None: 0, "rms": 1, "layer": 2}


def residual_norm_quantize_rows(branch: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                                bias: torch.Tensor | None = None, *, norm: str = "rms", eps: float = 1e-6,
                                post_norm: str | None = None, post_weight: torch.Tensor | None = None,
                                post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                                residual_scale: float = 1.0, mod_scale: torch.Tensor | None = None,
                                mod_shift: torch.Tensor | None = None, vector_rows: torch.Tensor | None = None,
                                quantize: bool = True, return_normalized: bool = False):
    """The norms behind and before a block, its gate and residual, and the next projections' quantizer in one launch
    (``sacq_residual_norm``).  For the output ``branch`` of a block and its input ``residual``, bf16 ``[M, K]``::

        r = residual_scale * residual + gate * (norm_post(branch) * post_weight + post_bias)
        h = (norm(r) * weight + bias) * (1 + mod_scale) + mod_shift

    ``norm``: ``"rms"`` or ``"layer"``, ``post_norm``: one of them, or ``None`` for the branch as it is; weights and biases are bf16 ``[K]`` or
    ``None``.  ``gate``, ``mod_scale`` and ``mod_shift`` are bf16 ``[K]``, or ``[R, K]`` with ``vector_rows`` (int32 ``[M]``, the row of them that
    each token takes; one outside of ``[0, R)`` makes its token NaN).  Returns ``(r, q, scale)`` with ``r`` in bf16 and the FP8 rows of ``h``, with
    ``return_normalized`` ``(r, q, scale, h)``, or with ``quantize=False`` ``(r, h)``.  Sums and everything in between are fp32, and each
    result is rounded once: ``q`` is made from the fp32 ``h``, not from its bf16 rounding as in ``layernorm_quantize_rows``."""
    if norm not in ("rms", "layer") or post_norm not in _NORMS:
        raise ValueError(f"unknown norm {norm!r} or post_norm {post_norm!r}")
    args = (_NORMS[norm], _NORMS[post_norm], float(eps), float(residual_scale), bool(quantize), bool(return_normalized))
    made = _lib.native().residual_norm_quantize_rows(branch, residual, weight, bias, post_weight, post_bias, gate, mod_scale,
                                                     mod_shift, vector_rows, *args)
    if made is not None:
        return made
    from .attention import refuse_grad
    for t, what in ((branch, "branch"), (residual, "residual")):
        if not isinstance(t, torch.Tensor) or t.ndim != 2 or t.dtype != torch.bfloat16 or not t.is_cuda:
            raise TypeError(f"{what} must be a 2-D bfloat16 CUDA tensor")
    if branch.shape != residual.shape or branch.device != residual.device:
        raise ValueError("branch and residual must have one shape and device")
    m, k = branch.shape
    vectors = {"weight": weight, "bias": bias, "post_weight": post_weight, "post_bias": post_bias}
    tables = {"gate": gate, "mod_scale": mod_scale, "mod_shift": mod_shift}
    refuse_grad("residual_norm_quantize_rows", branch, residual, *vectors.values(), *tables.values())
    if post_norm is None and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need a post_norm")
    if (mod_scale is None) != (mod_shift is None):
        raise ValueError("modulation needs both its scale and its shift")
    if not eps >= 0.0:
        raise ValueError("eps must be non-negative")
    for name, t in {**vectors, **tables}.items():
        if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.bfloat16 or t.device != branch.device):
            raise TypeError(f"{name} must be a bfloat16 tensor on branch's device")
    for name, t in vectors.items():
        if t is not None:
            if t.numel() != k:
                raise ValueError(f"{name} must have {k} elements")
            vectors[name] = t.reshape(-1).contiguous()
    rows = None
    for name, t in tables.items():
        if t is None:
            continue
        if vector_rows is None:
            if t.numel() != k:
                raise ValueError(f"{name} must have {k} elements, or rows of them with vector_rows")
            tables[name] = t.reshape(-1).contiguous()
        else:
            if t.ndim != 2 or t.shape[1] != k or t.shape[0] == 0 or (rows is not None and t.shape[0] != rows):
                raise ValueError(f"{name} must be [R, {k}], with one R for all")
            rows = t.shape[0]
            tables[name] = t.contiguous()
    if vector_rows is not None:
        if rows is None:
            raise ValueError("vector_rows without a gate or a modulation")
        if not isinstance(vector_rows, torch.Tensor) or vector_rows.dtype != torch.int32 or vector_rows.device != branch.device:
            raise TypeError("vector_rows must be an int32 tensor on branch's device")
        if vector_rows.numel() != m:
            raise ValueError("vector_rows must have one entry per row")
        vector_rows = vector_rows.reshape(-1).contiguous()
    branch, residual = (t if t.stride(1) == 1 and t.stride(0) >= k else t.contiguous() for t in (branch, residual))
    if m == 0 or k == 0:
        y = torch.empty_like(branch)
        q, s = torch.empty((m, k), dtype=torch.float8_e4m3fn, device=y.device), torch.ones((m, 1), device=y.device)
        return (y, torch.empty_like(y)) if not quantize else (y, q, s, torch.empty_like(y)) if return_normalized else (y, q, s)
    made = _lib.native().residual_norm_quantize_rows(branch, residual, *vectors.values(), *tables.values(), vector_rows, *args)
    if made is None:
        raise ValueError("residual_norm_quantize_rows: unsupported arguments")
    return made
