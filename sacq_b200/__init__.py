"""sacq_b200 -- B200 (sm_100a) implementation of SACQ's packed vector-codebook
quantized-linear forward (W1.5A8): hand-written CUDA kernels behind a C ABI, with a
PyTorch module that keeps the reference's payload format and module interface.

Importing the package does not need a GPU; constructing a layer or calling a kernel
does, and fails loudly when the CUDA library has not been built."""
from .packing import index_bits_for, index_window_bytes, pack_indices, pack_payload, unpack_indices  # noqa: F401

__all__ = [
    "PrecomputedPackedVectorCodebookLinear", "forward_shared", "linear_a8_multi", "quantize_rows", "act_quantize_rows", "modulate_quantize_rows", "layernorm_quantize_rows", "pack_indices", "unpack_indices",
    "pack_payload", "index_bits_for", "index_window_bytes", "attention_packed", "rotate_heads", "rotary_frequencies",
    "residual_norm_quantize_rows", "block_steps_status",
]


# public names that need the CUDA library, and the module each is in; looked up on first use
_LAZY = {
    "PrecomputedPackedVectorCodebookLinear": "linear", "forward_shared": "linear", "linear_a8_multi": "linear",
    "layernorm_quantize_rows": "activation", "modulate_quantize_rows": "activation", "act_quantize_rows": "activation",
    "quantize_rows": "activation", "residual_norm_quantize_rows": "activation", "attention_packed": "attention", "block_steps_status": "attention",
    "rotate_heads": "rotary", "rotary_frequencies": "rotary",
}


def __getattr__(name):
    if name not in _LAZY:
        raise AttributeError(name)
    from importlib import import_module
    found = globals()[name] = getattr(import_module("." + _LAZY[name], __name__), name)   # from now on a plain name
    return found
