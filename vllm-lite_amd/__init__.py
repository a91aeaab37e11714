"""MI355X paged attention for vllm-lite: HIP kernels behind a C ABI.

The product is ``libpa.so`` (built from ``csrc/`` by ``build_lib.build``).
This package is the thin Python face of it: ctypes bindings (``_lib``),
torch-tensor wrappers of the stateless entry points (``ops``) and the
``PagedKvCache`` mirror of the reference's cache object (``kv_cache``).
There is no fallback path: importing the wrappers without a built library
raises.
"""
from . import _lib
from .ops import (
    BLOCK_SIZE,
    Int8Cache,
    MxRows,
    MxWeight,
    PaError,
    append_int8,
    argmax,
    block_hash,
    decode,
    decode_int8,
    decode_int8_workspace_size,
    decode_workspace_size,
    prefill,
    prefill_int8,
    read_kv,
    read_kv_int8,
    reshape_and_cache,
    reshape_and_cache_fp8,
    rope_inv_freq,
    layer_norm,
    linear,
    linear_mx,
    quantize_mx,
    rms_norm,
    rms_norm_mx,
    rope_reshape_and_cache,
    sample,
    sample_workspace_size,
    silu_mul,
    slot_mapping,
)
from .kv_cache import PagedKvCache, StepBatch

__all__ = [
    "BLOCK_SIZE",
    "Int8Cache",
    "MxRows",
    "MxWeight",
    "PaError",
    "PagedKvCache",
    "StepBatch",
    "append_int8",
    "argmax",
    "block_hash",
    "decode",
    "decode_int8",
    "decode_int8_workspace_size",
    "decode_workspace_size",
    "prefill",
    "prefill_int8",
    "read_kv",
    "read_kv_int8",
    "reshape_and_cache",
    "reshape_and_cache_fp8",
    "rope_inv_freq",
    "layer_norm",
    "linear",
    "linear_mx",
    "quantize_mx",
    "rms_norm",
    "rms_norm_mx",
    "rope_reshape_and_cache",
    "sample",
    "sample_workspace_size",
    "silu_mul",
    "slot_mapping",
]
