"""torch-tensor wrappers of the stateless C entry points of libpa.so.

Tensors are passed by device pointer; work goes on the current HIP stream of
the tensors' device.  Each wrapper checks dtype, device, contiguity and
shape before calling, and raises PaError with the library's message when a
call returns a non-zero status.
"""
import ctypes as C
import math

import torch

from . import _lib

BLOCK_SIZE = 16
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
# FP8-E4M3 caches (the reference's codes) are uint8 tensors; q / out are bf16.
FP8 = 2


class PaError(RuntimeError):
    """A libpa entry point returned a negative pa_status."""

    def __init__(self, fn, code, msg):
        super().__init__(f"{fn} failed ({code}): {msg}")
        self.code = code


def _check(fn, rc):
    if rc != 0:
        raise PaError(fn, rc, _lib.load().pa_last_error().decode())


def _stream(t):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _dev(*ts):
    for t in ts:
        if not (t.is_cuda and t.is_contiguous()):
            raise ValueError("expected contiguous device tensors")


def _dtype_code(t):
    if t.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {t.dtype}")
    return _DTYPES[t.dtype]


def new_cache(num_blocks, num_kv_heads, head_dim, dtype, device="cuda"):
    """Zeroed (k_cache [NB, H, 16, D], v_cache [NB, H, D, 16]) for one layer;
    dtype torch.uint8 makes FP8-E4M3 caches."""
    k = torch.zeros(num_blocks, num_kv_heads, BLOCK_SIZE, head_dim, dtype=dtype, device=device)
    v = torch.zeros(num_blocks, num_kv_heads, head_dim, BLOCK_SIZE, dtype=dtype, device=device)
    return k, v


def _cache_dims(k_cache, v_cache):
    nb, h, bs, d = k_cache.shape
    if bs != BLOCK_SIZE or tuple(v_cache.shape) != (nb, h, d, BLOCK_SIZE):
        raise ValueError("caches must be K [NB, H, 16, D] and V [NB, H, D, 16]")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError("K and V caches differ in dtype")
    return nb, h, d


def _rows_ok(x, h, d):
    """Token rows [H, D] of x [T, H, D]: contiguous within a row, and rows
    that do not overlap (a token stride of at least H * D; the C ABI reads a
    stride of 0 as "contiguous")."""
    return (x.stride(2) == 1 and x.stride(1) == d and
            (x.shape[0] <= 1 or x.stride(0) >= h * d))


def reshape_and_cache(key, value, k_cache, v_cache, slot_mapping):
    """Scatter key/value [T, H, D] into the caches at slot_mapping [T] (int64)."""
    _dev(k_cache, v_cache, slot_mapping)
    nb, h, d = _cache_dims(k_cache, v_cache)
    t = key.shape[0]
    if key.shape[1:] != (h, d) or value.shape != key.shape or slot_mapping.shape != (t,):
        raise ValueError("key/value must be [T, H, D] matching the cache; slot_mapping [T]")
    if slot_mapping.dtype != torch.int64 or key.dtype != k_cache.dtype or value.dtype != k_cache.dtype:
        raise ValueError("dtype mismatch")
    if not (_rows_ok(key, h, d) and _rows_ok(value, h, d)):
        raise ValueError("key/value rows must be contiguous [H, D], not overlapping")
    lib = _lib.load()
    _check("pa_reshape_and_cache", lib.pa_reshape_and_cache(
        _ptr(key), _ptr(value), _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), t, h, d, nb,
        key.stride(0), value.stride(0), _dtype_code(k_cache), _stream(k_cache)))


def _cache_code(k_cache, q=None):
    """dtype code of a (q, cache) pair: uint8 caches are FP8 with bf16 q."""
    if k_cache.dtype == torch.uint8:
        if q is not None and q.dtype != torch.bfloat16:
            raise ValueError("FP8 caches take bf16 q")
        return FP8
    if q is not None and q.dtype != k_cache.dtype:
        raise ValueError("q must be in the cache dtype")
    return _dtype_code(k_cache)


def reshape_and_cache_fp8(key, value, k_cache, v_cache, slot_mapping, block_flags=None):
    """Quantise key/value [T, H, D] (f32 or bf16) into uint8 FP8 caches at
    slot_mapping [T] (int64), with the reference's E4M3 encoder.
    block_flags (uint8 [NB]): pa_reshape_and_cache_fp8_flagged, which also
    sets the flag of every block that receives a NaN / inf code."""
    _dev(k_cache, v_cache, slot_mapping)
    nb, h, d = _cache_dims(k_cache, v_cache)
    if k_cache.dtype != torch.uint8:
        raise ValueError("FP8 caches are uint8")
    t = key.shape[0]
    if key.shape[1:] != (h, d) or value.shape != key.shape or slot_mapping.shape != (t,):
        raise ValueError("key/value must be [T, H, D] matching the cache; slot_mapping [T]")
    if slot_mapping.dtype != torch.int64 or value.dtype != key.dtype:
        raise ValueError("dtype mismatch")
    if not (_rows_ok(key, h, d) and _rows_ok(value, h, d)):
        raise ValueError("key/value rows must be contiguous [H, D], not overlapping")
    lib = _lib.load()
    if block_flags is not None:
        _flags(block_flags, nb)
        _check("pa_reshape_and_cache_fp8_flagged", lib.pa_reshape_and_cache_fp8_flagged(
            _ptr(key), _ptr(value), _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), t, h, d,
            nb, key.stride(0), value.stride(0), _dtype_code(key), _ptr(block_flags),
            _stream(k_cache)))
        return
    _check("pa_reshape_and_cache_fp8", lib.pa_reshape_and_cache_fp8(
        _ptr(key), _ptr(value), _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), t, h, d, nb,
        key.stride(0), value.stride(0), _dtype_code(key), _stream(k_cache)))


def _flags(block_flags, nb):
    _dev(block_flags)
    if block_flags.dtype != torch.uint8 or block_flags.shape != (nb,):
        raise ValueError("block_flags must be uint8 [num_blocks]")


def slot_mapping(block_tables, positions, cu_seq_tokens):
    """Device slot mapping from block tables [B, MBS] (int32), positions [T]
    (int64) and cumulative token counts [B + 1] (int32)."""
    _dev(block_tables, positions, cu_seq_tokens)
    b, mbs = block_tables.shape
    out = torch.empty(positions.shape[0], dtype=torch.int64, device=positions.device)
    lib = _lib.load()
    _check("pa_slot_mapping", lib.pa_slot_mapping(
        _ptr(block_tables), mbs, _ptr(positions), _ptr(cu_seq_tokens), b, positions.shape[0],
        _ptr(out), _stream(positions)))
    return out


def read_kv(k_cache, v_cache, block_ids, seq_len):
    """Gather one sequence's first seq_len tokens -> (k, v) [seq_len, H, D]
    (f32 dequantised values for FP8 caches)."""
    _dev(k_cache, v_cache, block_ids)
    nb, h, d = _cache_dims(k_cache, v_cache)
    odt = torch.float32 if k_cache.dtype == torch.uint8 else k_cache.dtype
    out_k = torch.empty(seq_len, h, d, dtype=odt, device=k_cache.device)
    out_v = torch.empty_like(out_k)
    lib = _lib.load()
    _check("pa_read_kv", lib.pa_read_kv(
        _ptr(k_cache), _ptr(v_cache), _ptr(block_ids), block_ids.shape[0], seq_len, h, d, nb,
        _ptr(out_k), _ptr(out_v), _cache_code(k_cache), _stream(k_cache)))
    return out_k, out_v


def block_hash(k_cache, block_ids):
    """Reference block-content hash of each listed block (f32 cache);
    returns int64 holding the u64 bit patterns."""
    _dev(k_cache, block_ids)
    if k_cache.dtype != torch.float32:
        raise ValueError("block_hash is defined on f32 caches")
    nb, h, _, d = k_cache.shape
    out = torch.empty(block_ids.shape[0], dtype=torch.int64, device=k_cache.device)
    lib = _lib.load()
    _check("pa_block_hash", lib.pa_block_hash(
        _ptr(k_cache), _ptr(block_ids), block_ids.shape[0], h, d, nb, _ptr(out),
        _stream(k_cache)))
    return out


def decode_workspace_size(num_seqs, num_heads, head_dim, max_context_len):
    return int(_lib.load().pa_decode_workspace_size(num_seqs, num_heads, head_dim,
                                                     max_context_len))


def decode(q, k_cache, v_cache, block_tables, context_lens, max_context_len, scale=None,
           out=None, workspace=None, block_scales=None, block_flags=None):
    """Decode attention: q [B, Hq, D] -> out [B, Hq, D].  block_scales
    (f32 [NB]) marks the f32 caches as quantised (pa_decode_quantized);
    block_flags (uint8 [NB]) FP8 caches written with flags
    (pa_decode_fp8_flagged)."""
    _dev(q, k_cache, v_cache, block_tables, context_lens)
    nb, hkv, d = _cache_dims(k_cache, v_cache)
    b, hq, dq = q.shape
    if dq != d:
        raise ValueError("q must be [B, Hq, D]")
    code = _cache_code(k_cache, q)
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise ValueError("block_tables / context_lens must be int32")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    need = decode_workspace_size(b, hq, d, max_context_len)
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    lib = _lib.load()
    if block_scales is not None:
        _quant_scales(block_scales, k_cache, nb)
        _check("pa_decode_quantized", lib.pa_decode_quantized(
            _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_scales),
            _ptr(block_tables), block_tables.shape[1], _ptr(context_lens), max_context_len, b, hq,
            hkv, d, nb, float(scale), _ptr(workspace), ws_bytes, _stream(q)))
        return out
    if block_flags is not None:
        if k_cache.dtype != torch.uint8:
            raise ValueError("block_flags are for FP8 caches")
        _flags(block_flags, nb)
        _check("pa_decode_fp8_flagged", lib.pa_decode_fp8_flagged(
            _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables),
            block_tables.shape[1], _ptr(context_lens), max_context_len, b, hq, hkv, d, nb,
            float(scale), _ptr(workspace), ws_bytes, _ptr(block_flags), _stream(q)))
        return out
    _check("pa_decode", lib.pa_decode(
        _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables),
        block_tables.shape[1], _ptr(context_lens), max_context_len, b, hq, hkv, d, nb,
        float(scale), _ptr(workspace), ws_bytes, code, _stream(q)))
    return out


def _quant_scales(block_scales, k_cache, nb):
    _dev(block_scales)
    if block_scales.dtype != torch.float32 or block_scales.shape != (nb,):
        raise ValueError("block_scales must be f32 [num_blocks]")
    if k_cache.dtype != torch.float32:
        raise ValueError("quantised caches are f32")


def prefill(q, k_cache, v_cache, block_tables, cu_q_lens, past_lens, max_q_len, scale=None,
            out=None, block_scales=None):
    """Chunked causal prefill: q [total_q, Hq, D] -> out [total_q, Hq, D].
    block_scales (f32 [NB]) marks the f32 caches as quantised."""
    _dev(q, k_cache, v_cache, block_tables, cu_q_lens, past_lens)
    nb, hkv, d = _cache_dims(k_cache, v_cache)
    tq, hq, dq = q.shape
    if dq != d:
        raise ValueError("q must be [total_q, Hq, D]")
    code = _cache_code(k_cache, q)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty_like(q)
    lib = _lib.load()
    if block_scales is not None:
        _quant_scales(block_scales, k_cache, nb)
        _check("pa_prefill_quantized", lib.pa_prefill_quantized(
            _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_scales),
            _ptr(block_tables), block_tables.shape[1], _ptr(cu_q_lens), _ptr(past_lens),
            block_tables.shape[0], tq, max_q_len, hq, hkv, d, nb, float(scale), _stream(q)))
        return out
    _check("pa_prefill", lib.pa_prefill(
        _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables),
        block_tables.shape[1], _ptr(cu_q_lens), _ptr(past_lens), block_tables.shape[0], tq,
        max_q_len, hq, hkv, d, nb, float(scale), code, _stream(q)))
    return out


ROPE_TYPES = {"default": 0, "linear": 1, "yarn": 2, "dynamic": 3, "su": 4}


def rope_inv_freq(head_dim, theta, rope_type="default", factor=1.0, original_max_position=0,
                  cur_seq_len=0, short_factor=None, long_factor=None):
    """Host RoPE inverse-frequency table (numpy float32 [head_dim // 2])."""
    import numpy as np

    out = np.zeros(head_dim // 2, dtype=np.float32)

    def arr(a):
        if a is None:
            return None
        a = np.ascontiguousarray(a, dtype=np.float32)
        return a.ctypes.data_as(C.c_void_p)

    sf = None if short_factor is None else np.ascontiguousarray(short_factor, dtype=np.float32)
    lf = None if long_factor is None else np.ascontiguousarray(long_factor, dtype=np.float32)
    lib = _lib.load()
    _check("pa_rope_inv_freq", lib.pa_rope_inv_freq(
        head_dim, float(theta), ROPE_TYPES[rope_type], float(factor), int(original_max_position),
        int(cur_seq_len), arr(sf), arr(lf), out.ctypes.data_as(C.c_void_p)))
    return out


def rope_reshape_and_cache(q, key, value, k_cache, v_cache, slot_mapping, positions, inv_freq):
    """Rotate q [T, Hq, D] in place; rotate key [T, Hkv, D] into the K cache
    and copy value into the V cache at slot_mapping (int64); positions int64,
    inv_freq float32 [D/2] on the device."""
    _dev(k_cache, v_cache, slot_mapping, positions, inv_freq)
    nb, h, d = _cache_dims(k_cache, v_cache)
    t, hq, dq = q.shape
    if dq != d or key.shape[1:] != (h, d) or value.shape != key.shape or key.shape[0] != t:
        raise ValueError("q [T, Hq, D], key/value [T, Hkv, D] must match the cache")
    if positions.shape != (t,) or slot_mapping.shape != (t,) or inv_freq.shape != (d // 2,):
        raise ValueError("positions / slot_mapping [T], inv_freq [D/2]")
    if positions.dtype != torch.int64 or slot_mapping.dtype != torch.int64 or \
            inv_freq.dtype != torch.float32:
        raise ValueError("positions / slot_mapping int64, inv_freq float32")
    for x in (q, key, value):
        if x.dtype != k_cache.dtype or not x.is_cuda or not _rows_ok(x, x.shape[1], d):
            raise ValueError("q/key/value rows must be contiguous [H, D] in the cache dtype, "
                             "not overlapping")
    lib = _lib.load()
    _check("pa_rope_reshape_and_cache", lib.pa_rope_reshape_and_cache(
        _ptr(q), q.stride(0), _ptr(key), key.stride(0), _ptr(value), value.stride(0),
        _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), _ptr(positions), _ptr(inv_freq), t, hq,
        h, d, nb, _dtype_code(k_cache), _stream(q)))


def _norm_args(residual, weight, add, out, bias=None):
    _dev(residual, weight)
    rows, hidden = residual.shape
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (hidden,) or t.dtype != residual.dtype):
            raise ValueError(f"{name} must be [hidden] in the residual dtype")
    if bias is not None:
        _dev(bias)
    if add is not None:
        _dev(add)
        if add.shape != residual.shape or add.dtype != residual.dtype:
            raise ValueError("add must match residual")
    if out is None:
        out = torch.empty_like(residual)
    return rows, hidden, out


def rms_norm(residual, weight, eps, add=None, out=None):
    """pa_rms_norm: residual += add (in place, when given), then
    out = residual / sqrt(mean(residual^2) + eps) * weight; [rows, hidden]."""
    rows, hidden, out = _norm_args(residual, weight, add, out)
    lib = _lib.load()
    _check("pa_rms_norm", lib.pa_rms_norm(
        _ptr(out), _ptr(residual), _ptr(add), _ptr(weight), rows, hidden, float(eps),
        _dtype_code(residual), _stream(residual)))
    return out


def layer_norm(residual, weight, eps, bias=None, add=None, out=None):
    """pa_layer_norm (LnLayerNorm, crates/model/src/components/norm/layer_norm.rs:26-39):
    residual += add (in place, when given), then
    out = (residual - mean) / sqrt(var + eps) * weight + bias; [rows, hidden]."""
    rows, hidden, out = _norm_args(residual, weight, add, out, bias)
    lib = _lib.load()
    _check("pa_layer_norm", lib.pa_layer_norm(
        _ptr(out), _ptr(residual), _ptr(add), _ptr(weight), _ptr(bias), rows, hidden,
        float(eps), _dtype_code(residual), _stream(residual)))
    return out


def silu_mul(gate_up, out=None):
    """pa_silu_mul: gate_up [rows, 2 * inter] -> silu(gate) * up [rows, inter]."""
    _dev(gate_up)
    rows, two = gate_up.shape
    inter = two // 2
    if out is None:
        out = torch.empty(rows, inter, dtype=gate_up.dtype, device=gate_up.device)
    lib = _lib.load()
    _check("pa_silu_mul", lib.pa_silu_mul(_ptr(out), _ptr(gate_up), rows, inter,
                                          _dtype_code(gate_up), _stream(gate_up)))
    return out


def argmax(logits, out=None):
    """pa_argmax: greedy token ids of logit rows [rows, vocab] (bf16 or f32,
    unit stride along the vocab) -> int64 [rows]; the first index of the
    largest value, NaN never chosen, 0 for a row with nothing above -inf
    (argmax_logits, crates/traits/src/sampling.rs:439-453)."""
    if not logits.is_cuda:
        raise ValueError("argmax: expected a device tensor")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("argmax: logits must be [rows, vocab] with unit column stride")
    rows, cols = logits.shape
    if rows > 1 and logits.stride(0) < cols:
        logits = logits.contiguous()  # rows that overlap (e.g. an expanded view)
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    lib = _lib.load()
    _check("pa_argmax", lib.pa_argmax(_ptr(out), _ptr(logits), rows, cols,
                                      logits.stride(0) if rows > 1 else cols,
                                      _dtype_code(logits), _stream(logits)))
    return out


def sample_workspace_size(rows):
    return _lib.load().pa_sample_workspace_size(rows)


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None,
           workspace=None):
    """pa_sample: token ids drawn from logit rows [rows, vocab] (bf16 or f32, unit
    stride along the vocab) with the uniform numbers `uniform` (f32 [rows], in
    [0, 1)) -> int64 [rows].  temperature, top_p, min_p (f32 [rows]) and top_k
    (int32 [rows]): each row's settings, None for 1, off, off, off; a temperature
    of 0 is the argmax.  workspace: sample_workspace_size(rows) bytes (uint8)."""
    if not logits.is_cuda:
        raise ValueError("sample: expected a device tensor")
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("sample: logits must be [rows, vocab] with unit column stride")
    rows, cols = logits.shape
    device = logits.device
    code = _dtype_code(logits)
    if not 0 < cols <= 1 << 22 or rows > 65535:
        raise ValueError(f"sample: {rows} rows of {cols} (at most 65535 of 2^22)")
    if rows > 1 and logits.stride(0) < cols:
        logits = logits.contiguous()  # rows that overlap (e.g. an expanded view)
    ptrs = []
    for name, t, dtype in (("uniform", uniform, torch.float32),
                           ("temperature", temperature, torch.float32),
                           ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
        if t is None and name != "uniform":
            ptrs.append(None)
            continue
        if t is None or not _mx_like(t, (rows,), dtype, device):
            raise ValueError(f"{name}: expected a contiguous {dtype} tensor [{rows}] on {device}")
        ptrs.append(t.data_ptr())
    if out is None:
        out = torch.empty_strided((rows,), (1,), dtype=torch.int64, device=device)
    elif not _mx_like(out, (rows,), torch.int64, device):
        _mx_refuse("out", out, (rows,), torch.int64, device)
    if workspace is None:
        workspace = torch.empty_strided((sample_workspace_size(rows),), (1,), dtype=torch.uint8,
                                        device=device)
    elif workspace.device != device or workspace.dtype != torch.uint8 or \
            not workspace.is_contiguous():
        raise ValueError(f"workspace: expected a contiguous uint8 tensor on {device}")
    _mx_call("pa_sample", device, out.data_ptr(), logits.data_ptr(), *ptrs, rows, cols,
             logits.stride(0) if rows > 1 else cols, workspace.data_ptr(), workspace.numel(), code)
    return out


ACT_NONE, ACT_SILU_MUL = 0, 1
LINEAR_RMS_IN, LINEAR_ADD_OUT = 1, 2


class PackedWeight:
    """A bf16 weight [N, K] repacked by pa_linear_pack (see pa_dense.h); pass
    it to linear() in place of the row-major tensor.  col_scale [K] (bf16):
    folded into the columns (a norm weight in front of the projection).
    rope_heads=(num_heads, num_kv_heads, head_dim): the fused QKV weight
    packed by pa_linear_pack_qkv for linear_rope_cache (rotation pairs in
    one wavefront); linear() does not take it."""

    def __init__(self, weight, col_scale=None, rope_heads=None):
        _dev(weight)
        if not weight.is_contiguous():
            raise ValueError("pa_linear_pack takes a contiguous weight")
        if col_scale is not None and (col_scale.shape != (weight.shape[1],) or
                                      col_scale.dtype != weight.dtype):
            raise ValueError("col_scale must be [K] in the weight's dtype")
        self.shape = tuple(weight.shape)
        self.dtype = weight.dtype
        self.data = torch.empty_like(weight)
        self.rope_heads = tuple(rope_heads) if rope_heads is not None else None
        lib = _lib.load()
        if rope_heads is None:
            _check("pa_linear_pack", lib.pa_linear_pack(
                _ptr(self.data), _ptr(weight), _ptr(col_scale), weight.shape[0],
                weight.shape[1], _dtype_code(weight), _stream(weight)))
        else:
            hq, hkv, d = rope_heads
            if weight.shape[0] != (hq + 2 * hkv) * d:
                raise ValueError(f"weight {self.shape} is not a fused QKV weight of "
                                 f"{hq} + 2 x {hkv} heads of {d}")
            _check("pa_linear_pack_qkv", lib.pa_linear_pack_qkv(
                _ptr(self.data), _ptr(weight), _ptr(col_scale), hq, hkv, d, weight.shape[1],
                _dtype_code(weight), _stream(weight)))


def linear_rope_cache(x, weight, bias, positions, slot_mapping, inv_freq, k_cache, v_cache,
                      rms_eps=None, out=None):
    """pa_linear_rope_cache: the fused QKV projection of x [rows, K] with q and
    k rotated (positions [rows] int64, inv_freq [D/2] f32) and each token's
    k / v written to its slot (slot_mapping [rows] int64) of the caches
    (k_cache [NB, Hkv, 16, D], token-minor v_cache [NB, Hkv, D, 16], bf16).
    weight: PackedWeight(w_qkv, rope_heads=(Hq, Hkv, D)).  Returns out
    [rows, (Hq + 2 Hkv) D] (rotated q and k, v)."""
    if not isinstance(weight, PackedWeight) or weight.rope_heads is None:
        raise ValueError("linear_rope_cache takes a PackedWeight with rope_heads")
    hq, hkv, d = weight.rope_heads
    _dev(x, weight.data, positions, slot_mapping, inv_freq, k_cache, v_cache)
    rows, k = x.shape
    if weight.shape[1] != k:
        raise ValueError(f"weight {weight.shape} does not match x {tuple(x.shape)}")
    if positions.shape != (rows,) or slot_mapping.shape != (rows,) or \
            positions.dtype != torch.int64 or slot_mapping.dtype != torch.int64:
        raise ValueError("positions / slot_mapping must be int64 [rows]")
    if k_cache.shape[1:] != (hkv, BLOCK_SIZE, d) or v_cache.shape != (k_cache.shape[0], hkv, d,
                                                                       BLOCK_SIZE):
        raise ValueError("caches must be [NB, Hkv, 16, D] and [NB, Hkv, D, 16]")
    if bias is not None:
        _dev(bias)
        if bias.shape != (weight.shape[0],):
            raise ValueError("bias must be [(Hq + 2 Hkv) D]")
    if out is None:
        out = torch.empty(rows, weight.shape[0], dtype=x.dtype, device=x.device)
    _check("pa_linear_rope_cache", _lib.load().pa_linear_rope_cache(
        _ptr(out), _ptr(x), _ptr(weight.data), _ptr(bias), rows, hq, hkv, d, k,
        LINEAR_RMS_IN if rms_eps is not None else 0,
        float(rms_eps) if rms_eps is not None else 0.0, _ptr(positions), _ptr(slot_mapping),
        _ptr(inv_freq), _ptr(k_cache), _ptr(v_cache), k_cache.shape[0], _dtype_code(x),
        _stream(x)))
    return out


def linear_workspace_size(rows, n, k, act=ACT_NONE):
    """pa_linear_workspace_size: bytes of pa_linear's K-split workspace for
    this shape (0: the shape does not split)."""
    return _lib.load().pa_linear_workspace_size(rows, n, k, act)


def linear_workspace(rows, n, k, act=ACT_NONE, device="cuda"):
    """A zeroed workspace for pa_linear's K split at this shape (uint8 device
    tensor), or None when the shape does not split.  One workspace serves
    any number of calls that run one after another (each leaves its
    counters zero), e.g. every layer of a model, if it is sized for the
    largest of them."""
    nbytes = linear_workspace_size(rows, n, k, act)
    return torch.zeros(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def linear(x, weight, bias=None, act=ACT_NONE, out=None, rms_eps=None, add_to_out=False,
           workspace=None):
    """pa_linear: x [rows, K] bf16, weight [N, K] (or the fused gate|up
    [2 N, K] with act=ACT_SILU_MUL), row-major or a PackedWeight -> out
    [rows, N] bf16.  rms_eps: RMS-normalise the rows of x on the fly (the
    norm weight folded into a PackedWeight's col_scale); add_to_out: out is
    the residual stream, updated in place with the result; workspace: from
    linear_workspace (K split over several workgroups per tile) or None."""
    packed = isinstance(weight, PackedWeight)
    if packed and weight.rope_heads is not None:
        raise ValueError("a weight packed with rope_heads is for linear_rope_cache")
    wt = weight.data if packed else weight
    _dev(x, wt)
    rows, k = x.shape
    n = weight.shape[0] // (2 if act == ACT_SILU_MUL else 1)
    if weight.shape[1] != k:
        raise ValueError(f"weight {tuple(weight.shape)} does not match x {tuple(x.shape)}")
    if not (x.is_contiguous() and wt.is_contiguous()):
        raise ValueError("pa_linear takes contiguous x and weight")
    if bias is not None and (bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError(f"bias {tuple(bias.shape)} does not match {n} outputs")
    if out is None:
        if add_to_out:
            raise ValueError("add_to_out needs out")
        out = torch.empty(rows, n, dtype=x.dtype, device=x.device)
    if workspace is not None:
        _dev(workspace)
        if workspace.dtype != torch.uint8:
            raise ValueError("workspace: expected a uint8 tensor from linear_workspace")
    flags = (LINEAR_RMS_IN if rms_eps is not None else 0) | (LINEAR_ADD_OUT if add_to_out else 0)
    lib = _lib.load()
    _check("pa_linear", lib.pa_linear(_ptr(out), _ptr(x), _ptr(wt),
                                      _ptr(bias) if bias is not None else None, rows, n, k, act,
                                      1 if packed else 0, flags,
                                      float(rms_eps) if rms_eps is not None else 0.0,
                                      _ptr(workspace) if workspace is not None else None,
                                      workspace.numel() if workspace is not None else 0,
                                      _dtype_code(x), _stream(x)))
    return out


# ---- the projections in MXFP8 (pa_dense.h) ---------------------------------


def _mx_call(fn, device, *args):
    """Calls a libpa entry point on the current stream of `device`, with that
    device current.  Pointers as plain integers, and the raw stream: a decode
    step's calls are a few microseconds each, of which the objects in between
    would be most (quantize_mx of 32 rows: 12.7 us with them)."""
    index = device.index
    call = getattr(_lib.load(), fn)
    if torch._C._cuda_getDevice() == index:  # a tensor of `device` exists: CUDA is up
        rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _check(fn, rc)


def _mx_like(t, shape, dtype, device):
    return (t.shape == shape and t.dtype == dtype and t.device == device and
            t.is_contiguous())


def _mx_refuse(name, t, shape, dtype, device):
    raise ValueError(f"{name}: expected a contiguous {dtype} tensor {tuple(shape)} on {device}, "
                     f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _mx_sizes(rows, cols):
    """Refuses what the entry points cannot take (int32 rows, 2^22 columns)
    before ctypes cuts it to 32 bits."""
    if not 0 <= rows < 1 << 31 or not 0 < cols <= 1 << 22:
        raise ValueError(f"MXFP8 of {rows} x {cols}")


class MxRows:
    """MXFP8 rows [rows, cols]: codes uint8 [rows, Kp] (Kp = cols rounded up to
    128), scales uint8 [Kp / 128, R, 4] (R = rows rounded up to 16), see
    pa_dense.h."""

    __slots__ = ("codes", "scales", "rows", "cols")

    def __init__(self, codes, scales, rows, cols):
        _mx_sizes(rows, cols)
        self.codes, self.scales, self.rows, self.cols = codes, scales, rows, cols
        kp = -(-cols // 128) * 128
        if codes.shape != (rows, kp) or scales.shape != (kp // 128, -(-rows // 16) * 16, 4):
            raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are "
                             f"not MXFP8 rows of {rows} x {cols}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not codes.is_cuda:
            raise ValueError("MXFP8 rows are uint8 device tensors")
        if codes.device != scales.device or not (codes.is_contiguous() and
                                                 scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous, on one device")

    @classmethod
    def empty(cls, rows, cols, device="cuda"):
        """Rows whose arrays are allocated and not filled."""
        _mx_sizes(rows, cols)
        self = cls.__new__(cls)
        kp = -(-cols // 128) * 128
        pad = -(-rows // 16) * 16
        # a microsecond less than torch.empty, of a decode step's call of nine
        self.codes = torch.empty_strided((rows, kp), (kp, 1), dtype=torch.uint8, device=device)
        self.scales = torch.empty_strided((kp // 128, pad, 4), (pad * 4, 4, 1),
                                          dtype=torch.uint8, device=device)
        self.rows, self.cols = rows, cols
        return self


def _mx_out(out, rows, cols, device):
    if out is None:
        return MxRows.empty(rows, cols, device)
    if (out.rows, out.cols) != (rows, cols) or out.codes.device != device:
        raise ValueError(f"out holds {out.rows} x {out.cols} on {out.codes.device}, not "
                         f"{rows} x {cols} on {device}")
    return out


def quantize_mx(x, out=None):
    """pa_quantize_mx: x [rows, cols] (bf16 or f32, unit stride along a row,
    rows that do not overlap) -> MxRows."""
    if not x.is_cuda or x.dim() != 2:
        raise ValueError("quantize_mx: expected a device tensor [rows, cols]")
    rows, cols = x.shape
    pitch, step = x.stride()
    if (cols > 1 and step != 1) or (rows > 1 and pitch < cols):
        raise ValueError("quantize_mx: rows must have unit stride and not overlap")
    code = _dtype_code(x)
    device = x.device
    out = _mx_out(out, rows, cols, device)
    _mx_call("pa_quantize_mx", device, out.codes.data_ptr(), out.scales.data_ptr(),
             x.data_ptr(), rows, cols, pitch if rows > 1 else cols, code)
    return out


def rms_norm_mx(residual, weight, eps, add=None, residual_out=None, out=None):
    """pa_rms_norm_mx: residual + add (when given; into residual_out, by
    default residual itself), then its RMSNorm as MxRows; [rows, hidden]."""
    if not residual.is_cuda or residual.dim() != 2 or not residual.is_contiguous():
        raise ValueError("rms_norm_mx: expected a contiguous device tensor [rows, hidden]")
    shape, dtype, device = residual.shape, residual.dtype, residual.device
    rows, hidden = shape
    code = _dtype_code(residual)
    total = None
    if not _mx_like(weight, (hidden,), dtype, device):
        _mx_refuse("weight", weight, (hidden,), dtype, device)
    if add is not None:
        if not _mx_like(add, shape, dtype, device):
            _mx_refuse("add", add, shape, dtype, device)
        if residual_out is None:
            residual_out = residual
        elif not _mx_like(residual_out, shape, dtype, device):
            _mx_refuse("residual_out", residual_out, shape, dtype, device)
        add, total = add.data_ptr(), residual_out.data_ptr()
    elif residual_out is not None:
        raise ValueError("residual_out holds the sum with add")
    out = _mx_out(out, rows, hidden, device)
    _mx_call("pa_rms_norm_mx", device, out.codes.data_ptr(), out.scales.data_ptr(), total,
             residual.data_ptr(), add, weight.data_ptr(), rows, hidden, eps, code)
    return out


class MxWeight:
    """A weight [N, K] (bf16 or f32, contiguous) quantised to MXFP8 in the
    layout that linear_mx reads (pa_linear_mx_pack)."""

    def __init__(self, weight):
        if not weight.is_cuda or weight.dim() != 2 or not weight.is_contiguous():
            raise ValueError("MxWeight: expected a contiguous device tensor [N, K]")
        lib = _lib.load()
        n, k = self.shape = tuple(weight.shape)
        _mx_sizes(n, k)
        code = _dtype_code(weight)
        self.codes = torch.empty(lib.pa_mx_weight_bytes(n, k), dtype=torch.uint8,
                                 device=weight.device)
        self.scales = torch.empty(lib.pa_mx_scale_bytes(n, k), dtype=torch.uint8,
                                  device=weight.device)
        _mx_call("pa_linear_mx_pack", weight.device, self.codes.data_ptr(),
                 self.scales.data_ptr(), weight.data_ptr(), n, k, code)

    @classmethod
    def from_packed(cls, codes, scales, rows, cols):
        """A weight [rows, cols] whose packed codes and scales (flat uint8)
        are at hand, e.g. from a checkpoint."""
        _mx_sizes(rows, cols)
        self = cls.__new__(cls)
        self.shape, self.codes, self.scales = (rows, cols), codes, scales
        size = -(-rows // 16) * 16 * (-(-cols // 128) * 128)  # pa_mx_weight_bytes
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or not codes.is_cuda or \
                rows == 0 or codes.shape != (size,) or scales.shape != (size // 32,):
            raise ValueError(f"not the packed MXFP8 codes and scales of {rows} x {cols}")
        if codes.device != scales.device or not (codes.is_contiguous() and
                                                 scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous, on one device")
        return self

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


def linear_mx(x, weight, bias=None, act=ACT_NONE, residual=None, out=None, mx_out=False):
    """pa_linear_mx: x MxRows [rows, K], weight MxWeight [N, K] (or the fused
    gate|up [2 N, K] with act=ACT_SILU_MUL) -> [rows, N] bf16, with bias [N]
    and residual [rows, N] (bf16; out may be the residual itself) added before
    the one rounding; mx_out (with ACT_SILU_MUL): -> MxRows."""
    if not isinstance(x, MxRows) or not isinstance(weight, MxWeight):
        raise ValueError("linear_mx takes MxRows and an MxWeight")
    device, rows, k = x.codes.device, x.rows, x.cols
    n, wk = weight.shape
    if act == ACT_SILU_MUL:
        n, odd = divmod(n, 2)
        if odd:
            raise ValueError(f"weight {weight.shape} is not a gate|up matrix")
    elif mx_out:
        raise ValueError("an MXFP8 output needs the SwiGLU epilogue")
    if wk != k or weight.codes.device != device:
        raise ValueError(f"weight {weight.shape} on {weight.codes.device} does not match x "
                         f"{rows} x {k} on {device}")
    bf16, shape = torch.bfloat16, (rows, n)
    if bias is not None:
        if not _mx_like(bias, (n,), bf16, device):
            _mx_refuse("bias", bias, (n,), bf16, device)
        bias = bias.data_ptr()
    if residual is not None:
        if not _mx_like(residual, shape, bf16, device):
            _mx_refuse("residual", residual, shape, bf16, device)
        residual = residual.data_ptr()
    if mx_out:
        out = _mx_out(out, rows, n, device)
        data, scales = out.codes.data_ptr(), out.scales.data_ptr()
    else:
        if out is None:
            out = torch.empty_strided(shape, (n, 1), dtype=bf16, device=device)
        elif not _mx_like(out, shape, bf16, device):
            _mx_refuse("out", out, shape, bf16, device)
        data, scales = out.data_ptr(), None
    _mx_call("pa_linear_mx", device, data, scales, x.codes.data_ptr(), x.scales.data_ptr(),
             weight.codes.data_ptr(), weight.scales.data_ptr(), bias, residual, rows, n, k, act)
    return out


# ---- the int8 cache (pa.h) --------------------------------------------------


def _int8_like(t, shape, dtype, index):
    """A contiguous tensor of `shape` on the device of this index: _mx_like for calls
    that are as long as their checks (a device's index compares in half the time)."""
    return (t.dtype is dtype and t.get_device() == index and t.is_contiguous() and
            t.shape == shape)


class Int8Cache:
    """One layer's int8 cache: codes k int8 [NB, H, 16, D] and v int8
    [NB, H, D, 16], scale bytes k_scales and v_scales uint8 [NB, H]; a value is
    code * 2^(byte - 127), see pa.h.  Int8Cache.empty makes a zeroed one."""

    __slots__ = ("k", "v", "k_scales", "v_scales", "num_blocks", "num_kv_heads", "head_dim")

    def __init__(self, k, v, k_scales, v_scales):
        shape = k.shape
        if len(shape) != 4 or shape[2] != BLOCK_SIZE:
            raise ValueError("k must be [NB, H, 16, D]")
        nb, h, _, d = shape
        if not k.is_cuda:
            raise ValueError("an int8 cache is on the device")
        i, codes, scales = k.get_device(), torch.int8, torch.uint8
        if not (_int8_like(k, shape, codes, i) and
                _int8_like(v, (nb, h, d, BLOCK_SIZE), codes, i) and
                _int8_like(k_scales, (nb, h), scales, i) and
                _int8_like(v_scales, (nb, h), scales, i)):
            for name, x, s, dtype in (("k", k, shape, codes),
                                      ("v", v, (nb, h, d, BLOCK_SIZE), codes),
                                      ("k_scales", k_scales, (nb, h), scales),
                                      ("v_scales", v_scales, (nb, h), scales)):
                if not _int8_like(x, s, dtype, i):
                    _mx_refuse(name, x, s, dtype, k.device)
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.num_blocks, self.num_kv_heads, self.head_dim = nb, h, d

    @classmethod
    def empty(cls, num_blocks, num_kv_heads, head_dim, device="cuda"):
        """A zeroed cache."""
        def zeros(*shape, dtype=torch.int8):
            return torch.zeros(shape, dtype=dtype, device=device)

        nb, h, d = num_blocks, num_kv_heads, head_dim
        return cls(zeros(nb, h, BLOCK_SIZE, d), zeros(nb, h, d, BLOCK_SIZE),
                   zeros(nb, h, dtype=torch.uint8), zeros(nb, h, dtype=torch.uint8))

    def _ptrs(self):
        return (self.k.data_ptr(), self.v.data_ptr(), self.k_scales.data_ptr(),
                self.v_scales.data_ptr())


def _int8_index(name, t, n, index):
    if not _int8_like(t, (n,), torch.int32, index):
        _mx_refuse(name, t, (n,), torch.int32, f"cuda:{index}")
    return t.data_ptr()


def _int8_tables(tables, index):
    shape = tables.shape
    if len(shape) != 2:
        raise ValueError("block_tables must be [num_seqs, max_blocks_per_seq]")
    if not _int8_like(tables, shape, torch.int32, index):
        _mx_refuse("block_tables", tables, shape, torch.int32, f"cuda:{index}")
    return shape


def append_int8(cache, key, value, block_tables, cu_seq_tokens, context_lens, max_tokens, q=None,
                inv_freq=None):
    """pa_append_int8: quantises key / value [T, H, D] (bf16 or f32, rows that may
    be strided views) into the cache's blocks.  Sequence s owns rows
    cu_seq_tokens[s] .. [s + 1] and has context_lens[s] tokens with them
    (block_tables [B, MBS], cu_seq_tokens [B + 1], context_lens [B], int32);
    max_tokens: the most of any sequence.  With inv_freq (f32 [D / 2]), q
    [T, Hq, D] is rotated in place and the keys on their way."""
    device, h, d = cache.k.device, cache.num_kv_heads, cache.head_dim
    index = device.index
    b, mbs = _int8_tables(block_tables, index)
    shape, dtype = key.shape, key.dtype
    t, code = shape[0] if shape else 0, _dtype_code(key)
    if (q is None) != (inv_freq is None):
        raise ValueError("q is rotated with inv_freq: both or neither")
    hq = 0 if q is None else q.shape[1] if q.dim() == 3 else 0

    def stride(name, x, heads):
        if (x.shape != (t, heads, d) or heads == 0 or x.dtype is not dtype or
                x.get_device() != index):
            raise ValueError(f"{name}: expected {dtype} [{t}, {heads or 'Hq'}, {d}] on "
                             f"{device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
        row, head, one = x.stride()
        if one != 1 or head != d or (t > 1 and row < heads * d):
            raise ValueError(f"{name}: rows must be contiguous [H, D], not overlapping")
        return row if t > 1 else 0

    ks, vs = stride("key", key, h), stride("value", value, h)
    qs = 0 if q is None else stride("q", q, hq)
    if inv_freq is not None and not _mx_like(inv_freq, (d // 2,), torch.float32, device):
        _mx_refuse("inv_freq", inv_freq, (d // 2,), torch.float32, device)
    _mx_call("pa_append_int8", device, *cache._ptrs(), key.data_ptr(), ks, value.data_ptr(), vs,
             None if q is None else q.data_ptr(), qs,
             None if inv_freq is None else inv_freq.data_ptr(), block_tables.data_ptr(), mbs,
             _int8_index("cu_seq_tokens", cu_seq_tokens, b + 1, index),
             _int8_index("context_lens", context_lens, b, index), b, t, max_tokens, hq, h, d,
             cache.num_blocks, code)


def read_kv_int8(cache, block_ids, seq_len):
    """pa_read_kv_int8: one sequence's first seq_len tokens as f32 (k, v)
    [seq_len, H, D]; block_ids int32."""
    device = cache.k.device
    if block_ids.dim() != 1:
        raise ValueError("block_ids must be one-dimensional")
    ids = _int8_index("block_ids", block_ids, block_ids.shape[0], device.index)
    shape = (seq_len, cache.num_kv_heads, cache.head_dim)
    out_k, out_v = (torch.empty(shape, dtype=torch.float32, device=device) for _ in range(2))
    _mx_call("pa_read_kv_int8", device, *cache._ptrs(), ids, block_ids.shape[0], seq_len,
             cache.num_kv_heads, cache.head_dim, cache.num_blocks, out_k.data_ptr(),
             out_v.data_ptr())
    return out_k, out_v


def decode_int8_workspace_size(num_seqs, num_heads, num_kv_heads, head_dim, max_context_len):
    return _lib.load().pa_decode_int8_workspace_size(num_seqs, num_heads, num_kv_heads, head_dim,
                                                     max_context_len)


def _int8_q(q, cache, out):
    index, shape = cache.k.get_device(), q.shape
    if len(shape) != 3 or shape[2] != cache.head_dim:
        raise ValueError("q must be [rows, Hq, D]")
    if not _int8_like(q, shape, torch.bfloat16, index):
        _mx_refuse("q", q, shape, torch.bfloat16, f"cuda:{index}")
    if out is None:
        return torch.empty_like(q), shape
    if not _int8_like(out, shape, torch.bfloat16, index):
        _mx_refuse("out", out, shape, torch.bfloat16, f"cuda:{index}")
    return out, shape


def decode_int8(q, cache, block_tables, context_lens, max_context_len, scale=None, out=None,
                workspace=None):
    """pa_decode_int8: q [B, Hq, D] bf16 -> out [B, Hq, D]."""
    device = cache.k.device
    index = device.index
    out, (n, hq, d) = _int8_q(q, cache, out)
    b, mbs = _int8_tables(block_tables, index)
    if b != n:
        raise ValueError(f"block_tables of {b} sequences, q of {n}")
    lens = _int8_index("context_lens", context_lens, b, index)
    if workspace is None:
        need = decode_int8_workspace_size(b, hq, cache.num_kv_heads, d, max_context_len)
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.device != device or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous on {device}")
    _mx_call("pa_decode_int8", device, out.data_ptr(), q.data_ptr(), *cache._ptrs(),
             block_tables.data_ptr(), mbs, lens, max_context_len, b, hq, cache.num_kv_heads, d,
             cache.num_blocks, 1.0 / math.sqrt(d) if scale is None else scale,
             None if workspace is None else workspace.data_ptr(),
             0 if workspace is None else workspace.numel() * workspace.element_size())
    return out


def prefill_int8(q, cache, block_tables, cu_q_lens, past_lens, max_q_len, scale=None, out=None):
    """pa_prefill_int8: q [total_q, Hq, D] bf16 -> out [total_q, Hq, D]."""
    device = cache.k.device
    index = device.index
    out, (n, hq, d) = _int8_q(q, cache, out)
    b, mbs = _int8_tables(block_tables, index)
    _mx_call("pa_prefill_int8", device, out.data_ptr(), q.data_ptr(), *cache._ptrs(),
             block_tables.data_ptr(), mbs, _int8_index("cu_q_lens", cu_q_lens, b + 1, index),
             _int8_index("past_lens", past_lens, b, index), b, n, max_q_len, hq,
             cache.num_kv_heads, d, cache.num_blocks,
             1.0 / math.sqrt(d) if scale is None else scale)
    return out
