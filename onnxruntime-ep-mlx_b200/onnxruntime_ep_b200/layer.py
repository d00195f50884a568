"""The operators around paged attention in one decoder layer (include/b200_layer.h):
``skip_rms_norm``, ``rotary_append`` and ``shared_prefix_attention``.

Torch only owns device memory and the current stream; the work runs in ``libb200_paged.so``.
Argument errors raise ``B200Error``.  Errors that only the device can see (a slot, position, length
or block id out of range) set a status word; ``check_status=True`` synchronises and raises them.
Every function takes ``stream=`` (default: the current stream).  The first call on a device, and the
first on a stream, allocate their status word and scratch: make them before a graph capture.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _capi
from ._capi import LIB, B200_ERR_WORKSPACE, B200Error, check
from .paged import _DTYPES

_FP8 = torch.float8_e4m3fn
_ACT = {torch.float16: _capi.DTYPE_FLOAT16, torch.bfloat16: _capi.DTYPE_BFLOAT16}
_TABLE = {**_ACT, torch.float32: _capi.DTYPE_FLOAT}
_INDEX = {torch.int32: _capi.DTYPE_INT32, torch.int64: _capi.DTYPE_INT64}
_DENSE = torch.contiguous_format
_E4M3 = _capi.DTYPE_FLOAT8E4M3FN

# The parameter structs of include/b200_layer.h as packed bytes (a decode step makes these calls for
# every layer: packing costs a fraction of filling a ctypes structure field by field).
_NORM = struct.Struct("@5if4q6P")
_ROPE = struct.Struct("@19i6q13PNP")
_PREFIX = struct.Struct("@3i2f9i2q10PNP")
for _which, _layout in enumerate((_NORM, _ROPE, _PREFIX)):
    if LIB.b200_layer_struct_size(_which) != _layout.size:
        raise ImportError("libb200_paged.so: a parameter layout of include/b200_layer.h differs from the binding")

_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice

# one status word per device, zeroed here once: calls only set bits, b200_layer_read_status clears
_status: dict[int, int] = {}
_status_words: list[torch.Tensor] = []

# Scratch per (device, stream), so calls on different streams never share it.  A buffer that became
# too small is kept: a captured graph may still use it (sizes at least double, so the kept ones
# together stay below the current one).
_scratch: dict[tuple[int, int], list[torch.Tensor]] = {}


def _bad(message: str) -> B200Error:
    return B200Error(_capi.B200_ERR_INVALID_ARGUMENT, message)


def _status_ptr(device: int) -> int:
    pointer = _status.get(device)
    if pointer is None:
        word = torch.zeros(1, dtype=torch.int32, device=f"cuda:{device}")
        torch.cuda.synchronize(device)  # zeroed before any stream uses it
        _status_words.append(word)
        pointer = _status[device] = word.data_ptr()
    return pointer


def _on_stream(stream, fn, *args, **kwargs):
    """``fn`` with ``stream`` current, so what it allocates belongs to the stream that uses it."""
    with torch.cuda.stream(stream):
        return fn(*args, **kwargs)


def _call(entry, params, device, check_status=False):
    """Run one library call on the device's current stream."""
    if device != _current_device():
        with torch.cuda.device(device):
            return _call(entry, params, device, check_status)
    stream = _raw_stream(device)
    code = entry(params, stream)
    if code:
        check(code)
    if check_status:
        check(LIB.b200_layer_read_status(_status_ptr(device), stream))


def _call_with_scratch(op, entry, size_entry, layout, fields, device, workspace, check_status):
    """``_call`` for an operator with a workspace: the last three fields are the workspace, its bytes and
    the status word.  Without a caller's workspace it runs in the current stream's own buffer, which
    grows when the library finds it too small."""
    status = _status_ptr(device)
    if workspace is not None:
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.get_device() != device:
            raise B200Error(B200_ERR_WORKSPACE, f"{op}: workspace must be a contiguous uint8 tensor on the caches' device")
        params = layout.pack(*fields, workspace.data_ptr(), workspace.numel(), status)
        return _call(entry, params, device, check_status)
    kept = _scratch.setdefault((device, _raw_stream(device)), [])
    while True:
        last = kept[-1] if kept else None
        params = layout.pack(*fields, last.data_ptr() if kept else 0, last.numel() if kept else 0, status)
        try:
            return _call(entry, params, device, check_status)
        except B200Error as e:
            need = ctypes.c_size_t(0)
            if e.code != B200_ERR_WORKSPACE or size_entry(params, ctypes.byref(need)) or (
                    kept and need.value <= kept[-1].numel()):
                raise
            size = max(need.value, 1 << 20, 2 * kept[-1].numel() if kept else 0)
            kept.append(torch.empty(size, dtype=torch.uint8, device=f"cuda:{device}"))


def _rows(op, name, t, rows, width, dtype, device):
    """Row stride of a [rows, width] tensor of ``dtype`` on ``device`` whose rows are contiguous."""
    if t.dtype is dtype and t.get_device() == device and t.shape == (rows, width):
        if t.is_contiguous():
            return width
        stride, inner = t.stride()
        if (inner == 1 or width == 1) and (stride != 0 or rows == 1):
            return stride if rows > 1 else width
        if stride == 0:  # the library reads a stride of 0 as dense rows
            raise _bad(f"{op}: {name} must not be a broadcast row")
        raise _bad(f"{op}: {name} rows must be contiguous")
    raise _bad(f"{op}: {name} must be a [{rows}, {width}] tensor of {dtype} on cuda:{device}")


def _dense(op, name, t, shape, dtype, device):
    """Address of a contiguous tensor of this shape and type on ``device``."""
    if t is not None and t.dtype is dtype and t.get_device() == device and t.is_contiguous() and t.shape == shape:
        return t.data_ptr()
    raise _bad(f"{op}: {name} must be a contiguous {tuple(shape)} tensor of {dtype} on cuda:{device}")


def _device(op, t):
    device = t.get_device()
    if device < 0:
        raise _bad(f"{op}: tensors must be on a CUDA device")
    return device


def skip_rms_norm(x, residual, weight, *, epsilon=1e-6, out_dtype=None, group_size=0, output=None, scales=None,
                  residual_output=None, stream=None):
    """``s = x + residual`` (fp32), ``y = s / sqrt(mean(s^2) + epsilon) * weight`` per row.

    ``x`` and ``residual`` (or ``None``) are ``[rows, hidden]`` in fp16 / bf16 with contiguous rows.
    Returns ``(y in x's type, s in x's type)``, or with ``out_dtype=torch.float8_e4m3fn``
    ``(codes, scales, s in x's type)``: ``codes * scales`` stands for ``y``, ``scales`` is fp32
    ``[rows, groups]`` with one scale per row (``group_size=0``) or per ``group_size`` channels.
    """
    if stream is not None:
        return _on_stream(stream, skip_rms_norm, x, residual, weight, epsilon=epsilon, out_dtype=out_dtype,
                          group_size=group_size, output=output, scales=scales, residual_output=residual_output)
    op = "SkipRmsNorm"
    dtype = x.dtype
    act = _ACT.get(dtype)
    if act is None or x.dim() != 2:
        raise _bad(f"{op}: x must be a [rows, hidden] tensor of fp16 or bf16")
    rows, hidden = x.shape
    device = _device(op, x)
    stride = _rows(op, "x", x, rows, hidden, dtype, device)
    r_ptr = r_stride = s_ptr = 0
    if residual is not None:
        r_stride = _rows(op, "residual", residual, rows, hidden, dtype, device)
        r_ptr = residual.data_ptr()
    w_ptr = _dense(op, "weight", weight, (hidden,), dtype, device)
    fp8 = out_dtype is _FP8
    if not fp8 and out_dtype is not None and out_dtype is not dtype:
        raise _bad(f"{op}: out_dtype must be x's type or float8_e4m3fn")
    o_stride = ro_stride = hidden
    if output is None:
        output = torch.empty_like(x, dtype=_FP8, memory_format=_DENSE) if fp8 else torch.empty_like(x, memory_format=_DENSE)
    else:
        o_stride = _rows(op, "output", output, rows, hidden, _FP8 if fp8 else dtype, device)
    if fp8:
        groups = -(-hidden // group_size) if group_size > 0 else 1
        if scales is None:
            scales = x.new_empty((rows, groups), dtype=torch.float32)
            s_ptr = scales.data_ptr()
        else:
            s_ptr = _dense(op, "scales", scales, (rows, groups), torch.float32, device)
    if residual_output is None:
        residual_output = torch.empty_like(x, memory_format=_DENSE)
    else:
        ro_stride = _rows(op, "residual_output", residual_output, rows, hidden, dtype, device)
    params = _NORM.pack(rows, hidden, act, _E4M3 if fp8 else act, group_size, epsilon, stride, r_stride, o_stride,
                        ro_stride, x.data_ptr(), r_ptr, w_ptr, output.data_ptr(), s_ptr,
                        residual_output.data_ptr())
    _call(LIB.b200_skip_rms_norm, params, device)
    return (output, scales, residual_output) if fp8 else (output, residual_output)


def rotary_append(query, key, value, key_cache, value_cache, position_ids, cos_cache, sin_cache, slot_mapping, *,
                  num_heads, kv_num_heads, axis_sections=None, rotary_interleaved=0, rotary_offset=0, k_scale=None,
                  v_scale=None, output=None, workspace=None, check_status=False, stream=None):
    """Rotate the new queries and keys and append keys and values to the paged caches (in place).

    ``query`` is ``[tokens, num_heads * d]``; ``key`` and ``value`` are ``[tokens, kv_num_heads * d]``,
    or both ``None`` for packed QKV rows.  ``position_ids`` (int32 / int64) is ``[tokens]`` or
    ``[axes, tokens]``; ``axis_sections`` gives the rotary pairs of each axis (time, height, width,
    ...), in order.  ``cos_cache`` / ``sin_cache`` are ``[positions, rotary_dim / 2]`` in the
    activations' type or fp32.  ``slot_mapping`` (int32) names each token's cache slot, -1 for none;
    of several tokens with one slot the last is stored.  fp8 e4m3 caches take ``k_scale`` and
    ``v_scale`` ``[blocks, kv_num_heads]``.  Returns ``(rotated query, key_cache, value_cache)``.
    """
    if stream is not None:
        return _on_stream(stream, rotary_append, query, key, value, key_cache, value_cache, position_ids, cos_cache,
                          sin_cache, slot_mapping, num_heads=num_heads, kv_num_heads=kv_num_heads,
                          axis_sections=axis_sections, rotary_interleaved=rotary_interleaved, rotary_offset=rotary_offset,
                          k_scale=k_scale, v_scale=v_scale, output=output, workspace=workspace, check_status=check_status)
    op = "RotaryAppend"
    dtype = query.dtype
    act = _ACT.get(dtype)
    if act is None or query.dim() != 2:
        raise _bad(f"{op}: query must be a [tokens, hidden] tensor of fp16 or bf16")
    H, KV = num_heads, kv_num_heads
    shape = key_cache.shape
    if len(shape) != 4 or shape[2] != KV:
        raise _bad(f"{op}: key_cache must be [blocks, block_size, kv_num_heads, head_size]")
    nt = query.shape[0]
    blocks, block_size, _, d = shape
    device = _device(op, query)
    q_ptr = query.data_ptr()
    if key is None and value is None:
        q_stride = k_stride = v_stride = _rows(op, "packed query", query, nt, (H + 2 * KV) * d, dtype, device)
        k_ptr, v_ptr = q_ptr + 2 * H * d, q_ptr + 2 * (H + KV) * d
    elif key is None or value is None:
        raise _bad(f"{op}: key and value must be given together")
    else:
        q_stride = _rows(op, "query", query, nt, H * d, dtype, device)
        k_stride = _rows(op, "key", key, nt, KV * d, dtype, device)
        v_stride = _rows(op, "value", value, nt, KV * d, dtype, device)
        k_ptr, v_ptr = key.data_ptr(), value.data_ptr()
    kc_ptr = _dense(op, "key_cache", key_cache, shape, key_cache.dtype, device)
    vc_ptr = _dense(op, "value_cache", value_cache, shape, key_cache.dtype, device)
    cache = _DTYPES.get(key_cache.dtype)
    ks_ptr = vs_ptr = 0
    if cache != act:
        if cache != _E4M3:
            raise _bad(f"{op}: the cache must have the activations' type or fp8 e4m3")
        ks_ptr = _dense(op, "k_scale", k_scale, (blocks, KV), torch.float32, device)
        vs_ptr = _dense(op, "v_scale", v_scale, (blocks, KV), torch.float32, device)
    table = _TABLE.get(cos_cache.dtype)
    tables = cos_cache.shape
    if table is None or len(tables) != 2:
        raise _bad(f"{op}: cos_cache must be [positions, rotary_dim / 2] of the activations' type or fp32")
    positions, half = tables
    cos_ptr = _dense(op, "cos_cache", cos_cache, tables, cos_cache.dtype, device)
    sin_ptr = _dense(op, "sin_cache", sin_cache, tables, cos_cache.dtype, device)
    index = _INDEX.get(position_ids.dtype)
    places = position_ids.shape
    rank = len(places)
    if index is None or rank not in (1, 2) or places[-1] != nt or position_ids.get_device() != device:
        raise _bad(f"{op}: position_ids must be an int32 or int64 [tokens] or [axes, tokens] tensor on cuda:{device}")
    if position_ids.is_contiguous():
        axis_stride, token_stride = nt, 1
    else:
        if nt > 1 and position_ids.stride(-1) == 0:  # the library reads a token stride of 0 as 1
            position_ids = position_ids.contiguous()
        axis_stride, token_stride = position_ids.stride(0), position_ids.stride(-1)
    axes = 1 if rank == 1 else places[0]
    if axis_sections is None:
        named, sections = 1, (half, 0, 0, 0)
    else:
        named, sections = len(axis_sections), (*axis_sections, 0, 0, 0)[:4]
    if named != axes or axes > 4:
        raise _bad(f"{op}: axis_sections must name the pairs of each of the {axes} position axes (at most 4)")
    slot_ptr = _dense(op, "slot_mapping", slot_mapping, (nt,), torch.int32, device)
    if output is None:
        output = torch.empty_like(query, memory_format=_DENSE) if key is not None else query.new_empty((nt, H * d))
        o_stride = H * d
    else:
        o_stride = _rows(op, "output", output, nt, H * d, dtype, device)
    fields = (H, KV, d, 2 * half, rotary_offset, rotary_interleaved, positions, axes, *sections, act, cache, table, index,
              nt, blocks, block_size, q_stride, k_stride, v_stride, o_stride, axis_stride, token_stride, q_ptr, k_ptr, v_ptr,
              output.data_ptr(), kc_ptr, vc_ptr, position_ids.data_ptr(), cos_ptr, sin_ptr, slot_ptr, ks_ptr, vs_ptr)
    if nt <= _capi.ROTARY_APPEND_SCAN_TOKENS:
        _call(LIB.b200_rotary_append, _ROPE.pack(*fields, 0, 0, _status_ptr(device)), device, check_status)
    else:
        _call_with_scratch(op, LIB.b200_rotary_append, LIB.b200_rotary_append_workspace_size, _ROPE, fields, device,
                           workspace, check_status)
    return output, key_cache, value_cache


def shared_prefix_attention(query, key_cache, value_cache, cumulative_sequence_length, past_seqlens, block_table,
                            prefix_block_table, *, prefix_length, num_heads, kv_num_heads, scale=0.0, softcap=0.0,
                            head_sink=None, output=None, workspace=None, num_sms=0, check_status=False, stream=None):
    """Causal attention of a batch whose sequences share the ``prefix_length`` keys of
    ``prefix_block_table``; sequence ``b`` continues with its own ``past_seqlens[b]`` keys and its new
    tokens, paged by row ``b`` of ``block_table``.

    Every key is read from the caches (``[blocks, block_size, kv_num_heads, d]``, fp16 / bf16), the
    new tokens' included: append them first.  Metadata are int32 device tensors.  Returns the output
    ``[tokens, num_heads * d]``.  The scratch is the current stream's own buffer unless ``workspace``
    (uint8, at least ``b200_shared_prefix_attention_workspace_size`` bytes) is given.
    """
    if stream is not None:
        return _on_stream(stream, shared_prefix_attention, query, key_cache, value_cache, cumulative_sequence_length,
                          past_seqlens, block_table, prefix_block_table, prefix_length=prefix_length, num_heads=num_heads,
                          kv_num_heads=kv_num_heads, scale=scale, softcap=softcap, head_sink=head_sink, output=output,
                          workspace=workspace, num_sms=num_sms, check_status=check_status)
    op = "SharedPrefixAttention"
    dtype = query.dtype
    act = _ACT.get(dtype)
    if act is None or query.dim() != 2:
        raise _bad(f"{op}: query must be a [tokens, hidden] tensor of fp16 or bf16")
    H, KV = num_heads, kv_num_heads
    shape = key_cache.shape
    if len(shape) != 4 or shape[2] != KV:
        raise _bad(f"{op}: key_cache must be [blocks, block_size, kv_num_heads, head_size]")
    nt = query.shape[0]
    blocks, block_size, _, d = shape
    device = _device(op, query)
    q_stride = _rows(op, "query", query, nt, H * d, dtype, device)
    kc_ptr = _dense(op, "key_cache", key_cache, shape, dtype, device)
    vc_ptr = _dense(op, "value_cache", value_cache, shape, dtype, device)
    if block_table.dim() != 2:
        raise _bad(f"{op}: block_table must be [batch, blocks]")
    batch, columns = tables = block_table.shape
    bt_ptr = _dense(op, "block_table", block_table, tables, torch.int32, device)
    past_ptr = _dense(op, "past_seqlens", past_seqlens, (batch,), torch.int32, device)
    cum_ptr = _dense(op, "cumulative_sequence_length", cumulative_sequence_length, (batch + 1,), torch.int32, device)
    pt_ptr = prefix_blocks = sink_ptr = 0
    if prefix_block_table is not None:
        prefix_blocks = prefix_block_table.numel()
        pt_ptr = _dense(op, "prefix_block_table", prefix_block_table, (prefix_blocks,), torch.int32, device)
    if head_sink is not None:
        sink_ptr = _dense(op, "head_sink", head_sink, (H,), dtype, device)
    if output is None:
        output = torch.empty_like(query, memory_format=_DENSE)
        o_stride = H * d
    else:
        o_stride = _rows(op, "output", output, nt, H * d, dtype, device)
    fields = (H, KV, d, scale, softcap, act, nt, batch, blocks, block_size, columns, prefix_length, prefix_blocks, num_sms,
              q_stride, o_stride, query.data_ptr(), kc_ptr, vc_ptr, cum_ptr, past_ptr, bt_ptr, pt_ptr, sink_ptr,
              output.data_ptr())
    _call_with_scratch(op, LIB.b200_shared_prefix_attention, LIB.b200_shared_prefix_attention_workspace_size, _PREFIX,
                       fields, device, workspace, check_status)
    return output
