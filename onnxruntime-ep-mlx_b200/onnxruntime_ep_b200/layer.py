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
import functools

import torch

from . import _capi
from ._capi import LIB, B200Error, RotaryAppendParams, SharedPrefixParams, SkipRmsNormParams, check
from .paged import _DTYPES

_FP8 = torch.float8_e4m3fn
_ACT = {torch.float16: _capi.DTYPE_FLOAT16, torch.bfloat16: _capi.DTYPE_BFLOAT16}
_TABLE = {**_ACT, torch.float32: _capi.DTYPE_FLOAT}
_INDEX = {torch.int32: _capi.DTYPE_INT32, torch.int64: _capi.DTYPE_INT64}
_byref = ctypes.byref

# one status word per device, zeroed here once: calls only set bits, b200_layer_read_status clears
_status: dict[int, torch.Tensor] = {}


# Scratch per (device, stream), so calls on different streams never share it.  A buffer that became
# too small is kept: a captured graph may still use it (sizes at least double, so the kept ones
# together stay below the current one).
_scratch: dict[tuple[int, int], list[torch.Tensor]] = {}


def _bad(message: str) -> B200Error:
    return B200Error(_capi.B200_ERR_INVALID_ARGUMENT, message)


def _status_ptr(device: torch.device) -> int:
    word = _status.get(device.index)
    if word is None:
        word = _status[device.index] = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.synchronize(device)  # zeroed before any stream uses it
    return word.data_ptr()


def _on_stream(fn):
    """Give ``fn`` a ``stream`` argument: it runs with that stream current, so what it allocates belongs
    to the stream that uses it."""

    @functools.wraps(fn)
    def wrapped(*args, stream=None, **kwargs):
        if stream is None:
            return fn(*args, **kwargs)
        with torch.cuda.stream(stream):
            return fn(*args, **kwargs)

    return wrapped


def _call(entry, params, device, check_status=False):
    """Run one library call on the device's current stream."""
    handle = torch.cuda.current_stream(device).cuda_stream
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            check(entry(_byref(params), handle))
            if check_status:
                check(LIB.b200_layer_read_status(_status_ptr(device), handle))
        return
    check(entry(_byref(params), handle))
    if check_status:
        check(LIB.b200_layer_read_status(_status_ptr(device), handle))


def _same_device(op, device, **tensors):
    if device.type != "cuda":
        raise _bad(f"{op}: tensors must be on a CUDA device")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise _bad(f"{op}: {name} is on another device")


def _rows(op, name, t, width):
    """Row stride of a 2-D tensor whose rows are contiguous."""
    if t.dim() != 2 or t.shape[1] != width:
        raise _bad(f"{op}: {name} must be [rows, {width}]")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise _bad(f"{op}: {name} rows must be contiguous")
    if t.shape[0] <= 1:
        return width
    if t.stride(0) == 0:  # the library reads a stride of 0 as dense rows
        raise _bad(f"{op}: {name} must not be a broadcast row")
    return t.stride(0)


def _dense(op, name, t, shape, dtype):
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise _bad(f"{op}: {name} must be a contiguous {tuple(shape)} tensor of {dtype}")


def _workspace(op, device, need, workspace):
    """(pointer, bytes) of the caller's workspace or of the current stream's own one."""
    if not need:
        return None, 0
    if workspace is None:
        kept = _scratch.setdefault((device.index, torch.cuda.current_stream(device).cuda_stream), [])
        if not kept or kept[-1].numel() < need:
            size = max(need, 1 << 20, 2 * kept[-1].numel() if kept else 0)
            kept.append(torch.empty(size, dtype=torch.uint8, device=device))
        workspace = kept[-1]
    elif workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.numel() < need:
        raise B200Error(_capi.B200_ERR_WORKSPACE, f"{op}: workspace must be a contiguous uint8 tensor of at least {need} bytes")
    return workspace.data_ptr(), workspace.numel()


@_on_stream
def skip_rms_norm(x, residual, weight, *, epsilon=1e-6, out_dtype=None, group_size=0, output=None, scales=None,
                  residual_output=None):
    """``s = x + residual`` (fp32), ``y = s / sqrt(mean(s^2) + epsilon) * weight`` per row.

    ``x`` and ``residual`` (or ``None``) are ``[rows, hidden]`` in fp16 / bf16 with contiguous rows.
    Returns ``(y in x's type, s in x's type)``, or with ``out_dtype=torch.float8_e4m3fn``
    ``(codes, scales, s in x's type)``: ``codes * scales`` stands for ``y``, ``scales`` is fp32
    ``[rows, groups]`` with one scale per row (``group_size=0``) or per ``group_size`` channels.
    """
    op = "SkipRmsNorm"
    dtype = x.dtype
    act = _ACT.get(dtype)
    if act is None or x.dim() != 2:
        raise _bad(f"{op}: x must be a [rows, hidden] tensor of fp16 or bf16")
    rows, hidden = x.shape
    device = x.device
    _same_device(op, device, residual=residual, weight=weight, output=output, scales=scales,
                 residual_output=residual_output)
    stride = _rows(op, "x", x, hidden)
    r_stride = 0
    if residual is not None:
        if residual.dtype != dtype or residual.shape[0] != rows:
            raise _bad(f"{op}: residual must have x's shape and type")
        r_stride = _rows(op, "residual", residual, hidden)
    if weight.dtype != dtype or weight.shape != (hidden,) or not weight.is_contiguous():
        raise _bad(f"{op}: weight must be a contiguous [hidden] tensor of x's type")
    fp8 = out_dtype == _FP8
    if not fp8 and out_dtype is not None and out_dtype != dtype:
        raise _bad(f"{op}: out_dtype must be x's type or float8_e4m3fn")
    if output is None:
        output = torch.empty((rows, hidden), dtype=_FP8 if fp8 else dtype, device=device)
        o_stride = hidden
    else:
        if output.dtype != (_FP8 if fp8 else dtype) or output.shape[0] != rows:
            raise _bad(f"{op}: output has another shape or type")
        o_stride = _rows(op, "output", output, hidden)
    group_size = int(group_size)
    if fp8:
        groups = -(-hidden // group_size) if group_size > 0 else 1
        if scales is None:
            scales = torch.empty((rows, groups), dtype=torch.float32, device=device)
        else:
            _dense(op, "scales", scales, (rows, groups), torch.float32)
    if residual_output is None:
        residual_output = torch.empty((rows, hidden), dtype=dtype, device=device)
        ro_stride = hidden
    else:
        if residual_output.dtype != dtype or residual_output.shape[0] != rows:
            raise _bad(f"{op}: residual_output has another shape or type")
        ro_stride = _rows(op, "residual_output", residual_output, hidden)
    p = SkipRmsNormParams(
        rows, hidden, act, _capi.DTYPE_FLOAT8E4M3FN if fp8 else act, group_size, epsilon, stride, r_stride, o_stride,
        ro_stride, x.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(),
        output.data_ptr(), scales.data_ptr() if fp8 else None, residual_output.data_ptr())
    _call(LIB.b200_skip_rms_norm, p, device)
    return (output, scales, residual_output) if fp8 else (output, residual_output)


@_on_stream
def rotary_append(query, key, value, key_cache, value_cache, position_ids, cos_cache, sin_cache, slot_mapping, *,
                  num_heads, kv_num_heads, axis_sections=None, rotary_interleaved=0, rotary_offset=0, k_scale=None,
                  v_scale=None, output=None, workspace=None, check_status=False):
    """Rotate the new queries and keys and append keys and values to the paged caches (in place).

    ``query`` is ``[tokens, num_heads * d]``; ``key`` and ``value`` are ``[tokens, kv_num_heads * d]``,
    or both ``None`` for packed QKV rows.  ``position_ids`` (int32 / int64) is ``[tokens]`` or
    ``[axes, tokens]``; ``axis_sections`` gives the rotary pairs of each axis (time, height, width,
    ...), in order.  ``cos_cache`` / ``sin_cache`` are ``[positions, rotary_dim / 2]`` in the
    activations' type or fp32.  ``slot_mapping`` (int32) names each token's cache slot, -1 for none;
    of several tokens with one slot the last is stored.  fp8 e4m3 caches take ``k_scale`` and
    ``v_scale`` ``[blocks, kv_num_heads]``.  Returns ``(rotated query, key_cache, value_cache)``.
    """
    op = "RotaryAppend"
    act = _ACT.get(query.dtype)
    if act is None or query.dim() != 2:
        raise _bad(f"{op}: query must be a [tokens, hidden] tensor of fp16 or bf16")
    H, KV = int(num_heads), int(kv_num_heads)
    if key_cache.dim() != 4 or key_cache.shape[2] != KV:
        raise _bad(f"{op}: key_cache must be [blocks, block_size, kv_num_heads, head_size]")
    nt = query.shape[0]
    blocks, block_size, _, d = key_cache.shape
    device = query.device
    _same_device(op, device, key=key, value=value, key_cache=key_cache, value_cache=value_cache,
                 position_ids=position_ids, cos_cache=cos_cache, sin_cache=sin_cache, slot_mapping=slot_mapping,
                 k_scale=k_scale, v_scale=v_scale, output=output, workspace=workspace)
    if key is None and value is None:
        q_stride = k_stride = v_stride = _rows(op, "packed query", query, (H + 2 * KV) * d)
        q_ptr = query.data_ptr()
        k_ptr, v_ptr = q_ptr + 2 * H * d, q_ptr + 2 * (H + KV) * d
    elif key is None or value is None:
        raise _bad(f"{op}: key and value must be given together")
    else:
        if key.dtype != query.dtype or value.dtype != query.dtype or key.shape[0] != nt or value.shape[0] != nt:
            raise _bad(f"{op}: key and value must have the query's tokens and type")
        q_stride = _rows(op, "query", query, H * d)
        k_stride, v_stride = _rows(op, "key", key, KV * d), _rows(op, "value", value, KV * d)
        q_ptr, k_ptr, v_ptr = query.data_ptr(), key.data_ptr(), value.data_ptr()
    cache_dtype = _DTYPES.get(key_cache.dtype)
    if value_cache.dtype != key_cache.dtype or value_cache.shape != key_cache.shape or not (
            key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise _bad(f"{op}: key_cache and value_cache must be contiguous and alike")
    if cache_dtype not in (act, _capi.DTYPE_FLOAT8E4M3FN):
        raise _bad(f"{op}: the cache must have the activations' type or fp8 e4m3")
    ks_ptr = vs_ptr = None
    if cache_dtype != act:
        if k_scale is None or v_scale is None:
            raise _bad(f"{op}: fp8 caches require k_scale and v_scale")
        _dense(op, "k_scale", k_scale, (blocks, KV), torch.float32)
        _dense(op, "v_scale", v_scale, (blocks, KV), torch.float32)
        ks_ptr, vs_ptr = k_scale.data_ptr(), v_scale.data_ptr()
    table = _TABLE.get(cos_cache.dtype)
    if (table is None or cos_cache.dim() != 2 or sin_cache.dtype != cos_cache.dtype
            or sin_cache.shape != cos_cache.shape or not (cos_cache.is_contiguous() and sin_cache.is_contiguous())):
        raise _bad(f"{op}: cos_cache and sin_cache must be contiguous [positions, rotary_dim / 2] tensors alike")
    half = cos_cache.shape[1]
    index = _INDEX.get(position_ids.dtype)
    if index is None or position_ids.dim() not in (1, 2) or position_ids.shape[-1] != nt:
        raise _bad(f"{op}: position_ids must be an int32 or int64 [tokens] or [axes, tokens] tensor")
    if nt > 1 and position_ids.stride(-1) == 0:  # the library reads a token stride of 0 as 1
        position_ids = position_ids.contiguous()
    axes = 1 if position_ids.dim() == 1 else position_ids.shape[0]
    sections = (half,) if axis_sections is None else tuple(axis_sections)
    if len(sections) != axes or axes > 4:
        raise _bad(f"{op}: axis_sections must name the pairs of each of the {axes} position axes (at most 4)")
    if slot_mapping.dtype != torch.int32 or slot_mapping.shape != (nt,) or not slot_mapping.is_contiguous():
        raise _bad(f"{op}: slot_mapping must be a contiguous int32 [tokens] tensor")
    if output is None:
        output = torch.empty((nt, H * d), dtype=query.dtype, device=device)
        o_stride = H * d
    else:
        if output.dtype != query.dtype or output.shape[0] != nt:
            raise _bad(f"{op}: output has another shape or type")
        o_stride = _rows(op, "output", output, H * d)
    p = RotaryAppendParams(
        H, KV, d, 2 * half, int(rotary_offset), int(rotary_interleaved), cos_cache.shape[0], axes, sections,
        act, cache_dtype, table, index, nt, blocks, block_size, q_stride, k_stride, v_stride, o_stride,
        position_ids.stride(0) if axes > 1 else 0, position_ids.stride(-1), q_ptr, k_ptr, v_ptr, output.data_ptr(),
        key_cache.data_ptr(), value_cache.data_ptr(), position_ids.data_ptr(), cos_cache.data_ptr(),
        sin_cache.data_ptr(), slot_mapping.data_ptr(), ks_ptr, vs_ptr)
    p.device_status = _status_ptr(device)
    if nt > _capi.ROTARY_APPEND_SCAN_TOKENS:
        need = ctypes.c_size_t(0)
        check(LIB.b200_rotary_append_workspace_size(_byref(p), _byref(need)))
        p.workspace, p.workspace_bytes = _workspace(op, device, need.value, workspace)
    _call(LIB.b200_rotary_append, p, device, check_status)
    return output, key_cache, value_cache


@_on_stream
def shared_prefix_attention(query, key_cache, value_cache, cumulative_sequence_length, past_seqlens, block_table,
                            prefix_block_table, *, prefix_length, num_heads, kv_num_heads, scale=0.0, softcap=0.0,
                            head_sink=None, output=None, workspace=None, num_sms=0, check_status=False):
    """Causal attention of a batch whose sequences share the ``prefix_length`` keys of
    ``prefix_block_table``; sequence ``b`` continues with its own ``past_seqlens[b]`` keys and its new
    tokens, paged by row ``b`` of ``block_table``.

    Every key is read from the caches (``[blocks, block_size, kv_num_heads, d]``, fp16 / bf16), the
    new tokens' included: append them first.  Metadata are int32 device tensors.  Returns the output
    ``[tokens, num_heads * d]``.  The scratch is the current stream's own buffer unless ``workspace``
    (uint8, at least ``b200_shared_prefix_attention_workspace_size`` bytes) is given.
    """
    op = "SharedPrefixAttention"
    act = _ACT.get(query.dtype)
    if act is None or query.dim() != 2:
        raise _bad(f"{op}: query must be a [tokens, hidden] tensor of fp16 or bf16")
    H, KV = int(num_heads), int(kv_num_heads)
    if key_cache.dim() != 4 or key_cache.shape[2] != KV:
        raise _bad(f"{op}: key_cache must be [blocks, block_size, kv_num_heads, head_size]")
    nt = query.shape[0]
    blocks, block_size, _, d = key_cache.shape
    device = query.device
    _same_device(op, device, key_cache=key_cache, value_cache=value_cache,
                 cumulative_sequence_length=cumulative_sequence_length, past_seqlens=past_seqlens,
                 block_table=block_table, prefix_block_table=prefix_block_table, head_sink=head_sink, output=output,
                 workspace=workspace)
    if value_cache.shape != key_cache.shape or key_cache.dtype != query.dtype or value_cache.dtype != query.dtype or not (
            key_cache.is_contiguous() and value_cache.is_contiguous()):
        raise _bad(f"{op}: key_cache and value_cache must be contiguous, alike and of the query's type")
    for name, t, rank in (("cumulative_sequence_length", cumulative_sequence_length, 1), ("past_seqlens", past_seqlens, 1),
                          ("block_table", block_table, 2), ("prefix_block_table", prefix_block_table, 1)):
        if t is None and name == "prefix_block_table" and int(prefix_length) == 0:
            continue
        if t is None or t.dtype != torch.int32 or t.dim() != rank or not t.is_contiguous():
            raise _bad(f"{op}: {name} must be a contiguous int32 tensor of rank {rank}")
    batch = past_seqlens.shape[0]
    if cumulative_sequence_length.shape[0] != batch + 1 or block_table.shape[0] != batch:
        raise _bad(f"{op}: inconsistent cumulative lengths, past lengths or block table")
    if head_sink is not None and (head_sink.dtype != query.dtype or head_sink.shape != (H,) or not head_sink.is_contiguous()):
        raise _bad(f"{op}: head_sink must be a contiguous [num_heads] tensor of the query's type")
    q_stride = _rows(op, "query", query, H * d)
    if output is None:
        output = torch.empty((nt, H * d), dtype=query.dtype, device=device)
        o_stride = H * d
    else:
        if output.dtype != query.dtype or output.shape[0] != nt:
            raise _bad(f"{op}: output has another shape or type")
        o_stride = _rows(op, "output", output, H * d)
    p = SharedPrefixParams(
        H, KV, d, scale or 0.0, softcap, act, nt, batch, blocks, block_size, block_table.shape[1], int(prefix_length),
        0 if prefix_block_table is None else prefix_block_table.shape[0], int(num_sms), q_stride, o_stride,
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), cumulative_sequence_length.data_ptr(),
        past_seqlens.data_ptr(), block_table.data_ptr(),
        None if prefix_block_table is None else prefix_block_table.data_ptr(),
        None if head_sink is None else head_sink.data_ptr(), output.data_ptr())
    p.device_status = _status_ptr(device)
    need = ctypes.c_size_t(0)
    check(LIB.b200_shared_prefix_attention_workspace_size(_byref(p), _byref(need)))
    p.workspace, p.workspace_bytes = _workspace(op, device, need.value, workspace)
    _call(LIB.b200_shared_prefix_attention, p, device, check_status)
    return output
