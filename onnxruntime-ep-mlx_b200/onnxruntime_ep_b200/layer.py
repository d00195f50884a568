"""The operators around paged attention in one decoder layer (include/b200_layer.h):
``skip_rms_norm``, ``rotary_append`` and ``shared_prefix_attention``.

Torch only owns device memory and the current stream; the work runs in ``libb200_paged.so``, called
through the native binding ``_layer``, which checks the tensors and allocates the outputs.  Argument
errors raise ``B200Error``.  Errors that only the device can see (a slot, position, length or block id
out of range) set the status word of the stream; ``check_status=True`` synchronises and raises what the
stream's calls have reported, as does ``check_status(stream)``.  A captured call reports to the stream that
it was captured on.  Every function
takes ``stream=`` (default: the current stream).  Scratch belongs to the stream of the calls; calls that
are captured in a CUDA graph get scratch of that graph, which lives as long as the graph, so graphs may
be replayed at the same time as each other and as other calls.  The first call on a device allocates its
status word: make it before a graph capture.
"""

from __future__ import annotations

import importlib

import torch

from . import _capi
from ._capi import B200Error


class _Binding:
    """The native module ``_layer``, loaded at the first use: it is built against one torch, and the rest of
    the package needs neither it nor that torch."""

    def __getattr__(self, name):
        try:
            module = importlib.import_module("._layer", __package__)
        except ImportError as e:
            raise ImportError(f"onnxruntime_ep_b200/_layer.so cannot be loaded ({e}): build it against this torch with "
                              "`make -C onnxruntime-ep-mlx_b200/csrc`") from e
        module.set_error_class(B200Error)
        globals()["_layer"] = module
        return getattr(module, name)


_layer = _Binding()

_FP8 = torch.float8_e4m3fn


def _on_stream(stream, fn, *args, **kwargs):
    """``fn`` with ``stream`` current, so what it allocates belongs to the stream that uses it."""
    with torch.cuda.stream(stream):
        return fn(*args, **kwargs)


def check_status(stream=None):
    """Synchronise ``stream`` (default: the current one) and raise what its calls have reported since the last
    check.  For the calls in a CUDA graph, ``stream`` is the one they were captured on: wait for the replays
    first, then check it."""
    stream = stream if stream is not None else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        _layer.read_status(stream.device.index)


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
    fp8 = out_dtype is _FP8
    if not fp8 and out_dtype is not None and out_dtype is not x.dtype:
        raise B200Error(_capi.B200_ERR_INVALID_ARGUMENT, "SkipRmsNorm: out_dtype must be x's type or float8_e4m3fn")
    return _layer.skip_rms_norm(x, residual, weight, epsilon, fp8, group_size, output, scales, residual_output)


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
    result = _layer.rotary_append(query, key, value, key_cache, value_cache, position_ids, cos_cache, sin_cache,
                                  slot_mapping, num_heads, kv_num_heads, axis_sections, rotary_interleaved, rotary_offset,
                                  k_scale, v_scale, output, workspace)
    if check_status:
        _layer.read_status(query.get_device())
    return result


def shared_prefix_attention(query, key_cache, value_cache, cumulative_sequence_length, past_seqlens, block_table,
                            prefix_block_table, *, prefix_length, num_heads, kv_num_heads, scale=0.0, softcap=0.0,
                            head_sink=None, output=None, workspace=None, num_sms=0, check_status=False, stream=None):
    """Causal attention of a batch whose sequences share the ``prefix_length`` keys of
    ``prefix_block_table``; sequence ``b`` continues with its own ``past_seqlens[b]`` keys and its new
    tokens, paged by row ``b`` of ``block_table``.

    Every key is read from the caches (``[blocks, block_size, kv_num_heads, d]``, fp16 / bf16), the
    new tokens' included: append them first.  Metadata are int32 device tensors.  Returns the output
    ``[tokens, num_heads * d]``.  The scratch is the current stream's own buffer, or in a graph capture
    the graph's, unless ``workspace`` (uint8, at least ``b200_shared_prefix_attention_workspace_size``
    bytes, aligned to 16) is given.
    """
    if stream is not None:
        return _on_stream(stream, shared_prefix_attention, query, key_cache, value_cache, cumulative_sequence_length,
                          past_seqlens, block_table, prefix_block_table, prefix_length=prefix_length, num_heads=num_heads,
                          kv_num_heads=kv_num_heads, scale=scale, softcap=softcap, head_sink=head_sink, output=output,
                          workspace=workspace, num_sms=num_sms, check_status=check_status)
    result = _layer.shared_prefix_attention(query, key_cache, value_cache, cumulative_sequence_length, past_seqlens,
                                            block_table, prefix_block_table, prefix_length, num_heads, kv_num_heads, scale,
                                            softcap, head_sink, output, workspace, num_sms)
    if check_status:
        _layer.read_status(query.get_device())
    return result
