"""Host-side checks of the decoder-layer operators (include/b200_layer.h): every refusal comes before
anything touches a device, with its code and message."""

import ctypes

import pytest

from onnxruntime_ep_b200 import _capi

BF16, FP16, FP32, E4M3 = (_capi.DTYPE_BFLOAT16, _capi.DTYPE_FLOAT16, _capi.DTYPE_FLOAT, _capi.DTYPE_FLOAT8E4M3FN)
LIB = _capi.LIB
INVALID, UNSUPPORTED, WORKSPACE = (_capi.B200_ERR_INVALID_ARGUMENT, _capi.B200_ERR_UNSUPPORTED, _capi.B200_ERR_WORKSPACE)


def norm():
    p = _capi.SkipRmsNormParams(rows=2, hidden=64, dtype=BF16, out_dtype=BF16, epsilon=1e-6)
    p.x, p.residual, p.weight, p.out, p.residual_out, p.scales = 0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 0x6000
    return p


def rope():
    p = _capi.RotaryAppendParams(num_heads=4, kv_num_heads=2, head_size=64, rotary_dim=64, rotary_positions=128, axes=1,
                                 axis_pairs=(32,), act_dtype=BF16, cache_dtype=BF16, table_dtype=BF16,
                                 position_dtype=_capi.DTYPE_INT64, num_tokens=3, num_blocks=8, block_size=16)
    for i, f in enumerate(("query", "key", "value", "output", "key_cache", "value_cache", "position_ids", "cos_cache",
                           "sin_cache", "slot_mapping")):
        setattr(p, f, 0x1000 * (i + 1))
    return p


def prefix():
    p = _capi.SharedPrefixParams(num_heads=4, kv_num_heads=2, head_size=64, act_dtype=FP16, num_tokens=3, batch=2,
                                 num_blocks=8, block_size=16, max_blocks_per_seq=2, prefix_length=40, prefix_blocks=3)
    for i, f in enumerate(("query", "key_cache", "value_cache", "cumulative_sequence_length", "past_seqlens",
                           "block_table", "prefix_block_table", "output")):
        setattr(p, f, 0x1000 * (i + 1))
    return p


def test_struct_layouts():
    for which, cls in enumerate((_capi.SkipRmsNormParams, _capi.RotaryAppendParams, _capi.SharedPrefixParams)):
        assert LIB.b200_layer_struct_size(which) == ctypes.sizeof(cls)
    assert LIB.b200_layer_struct_size(3) == 0


@pytest.mark.parametrize("entry", ["b200_skip_rms_norm", "b200_rotary_append", "b200_shared_prefix_attention"])
def test_null_params(entry):
    assert getattr(LIB, entry)(None, None) == INVALID
    assert LIB.b200_layer_read_status(None, None) == INVALID


REFUSED = [
    (norm, "b200_skip_rms_norm", INVALID, dict(hidden=0), "hidden > 0"),
    (norm, "b200_skip_rms_norm", INVALID, dict(rows=-1), "rows >= 0"),
    (norm, "b200_skip_rms_norm", UNSUPPORTED, dict(hidden=32769), "hidden above 32768"),
    (norm, "b200_skip_rms_norm", INVALID, dict(dtype=FP32, out_dtype=FP32), "fp16 or bf16"),
    (norm, "b200_skip_rms_norm", INVALID, dict(out_dtype=FP16), "out must be x's type or fp8"),
    (norm, "b200_skip_rms_norm", INVALID, dict(epsilon=-1.0), "epsilon"),
    (norm, "b200_skip_rms_norm", INVALID, dict(epsilon=float("nan")), "epsilon"),
    (norm, "b200_skip_rms_norm", INVALID, dict(group_size=64), "group_size needs an fp8 output"),
    (norm, "b200_skip_rms_norm", INVALID, dict(out_dtype=E4M3, group_size=48), "power of two from 32 to 1024"),
    (norm, "b200_skip_rms_norm", INVALID, dict(out_dtype=E4M3, group_size=16), "power of two from 32 to 1024"),
    (norm, "b200_skip_rms_norm", INVALID, dict(out_dtype=E4M3, group_size=-32), "power of two from 32 to 1024"),
    (norm, "b200_skip_rms_norm", INVALID, dict(x_row_stride=-64), "negative row stride"),
    (norm, "b200_skip_rms_norm", INVALID, dict(out_row_stride=63), "output rows overlap"),
    (norm, "b200_skip_rms_norm", INVALID, dict(residual_out_row_stride=63), "output rows overlap"),
    (norm, "b200_skip_rms_norm", INVALID, dict(weight=None), "x, weight and out"),
    (norm, "b200_skip_rms_norm", INVALID, dict(out_dtype=E4M3, scales=None), "requires scales"),
    (norm, "b200_skip_rms_norm", INVALID, dict(out_dtype=E4M3, out=0x1000), "cannot share"),
    (norm, "b200_skip_rms_norm", INVALID, dict(residual_out=0x4000), "must differ"),
    (rope, "b200_rotary_append", INVALID, dict(num_heads=0), "must be positive"),
    (rope, "b200_rotary_append", INVALID, dict(num_tokens=-1), "must not be negative"),
    (rope, "b200_rotary_append", UNSUPPORTED, dict(num_tokens=(1 << 29) + 1), "2^29 tokens"),
    (rope, "b200_rotary_append", INVALID, dict(block_size=0), "block geometry"),
    (rope, "b200_rotary_append", UNSUPPORTED, dict(num_blocks=1 << 28), "exceeds int32"),
    (rope, "b200_rotary_append", INVALID, dict(act_dtype=FP32), "fp16 or bf16"),
    (rope, "b200_rotary_append", INVALID, dict(cache_dtype=FP16), "the activations' type or fp8"),
    (rope, "b200_rotary_append", INVALID, dict(table_dtype=FP16), "the activations' type or fp32"),
    (rope, "b200_rotary_append", INVALID, dict(position_dtype=FP32), "int32 or int64"),
    (rope, "b200_rotary_append", INVALID, dict(rotary_dim=63), "must be even"),
    (rope, "b200_rotary_append", INVALID, dict(rotary_dim=66), "must not exceed head_size"),
    (rope, "b200_rotary_append", INVALID, dict(rotary_offset=2), "must not exceed head_size"),
    (rope, "b200_rotary_append", INVALID, dict(rotary_offset=-2), "must not exceed head_size"),
    (rope, "b200_rotary_append", INVALID, dict(rotary_positions=0), "must not be empty"),
    (rope, "b200_rotary_append", INVALID, dict(axes=0), "1 to 4"),
    (rope, "b200_rotary_append", INVALID, dict(axes=5), "1 to 4"),
    (rope, "b200_rotary_append", INVALID, dict(axes=2, axis_pairs=(32, 1)), "sum to rotary_dim / 2"),
    (rope, "b200_rotary_append", INVALID, dict(axis_pairs=(31,)), "sum to rotary_dim / 2"),
    (rope, "b200_rotary_append", INVALID, dict(axes=2, axis_pairs=(40, -8)), "must not be negative"),
    (rope, "b200_rotary_append", INVALID, dict(output_row_stride=255), "output rows overlap"),
    (rope, "b200_rotary_append", INVALID, dict(slot_mapping=None), "missing required tensor"),
    (rope, "b200_rotary_append", INVALID, dict(cache_dtype=E4M3), "k_scale and v_scale"),
    (rope, "b200_rotary_append", WORKSPACE, dict(num_tokens=8193), "workspace"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(num_heads=3), "num_heads/kv_num_heads"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(head_size=0), "head_size must be positive"),
    (prefix, "b200_shared_prefix_attention", UNSUPPORTED, dict(head_size=257), "head_size above 256"),
    (prefix, "b200_shared_prefix_attention", UNSUPPORTED, dict(num_heads=65538), "65535 heads"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(act_dtype=E4M3), "fp16 or bf16"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(num_blocks=0), "block geometry"),
    (prefix, "b200_shared_prefix_attention", UNSUPPORTED, dict(num_blocks=1 << 28), "slot count exceeds int32"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(batch=0), "batch must be positive"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(num_tokens=-1), "not negative"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(prefix_length=49), "exceeds prefix_block_table"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(prefix_length=-1), "exceeds prefix_block_table"),
    (prefix, "b200_shared_prefix_attention", UNSUPPORTED, dict(max_blocks_per_seq=1 << 28), "keys exceed int32"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(scale=float("inf")), "scale must be finite"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(softcap=-1.0), "softcap"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(softcap=float("nan")), "softcap"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(output_row_stride=255), "output rows overlap"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(past_seqlens=None), "missing required tensor"),
    (prefix, "b200_shared_prefix_attention", INVALID, dict(prefix_block_table=None), "missing required tensor"),
]


@pytest.mark.parametrize("make,entry,code,change,message", REFUSED, ids=lambda v: str(v) if isinstance(v, dict) else "")
def test_refusals(make, entry, code, change, message):
    p = make()
    for name, value in change.items():
        if name == "axis_pairs":
            value = (ctypes.c_int32 * 4)(*value)
        setattr(p, name, value)
    assert getattr(LIB, entry)(ctypes.byref(p), None) == code
    assert message in LIB.b200_last_error().decode()


def test_workspace_sizes():
    n = ctypes.c_size_t(7)
    p = rope()
    assert LIB.b200_rotary_append_workspace_size(ctypes.byref(p), ctypes.byref(n)) == _capi.B200_OK and n.value == 0
    p.num_tokens = _capi.ROTARY_APPEND_SCAN_TOKENS + 1
    assert LIB.b200_rotary_append_workspace_size(ctypes.byref(p), ctypes.byref(n)) == _capi.B200_OK
    assert n.value >= 8 * p.num_tokens
    assert LIB.b200_rotary_append_workspace_size(ctypes.byref(p), None) == INVALID
    q = prefix()
    assert LIB.b200_shared_prefix_attention_workspace_size(ctypes.byref(q), ctypes.byref(n)) == _capi.B200_OK
    assert LIB.b200_shared_prefix_attention_workspace_size(None, ctypes.byref(n)) == INVALID


def test_empty_calls_touch_nothing():
    p = norm()
    p.rows, p.x, p.out = 0, None, None
    assert LIB.b200_skip_rms_norm(ctypes.byref(p), None) == _capi.B200_OK
    r = rope()
    r.num_tokens, r.query = 0, None
    assert LIB.b200_rotary_append(ctypes.byref(r), None) == _capi.B200_OK
    a = prefix()
    a.num_tokens, a.query = 0, None
    assert LIB.b200_shared_prefix_attention(ctypes.byref(a), None) == _capi.B200_OK


@pytest.mark.parametrize("make,name,change,align", [(rope, "rotary_append", dict(num_tokens=8193), 4),
                                                    (prefix, "shared_prefix_attention", {}, 16)])
def test_misaligned_workspaces_are_refused(make, name, change, align):
    p = make()
    for field, value in change.items():
        setattr(p, field, value)
    n = ctypes.c_size_t(0)
    assert getattr(LIB, f"b200_{name}_workspace_size")(ctypes.byref(p), ctypes.byref(n)) == _capi.B200_OK and n.value
    p.workspace_bytes = n.value + 64
    for off in {1, 2, align // 2, align - 1, align + 1}:
        p.workspace = 0x100000 + off
        assert getattr(LIB, f"b200_{name}")(ctypes.byref(p), None) == WORKSPACE
        assert f"aligned to {align} bytes" in LIB.b200_last_error().decode()


@pytest.mark.parametrize("make,entry,change,fields", [
    (norm, "b200_skip_rms_norm", {}, dict(x=1, residual=1, weight=1, out=1, residual_out=1)),
    (norm, "b200_skip_rms_norm", dict(out_dtype=E4M3), dict(x=1, scales=2)),
    (rope, "b200_rotary_append", dict(table_dtype=FP32),
     dict(query=1, key=1, value=1, output=1, key_cache=1, value_cache=1, cos_cache=2, sin_cache=2, position_ids=4,
          slot_mapping=2, device_status=2)),
    (rope, "b200_rotary_append", dict(cache_dtype=E4M3, k_scale=0x20000, v_scale=0x21000, position_dtype=_capi.DTYPE_INT32),
     dict(cos_cache=1, sin_cache=1, position_ids=2, k_scale=2, v_scale=2)),
    (prefix, "b200_shared_prefix_attention", {},
     dict(query=1, key_cache=1, value_cache=1, head_sink=1, output=1, cumulative_sequence_length=2, past_seqlens=2,
          block_table=2, prefix_block_table=2, device_status=2)),
])
def test_misaligned_tensors_are_refused(make, entry, change, fields):
    for field, off in fields.items():
        p = make()
        for name, value in change.items():
            setattr(p, name, value)
        setattr(p, field, (getattr(p, field) or 0x30000) + off)
        assert getattr(LIB, entry)(ctypes.byref(p), None) == INVALID, field
        assert "not aligned to its elements" in LIB.b200_last_error().decode()
    assert LIB.b200_layer_read_status(0x30002, None) == INVALID


@pytest.mark.parametrize("num_sms", [1025, 200_000_000, 2 ** 31 - 1])
def test_num_sms_is_bounded(num_sms):
    p, n = prefix(), ctypes.c_size_t(0)
    p.num_sms, p.workspace, p.workspace_bytes = num_sms, 0x100000, 1 << 62
    assert LIB.b200_shared_prefix_attention(ctypes.byref(p), None) == INVALID
    assert "num_sms" in LIB.b200_last_error().decode()
    assert LIB.b200_shared_prefix_attention_workspace_size(ctypes.byref(p), ctypes.byref(n)) == INVALID
    p.num_sms = 1024
    assert LIB.b200_shared_prefix_attention_workspace_size(ctypes.byref(p), ctypes.byref(n)) == _capi.B200_OK and n.value < 1 << 40


def test_an_empty_batch_is_an_empty_call():
    p, n = prefix(), ctypes.c_size_t(7)
    p.num_tokens, p.batch = 0, 0
    for field in ("query", "output", "cumulative_sequence_length", "past_seqlens", "block_table"):
        setattr(p, field, None)
    assert LIB.b200_shared_prefix_attention(ctypes.byref(p), None) == _capi.B200_OK
    assert LIB.b200_shared_prefix_attention_workspace_size(ctypes.byref(p), ctypes.byref(n)) == _capi.B200_OK and n.value == 0
    for batch, tokens in ((0, 1), (-1, 0)):
        p.batch, p.num_tokens = batch, tokens
        assert LIB.b200_shared_prefix_attention(ctypes.byref(p), None) == INVALID
