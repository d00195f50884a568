"""The decoder-layer operators (include/b200_layer.h) against plain implementations in 64 bits.

Tolerances (fixed before the first run).  16-bit outputs: half a unit in the last place of the
output's own rounding is always allowed (oracle.tolerance); beyond it
 * norm: fp32 sums of up to 32768 squares in blocks (each thread at most 32 in a row, then two
   32-way trees) and six roundings: 2^-17 of the value;
 * rotation: three roundings of terms up to |x0| + |x1|: 2^-21 of that sum;
 * attention: 2e-3, this library's bound for 16-bit paged attention on N(0, 1) values.
fp8 codes: the code of a value within 2^-17 of the exact one: |code * scale - y| at most half a step of
e4m3 (2^-4 of the magnitude, 2^-10 of a subnormal unit) plus that.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from onnxruntime_ep_b200 import (B200Error, kv_append, paged_attention, rotary_append, shared_prefix_attention,  # noqa: E402
                                 skip_rms_norm)
from oracle import tolerance  # noqa: E402
from onnxruntime_ep_b200 import layer  # noqa: E402

FP8 = torch.float8_e4m3fn
BITS = {torch.bfloat16: 8, torch.float16: 11}
HALF_STEP = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # of subnormal outputs
TYPES = [torch.bfloat16, torch.float16]


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def close16(got, want, allowed):
    """Every |got - want| within half an output ulp plus `allowed` (a number or a tensor)."""
    a, b = got.double().cpu().numpy(), want.cpu().numpy()
    half = tolerance.half_ulp(np.maximum(np.abs(a), np.abs(b)), BITS[got.dtype])
    off = np.abs(a - b) - np.maximum(half, HALF_STEP[got.dtype])
    allowed = allowed.cpu().numpy() if isinstance(allowed, torch.Tensor) else allowed
    assert (off <= allowed).all(), float((off - allowed).max())


# ------------------------------------------------------------------------------------- norm
def norm64(x, r, w, eps=1e-6):
    s = x.double() + (0 if r is None else r.double())
    return s, s / (s.pow(2).mean(1, keepdim=True) + eps).sqrt() * w.double()


def check_codes(codes, scales, y, group):
    n, h = y.shape
    width = h if group == 0 else group
    groups = -(-h // width)
    pad = torch.zeros(n, groups * width - h, device="cuda", dtype=torch.float64)
    yp = torch.cat([y, pad], 1).view(n, groups, width)
    want = yp.abs().amax(-1).clamp(min=1e-12) / 448
    assert scales.shape == (n, groups)
    assert ((scales.double() - want).abs() <= want * 2.0 ** -17).all()
    value = torch.cat([codes.double(), pad], 1).view(n, groups, width) * scales.double()[..., None]
    step = torch.maximum(yp.abs() * 2.0 ** -4, scales.double()[..., None] * 2.0 ** -10)
    assert ((value - yp).abs() <= step * (1 + 2.0 ** -12) + yp.abs() * 2.0 ** -17).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (2, 32), (5, 33), (4, 100), (1, 4096), (7, 2880), (9, 4828),
                                         (3, 5001), (2, 8192), (2, 16384), (3, 20004), (2, 32768), (2, 32767)])
def test_norm(rows, hidden, dtype):
    g = gen(hidden)
    x, r, w = normal(g, rows, hidden, dtype=dtype), normal(g, rows, hidden, dtype=dtype, scale=3), normal(g, hidden, dtype=dtype)
    s, y = norm64(x, r, w)
    out, res = skip_rms_norm(x, r, w)
    close16(res, s, s.abs() * 2.0 ** -23)
    close16(out, y, y.abs() * 2.0 ** -17)
    out, res = skip_rms_norm(x, None, w)
    assert torch.equal(res, x)
    close16(out, norm64(x, None, w)[1], norm64(x, None, w)[1].abs() * 2.0 ** -17)


@pytest.mark.parametrize("group", [0, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 31), (2, 128), (5, 130), (7, 2880), (9, 4828), (3, 5001), (2, 8192),
                                         (2, 20000), (2, 32767)])
def test_norm_fp8(rows, hidden, group):
    g = gen(hidden + group)
    x, r, w = normal(g, rows, hidden), normal(g, rows, hidden), normal(g, hidden)
    s, y = norm64(x, r, w)
    codes, scales, res = skip_rms_norm(x, r, w, out_dtype=FP8, group_size=group)
    close16(res, s, s.abs() * 2.0 ** -23)
    check_codes(codes, scales, y, group)


def test_norm_many_rows_and_batch_invariance():
    g = gen(1)
    x, r, w = normal(g, 70001, 64), normal(g, 70001, 64), normal(g, 64)
    out, res = skip_rms_norm(x, r, w)
    s, y = norm64(x, r, w)
    close16(out, y, y.abs() * 2.0 ** -17)
    one, one_res = skip_rms_norm(x[70000:], r[70000:], w)
    assert torch.equal(one, out[70000:]) and torch.equal(one_res, res[70000:])


@pytest.mark.parametrize("rows,hidden", [(2001, 301), (1500, 2881), (900, 4002), (700, 8191), (650, 12290), (3000, 129), (900, 1031), (700, 256), (700, 1024),
                                         (650, 16391), (1300, 15), (601, 8200)])
@pytest.mark.parametrize("group", [None, 0, 32, 128])
def test_norm_many_odd_rows(rows, hidden, group):
    """Rows off 16 bytes in CTAs that walk: every row, first and last channels included."""
    g = gen(hidden)
    x, r, w = normal(g, rows, hidden), normal(g, rows, hidden), normal(g, hidden)
    s, y = norm64(x, r, w)
    if group is None:
        out, res = skip_rms_norm(x, r, w)
        close16(out, y, y.abs() * 2.0 ** -17)
        keep = x.clone(), r.clone()
        skip_rms_norm(keep[0], keep[1], w, output=keep[0], residual_output=keep[1])
        assert torch.equal(keep[0], out) and torch.equal(keep[1], res)
    else:
        codes, scales, res = skip_rms_norm(x, r, w, out_dtype=FP8, group_size=group)
        check_codes(codes, scales, y, group)
    close16(res, s, s.abs() * 2.0 ** -23)


@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (4, 4), (0, 1), (3, 2)])
def test_norm_strides_alignment_and_in_place(pad, shift):
    g = gen(pad + 10 * shift)
    rows, hidden = 6, 1024
    base = normal(g, rows * (hidden + pad) + shift + 8)
    x = base[shift:shift + rows * (hidden + pad)].view(rows, hidden + pad)[:, :hidden]
    r = normal(g, rows, hidden + pad)[:, :hidden]
    w = normal(g, hidden + shift)[shift:]
    s, y = norm64(x, r, w)
    codes = torch.empty(rows, hidden + pad, device="cuda", dtype=FP8)[:, :hidden]
    got, scales, _ = skip_rms_norm(x, r, w, out_dtype=FP8, group_size=128, output=codes)
    check_codes(got, scales, y, 128)
    out, res = skip_rms_norm(x, r, w, output=x, residual_output=r)
    assert out.data_ptr() == x.data_ptr() and res.data_ptr() == r.data_ptr()
    close16(out, y, y.abs() * 2.0 ** -17)
    close16(res, s, s.abs() * 2.0 ** -23)


@pytest.mark.parametrize("group", [0, 64, 512])
def test_norm_zero_nan_inf_rows(group):
    g = gen(5)
    x, w = normal(g, 5, 512), normal(g, 512)
    x[0] = 0
    x[1, 70] = float("nan")
    x[2, 300] = float("inf")
    clean = x.clone()
    clean[1:3] = 1
    codes, scales, _ = skip_rms_norm(x, None, w, out_dtype=FP8, group_size=group)
    want, want_scales, _ = skip_rms_norm(clean, None, w, out_dtype=FP8, group_size=group)
    assert torch.isnan(scales[1]).all() and torch.isnan(codes[1].float()).all()  # the sum is NaN for all channels
    keep = [3, 4]  # the other rows do not see them
    assert torch.equal(codes[keep].view(torch.uint8), want[keep].view(torch.uint8))
    assert torch.equal(scales[keep], want_scales[keep])
    assert (codes[0].float() == 0).all() and (scales[0] > 0).all()  # a row of zeros still has scales
    out, res = skip_rms_norm(x, None, w)
    assert (out[0] == 0).all() and torch.isnan(out[1]).all()
    assert torch.isnan(out[2, 300]) and (out[2, :300] == 0).all()  # x / inf


def test_norm_refusals():
    x = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    for call in (lambda: skip_rms_norm(x.float(), x, w), lambda: skip_rms_norm(x, x.half(), w),
                 lambda: skip_rms_norm(x, x[:1], w), lambda: skip_rms_norm(x, x, w[:32]),
                 lambda: skip_rms_norm(x.t(), x, w), lambda: skip_rms_norm(x.cpu(), x, w),
                 lambda: skip_rms_norm(x[:1].expand(2, 64), x, w), lambda: skip_rms_norm(x, x, w, group_size=32),
                 lambda: skip_rms_norm(x, x, w, out_dtype=torch.int8),
                 lambda: skip_rms_norm(x, x, w, out_dtype=FP8, scales=torch.zeros(2, 2, device="cuda"))):
        with pytest.raises(B200Error):
            call()
    out, res = skip_rms_norm(x[:0], x[:0], w)
    assert out.shape == (0, 64) and res.shape == (0, 64)


# ------------------------------------------------------------------------------------- rotary append
def rope_case(seed, nt, H, KV, d, rot, *, axes=1, interleaved=0, offset=0, packed=False, dtype=torch.bfloat16,
              cache="same", bs=16, skip=0.1, table=None, index=torch.int64, positions=97):
    g = gen(seed)
    blocks = -(-nt // bs) + 2
    qkv = normal(g, nt, (H + 2 * KV) * d, dtype=dtype)
    parts = qkv.split([H * d, KV * d, KV * d], 1)
    kc, vc = normal(g, blocks, bs, KV, d, dtype=dtype), normal(g, blocks, bs, KV, d, dtype=dtype)
    ks = vs = None
    if cache == "fp8":
        kc, vc = kc.to(FP8), vc.to(FP8)
        ks, vs = (torch.rand(blocks, KV, device="cuda", generator=g) * 0.02 + 0.004 for _ in range(2))
    angle = torch.randn(positions, rot // 2, device="cuda", generator=g) * 3
    slots = torch.randperm(blocks * bs, device="cuda", generator=g)[:nt].int()
    slots[torch.rand(nt, device="cuda", generator=g) < skip] = -1
    sections = [rot // 2 // axes] * axes
    sections[-1] += rot // 2 - sum(sections)
    return dict(H=H, KV=KV, d=d, rot=rot, offset=offset, interleaved=interleaved, qkv=qkv, packed=packed,
                q=parts[0].contiguous(), k=parts[1].contiguous(), v=parts[2].contiguous(), kc=kc, vc=vc, ks=ks, vs=vs,
                cos=angle.cos().to(table or dtype), sin=angle.sin().to(table or dtype), slots=slots, sections=sections,
                pos=torch.randint(0, positions, (axes, nt), device="cuda", generator=g).to(index), bs=bs)


def rope_call(c, kc, vc, **kw):
    q, k, v = (c["qkv"], None, None) if c["packed"] else (c["q"], c["k"], c["v"])
    pos = c["pos"] if len(c["sections"]) > 1 else c["pos"][0]
    kw.setdefault("check_status", True)
    return rotary_append(q, k, v, kc, vc, pos, c["cos"], c["sin"], c["slots"], num_heads=c["H"], kv_num_heads=c["KV"],
                         axis_sections=c["sections"] if len(c["sections"]) > 1 else None,
                         rotary_interleaved=c["interleaved"], rotary_offset=c["offset"], k_scale=c["ks"],
                         v_scale=c["vs"], **kw)


def rotate64(c, x, heads):
    """(rotated rows, |x0| + |x1| of each channel's pair) in 64 bits."""
    nt, half = x.shape[0], c["rot"] // 2
    x = x.double().view(nt, heads, c["d"])
    y, mag = x.clone(), torch.zeros_like(x)
    pair = 0
    for axis, count in enumerate(c["sections"]):
        for i in range(pair, pair + count):
            a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
            a, b = a + c["offset"], b + c["offset"]
            co, si = c["cos"].double()[c["pos"][axis].long(), i], c["sin"].double()[c["pos"][axis].long(), i]
            y[:, :, a] = x[:, :, a] * co[:, None] - x[:, :, b] * si[:, None]
            y[:, :, b] = x[:, :, b] * co[:, None] + x[:, :, a] * si[:, None]
            mag[:, :, a] = mag[:, :, b] = x[:, :, a].abs() + x[:, :, b].abs()
        pair += count
    return y, mag


def last_writers(slots):
    """Tokens whose slot no later token names."""
    s = slots.cpu().numpy()
    last = {}
    for t, slot in enumerate(s):
        if slot >= 0:
            last[int(slot)] = t
    return torch.tensor(sorted(last.values()), device="cuda", dtype=torch.long)


def check_rope(c):
    kc, vc = c["kc"].clone(), c["vc"].clone()
    out, kc2, vc2 = rope_call(c, kc, vc)
    assert kc2.data_ptr() == kc.data_ptr() and vc2.data_ptr() == vc.data_ptr()
    nt, KV, d = out.shape[0], c["KV"], c["d"]
    want, mag = rotate64(c, c["q"], c["H"])
    close16(out, want.view(nt, -1), (mag * 2.0 ** -21).view(nt, -1))
    tokens = last_writers(c["slots"])
    slot = c["slots"][tokens].long()
    key, kmag = rotate64(c, c["k"], KV)
    value = c["v"].double().view(nt, KV, d)
    for cache, before, rows, rmag, scale in ((kc, c["kc"], key, kmag, c["ks"]), (vc, c["vc"], value, value * 0, c["vs"])):
        got = cache.view(-1, KV, d)[slot]
        if scale is None:
            close16(got, rows[tokens], rmag[tokens] * 2.0 ** -21)
        else:
            s = scale.double()[slot // c["bs"]][..., None]
            y = (rows[tokens] / s).clamp(-448, 448)
            step = torch.maximum(y.abs() * 2.0 ** -4, torch.full_like(y, 2.0 ** -10))
            assert ((got.double() - y).abs() <= step * (1 + 2.0 ** -12) + rmag[tokens] / s * 2.0 ** -21).all()
        # nothing else changed
        rest = torch.ones(cache.view(-1, KV, d).shape[0], dtype=torch.bool, device="cuda")
        rest[slot] = False
        assert torch.equal(cache.view(-1, KV, d)[rest].view(torch.uint8), before.view(-1, KV, d)[rest].view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("nt,H,KV,d,rot,kw", [
    (1, 32, 8, 128, 128, {}),
    (128, 32, 8, 128, 128, dict(packed=True)),
    (33, 14, 2, 64, 32, dict(interleaved=1)),
    (40, 4, 4, 80, 80, dict(axes=3)),
    (17, 6, 2, 96, 48, dict(axes=2, interleaved=1, offset=16)),
    (9, 3, 1, 256, 64, dict(offset=8, packed=True)),
    (21, 5, 5, 72, 40, dict(offset=24, axes=4)),
    (300, 2, 1, 18, 6, dict(offset=3, interleaved=1)),
    (5, 1, 1, 2, 2, dict(packed=True)),
    (19, 7, 1, 64, 64, dict(axes=3, index=torch.int32, table=torch.float32)),
    (64, 40, 8, 128, 96, dict(offset=16, table=torch.float32, packed=True)),
    (70, 128, 1, 640, 64, dict(offset=512)),
])
def test_rope(nt, H, KV, d, rot, kw, cache, dtype):
    check_rope(rope_case(nt + d, nt, H, KV, d, rot, cache=cache, dtype=dtype, **kw))


@pytest.mark.parametrize("nt", [50, 1000, 8192, 8193, 20000])
@pytest.mark.parametrize("cache", ["same", "fp8"])
def test_rope_last_token_of_a_slot_wins(nt, cache):
    c = rope_case(nt, nt, 2, 1, 32, 32, cache=cache, skip=0.05)
    g = gen(3)
    again = torch.randint(0, nt, (nt // 3,), device="cuda", generator=g)
    c["slots"][again] = c["slots"][torch.randint(0, nt, (nt // 3,), device="cuda", generator=g)]
    c["slots"][nt // 2:nt // 2 + 9] = c["slots"].max()  # a run inside one tile
    check_rope(c)


def test_rope_strided_rows_and_in_place_query():
    c = rope_case(4, 37, 8, 2, 64, 64)
    want, _, _ = rope_call(c, c["kc"].clone(), c["vc"].clone())
    for pad in (8, 3):  # rows on 16 bytes and off them
        wide = {n: torch.nn.functional.pad(c[n], (0, pad))[:, :c[n].shape[1]] for n in "qkv"}
        kc, vc = c["kc"].clone(), c["vc"].clone()
        out, _, _ = rope_call({**c, **wide}, kc, vc, output=wide["q"])
        assert out.data_ptr() == wide["q"].data_ptr() and torch.equal(out, want)
        kc2, vc2 = c["kc"].clone(), c["vc"].clone()
        rope_call(c, kc2, vc2)
        assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    # positions with strides of their own: one row of positions for three axes, and a transposed array
    c3 = rope_case(5, 37, 8, 2, 64, 64, axes=3)
    c3["pos"] = c3["pos"][:1].expand(3, 37)
    check_rope(c3)
    c3["pos"] = c3["pos"].contiguous().t().contiguous().t()
    check_rope(c3)
    c3["pos"] = c3["pos"][:, :1].expand(3, 37)
    check_rope(c3)


def test_rope_codes_match_kv_append():
    """Values, and keys at position 0 (cos 1, sin 0), get the bytes that kv_append writes."""
    c = rope_case(6, 60, 4, 2, 128, 128, cache="fp8", skip=0.0)
    c["cos"][0], c["sin"][0] = 1, 0
    c["pos"].zero_()
    kc, vc = c["kc"].clone(), c["vc"].clone()
    rope_call(c, kc, vc)
    kc2, vc2 = c["kc"].clone(), c["vc"].clone()
    cum = torch.tensor([0, 60], dtype=torch.int32)
    table = torch.arange(kc.shape[0], dtype=torch.int32)[None]
    kv_append(c["k"], c["v"], kc2, vc2, cum, torch.zeros(1, dtype=torch.int32), table, c["slots"], kv_num_heads=2,
              k_scale=c["ks"], v_scale=c["vs"])
    assert torch.equal(kc.view(torch.uint8), kc2.view(torch.uint8))
    assert torch.equal(vc.view(torch.uint8), vc2.view(torch.uint8))


@pytest.mark.parametrize("d,rot", [(64, 64), (18, 6)])
def test_rope_bad_slots_and_positions(d, rot):
    c = rope_case(7, 12, 2, 1, d, rot, skip=0.0)
    good = c["slots"].clone()
    for bad in (-2, c["kc"].shape[0] * c["bs"], 2 ** 31 - 1):
        c["slots"] = good.clone()
        c["slots"][5] = bad
        kc, vc = c["kc"].clone(), c["vc"].clone()
        with pytest.raises(B200Error, match="slot_mapping must contain -1 or valid"):
            rope_call(c, kc, vc)
        slots = good.clone()
        slots[5] = -1  # the token is not cached, every other one is
        kc2, vc2 = c["kc"].clone(), c["vc"].clone()
        rope_call({**c, "slots": slots}, kc2, vc2)
        assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    c["slots"] = good
    for bad in (-1, 97, 2 ** 40):
        pos = c["pos"].clone()
        pos[0, 3] = bad
        kc, vc = c["kc"].clone(), c["vc"].clone()
        with pytest.raises(B200Error, match="rotary position exceeds"):
            rope_call({**c, "pos": pos}, kc, vc)
        out, _, _ = rope_call({**c, "pos": pos}, kc, vc, check_status=False)
        assert torch.equal(out[3], c["q"][3])  # left unrotated
        assert torch.equal(kc.view(-1, d)[good[3].long()], c["k"][3])
        with pytest.raises(B200Error):  # the word is cleared by this read
            rope_call({**c, "pos": pos}, kc, vc)
    rope_call(c, c["kc"].clone(), c["vc"].clone())


def test_rope_refusals():
    c = rope_case(8, 4, 2, 1, 32, 32)
    for change in (dict(sections=[8, 7]), dict(slots=c["slots"].long()), dict(pos=c["pos"].float()),
                   dict(cos=c["cos"].half()), dict(k=c["k"][:3]), dict(v=c["v"].half()), dict(KV=2),
                   dict(q=c["q"][:, :32]), dict(kc=c["kc"].half()), dict(vc=c["vc"][:1])):
        bad = {**c, **change}
        with pytest.raises(B200Error):
            rope_call(bad, bad["kc"], bad["vc"])
    out, _, _ = rope_call({**c, "q": c["q"][:0], "k": c["k"][:0], "v": c["v"][:0], "slots": c["slots"][:0],
                           "pos": c["pos"][:, :0]}, c["kc"], c["vc"])
    assert out.shape == (0, 64)


# ------------------------------------------------------------------------------------- shared prefix
def prefix_case(seed, past, new, P, H, KV, d, *, bs=16, dtype=torch.bfloat16, scale=1.0, spare_blocks=1, fill=None,
                sink=False, extra_columns=2):
    """Caches with random pages; slots past a sequence's or the prefix's end hold `fill`."""
    g = gen(seed)
    own = [-(-(p + n) // bs) for p, n in zip(past, new)]
    pb = -(-P // bs)
    total = pb + sum(own) + spare_blocks
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int()
    kc, vc = normal(g, total, bs, KV, d, dtype=dtype, scale=scale), normal(g, total, bs, KV, d, dtype=dtype)
    table = torch.full((len(past), max(own + [0]) + extra_columns), -1, dtype=torch.int32)
    used = torch.zeros(total * bs, dtype=torch.bool)

    def mark(blocks, count):
        slots = (blocks.long()[:, None] * bs + torch.arange(bs)).flatten()[:count]
        used[slots] = True

    mark(order[:pb], P)
    at = pb
    for b, n in enumerate(own):
        table[b, :n] = order[at:at + n]
        mark(order[at:at + n], past[b] + new[b])
        at += n
    if fill is not None:
        kc.view(-1, KV, d)[~used.cuda()] = fill
        vc.view(-1, KV, d)[~used.cuda()] = fill
    nt = sum(new)
    cum = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    return dict(q=normal(g, nt, H * d, dtype=dtype, scale=scale), kc=kc, vc=vc, cum=cum.cuda(),
                past=torch.tensor(past, dtype=torch.int32).cuda(), table=table.cuda(), ptable=order[:pb].cuda(), P=P, H=H,
                KV=KV, d=d, bs=bs, new=new, pasts=past, sink=normal(g, H, dtype=dtype, scale=2) if sink else None)


def prefix_call(c, **kw):
    kw.setdefault("check_status", True)
    return shared_prefix_attention(c["q"], c["kc"], c["vc"], c["cum"], c["past"], c["table"], c["ptable"],
                                   prefix_length=c["P"], num_heads=c["H"], kv_num_heads=c["KV"], head_sink=c["sink"], **kw)


def prefix64(c, scale=0.0, softcap=0.0):
    H, KV, d, P, bs = c["H"], c["KV"], c["d"], c["P"], c["bs"]
    g = H // KV
    out = torch.zeros(c["q"].shape[0], H, d, dtype=torch.float64, device="cuda")

    def rows(cache, table, n):
        return cache[table[:-(-n // bs)].long()].reshape(-1, KV, d)[:n].double()

    at = 0
    for b, (p, n) in enumerate(zip(c["pasts"], c["new"])):
        if n == 0:
            continue
        k = torch.cat([rows(c["kc"], c["ptable"], P), rows(c["kc"], c["table"][b], p + n)])
        v = torch.cat([rows(c["vc"], c["ptable"], P), rows(c["vc"], c["table"][b], p + n)])
        q = c["q"][at:at + n].double().view(n, KV, g, d)
        x = torch.einsum("nkgd,skd->nkgs", q, k) * (scale or d ** -0.5)
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        late = torch.arange(P + p + n, device="cuda")[None] > P + p + torch.arange(n, device="cuda")[:, None]
        x = x.masked_fill(late[:, None, None], float("-inf"))
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - m)
        total = e.sum(-1, keepdim=True)
        if c["sink"] is not None:
            total = total + torch.exp(c["sink"].double().view(1, KV, g, 1) - m)
        out[at:at + n] = torch.einsum("nkgs,skd->nkgd", e / total, v).reshape(n, H, d)
        at += n
    return out.view(-1, H * d)


def check_prefix(c, **kw):
    got = prefix_call(c, **kw)
    close16(got, prefix64(c, kw.get("scale", 0.0), kw.get("softcap", 0.0)), 2e-3)
    return got


SHAPES = [  # past, new, prefix, heads, kv heads, head size
    ([0], [1], 0, 1, 1, 64),
    ([0], [1], 1, 4, 1, 128),
    ([5, 0, 31], [1, 1, 1], 16, 8, 2, 128),
    ([0, 100, 17, 250], [1, 1, 1, 1], 127, 32, 8, 128),
    ([63, 200, 0], [2, 1, 4], 129, 28, 4, 128),
    ([1, 2, 3, 4, 5], [1, 0, 1, 0, 2], 300, 6, 2, 64),
    ([0, 40], [70, 3], 256, 16, 16, 64),
    ([10, 0, 77], [33, 128, 200], 513, 8, 1, 128),
    ([0], [600], 0, 4, 2, 128),
    ([129], [1], 2000, 64, 4, 128),
    ([3, 9], [1, 5], 1111, 40, 1, 64),
    ([50], [20], 400, 48, 16, 128),
    ([7] * 130, [1] * 130, 640, 8, 2, 64),
    ([0, 20], [1, 9], 77, 6, 3, 80),
    ([11, 0], [1, 40], 130, 4, 2, 256),
    ([0, 2], [3, 1], 9, 3, 1, 17),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("past,new,P,H,KV,d", SHAPES)
def test_prefix(past, new, P, H, KV, d, dtype):
    check_prefix(prefix_case(P + H, past, new, P, H, KV, d, dtype=dtype))


@pytest.mark.parametrize("bs", [1, 8, 16, 24, 32, 48, 64, 128, 256])
def test_prefix_block_sizes(bs):
    check_prefix(prefix_case(bs, [0, 90, 300], [1, 40, 2], 333, 8, 2, 128, bs=bs))


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -3e38])
@pytest.mark.parametrize("past,new,P", [([0, 37, 5], [1, 1, 2], 100), ([3, 0], [50, 130], 17), ([15], [1], 0)])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_prefix_unused_slots_do_not_matter(past, new, P, d, fill):
    c = prefix_case(P, past, new, P, 8, 2, d, fill=0.0)
    want = check_prefix(c)
    c = prefix_case(P, past, new, P, 8, 2, d, fill=fill)
    assert torch.equal(prefix_call(c), want)


@pytest.mark.parametrize("d", [64, 128, 96])
def test_prefix_softcap_scale_sink(d):
    c = prefix_case(d, [0, 90, 33], [1, 1, 60], 500, 14, 2, d, scale=2.0, sink=True)
    check_prefix(c, softcap=20.0)
    check_prefix(c, scale=0.05)
    check_prefix(c, scale=0.2, softcap=5.0)
    check_prefix(c, scale=-0.1)


@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("B", [5, 140])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_prefix_nan_scores(d, B, softcap):
    """A NaN in a query, in a key of the prefix or in an own key: NaN in the rows that see it, in no other."""
    H, KV, P = 16, 2, 300
    new = [1] * (B - 2) + [3, 40]
    c = prefix_case(d, [4] * B, new, P, H, KV, d)
    clean = prefix_call(c, softcap=softcap).view(-1, H, d)
    q, kc = c["q"].clone(), c["kc"].clone()
    c["q"].view(-1, H, d)[2, 5, 7] = float("nan")
    touched = torch.zeros(clean.shape[0], H, dtype=torch.bool, device="cuda")
    touched[2, 5] = True
    def check():
        got = prefix_call(c, softcap=softcap).view(-1, H, d)
        assert torch.isnan(got[touched]).all()
        # the running maxima of other rows may have moved at other tiles: a unit of the output type
        torch.testing.assert_close(got[~touched], clean[~touched], rtol=2.0 ** -7, atol=1e-3)
    check()
    c["q"].copy_(q)
    for b, at, first in ((0, 3, 0), (1, 4, 1), (B - 2, 5, B - 1), (B - 1, 20, B + 17)):  # own key `at`, seen from token `first` on
        slot = int(c["table"][b][at // 16]) * 16 + at % 16
        c["kc"].view(-1, KV, d)[slot, 1, 3] = float("nan")
        touched.zero_()
        touched[first:len(touched) if b == B - 1 else first + (2 if b == B - 2 else 1), H // 2:] = True
        check()
        c["kc"].copy_(kc)
    for at in (0, 14, 15, 30, 31, 100, 127, 128, 299):
        slot = int(c["ptable"][at // 16]) * 16 + at % 16
        c["kc"].view(-1, KV, d)[slot, 1, 3] = float("nan")
        touched.zero_()
        touched[:, H // 2:] = True
        check()
        c["kc"].copy_(kc)


@pytest.mark.parametrize("cap", [0.5, 3.0, 40.0, 1e4])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_prefix_softcap_range(d, cap):
    """Scores far below, around and far above the cap."""
    c = prefix_case(d, [0, 90, 33, 7], [1, 1, 60, 2], 300, 16, 4, d, scale=2.0, dtype=torch.float16)
    check_prefix(c, softcap=cap)


def test_prefix_many_sequences():
    """More sequences than a window, a CTA or a scan step covers; some without tokens, some long."""
    g = np.random.default_rng(5)
    B = 2600
    new = [int(x) for x in g.choice([0, 1, 1, 1, 2, 5], B)]
    new[7], new[1500], new[2599] = 40, 130, 33
    past = [int(x) for x in g.integers(0, 40, B)]
    check_prefix(prefix_case(8, past, new, 150, 4, 1, 64))
    check_prefix(prefix_case(9, past, new, 40, 6, 2, 128))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [17, 1, 90, 3]])
def test_prefix_peaked_scores(new):
    """Scores up to about +-600: one key takes all the weight, wherever it lies."""
    c = prefix_case(9, [40, 0, 130, 5], new, 700, 8, 2, 128, scale=4.0)
    check_prefix(c, scale=1.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [None, 60000.0, 70000.0, 1e30, float("inf"), float("nan")])
def test_prefix_values_beyond_fp16(d, value):
    """Enough query tiles for the fp16 copy of the prefix's values, with and without a value that does not
    fit: then the call has to be the one on the bf16 values."""
    H, KV, B, P = 16, 2, 150, 400
    c = prefix_case(d, [3] * B, [1] * B, P, H, KV, d)
    if value is None:
        check_prefix(c)
        return
    c["vc"][c["ptable"][7].long(), 5, 1, 3] = value
    got, want = prefix_call(c).double().view(B, H, d), prefix64(c).view(B, H, d)
    touched = torch.zeros(B, H, d, dtype=torch.bool, device="cuda")
    touched[:, H // 2:, 3] = True  # kv head 1, channel 3
    close16(prefix_call(c).view(B, H, d)[~touched], want[~touched], 2e-3)
    if value == value and abs(value) < float("inf"):
        assert ((got[touched] - want[touched]).abs() <= want[touched].abs() * 2.0 ** -8 + 2e-3).all()
    else:
        assert not torch.isfinite(got[touched]).any()


def weighted_magnitude(c):
    """sum_j p_j |v_j| of every output channel, in 64 bits."""
    return prefix64({**c, "vc": c["vc"].abs()})


@pytest.mark.parametrize("B", [5, 150])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e-5, 1e-6, 1e-8, 1e-30])
def test_prefix_small_values(size, d, B):
    """bf16 values far below 1, with few and with many query tiles: the bound scales with them."""
    c = prefix_case(d, [3] * B, [1] * B, 400, 16, 2, d)
    c["vc"] = c["vc"] * size
    close16(prefix_call(c), prefix64(c), 2e-3 * size)


@pytest.mark.parametrize("B", [5, 150])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("by", ["head", "channel", "key"])
def test_prefix_values_of_mixed_size(by, d, B):
    """Values whose magnitude differs by kv head, by channel or by key over eight decades, and rows that one key
    all but fills: the bound, 2e-3 for values of order one, is one on every row's own sum of p |v|."""
    KV = 4
    c = prefix_case(d, [3] * B, [1] * B, 400, 16, KV, d, scale=4.0 if by == "key" else 1.0)
    blocks, bs = c["vc"].shape[:2]
    shape = dict(head=(1, 1, KV, 1), channel=(1, 1, 1, d), key=(blocks, bs, 1, 1))[by]
    size = 10.0 ** -(8 * torch.rand(shape, device="cuda", generator=gen(7)))
    c["vc"] = (c["vc"].float() * size).bfloat16()
    close16(prefix_call(c), prefix64(c), 2e-3 * weighted_magnitude(c))


def test_prefix_equals_whole_sequences():
    """The same keys as one block table per sequence, through paged_attention."""
    past, new, P, H, KV, d = [40, 7, 0], [1, 1, 1], 320, 32, 8, 128
    c = prefix_case(3, past, new, P, H, KV, d)
    got = check_prefix(c)
    k = torch.stack([c["kc"][c["table"][b, (p // 16)].long(), p % 16] for b, p in enumerate(past)]).reshape(3, -1)
    v = torch.stack([c["vc"][c["table"][b, (p // 16)].long(), p % 16] for b, p in enumerate(past)]).reshape(3, -1)
    table = torch.cat([c["ptable"][None].expand(3, -1), c["table"].clamp(min=0)], 1).contiguous()
    out, _, _ = paged_attention(c["q"], k, v, c["kc"].clone(), c["vc"].clone(), c["cum"], c["past"] + P, table,
                                num_heads=H, kv_num_heads=KV, check_status=True)
    assert (out.double() - got.double()).abs().max() <= 2e-3 * 2 + 2.0 ** -8


def test_prefix_strides_output_workspace_stream():
    c = prefix_case(4, [30, 0], [1, 40], 200, 8, 2, 128)
    want = check_prefix(c)
    wide = torch.nn.functional.pad(c["q"], (0, 24))[:, :1024]
    out = torch.full((41, 1024 + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    prefix_call({**c, "q": wide}, output=out[:, :1024])
    assert torch.equal(out[:, :1024], want) and (out[:, 1024:] == 7).all()
    ws = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    assert torch.equal(prefix_call(c, workspace=ws), want)
    ws.fill_(0xff)  # whatever the workspace holds
    assert torch.equal(prefix_call(c, workspace=ws), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = prefix_call(c, stream=side, check_status=False)
    side.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(prefix_call(c, num_sms=3), prefix_call(c, num_sms=3))
    close16(prefix_call(c, num_sms=1), prefix64(c), 2e-3)


def test_prefix_odd_row_alignment():
    """Queries and outputs whose rows start off 16 bytes."""
    c = prefix_case(4, [30, 0], [1, 40], 200, 8, 2, 64)
    want = check_prefix(c)
    for pad in (1, 2, 4):
        wide = torch.nn.functional.pad(c["q"], (0, pad))[:, :512]
        out = torch.zeros(41, 512 + pad, device="cuda", dtype=torch.bfloat16)[:, :512]
        close16(prefix_call({**c, "q": wide}, output=out), prefix64(c), 2e-3)
    flat = torch.cat([c["q"].flatten()[:1], c["q"].flatten()])[1:].view(41, 512)
    assert flat.data_ptr() % 16
    close16(prefix_call({**c, "q": flat}), prefix64(c), 2e-3)
    assert torch.equal(prefix_call(c), want)


def test_prefix_repeats_bit_for_bit():
    c = prefix_case(12, [500, 3, 900, 64] * 8, [1, 1, 2, 1] * 8, 3000, 32, 8, 128)
    want = prefix_call(c)
    for _ in range(5):
        assert torch.equal(prefix_call(c), want)


def test_prefix_offsets_beyond_32_bits():
    """Pages whose elements lie past 2^31 in the pool."""
    KV, d, bs = 8, 128, 16
    blocks = (1 << 31) // (bs * KV * d) + 64
    c = prefix_case(2, [20, 100], [1, 30], 150, 16, KV, d)
    n = c["kc"].shape[0]
    big = {}
    for name in ("kc", "vc"):
        big[name] = torch.empty(blocks, bs, KV, d, device="cuda", dtype=torch.bfloat16)
        big[name][blocks - n:] = c[name]
    far = {**c, **big, "table": torch.where(c["table"] >= 0, c["table"] + (blocks - n), -1), "ptable": c["ptable"] + (blocks - n)}
    assert torch.equal(prefix_call(far), prefix_call(c))
    q = rope_case(1, 6, 2, KV, d, 128)
    slots = torch.arange(6, device="cuda", dtype=torch.int32) + (blocks * bs - 40)
    rope_call({**q, "slots": slots}, big["kc"], big["vc"])
    assert torch.equal(big["vc"].view(-1, KV * d)[slots.long()], q["v"])


@pytest.mark.parametrize("change,message", [
    (lambda c: c["cum"].__setitem__(0, 1), "inconsistent"),
    (lambda c: c["cum"].__setitem__(3, 99), "inconsistent"),
    (lambda c: c["cum"].__setitem__(1, 40), "inconsistent"),
    (lambda c: c["past"].__setitem__(1, -4), "inconsistent"),
    (lambda c: c["past"].__setitem__(2, 5000), "inconsistent"),
    (lambda c: c["table"].__setitem__((0, 0), -1), "invalid physical block"),
    (lambda c: c["table"].__setitem__((1, 1), 10 ** 6), "invalid physical block"),
    (lambda c: c["ptable"].__setitem__(2, 1 << 20), "invalid physical block"),
    (lambda c: c["ptable"].__setitem__(0, -7), "invalid physical block"),
])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_prefix_invalid_metadata(change, message, d):
    c = prefix_case(6, [20, 40, 9], [1, 1, 30], 100, 8, 2, d)
    want = prefix_call(c)
    bad = {**c, "cum": c["cum"].clone(), "past": c["past"].clone(), "table": c["table"].clone(), "ptable": c["ptable"].clone()}
    change(bad)
    with pytest.raises(B200Error, match=message):
        prefix_call(bad)
    assert torch.equal(prefix_call(c), want)  # the next call is clean


def test_prefix_refusals():
    c = prefix_case(6, [20], [1], 100, 8, 2, 64)
    for change in (dict(q=c["q"].half()), dict(q=c["q"][:, :64]), dict(cum=c["cum"].long()), dict(past=c["past"][:0]),
                   dict(ptable=c["ptable"][:2]), dict(ptable=None), dict(kc=c["kc"].cpu()), dict(vc=c["vc"][1:]),
                   dict(H=6), dict(table=c["table"].t()), dict(sink=c["q"][0])):
        with pytest.raises((B200Error, ZeroDivisionError)):
            prefix_call({**c, **change})
    with pytest.raises(B200Error, match="workspace"):
        big = prefix_case(6, [20], [1], 100, 8, 2, 128)
        prefix_call(big, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_empty_calls():
    """No rows, no tokens, no sequences."""
    x = torch.empty(0, 256, device="cuda", dtype=torch.bfloat16)
    codes, scales, res = skip_rms_norm(x, x, torch.ones(256, device="cuda", dtype=torch.bfloat16), out_dtype=FP8, group_size=64)
    assert codes.shape == res.shape == (0, 256) and scales.shape == (0, 4)
    c = rope_case(1, 4, 4, 2, 64, 64)
    empty = {**c, "slots": c["slots"][:0], "pos": c["pos"][:, :0], **{n: c[n][:0] for n in "qkv"}}
    assert rope_call(empty, c["kc"], c["vc"])[0].shape == (0, 256)
    a = prefix_case(6, [20], [1], 100, 8, 2, 64)
    none = {**a, "q": a["q"][:0], "cum": a["cum"][:1], "past": a["past"][:0], "table": a["table"][:0]}
    assert prefix_call(none).shape == (0, 512)
    assert prefix_call({**a, "q": a["q"][:0], "cum": a["cum"] * 0}).shape == (0, 512)


def test_layer_in_a_graph():
    """The three operators captured in one CUDA graph and replayed on new inputs."""
    H, KV, d, B, P = 8, 2, 128, 5, 200
    c = prefix_case(1, [20, 0, 33, 7, 64], [1] * B, P, H, KV, d)
    g = gen(2)
    x, r, w = normal(g, B, 512), normal(g, B, 512), normal(g, 512)
    proj = normal(g, 512, (H + 2 * KV) * d, scale=0.05)
    angle = torch.randn(512, d // 2, device="cuda", generator=g)
    cos, sin = angle.cos().bfloat16(), angle.sin().bfloat16()
    slots = torch.stack([c["table"][b, p // 16] * 16 + p % 16 for b, p in enumerate(c["pasts"])]).int()
    pos = (c["past"] + P).long()

    def layer():
        y, res = skip_rms_norm(x, r, w)
        q, _, _ = rotary_append(y @ proj, None, None, c["kc"], c["vc"], pos, cos, sin, slots, num_heads=H, kv_num_heads=KV)
        return prefix_call({**c, "q": q}, check_status=False), res

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, res = layer()
    for seed in (3, 4):
        x.copy_(normal(gen(seed), B, 512))
        graph.replay()
        torch.cuda.synchronize()
        got, got_res = out.clone(), res.clone()
        want, want_res = layer()
        assert torch.equal(got, want) and torch.equal(got_res, want_res)
    del graph


def scratch_calls():
    """Two callables that need scratch, of different sizes: a rotation with more tokens than are searched and an
    attention call of four launches.  Each returns all that it wrote."""
    calls = []
    for seed, nt, prefix in ((5, 8500, ([300] * 40, [1] * 40, 3000, 32, 8, 128)), (6, 9000, ([5, 0, 90], [60, 1, 200], 1000, 16, 4, 64))):
        rope, attention = rope_case(seed, nt, 4, 1, 64, 64), prefix_case(seed, *prefix)
        rope["slots"][nt // 2:nt // 2 + 3000] = rope["slots"][:3000].clone()  # duplicates: the table decides

        def call(rope=rope, attention=attention):
            q, kc, vc = rope_call(rope, rope["kc"], rope["vc"], check_status=False)
            return q, kc, vc, prefix_call(attention, check_status=False)

        calls.append(call)
    return calls


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("on_side", [False, True])
def test_captured_graphs_have_scratch_of_their_own(on_side):
    """Two graphs captured on one stream (torch's default capture stream, or one that ran the calls before),
    replayed on two streams at once and beside eager calls on a third and on the capture stream."""
    calls = scratch_calls()
    capture = torch.cuda.Stream() if on_side else None
    wants = [[t.clone() for t in call()] for call in calls]
    if on_side:
        with torch.cuda.stream(capture):
            for call in calls:
                call()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=capture):
            outs.append(call())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    eager = prefix_case(8, [50, 7] * 20, [1] * 40, 2000, 32, 8, 128)
    want = prefix_call(eager)
    for _ in range(10):
        got = []
        for _ in range(4):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            got.append(prefix_call(eager, check_status=False))
            if on_side:
                with torch.cuda.stream(capture):
                    got.append(prefix_call(eager, check_status=False))
        torch.cuda.synchronize()
        assert same(outs[0], wants[0]) and same(outs[1], wants[1]) and all(torch.equal(g, want) for g in got)
    del graphs, graph


def bad_slots(c):
    return {**c, "slots": c["slots"].clone().fill_(1 << 30)}


def test_status_belongs_to_the_stream_of_the_call():
    """A bad call on one stream is not another stream's error, and stays its own stream's until read."""
    c, a = rope_case(3, 20, 4, 2, 64, 64), prefix_case(6, [20, 40], [1, 1], 100, 8, 2, 64)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    rope_call(bad_slots(c), c["kc"], c["vc"], check_status=False, stream=one)
    torch.cuda.synchronize()
    rope_call(c, c["kc"], c["vc"], stream=two)
    prefix_call(a, stream=two)
    prefix_call(a)
    layer.check_status(two)
    with pytest.raises(B200Error, match="slot_mapping"):
        prefix_call(a, stream=one)
    layer.check_status(one)  # read once
    rope_call(bad_slots(c), c["kc"], c["vc"], check_status=False, stream=one)
    with pytest.raises(B200Error, match="slot_mapping"):
        layer.check_status(one)


def test_status_of_a_graph_is_on_its_capture_stream():
    c = rope_case(3, 20, 4, 2, 64, 64)
    rope_call(c, c["kc"], c["vc"])  # the device's words exist
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    c["slots"] = c["slots"].clone()
    with torch.cuda.graph(graph, stream=side):
        rope_call(c, c["kc"], c["vc"], check_status=False)
    graph.replay()
    torch.cuda.synchronize()
    layer.check_status(side)
    c["slots"].fill_(-2)
    graph.replay()
    torch.cuda.synchronize()
    good = rope_case(4, 20, 4, 2, 64, 64)
    rope_call(good, good["kc"], good["vc"])
    with pytest.raises(B200Error, match="slot_mapping"):
        layer.check_status(side)
    layer.check_status(side)
    del graph


def test_scratch_of_a_graph_ends_with_it():
    """Captured again and again, the calls hold no more memory than one graph's."""
    import time

    call = scratch_calls()[0]
    call()

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call()
        graph.replay()
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated()

    first = capture()
    for _ in range(20):
        call()
        torch.cuda.synchronize()
        if capture() <= first:  # the driver reports a graph's end from a thread of its own
            break
        time.sleep(0.1)
    else:
        pytest.fail("scratch of deleted graphs is not freed")


def test_scratch_of_a_graph_lives_as_long_as_it():
    """Later eager calls, which free what ended graphs held, free nothing of a live one."""
    call = scratch_calls()[0]
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated()
        call()
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() == held
    del graph, outs


def test_first_call_of_a_process_in_a_capture_is_refused():
    import os
    import subprocess
    import sys

    code = """
import torch
from onnxruntime_ep_b200 import B200Error, shared_prefix_attention
q = torch.zeros(1, 128, device="cuda", dtype=torch.bfloat16)
kc = torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.bfloat16)
i = lambda *v: torch.tensor(v, device="cuda", dtype=torch.int32)
args = (q, kc, kc.clone(), i(0, 1), i(0), i(0)[None], i(1))
call = lambda: shared_prefix_attention(*args, prefix_length=16, num_heads=2, kv_num_heads=2, check_status=False)
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        call()
except B200Error as e:
    assert "cannot be captured" in str(e), e
else:
    raise AssertionError("captured")
call()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = call()
graph.replay()
torch.cuda.synchronize()
assert not out.any()
del graph
print("fine")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=os.path.join(root, "onnxruntime-ep-mlx_b200"))
    done = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "fine", done.stderr


def test_example_layer_against_whole_sequences():
    """The example's last decode step, recomputed from its caches with every sequence's keys in one piece."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "shared_prefix_decode.py")
    spec = importlib.util.spec_from_file_location("shared_prefix_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    H, KV, d = 8, 2, 128
    _, got, (layer, x, residual, past, table, ptable, P) = example.serve(batch=5, prefix=203, prompt=20, steps=6, hidden=512,
                                                                         heads=H, kv_heads=KV, head_size=d)
    # the step's own keys are in the cache: past counts them after the step
    codes, scales, _ = skip_rms_norm(x, residual, layer.norm, out_dtype=FP8)
    qkv = torch._scaled_mm(codes, layer.qkv.t(), scale_a=scales, scale_b=layer.qkv_scale, out_dtype=torch.bfloat16)
    q = qkv[:, :H * d].double().view(5, H, d)
    pos = P + past.long() - 1
    c, s = (t.double()[pos][:, None] for t in (layer.cos, layer.sin))
    a, b = q[..., :d // 2], q[..., d // 2:]
    q = torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().double()
    out = torch.empty(5, H, d, device="cuda", dtype=torch.float64)
    for i in range(5):
        n = int(past[i])
        rows = [torch.cat([cache[ptable.long()].reshape(-1, KV, d)[:P], cache[table[i].long()].reshape(-1, KV, d)[:n]]).double()
                for cache in (layer.key_cache, layer.value_cache)]
        scores = torch.einsum("kgd,skd->kgs", q[i].view(KV, H // KV, d), rows[0]) * d ** -0.5
        out[i] = torch.einsum("kgs,skd->kgd", scores.softmax(-1), rows[1]).reshape(H, d)
    want = out.view(5, H * d) @ layer.out.double()
    # bf16 attention output (2^-9 relative) and bf16 result: 2^-7 of the result's scale
    assert ((got.double() - want).abs() <= 2.0 ** -7 * want.abs().amax()).all()
