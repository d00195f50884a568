"""Measured cases of the decoder-layer operators: ``skip_rms_norm``, ``rotary_append`` and
``shared_prefix_attention``, with their plain forms in elementary torch operations and their
definitions in 64 bits.

``own`` chooses between the plain forms (False) and the package's kernels (True).
"""

from __future__ import annotations

import os
import random
import sys

import torch
import torch.nn.functional as F

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
AMAX_FLOOR = 1e-12  # smallest magnitude a scale is made from (an all-zero row or group)
EPSILON = 1e-6

_package = None


def package():
    global _package
    if _package is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnxruntime-ep-mlx_b200")
        for path in (os.path.join(os.getcwd(), "onnxruntime-ep-mlx_b200"), root):
            if os.path.isdir(path) and path not in sys.path:
                sys.path.insert(0, path)
        import onnxruntime_ep_b200
        _package = onnxruntime_ep_b200
    return _package


# --------------------------------------------------------------------------------------- cases
# norm: tokens, hidden, type of the activations, quant ("none", "row" or a group size in channels)
# rope: tokens, heads, kv heads, head size, rotated channels, axes, pair layout, packed QKV, share
#       of padding tokens (slot -1), cache ("same" or "fp8"), block size
# attn: sequences, heads, kv heads, head size, prefix keys, cached suffix keys from/to, new tokens
#       from/to, soft cap, sink, block size; `lens` seeds the ragged lengths


def listed():
    return [
        # one token of a chat: the norm before a layer's projection, where only latency counts
        dict(name="norm_token", op="norm", tokens=1, hidden=4096, type="bf16", quant="none"),
        # a decode batch of an odd-sized model whose projection takes e4m3 in groups of 128
        dict(name="norm_group_odd", op="norm", tokens=333, hidden=2880, type="fp16", quant="128"),
        # a prefill chunk whose projection takes e4m3 rows
        dict(name="norm_chunk_fp8", op="norm", tokens=16384, hidden=4096, type="bf16", quant="row"),
        # a decode batch: 128 sequences, one token each
        dict(name="rope_decode", op="rope", tokens=128, heads=32, kv=8, dim=128, rot=128, axes=1, interleaved=0,
             packed=0, skip=0.0, cache="same", block=16, type="bf16"),
        # an image's tokens: time, height and width positions, packed QKV, some padding
        dict(name="rope_image", op="rope", tokens=8192, heads=32, kv=8, dim=128, rot=128, axes=3, interleaved=0,
             packed=1, skip=0.02, cache="same", block=16, type="bf16"),
        # small heads, half of the channels rotated in neighbouring pairs, an odd number of tokens
        dict(name="rope_partial_odd", op="rope", tokens=1001, heads=14, kv=2, dim=64, rot=32, axes=1, interleaved=1,
             packed=0, skip=0.1, cache="same", block=32, type="fp16"),
        # prefill into an e4m3 cache
        dict(name="rope_fp8_cache", op="rope", tokens=4096, heads=64, kv=8, dim=128, rot=128, axes=1, interleaved=0,
             packed=1, skip=0.0, cache="fp8", block=16, type="bf16"),
        # a few sequences on a short system prompt
        dict(name="attn_few", op="attn", batch=4, heads=32, kv=8, dim=128, prefix=1024, past=1, past_to=64, new=1,
             new_to=1, softcap=0.0, sink=0, block=16, type="bf16", lens=1),
        # the ordinary decode batch: 128 sequences on a long shared prompt
        dict(name="attn_decode", op="attn", batch=128, heads=32, kv=8, dim=128, prefix=8192, past=32, past_to=1024,
             new=1, new_to=1, softcap=0.0, sink=0, block=16, type="bf16", lens=2),
        # drafted tokens are verified: 1 to 5 per sequence, 7 heads per kv head, ragged prefix, soft cap and sink
        dict(name="attn_verify_odd", op="attn", batch=31, heads=28, kv=4, dim=128, prefix=3001, past=0, past_to=700,
             new=1, new_to=5, softcap=30.0, sink=1, block=16, type="fp16", lens=3),
        # prompts of up to 512 tokens after a shared instruction, small heads
        dict(name="attn_prompts", op="attn", batch=16, heads=16, kv=16, dim=64, prefix=4096, past=0, past_to=0, new=17,
             new_to=512, softcap=0.0, sink=0, block=64, type="bf16", lens=4),
        # the largest: 256 sequences, 64 query heads, a shared document
        dict(name="attn_document", op="attn", batch=256, heads=64, kv=8, dim=128, prefix=16384, past=128, past_to=2048,
             new=1, new_to=1, softcap=0.0, sink=0, block=16, type="bf16", lens=5),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.random()
    if kind < 0.25:
        hidden = rng.choice([_log(rng, 256, 8192), 8 * _log(rng, 32, 1024), 1024 * rng.randint(1, 8)])
        tokens = _log(rng, 1, max(1, 16384 * 4096 // max(hidden, 4096)))
        return dict(op="norm", tokens=tokens, hidden=hidden, type=rng.choice(["bf16", "fp16"]),
                    quant=rng.choice(["none", "row", "128", "64"]))
    if kind < 0.55:
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 5, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
        axes = rng.choice([1, 1, 2, 3])
        rot = rng.choice([dim, dim, dim // 2])
        most = max(1, 8192 * 48 * 128 // ((heads + 2 * kv) * dim))
        return dict(op="rope", tokens=_log(rng, 1, min(16384, most)), heads=heads, kv=kv, dim=dim, rot=rot, axes=axes,
                    interleaved=rng.choice([0, 0, 1]), packed=rng.choice([0, 1]), skip=rng.choice([0.0, 0.05, 0.5]),
                    cache=rng.choice(["same", "same", "fp8"]), block=rng.choice([16, 32, 64]),
                    type=rng.choice(["bf16", "fp16"]))
    while True:
        kv = rng.choice([1, 2, 4, 8, 8])
        case = dict(op="attn", batch=_log(rng, 1, 256), heads=kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), kv=kv,
                    dim=rng.choice([64, 128, 128]), prefix=rng.choice([_log(rng, 16, 16384), 128 * _log(rng, 1, 128)]),
                    past=0, past_to=_log(rng, 1, 2048), new=1, new_to=rng.choice([1, 1, 4, _log(rng, 2, 512)]),
                    softcap=rng.choice([0.0, 0.0, 50.0]), sink=rng.choice([0, 0, 1]), block=rng.choice([16, 16, 32, 64]),
                    type=rng.choice(["bf16", "fp16"]), lens=rng.randint(1, 1 << 30))
        w = work(case)
        # the scores of the plain form have to fit as well: (tokens x heads) x keys
        scores = case["batch"] * case["heads"] * case["new_to"] * (case["prefix"] + case["past_to"] + case["new_to"])
        if w["flops"] < 1.3e11 and w["bytes"] < 1.1e9 and scores < 6e8:
            return case


def _lengths(case):
    """(cached suffix keys, new tokens) of every sequence."""
    r = random.Random(case["lens"])
    past = [r.randint(case["past"], case["past_to"]) for _ in range(case["batch"])]
    new = [r.randint(case["new"], case["new_to"]) for _ in range(case["batch"])]
    return past, new


def work(case):
    if case["op"] == "norm":
        n = case["tokens"] * case["hidden"]
        group = case["hidden"] if case["quant"] in ("none", "row") else int(case["quant"])
        scales = 0 if case["quant"] == "none" else 4 * case["tokens"] * -(-case["hidden"] // group)
        return {"bytes": n * (6 + (2 if case["quant"] == "none" else 1)) + scales + 2 * case["hidden"], "flops": 8 * n}
    if case["op"] == "rope":
        q, k = case["heads"] * case["dim"], case["kv"] * case["dim"]
        kept = round(case["tokens"] * (1 - case["skip"]))
        cached = kept * 2 * k
        size = 1 if case["cache"] == "fp8" else 2
        table = min(case["tokens"], POSITIONS) * case["rot"] * 2
        return {"bytes": 4 * case["tokens"] * q + cached * (2 + size) + case["tokens"] * (8 * case["axes"] + 4) + table,
                "flops": 3 * (case["tokens"] * case["heads"] + kept * case["kv"]) * case["rot"]}
    past, new = _lengths(case)
    d, heads, kv = case["dim"], case["heads"], case["kv"]
    keys = case["prefix"] + sum(p + n for p, n in zip(past, new))
    pairs = sum(n * (case["prefix"] + p) + n * (n + 1) // 2 for p, n in zip(past, new))
    return {"bytes": keys * kv * d * 4 + sum(new) * heads * d * 4, "flops": 4 * d * heads * pairs}


# --------------------------------------------------------------------------------------- inputs
POSITIONS = 8192  # rows of the cos / sin tables


def _normal(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _positions(n, axes, gen):
    """Decode: every token somewhere in its own sequence.  Prefill: consecutive; further axes are an
    image's rows and columns."""
    if n <= 256:
        return torch.randint(0, POSITIONS, (axes, n), device="cuda", generator=gen)
    pos = torch.randint(0, 64, (axes, n), device="cuda", generator=gen)
    pos[0] = (torch.randint(0, POSITIONS, (1,), device="cuda", generator=gen) + torch.arange(n, device="cuda")) % POSITIONS
    return pos


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]
    state = {"case": case}
    if case["op"] == "norm":
        n, h = case["tokens"], case["hidden"]
        state.update(x=_normal((n, h), t, gen, 0.7), residual=_normal((n, h), t, gen, 2.0),
                     weight=_normal((h,), t, gen, 0.1) + 1)
        return state
    if case["op"] == "rope":
        n, H, KV, d, rot, axes = (case[k] for k in ("tokens", "heads", "kv", "dim", "rot", "axes"))
        if case["packed"]:
            qkv = _normal((n, (H + 2 * KV) * d), t, gen)
            state.update(query=qkv, key=None, value=None)
        else:
            state.update(query=_normal((n, H * d), t, gen), key=_normal((n, KV * d), t, gen),
                         value=_normal((n, KV * d), t, gen))
        angle = torch.arange(POSITIONS, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(rot // 2, device="cuda") / (rot // 2))
        sections = [rot // 2 // axes] * axes
        sections[0] += rot // 2 - sum(sections)
        pair_axis = torch.repeat_interleave(torch.arange(axes, device="cuda"), torch.tensor(sections, device="cuda"))
        blocks = -(-n // case["block"]) + 3
        slots = torch.randperm(blocks * case["block"], device="cuda", generator=gen)
        slots = slots[slots != 0][:n].to(torch.int32)  # slot 0 stays unused
        skipped = torch.rand(n, device="cuda", generator=gen) < case["skip"]
        state.update(
            cos=angle.cos().to(t), sin=angle.sin().to(t), pair_axis=pair_axis,
            sections=None if axes == 1 else tuple(sections),
            positions=_positions(n, axes, gen),
            slots=torch.where(skipped, torch.full_like(slots, -1), slots))
        shape = (blocks, case["block"], KV, d)
        caches = [_normal(shape, t, gen), _normal(shape, t, gen)]
        scales = [None, None]
        if case["cache"] == "fp8":
            caches = [c.to(FP8) for c in caches]
            scales = [torch.rand((blocks, KV), device="cuda", generator=gen) * 0.02 + 0.005 for _ in caches]
        state.update(key_cache=caches[0], value_cache=caches[1], k_scale=scales[0], v_scale=scales[1])
        return state
    past, new = _lengths(case)
    B, H, KV, d, bs, P = (case[k] for k in ("batch", "heads", "kv", "dim", "block", "prefix"))
    own_blocks = [-(-(p + n) // bs) for p, n in zip(past, new)]
    prefix_blocks = -(-P // bs)
    total = prefix_blocks + sum(own_blocks)
    order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    width = max(own_blocks)
    counts = torch.tensor(own_blocks, device="cuda")
    column = torch.arange(width, device="cuda")
    used = column[None, :] < counts[:, None]
    first = torch.cumsum(counts, 0) - counts
    table = torch.where(used, order[prefix_blocks:][(first[:, None] + column[None, :]).clamp(max=sum(own_blocks) - 1)],
                        torch.zeros((), dtype=torch.int32, device="cuda"))
    cum = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    state.update(
        query=_normal((sum(new), H * d), t, gen, 2.0),
        key_cache=_normal((total, bs, KV, d), t, gen), value_cache=_normal((total, bs, KV, d), t, gen),
        cum=cum, past=torch.tensor(past, dtype=torch.int32, device="cuda"), table=table.contiguous(),
        prefix_table=order[:prefix_blocks].contiguous(),
        sink=_normal((H,), t, gen) if case["sink"] else None, widest_new=max(new))
    return state


# --------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if op == "norm":
        return (own_norm if own else plain_norm)(state, case)
    if op == "rope":
        return (own_rope if own else plain_rope)(state, case)
    return (own_attn if own else plain_attn)(state, case)


def own_norm(s, case):
    quant = case["quant"]
    if quant == "none":
        return package().skip_rms_norm(s["x"], s["residual"], s["weight"], epsilon=EPSILON)
    return package().skip_rms_norm(s["x"], s["residual"], s["weight"], epsilon=EPSILON, out_dtype=FP8,
                                   group_size=0 if quant == "row" else int(quant))


def own_rope(s, case):
    return package().rotary_append(
        s["query"], s["key"], s["value"], s["key_cache"], s["value_cache"], s["positions"], s["cos"], s["sin"],
        s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"], num_heads=case["heads"], kv_num_heads=case["kv"],
        axis_sections=s["sections"], rotary_interleaved=case["interleaved"])


def own_attn(s, case):
    return package().shared_prefix_attention(
        s["query"], s["key_cache"], s["value_cache"], s["cum"], s["past"], s["table"], s["prefix_table"],
        head_sink=s["sink"], prefix_length=case["prefix"], num_heads=case["heads"], kv_num_heads=case["kv"],
        softcap=case["softcap"])


def plain_norm(s, case):
    t = s["x"].dtype
    total = s["x"].float() + s["residual"].float()
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + EPSILON) * s["weight"].float()
    if case["quant"] == "none":
        return y.to(t), total.to(t)
    n, h = y.shape
    group = h if case["quant"] == "row" else int(case["quant"])
    y = F.pad(y, (0, -h % group)).view(n, -1, group)
    scale = y.abs().amax(-1).clamp(min=AMAX_FLOOR) / FP8_MAX
    code = (y / scale[..., None]).clamp(-FP8_MAX, FP8_MAX).view(n, -1)[:, :h].to(FP8)
    return code, scale, total.to(t)


def plain_rope(s, case):
    H, KV, d, rot = case["heads"], case["kv"], case["dim"], case["rot"]
    q, k, v = s["query"], s["key"], s["value"]
    if k is None:
        q, k, v = q.split([H * d, KV * d, KV * d], dim=1)
    n, t = q.shape[0], q.dtype
    pos = s["positions"][s["pair_axis"]].t()  # [tokens, pairs]
    pair = torch.arange(rot // 2, device=pos.device)
    c, si = s["cos"][pos, pair].float()[:, None], s["sin"][pos, pair].float()[:, None]

    def rotate(x, heads):
        x = x.reshape(n, heads, d).float()
        if case["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            r = torch.stack([a * c - b * si, b * c + a * si], -1).flatten(-2)
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            r = torch.cat([a * c - b * si, b * c + a * si], -1)
        return torch.cat([r, x[..., rot:]], -1)

    out = rotate(q, H).to(t).view(n, H * d)
    slot = s["slots"].long()
    valid = (slot >= 0)[:, None, None]
    slot = slot.clamp(min=0)  # skipped tokens write slot 0's own content back

    def store(cache, rows, scale):
        flat = cache.view(-1, KV, d)
        if scale is not None:
            rows = (rows / scale[slot // case["block"]][..., None]).clamp(-FP8_MAX, FP8_MAX)
            rows, flat = rows.to(FP8).view(torch.uint8), flat.view(torch.uint8)
        else:
            rows = rows.to(t)
        flat[slot] = torch.where(valid, rows, flat[:1])

    store(s["key_cache"], rotate(k, KV), s["k_scale"])
    store(s["value_cache"], v.reshape(n, KV, d).float(), s["v_scale"])
    return out, s["key_cache"], s["value_cache"]


def plain_attn(s, case):
    B, H, KV, d, P, cap = (case[k] for k in ("batch", "heads", "kv", "dim", "prefix", "softcap"))
    g, N, cum = H // KV, s["widest_new"], s["cum"].long()
    past, new = s["past"].long(), cum[1:] - cum[:-1]
    dev = cum.device

    def gather(cache, table):  # fp32 [..., keys, KV, d]
        return cache[table.long()].flatten(-4, -3).float()

    # queries padded to [B, N, H, d]
    i = torch.arange(N, device=dev)
    token = (cum[:-1, None] + i).clamp(max=s["query"].shape[0] - 1)
    q = s["query"][token].float().view(B, N, KV, g, d) * d ** -0.5
    kp, vp = (gather(s[c], s["prefix_table"])[:P] for c in ("key_cache", "value_cache"))
    ks, vs = (gather(s[c], s["table"]) for c in ("key_cache", "value_cache"))
    rows = q.permute(2, 0, 1, 3, 4)  # [KV, B, N, g, d]
    prefix = torch.matmul(rows.reshape(KV, B * N * g, d), kp.permute(1, 2, 0)).view(KV, B, N * g, P)
    suffix = torch.matmul(rows.reshape(KV, B, N * g, d), ks.permute(2, 0, 3, 1))  # [KV, B, N*g, S]
    scores = torch.cat([prefix, suffix], -1)
    if cap > 0:
        scores = cap * torch.tanh(scores / cap)
    key = torch.arange(ks.shape[1], device=dev)
    hidden = key[None, None, :] > (past[:, None] + i)[:, :, None]  # [B, N, S]
    hidden = hidden.repeat_interleave(g, 1)
    scores[..., P:].masked_fill_(hidden, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].float().view(KV, 1, 1, g).expand(KV, 1, N, g).reshape(KV, 1, N * g, 1)
        total = total + torch.exp(sink - top)
    # the pages' unused slots hold whatever was there: their weight is 0 and their values count as 0
    vs = vs.masked_fill((key[None, :] >= (past + new)[:, None])[:, :, None, None], 0.0)
    o = torch.matmul(e[..., :P].reshape(KV, B * N * g, P), vp.permute(1, 0, 2)).view(KV, B, N * g, d)
    o = (o + torch.matmul(e[..., P:], vs.permute(2, 0, 1, 3))) / total
    o = o.view(KV, B, N, g, d).permute(1, 2, 0, 3, 4).reshape(B * N, H * d).to(s["query"].dtype)
    # back to packed tokens
    nt = s["query"].shape[0]
    seq = torch.searchsorted(cum, torch.arange(nt, device=dev), right=True) - 1
    return o[seq * N + torch.arange(nt, device=dev) - cum[seq]]


# --------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": exact_norm, "rope": exact_rope, "attn": exact_attn}[case["op"]](s, case)


def exact_norm(s, case):
    x = s["x"].double() + s["residual"].double()
    y = x / (x.pow(2).sum(1, keepdim=True) / x.shape[1] + EPSILON).sqrt() * s["weight"].double()
    if case["quant"] == "none":
        return y, x
    parts = [y] if case["quant"] == "row" else list(y.split(int(case["quant"]), 1))
    scales = [torch.clamp(p.abs().max(1).values, min=AMAX_FLOOR) / FP8_MAX for p in parts]
    # the codes' values before their rounding to 8 bits
    codes = torch.cat([p / a[:, None] for p, a in zip(parts, scales)], 1)
    return codes, torch.stack(scales, 1), x


def exact_rope(s, case):
    H, KV, d, rot = case["heads"], case["kv"], case["dim"], case["rot"]
    q, k, v = s["query"], s["key"], s["value"]
    if k is None:
        k, v, q = q[:, H * d:(H + KV) * d], q[:, (H + KV) * d:], q[:, :H * d]
    n = q.shape[0]
    half = rot // 2
    where = [(2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half) for i in range(half)]
    first = torch.tensor([a for a, _ in where], device=q.device)
    second = torch.tensor([b for _, b in where], device=q.device)
    c = torch.empty((n, 1, half), dtype=torch.float64, device=q.device)
    si = torch.empty_like(c)
    at = 0
    for axis, count in enumerate(s["sections"] or (half,)):
        c[:, 0, at:at + count] = s["cos"].double()[s["positions"][axis], at:at + count]
        si[:, 0, at:at + count] = s["sin"].double()[s["positions"][axis], at:at + count]
        at += count

    def turned(x, heads):
        x = x.double().reshape(n, heads, d)
        y = x.clone()
        y[:, :, first] = x[:, :, first] * c - x[:, :, second] * si
        y[:, :, second] = x[:, :, second] * c + x[:, :, first] * si
        return y

    kept = torch.nonzero(s["slots"] >= 0)[:, 0]
    slot = s["slots"][kept].long()

    def stored(cache, rows, scale):
        flat = cache.double().reshape(-1, KV, d)
        rows = rows[kept]
        if scale is not None:  # the codes' values before their rounding to 8 bits
            rows = (rows / scale.double()[slot // case["block"]][:, :, None]).clamp(-FP8_MAX, FP8_MAX)
        flat[slot] = rows
        return flat.view(cache.shape)

    return (turned(q, H).reshape(n, H * d), stored(s["key_cache"], turned(k, KV), s["k_scale"]),
            stored(s["value_cache"], v.double().reshape(n, KV, d), s["v_scale"]))


def exact_attn(s, case):
    H, KV, d, P, bs, cap = (case[k] for k in ("heads", "kv", "dim", "prefix", "block", "softcap"))
    g = H // KV
    past, new = _lengths(case)
    out = torch.empty((sum(new), H, d), dtype=torch.float64, device="cuda")

    def rows(cache, table, count):
        return cache[table[:-(-count // bs)].long()].reshape(-1, KV, d)[:count].double().transpose(0, 1)

    kp, vp = rows(s["key_cache"], s["prefix_table"], P), rows(s["value_cache"], s["prefix_table"], P)
    at = 0
    for b, (p, n) in enumerate(zip(past, new)):
        k = torch.cat([kp, rows(s["key_cache"], s["table"][b], p + n)], 1)  # [KV, keys, d]
        v = torch.cat([vp, rows(s["value_cache"], s["table"][b], p + n)], 1)
        q = s["query"][at:at + n].double().view(n, KV, g, d).permute(1, 2, 0, 3).reshape(KV, g * n, d)
        x = q @ k.transpose(1, 2) / d ** 0.5
        if cap > 0:
            x = (x / cap).tanh() * cap
        x = x.view(KV, g, n, -1)
        late = torch.arange(P + p + n, device="cuda")[None, :] > (P + p + torch.arange(n, device="cuda"))[:, None]
        x = x.masked_fill(late, float("-inf"))
        if s["sink"] is not None:
            x = torch.cat([x, s["sink"].double().view(KV, g, 1, 1).expand(KV, g, n, 1)], -1)
        w = torch.softmax(x, -1)[..., :P + p + n]
        o = (w.reshape(KV, g * n, -1) @ v).view(KV, g, n, d)
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, H, d)
        at += n
    return out.view(sum(new), H * d)
