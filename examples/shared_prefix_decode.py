"""A decoder layer's attention half, served to a batch that shares one prompt.

    python examples/shared_prefix_decode.py [--batch 64] [--prefix 4096] [--steps 32]

One layer with random weights: residual + RMS norm (fp8 e4m3 rows for the fp8 QKV projection), the
rotation of the new queries and keys with the append to the paged cache, attention over the shared
prefix and each sequence's own keys, and the output projection.  The shared prompt goes in once as an
ordinary prefill, every sequence's own prompt follows as a ragged batch, then single tokens are decoded
from a captured CUDA graph.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onnxruntime-ep-mlx_b200"))
from onnxruntime_ep_b200 import rotary_append, shared_prefix_attention, skip_rms_norm  # noqa: E402

FP8 = torch.float8_e4m3fn


class Layer:
    """Weights, the paged cache of one layer and its block pool."""

    def __init__(self, *, hidden=2048, heads=16, kv_heads=4, head_size=128, blocks=4096, block_size=16,
                 positions=32768, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *shape, s=1.0: (torch.randn(*shape, device="cuda", generator=gen) * s).bfloat16()
        self.heads, self.kv_heads, self.head_size, self.block_size = heads, kv_heads, head_size, block_size
        self.norm = normal(hidden, s=0.1) + 1
        qkv = normal((heads + 2 * kv_heads) * head_size, hidden, s=hidden ** -0.5).float()
        self.qkv_scale = qkv.abs().amax(1, keepdim=True).t() / 448  # one scale per output channel
        self.qkv = (qkv / self.qkv_scale.t()).to(FP8)
        self.out = normal(heads * head_size, hidden, s=hidden ** -0.5)
        angle = torch.arange(positions, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(head_size // 2, device="cuda") / (head_size // 2))
        self.cos, self.sin = angle.cos(), angle.sin()  # fp32 tables
        self.key_cache = torch.zeros(blocks, block_size, kv_heads, head_size, device="cuda", dtype=torch.bfloat16)
        self.value_cache = torch.zeros_like(self.key_cache)

    def __call__(self, x, residual, positions, slots, cum, past, table, prefix_table, prefix_length):
        """(layer output, residual stream) of the packed new tokens ``x`` [tokens, hidden]."""
        codes, scales, residual = skip_rms_norm(x, residual, self.norm, out_dtype=FP8)
        qkv = torch._scaled_mm(codes, self.qkv.t(), scale_a=scales, scale_b=self.qkv_scale, out_dtype=torch.bfloat16)
        q, _, _ = rotary_append(qkv, None, None, self.key_cache, self.value_cache, positions, self.cos, self.sin, slots,
                                num_heads=self.heads, kv_num_heads=self.kv_heads)
        o = shared_prefix_attention(q, self.key_cache, self.value_cache, cum, past, table, prefix_table,
                                    prefix_length=prefix_length, num_heads=self.heads, kv_num_heads=self.kv_heads)
        return o @ self.out, residual


def slots_of(table, positions, block_size):
    """Cache slots of own positions in the rows of a block table (both [sequences, n] or [n])."""
    return (torch.gather(table, -1, positions // block_size) * block_size + positions % block_size).to(torch.int32)


def serve(*, batch=64, prefix=4096, prompt=48, steps=32, hidden=2048, heads=16, kv_heads=4, head_size=128, seed=0):
    """Prefill the shared prompt, the own prompts (ragged, up to ``prompt`` tokens) and ``steps`` single
    tokens.  Returns (milliseconds per decode step, last layer output, the layer and its metadata)."""
    bs = 16
    pages = -(-prefix // bs)
    own_pages = -(-(prompt + steps) // bs)
    layer = Layer(hidden=hidden, heads=heads, kv_heads=kv_heads, head_size=head_size, blocks=pages + batch * own_pages,
                  block_size=bs, seed=seed)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    rows = lambda n: torch.randn(n, hidden, device="cuda", generator=gen).bfloat16()
    order = torch.randperm(pages + batch * own_pages, device="cuda", generator=gen).to(torch.int32)
    prefix_table, table = order[:pages].contiguous(), order[pages:].view(batch, own_pages).contiguous()
    i32 = lambda x: torch.as_tensor(x, device="cuda").to(torch.int32)

    # the shared prompt: one sequence without a prefix of its own
    at = torch.arange(prefix, device="cuda")
    layer(rows(prefix), None, at, slots_of(prefix_table.long(), at, bs), i32([0, prefix]), i32([0]), prefix_table[None],
          None, 0)
    # every sequence's own prompt
    lengths = torch.randint(1, prompt + 1, (batch,), device="cuda", generator=gen)
    cum = torch.cat([lengths.new_zeros(1), lengths.cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(batch, device="cuda"), lengths)
    own = torch.arange(int(cum[-1]), device="cuda") - cum[seq]
    layer(rows(len(seq)), rows(len(seq)), prefix + own, slots_of(table[seq].long(), own[:, None], bs)[:, 0], i32(cum),
          i32(torch.zeros(batch)), table, prefix_table, prefix)

    # single tokens: inputs that the captured step reads
    past = i32(lengths)
    x, residual = rows(batch), rows(batch)
    cum = i32(torch.arange(batch + 1))

    def step():
        own = past.long()
        slots = slots_of(table.long(), own[:, None], bs)[:, 0]
        y, r = layer(x, residual, prefix + own, slots, cum, past, table, prefix_table, prefix)
        past.add_(1)
        return y, r

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # before the capture: the first call on a device allocates its status word
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, r = step()
    graph.replay()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(steps - 2):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    result = y.clone()
    del graph
    return begin.elapsed_time(end) / max(1, steps - 2), result, (layer, x, residual, past, table, prefix_table, prefix)


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--batch", type=int, default=64)
    parser.add_argument("--prefix", type=int, default=4096)
    parser.add_argument("--prompt", type=int, default=48)
    parser.add_argument("--steps", type=int, default=32)
    a = parser.parse_args()
    ms, _, _ = serve(batch=a.batch, prefix=a.prefix, prompt=a.prompt, steps=a.steps)
    print(f"{a.batch} sequences on a shared prompt of {a.prefix} tokens: {ms * 1e3:.1f} us per layer step, "
          f"{a.batch / ms * 1e3:.0f} tokens/s through one layer")
