"""The attention of a transformer layer as a server runs it: INT8 projections
around a paged 8-bit key/value cache.

  layer = CachedAttention(qkv, out, cache, angles, q_heads=32)
  y = layer(x, lengths, table)               # one new token for every sequence
  y = layer(x, lengths, table, offsets=...)  # prompts, or chunks of them

x -> fused W8A8 projection to queries, keys and values -> keys and queries
rotated and keys and values appended to the cache in one launch -> attention
over the cache -> fused W8A8 output projection.  Run as a module it serves a
few made-up prompts and tokens:

  python -m rdna2_ops.cached_attention
"""
from __future__ import annotations

import torch

from . import _args
from .convrot_checkpoint import Int8Linear, quantize_convrot
from .kv_cache import PagedKVCache
from .rotary import rope_table


class CachedAttention:
    """qkv: Int8Linear of (q_heads + 2 * kv_heads) * head_dim outputs, the
    queries' rows first, then the keys', then the values'.  out: Int8Linear of
    q_heads * head_dim inputs.  cache: this layer's PagedKVCache.  angles: a
    rope_table, or None for no rotation."""

    def __init__(self, qkv, out, cache, angles=None, *, q_heads, rotation_block=128, layout="half", window=None):
        _args.require(isinstance(qkv, Int8Linear) and isinstance(out, Int8Linear), TypeError,
                      "qkv and out must be Int8Linear")
        _args.require(isinstance(cache, PagedKVCache), TypeError, "cache must be a PagedKVCache")
        rows = (q_heads + 2 * cache.kv_heads) * cache.head_dim
        _args.require(qkv.out_features == rows, ValueError,
                      f"qkv has {qkv.out_features} outputs, expected {rows}")
        _args.require(out.in_features == q_heads * cache.head_dim, ValueError,
                      f"out has {out.in_features} inputs, expected {q_heads * cache.head_dim}")
        self.qkv, self.out, self.cache, self.angles = qkv, out, cache, angles
        self.q_heads, self.rotation_block, self.layout, self.window = q_heads, rotation_block, layout, window

    def __call__(self, x, lengths, table, *, offsets=None, max_new=None):
        """x [tokens, features] (fp16 or bf16), packed as PagedKVCache packs a
        call's tokens; lengths count them already.  Returns [tokens, out features]."""
        kv, heads = self.cache.kv_heads, self.q_heads
        both = self.qkv(x, rotation_block=self.rotation_block).view(x.shape[0], heads + 2 * kv, self.cache.head_dim)
        q, k, v = both[:, :heads], both[:, heads:heads + kv], both[:, heads + kv:]
        if self.angles is None:
            self.cache.append(k, v, lengths, table, offsets=offsets)
        else:
            q = self.cache.append(k, v, lengths, table, offsets=offsets, q=q, angles=self.angles, layout=self.layout)
        y = self.cache.attend(q, lengths, table, offsets=offsets, max_new=max_new, window=self.window)
        return self.out(y.view(x.shape[0], heads * self.cache.head_dim), rotation_block=self.rotation_block)


def main():
    torch.manual_seed(20261106)
    features, q_heads, kv_heads, head_dim, page = 1024, 8, 2, 128, 64
    prompts, steps = [300, 45, 1, 170], 20

    def linear(rows, columns):
        return quantize_convrot(torch.randn(rows, columns, device="cuda") * 0.02, rotation_block=128)

    need = [(n + steps + page - 1) // page for n in prompts]
    table = torch.full((len(prompts), max(need)), -1, dtype=torch.int32)
    pages = iter(torch.randperm(sum(need)).tolist())
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([next(pages) for _ in range(n)])
    table = table.cuda()
    layer = CachedAttention(linear((q_heads + 2 * kv_heads) * head_dim, features), linear(features, q_heads * head_dim),
                            PagedKVCache(sum(need), kv_heads, head_dim, page_size=page),
                            rope_table(max(prompts) + steps, head_dim), q_heads=q_heads)
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, *torch.tensor(prompts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(prompts), features, device="cuda").half()
    y = layer(x, lengths, table, offsets=offsets, max_new=max(prompts))
    rms = y.float().square().mean().sqrt().item()
    print(f"{len(prompts)} prompts, {sum(prompts)} tokens: output {tuple(y.shape)}, rms {rms:.4f}")
    x = y[(offsets[1:] - 1).long()]
    for _ in range(steps):
        lengths += 1
        x = layer(x, lengths, table)
        x = (x / x.float().square().mean(-1, keepdim=True).sqrt()).half()
    print(f"{steps} steps of {len(prompts)} tokens: lengths {lengths.tolist()}")


if __name__ == "__main__":
    main()
