"""One layer's attention over the 8-bit KV cache, operator by operator.

    python examples/kv8_cache.py                   # on the GPU where there is one
    python examples/kv8_cache.py --device cpu --prompt 100 --steps 3

A prompt is written and attended to in chunks, tokens are decoded one by one, and the request's rows then
leave the cache (``kv8_read``) and enter another one through its own pages, as a finished prefix that
moves to another engine does.  Prints how far the outputs are from attention over unrounded keys and values.
"""
import argparse
import math

import torch

from sglang_omni_b200 import ops
from sglang_omni_b200.ops.rope import rope_tables

PAGE = 64


def dense(q, k, v):
    """Attention of each row of q [n, Hq, D], the last n of the keys, in fp32."""
    g, n = q.shape[1] // k.shape[1], k.shape[0]
    s = torch.einsum("ahd,nhd->han", q.float(), k.float().repeat_interleave(g, 1)) / math.sqrt(q.shape[-1])
    i = torch.arange(n - q.shape[0], n, device=q.device)[:, None]
    p = s.masked_fill(torch.arange(n, device=q.device) > i, float("-inf")).softmax(-1)
    return torch.einsum("han,nhd->ahd", p, v.float().repeat_interleave(g, 1))


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--chunk", type=int, default=256)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args(argv)
    hq, hkv, d, n = 16, 4, 128, a.prompt + a.steps
    dev = torch.device(a.device)
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).bfloat16().to(dev)
    cos, sin = rope_tables(d, 1e6, n, dev)
    pages = -(-n // PAGE)
    table = (torch.randperm(pages, generator=g) + 1).int()[None].to(dev)          # page 0 stays the padding page
    pos = torch.arange(n, dtype=torch.int32, device=dev)
    slots = table[0, (pos // PAGE).long()] * PAGE + pos % PAGE
    cache = ops.KV8Cache.zeros(pages + 1, hkv, d, dev)
    worst = 0.0
    at = 0
    while at < n:
        new = min(a.chunk, a.prompt - at) if at < a.prompt else 1
        rows = slice(at, at + new)
        q = ops.kv8_store(qkv[rows], cache, slots[rows], hq, hkv, d, pos[rows], cos, sin)
        lens = torch.tensor([at + new], dtype=torch.int32, device=dev)
        if new > 1:
            cu = torch.tensor([0, new], dtype=torch.int32, device=dev)
            o = ops.kv8_prefill_attention(q, cache, table, cu, lens, hq, hkv, d)
        else:
            o = ops.kv8_decode_attention(q, cache, table, lens, hq, hkv, d)
        x = qkv[:at + new].float().view(at + new, -1, d)
        k = ops.rope.apply_rope_ref(x[:, hq:hq + hkv], pos[:at + new], cos, sin, d)
        want = dense(q.view(new, hq, d), k, x[:, hq + hkv:])
        worst = max(worst, float((o.view(new, hq, d).float() - want).norm() / want.norm()))
        at += new
    print(f"{n} tokens: outputs within {worst:.3f} of attention over the unrounded cache")
    k, v = ops.kv8_read(cache, slots)
    rows = torch.cat([k.new_zeros(n, hq * d), k.reshape(n, -1), v.reshape(n, -1)], 1).contiguous()
    moved = ops.KV8Cache.zeros(pages + 1, hkv, d, dev)
    there = pos + PAGE                                                            # other pages, in order
    ops.kv8_store(rows, moved, there, hq, hkv, d)
    same = all(torch.equal(x, y) for x, y in zip(ops.kv8_read(moved, there), (k, v)))
    print(f"moved to another cache: {'the same values' if same else 'VALUES CHANGED'}")
    return worst, same


if __name__ == "__main__":
    main()
