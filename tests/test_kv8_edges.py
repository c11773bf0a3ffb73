"""The 8-bit KV cache at the edges of its arguments: lengths, windows, exponents and queries that seldom occur."""
import pytest
import torch

from sglang_omni_b200 import ops
from test_kv8 import check_attention, make_cache, make_table

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def i32(device, *v):
    return torch.tensor(v, dtype=torch.int32, device=device)


def queries(rows, cols, seed, device):
    q = torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).bfloat16()
    return q.double() if device == "cpu" else q.cuda()      # the CPU form works in the type it is given


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width", [0, 2])
def test_lengths_beyond_the_block_table(device, width):
    """A request sees at most the keys that its block-table row can name, none where the row names none."""
    hq, hkv, d = 4, 2, 64
    cache = make_cache(4, hkv, d, device, seed=1)
    bt = i32(device, 2, 1)[None, :width].contiguous()
    q = queries(3, hq * d, 1, device)
    n = 64 * width
    out = ops.kv8_decode_attention(q[:1], cache, bt, i32(device, 1000), hq, hkv, d)
    chunk = ops.kv8_prefill_attention(q, cache, bt, i32(device, 0, 3), i32(device, 1000), hq, hkv, d)
    if width == 0:
        assert int(out.abs().max()) == 0 and int(chunk.abs().max()) == 0
        return
    check_attention(out, q[:1], cache, bt, [1], [n], hq, hkv, d, d ** -0.5, 0, 0)
    check_attention(chunk, q, cache, bt, [3], [n], hq, hkv, d, d ** -0.5, 0, 0)
