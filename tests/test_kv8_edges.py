"""The 8-bit KV cache at the edges of its arguments: lengths, windows, exponents and queries that seldom occur."""
import pytest
import torch

from sglang_omni_b200 import ops
from sglang_omni_b200.ops._ext import ext
from test_kv8 import check_attention, make_cache, make_table, to

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


@pytest.mark.gpu
def test_three_position_rows_without_sections():
    """Without sections every pair follows the first position row, whatever the kind of sections would be."""
    hq, hkv, d, n = 2, 1, 64, 9
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(2)).bfloat16()
    cos, sin = (torch.randn(2, 40, d // 2, generator=torch.Generator().manual_seed(3))).unbind(0)
    pos = torch.stack([torch.arange(n), torch.arange(n) + 11, torch.arange(n) + 23]).int()
    one = ops.KV8Cache.zeros(2, hkv, d, "cuda")
    want = ops.kv8_store(qkv.cuda(), one, i32("cuda", *range(n)), hq, hkv, d, pos[0].contiguous().cuda(), cos.cuda(), sin.cuda())
    for interleaved in (True, False):
        cache = ops.KV8Cache.zeros(2, hkv, d, "cuda")
        q = ops.kv8_store(qkv.cuda(), cache, i32("cuda", *range(n)), hq, hkv, d, pos.cuda(), cos.cuda(), sin.cuda(), interleaved=interleaved)
        assert torch.equal(q, want) and torch.equal(cache.k.view(torch.uint8), one.k.view(torch.uint8))
    for section in ([8, 24], [8, 8, 8, 8], [16, 24, -8]):
        with pytest.raises(RuntimeError):
            ops.kv8_store(qkv.cuda(), one, i32("cuda", *range(n)), hq, hkv, d, pos.cuda(), cos.cuda(), sin.cuda(), mrope_section=section)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 30])
@pytest.mark.parametrize("new,kv,width", [(100, 90, 4), (300, 130, 400), (600, 500, 400), (3, 2, 1)])
def test_windows_beyond_every_context(window, new, kv, width):
    """A window longer than the block table can name sees all keys, in chunks longer than their context too
    (whose first queries see none)."""
    hq, hkv, d = 32, 4, 64
    pages = (kv + 63) // 64
    cache = make_cache(pages + 2, hkv, d, "cuda", seed=4)
    bt = make_table([kv], pages + 2, seed=4, width=width).cuda()
    q = queries(new, hq * d, 4, "cuda")
    out = ops.kv8_prefill_attention(q, cache, bt, i32("cuda", 0, new), i32("cuda", kv), hq, hkv, d, window=window, sinks=2)
    check_attention(out, q, cache, bt, [new], [kv], hq, hkv, d, d ** -0.5, 0, 0)
    last = ops.kv8_decode_attention(q[-1:], cache, bt, i32("cuda", kv), hq, hkv, d, window=window, sinks=2)
    check_attention(last, q[-1:], cache, bt, [1], [kv], hq, hkv, d, d ** -0.5, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("new,past,width", [(1, 0, 1), (40, 0, 1), (40, 3000, 60), (300, 0, 200)])
@pytest.mark.parametrize("window", [0, 1])
def test_infinite_queries_that_see_few_keys(new, past, width, window):
    """A query with an infinity whose scores are all negative infinity has no softmax: NaN, not zeros."""
    hq, hkv, d = 16, 2, 128
    n = new + past
    cache = make_cache((n + 63) // 64 + 2, hkv, d, "cuda", seed=5)
    bt = make_table([n], (n + 63) // 64 + 2, seed=5, width=max(width, (n + 63) // 64)).cuda()
    q = queries(new, hq * d, 5, "cuda")
    for h in range(0, hq, 3):
        q[:, h * d + 5 * h] = float("inf") if h % 2 else float("-inf")
    out = ops.kv8_prefill_attention(q, cache, bt, i32("cuda", 0, new), i32("cuda", n), hq, hkv, d, window=window)
    assert torch.isnan(out.view(new, hq, d)[:, ::3]).all()
    check_attention(out, q, cache, bt, [new], [n], hq, hkv, d, d ** -0.5, window, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("new,width", [(1, 3), (40, 3), (300, 400)])
def test_exponents_outside_the_format(new, width):
    """Exponents that no write leaves (a cache made by hand) count as the nearest of the format, in every operator."""
    hq, hkv, d, n = 16, 2, 128, 190 if new < 300 else 330
    pages = (n + 63) // 64 + 1
    for case in range(2):
        cache = make_cache(pages, hkv, d, "cpu", seed=6)
        bt = make_table([n], pages, seed=6, width=max(width, pages))
        at = lambda j: (bt[0, j // 64], slice(None), j % 64)  # noqa: E731
        if case == 0:
            cache.k_exp[at(0)], cache.v_exp[at(0)] = -127, -61
            cache.k_exp[at(70)], cache.v_exp[at(70)] = -90, -127
            cache.k.view(torch.uint8)[at(100)], cache.k_exp[at(100)] = 0, 127        # zero keys: the score stays 0
            cache.k.view(torch.uint8)[at(101)], cache.k_exp[at(101)] = 0, 61
        else:
            cache.v_exp[at(1)], cache.v_exp[at(2)], cache.v_exp[at(90)] = 61, 127, 100
        dev = to(cache, "cuda")
        q = queries(new, hq * d, 6, "cuda")
        out = ops.kv8_prefill_attention(q, dev, bt.cuda(), i32("cuda", 0, new), i32("cuda", n), hq, hkv, d)
        check_attention(out, q, cache, bt, [new], [n], hq, hkv, d, d ** -0.5, 0, 0)
        last = ops.kv8_decode_attention(q[:1], dev, bt.cuda(), i32("cuda", n), hq, hkv, d)
        check_attention(last, q[:1], cache, bt, [1], [n], hq, hkv, d, d ** -0.5, 0, 0)
        slots = torch.tensor([int(bt[0, j // 64]) * 64 + j % 64 for j in range(n)], dtype=torch.int32)
        for a, b in zip(ops.kv8_read(dev, slots.cuda()), ops.kv8_read(cache, slots)):
            assert torch.equal(a.cpu(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("name,new,past,width,d", [
    ("in place", 900, 700, 25, 128), ("in place", 700, 900, 25, 128), ("in place", 600, 700, 21, 64), ("in place", 130, 3000, 60, 128),
    ("expanded", 900, 700, 400, 128), ("expanded", 900, 700, 400, 64), ("decode", 8, 900, 20, 128)])
def test_chunk_among_other_launches(name, new, past, width, d):
    """The same bits whatever runs around it: stores before and behind it, and itself, launched back to back."""
    hq, hkv, n = 16, 4, new + past
    pages = (n + 63) // 64
    cache, other = make_cache(pages + 2, hkv, d, "cuda", seed=9), ops.KV8Cache.zeros(20, hkv, d, "cuda")
    bt = make_table([n], pages + 2, seed=9, width=width).cuda()
    assert ext().kv8_chunk_form(new, 1, width, hq, hkv, d, 0, 0) == name
    rows = torch.randn(900, (8 + 2 * hkv) * d, generator=torch.Generator().manual_seed(10)).bfloat16().cuda()
    slots = torch.arange(900, dtype=torch.int32, device="cuda")
    cu, kl = i32("cuda", 0, new), i32("cuda", n)
    for size in (0.02, 3.0):                       # flat and sharp softmaxes
        q = (size * torch.randn(new, hq * d, generator=torch.Generator().manual_seed(11))).bfloat16().cuda()
        first = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d)
        check_attention(first, q, cache, bt, [new], [n], hq, hkv, d, d ** -0.5, 0, 0)
        for _ in range(8):
            outs = []
            for _ in range(8):
                ops.kv8_store(rows, other, slots, 8, hkv, d)
                outs.append(ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d))
            assert all(torch.equal(o, first) for o in outs)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [60, 900])
@pytest.mark.parametrize("d", [64, 128])
def test_dependent_launches_behind_a_chunk(new, d):
    """A GEMM and the next layer's store and attention, launched while the chunk attention runs, give what they
    give one by one."""
    hq, hkv, n = 16, 2, new + 700
    caches = [make_cache((n + 63) // 64 + 2, hkv, d, "cuda", seed=s) for s in (7, 8)]
    bt = make_table([n], (n + 63) // 64 + 2, seed=7, width=(n + 63) // 64).cuda()
    q = queries(new, hq * d, 7, "cuda")
    g = torch.Generator().manual_seed(8)
    w = (torch.randn((hq + 2 * hkv) * d, hq * d, generator=g) * d ** -0.5 / 4).bfloat16().cuda()
    slots = torch.tensor([int(bt[0, j // 64]) * 64 + j % 64 for j in range(n - new, n)], dtype=torch.int32, device="cuda")
    cu, kl = i32("cuda", 0, new), i32("cuda", n)

    def layers(wait):
        own = [to(c, "cpu") for c in caches]
        own = [to(c, "cuda") for c in own] * 3
        x, outs = q, []
        for c in own:
            x = ops.kv8_prefill_attention(x, c, bt, cu, kl, hq, hkv, d)
            wait()
            y = ops.linear(x, w)
            wait()
            x = ops.kv8_store(y, c, slots, hq, hkv, d)
            wait()
            outs += [y, x]
        return outs

    want = layers(torch.cuda.synchronize)
    for _ in range(3):
        for a, b in zip(layers(lambda: None), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("name,batch,new,width", [("in place", 33, 21, 30), ("in place", 70, 30, 30), ("expanded", 40, 130, 60)])
def test_more_requests_than_lanes(name, batch, new, width):
    """Row tiles are found over more than 32 requests, with empty ones among them and chunks beyond their context."""
    hq, hkv, d, window, sinks = 64, 2, 64, 500, 3
    q_lens = [0 if b % 11 == 5 else 1 + (b * 7) % new for b in range(batch)]
    kv_lens = [max(0, n + (-3 if b % 13 == 2 else (b * 97) % 700)) for b, n in enumerate(q_lens)]
    if name == "expanded":
        q_lens, window = [n + new for n in q_lens], 0
    pages = sum((n + 63) // 64 for n in kv_lens) + 2
    cache = make_cache(pages, hkv, d, "cuda", seed=12)
    bt = make_table(kv_lens, pages, seed=12, width=width).cuda()
    assert ext().kv8_chunk_form(sum(q_lens), batch, width, hq, hkv, d, window, sinks) == name
    q = queries(sum(q_lens), hq * d, 12, "cuda")
    cu = i32("cuda", *[sum(q_lens[:i]) for i in range(batch + 1)])
    out = ops.kv8_prefill_attention(q, cache, bt, cu, i32("cuda", *kv_lens), hq, hkv, d, window=window, sinks=sinks)
    check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)
