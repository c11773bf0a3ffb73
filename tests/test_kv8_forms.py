"""The chunk attention's form that expands its key blocks in a launch of their own: each test asserts that its
sizes take that form (tests/test_kv8.py covers the others)."""
import pytest
import torch

from sglang_omni_b200 import ops
from sglang_omni_b200.ops import kv8 as K
from sglang_omni_b200.ops._ext import ext
from test_kv8 import check_attention, make_cache, make_table, to

pytestmark = pytest.mark.gpu


def form(q_lens, bt, hq, hkv, d, window=0, sinks=0):
    return ext().kv8_chunk_form(sum(q_lens), len(q_lens), bt.shape[1], hq, hkv, d, window, sinks)


def lengths(q_lens, kv_lens):
    cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")
    return cu, torch.tensor(kv_lens, dtype=torch.int32, device="cuda")


def queries(q_lens, hq, d, seed):
    return torch.randn(sum(q_lens), hq * d, generator=torch.Generator().manual_seed(seed)).bfloat16()


@pytest.mark.parametrize("hq,hkv,d", [(40, 8, 128), (56, 8, 128), (34, 2, 128), (33, 1, 128), (40, 8, 64), (33, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 64), (150, 100), (1000, 3)])
def test_groups_that_do_not_divide_the_rows(hq, hkv, d, window, sinks):
    """Groups of 5, 7, 17 and 33 heads leave rows of a tile without a query; odd and even numbers of row tiles,
    requests without new tokens and from an empty cache."""
    q_lens, kv_lens = [700, 0, 257, 650], [700, 77, 1300, 651]
    pages = sum((n + 63) // 64 for n in kv_lens) + 2
    cache = make_cache(pages, hkv, d, "cuda", seed=20)
    bt = make_table(kv_lens, pages, seed=20, width=150).cuda()
    assert form(q_lens, bt, hq, hkv, d, window, sinks) == "expanded"
    q = queries(q_lens, hq, d, 20).cuda()
    cu, kl = lengths(q_lens, kv_lens)
    out = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, window=window, sinks=sinks)
    check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (120, 2)])
def test_rows_that_are_not_finite(d, window, sinks):
    """Marked key and value rows, and garbage codes and exponents past the context, touch only who sees them."""
    hq, hkv, n, new = 128, 8, 777, 500
    cache = make_cache(15, hkv, d, "cpu", seed=21)
    bt = make_table([n], 15, seed=21, width=100)
    for j, h, exps in ((600, 0, cache.k_exp), (650, 1, cache.v_exp), (700, 0, cache.v_exp), (1, 2, cache.k_exp)):
        exps[bt[0, j // 64], h, j % 64] = K.EXP_BAD
    for j in range(n, 832):
        cache.k.view(torch.uint8)[bt[0, j // 64], :, j % 64] = 0x7F
        cache.v.view(torch.uint8)[bt[0, j // 64], :, j % 64] = 0xFF
        cache.v_exp[bt[0, j // 64], :, j % 64] = 127
    assert form([new], bt, hq, hkv, d, window, sinks) == "expanded"
    q = queries([new], hq, d, 21).cuda()
    cu, kl = lengths([new], [n])
    out = ops.kv8_prefill_attention(q, to(cache, "cuda"), bt.cuda(), cu, kl, hq, hkv, d, window=window, sinks=sinks)
    assert not torch.isnan(out[:, 48 * d:]).any() and torch.isnan(out).any()
    check_attention(out, q, cache, bt, [new], [n], hq, hkv, d, d ** -0.5, window, sinks)


@pytest.mark.parametrize("d", [64, 128])
def test_queries_that_are_not_finite(d):
    hq, hkv, n, new = 32, 4, 500, 300
    cache = make_cache(10, hkv, d, "cuda", seed=22)
    bt = make_table([n], 10, seed=22, width=200).cuda()
    assert form([new], bt, hq, hkv, d) == "expanded"
    q = queries([new], hq, d, 22)
    clean = q.clone()
    hit = torch.zeros(new, hq, dtype=torch.bool)
    for t in (0, 16, 31, 150, new - 1):           # rows of a CTA's first and of its second query tile
        q[t, 3] = float("inf")
        q[t, 5 * d + 7] = float("nan")
        hit[t, 0] = hit[t, 5] = True
    cu, kl = lengths([new], [n])
    got = ops.kv8_prefill_attention(q.cuda(), cache, bt, cu, kl, hq, hkv, d).cpu().view(new, hq, d)
    want = ops.kv8_prefill_attention(clean.cuda(), cache, bt, cu, kl, hq, hkv, d).cpu().view(new, hq, d)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


def test_cache_past_32_bit_offsets():
    hq, hkv, d, n, pages = 8, 4, 128, 300, 66000               # codes: 2.16e9 bytes for K, as many for V
    cache = ops.KV8Cache.zeros(pages, hkv, d, "cuda")
    ids = [pages - 1, 5, pages - 2, 65999 // 2, pages - 3]
    bt = torch.zeros(1, 400, dtype=torch.int32)
    bt[0, :5] = torch.tensor(ids, dtype=torch.int32)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(23)).bfloat16()
    j = torch.arange(n)
    q = ops.kv8_store(qkv.cuda(), cache, (bt[0][j // 64].long() * 64 + j % 64).int().cuda(), hq, hkv, d)
    small = ops.KV8Cache.zeros(6, hkv, d, "cpu")
    ops.kv8_store(qkv, small, (j + 64).int(), hq, hkv, d)
    assert form([n], bt, hq, hkv, d) == "expanded"
    cu, kl = lengths([n], [n])
    out = ops.kv8_prefill_attention(q, cache, bt.cuda(), cu, kl, hq, hkv, d)
    check_attention(out, q, small, torch.tensor([[1, 2, 3, 4, 5]], dtype=torch.int32), [n], [n], hq, hkv, d, d ** -0.5, 0, 0)


def test_repeats_itself_on_other_streams_and_in_a_graph():
    """The same bits on every run, on a side stream, into a strided output and from a graph with changed lengths."""
    hq, hkv, d, q_lens, kv_lens = 32, 4, 128, [400, 250], [900, 251]
    cache = make_cache(24, hkv, d, "cuda", seed=24)
    bt = make_table(kv_lens, 24, seed=24, width=60).cuda()
    assert form(q_lens, bt, hq, hkv, d) == "expanded"
    q = queries(q_lens, hq, d, 24).cuda()
    cu, kl = lengths(q_lens, kv_lens)
    first = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    wide = torch.zeros(650, hq * d + 8, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, out=wide[:, :hq * d])
    side.synchronize()
    assert torch.equal(wide[:, :hq * d], first) and int(wide[:, hq * d:].abs().max()) == 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d)
    for a, lens in (([400, 250], kv_lens), ([650, 0], [660, 0]), ([3, 647], [70, 700])):
        c, n = lengths(a, lens)
        cu.copy_(c)
        kl.copy_(n)
        g.replay()
        torch.cuda.synchronize()
        check_attention(out, q, cache, bt, a, lens, hq, hkv, d, d ** -0.5, 0, 0)


def held_beside(f):
    """f's result and the bytes that it held at most beside what was there."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = f()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


def test_windows_need_scratch_for_what_they_see():
    """Wide block tables do not count where a window bounds the blocks (2000 pages of each request would be 1 GB)."""
    hq, hkv, d, window, sinks = 32, 8, 64, 1024, 70
    q_lens, kv_lens = [700, 1, 690, 640], [700, 5000, 3000, 1700]
    pages = sum((n + 63) // 64 for n in kv_lens) + 2
    cache = make_cache(pages, hkv, d, "cuda", seed=25)
    bt = make_table(kv_lens, pages, seed=25, width=2000).cuda()
    assert form(q_lens, bt, hq, hkv, d, window, sinks) == "expanded"
    q = queries(q_lens, hq, d, 25).cuda()
    cu, kl = lengths(q_lens, kv_lens)
    out, held = held_beside(lambda: ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, window=window, sinks=sinks))
    assert held < 2 * out.numel() + 24e6
    check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)


def test_without_room_for_the_scratch():
    """Where the expanded blocks find no room, the attention kernel expands them itself."""
    hq, hkv, d, q_lens, kv_lens = 16, 2, 128, [300, 200], [900, 200]
    cache = make_cache(25, hkv, d, "cuda", seed=26)
    bt = make_table(kv_lens, 25, seed=26, width=8000).cuda()              # 1 GB of blocks at most
    assert form(q_lens, bt, hq, hkv, d) == "expanded"
    q = queries(q_lens, hq, d, 26).cuda()
    cu, kl = lengths(q_lens, kv_lens)
    run = lambda: ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d)  # noqa: E731
    first, held = held_beside(run)
    assert held > 1e9
    del first
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (256 << 20)) / total)
    try:
        out, held = held_beside(run)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert held < 256 << 20
    check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, 0, 0)
