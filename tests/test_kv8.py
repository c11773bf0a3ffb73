"""The 8-bit paged KV cache: quantised write, read, decode and chunk attention against 64-bit oracles."""
import math

import pytest
import torch

from sglang_omni_b200 import ops
from sglang_omni_b200.ops import kv8 as K
from sglang_omni_b200.ops.rope import apply_rope_ref, rope_tables

PAGE = 64


# ------------------------------------------------------------------ oracles and inputs
def two(n):
    """2^n for whole n from its bits, fp64."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def hold64(x):
    """Rows [..., D] (fp64, finite) -> the values the format holds for them, written from its definition:
    the exponent by trial, the code as the nearest of all e4m3 values, ties to the even code."""
    amax = x.abs().amax(-1)
    e = torch.full(amax.shape, K.EXP_MAX)
    for t in range(K.EXP_MAX, K.EXP_MIN - 1, -1):
        e = torch.where(amax * 2.0 ** -t <= 448.0, torch.full_like(e, t), e)
    grid = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()     # 0 .. 448, ascending
    y = (x * two(-e)[..., None]).clamp(-448, 448)
    hi = torch.searchsorted(grid, y.abs().contiguous()).clamp(max=0x7E)
    lo = (hi - 1).clamp(min=0)
    dl, dh = y.abs() - grid[lo], grid[hi] - y.abs()
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(grid[pick], y) * two(e)[..., None], e


def make_cache(pages, hkv, d, device="cpu", seed=0, v_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    c = ops.KV8Cache.zeros(pages, hkv, d, "cpu")
    rows = torch.randn(2, pages, hkv, PAGE, d, generator=g) * torch.exp(torch.randn(2, pages, hkv, PAGE, 1, generator=g))
    rows[1] *= v_scale
    for codes, exps, x in ((c.k, c.k_exp, rows[0]), (c.v, c.v_exp, rows[1])):
        a, e = K.kv8_quantize_ref(x)
        codes.view(torch.uint8).copy_(a.view(torch.uint8))
        exps.copy_(e)
    return to(c, device)


def to(c, device):
    f = lambda t: t.to(device)  # noqa: E731
    return ops.KV8Cache(f(c.k.view(torch.uint8)).view(torch.float8_e4m3fn), f(c.v.view(torch.uint8)).view(torch.float8_e4m3fn),
                        f(c.k_exp), f(c.v_exp))


def make_table(kv_lens, pages, seed=0, width=None):
    g = torch.Generator().manual_seed(seed)
    need = [(n + 63) // 64 for n in kv_lens]
    ids = (torch.randperm(pages - 1, generator=g) + 1).tolist()
    bt = torch.zeros(len(kv_lens), width or max(1, max(need)), dtype=torch.int32)
    for b, n in enumerate(need):
        bt[b, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    return bt


def check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, scale, window, sinks):
    """|out - o| <= 2^-8 sum_j p_j |v_j| + 2^-8 |o|, per element: a weight is held in 16 bits with a relative
    rounding of at most 2^-9, the output once more with 2^-9 of itself; the exponential and the 32-bit sums
    stay far below (scores under 2^6 with a relative error of 2^-20), so twice those bounds is enough."""
    c = to(cache, "cpu")
    q64 = q.cpu().double()[:, :hq * d].reshape(-1, hq, d)
    want = K.kv8_attention_ref(q64, c, bt.cpu(), q_lens, kv_lens, hq, hkv, d, scale, window, sinks)
    size = K.kv8_attention_ref(q64, ops.KV8Cache(c.k, (c.v.view(torch.uint8) & 0x7F).view(torch.float8_e4m3fn), c.k_exp, c.v_exp),
                               bt.cpu(), q_lens, kv_lens, hq, hkv, d, scale, window, sinks)
    got = out.cpu().double().reshape(-1, hq, d)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    err = (got - want).abs()[ok]
    lim = (2.0 ** -8 * size + 2.0 ** -8 * want.abs())[ok] + 1e-30
    assert bool((err <= lim).all()), f"worst {(err / lim).max().item():.3f} of the bound"


# ------------------------------------------------------------------ CPU
def test_quantize_ref_is_the_nearest_code():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(300, 64, generator=g) * torch.exp(6 * torch.randn(300, 1, generator=g))
    x[0] = 0
    x[1, :] = 448.0
    x[2, 0], x[2, 1:] = 449.0, 1.0
    x[3] = torch.linspace(-30, 30, 64)
    codes, e = K.kv8_quantize_ref(x)
    want, we = hold64(x.double())
    assert torch.equal(e.long(), we)
    assert torch.equal(K.kv8_dequantize_ref(codes, e).double(), want)


def test_quantize_ref_marks_rows_that_are_not_finite():
    x = torch.ones(4, 64)
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    codes, e = K.kv8_quantize_ref(x)
    assert e.tolist()[1:3] == [K.EXP_BAD] * 2 and int(codes.view(torch.uint8)[1:3].max()) == 0
    y = K.kv8_dequantize_ref(codes, e)
    assert torch.isnan(y[1:3]).all() and torch.equal(y[[0, 3]], x[[0, 3]])
    big = torch.full((1, 64), 3e38)
    assert K.kv8_dequantize_ref(*K.kv8_quantize_ref(big)).max() == 448.0 * 2.0 ** 60     # saturates


def test_cpu_path_matches_dense_attention():
    hq, hkv, d, kv_lens = 4, 2, 64, [70, 1, 0]
    c = make_cache(5, hkv, d)
    bt = make_table(kv_lens, 5)
    q = torch.randn(3, hq * d, generator=torch.Generator().manual_seed(2))
    o = ops.kv8_decode_attention(q, c, bt, torch.tensor(kv_lens, dtype=torch.int32), hq, hkv, d)
    slots = bt[0, torch.arange(70) // 64] * 64 + torch.arange(70) % 64
    k, v = ops.kv8_read(c, slots.int())
    kk, vv = (t.float().repeat_interleave(2, 1).permute(1, 0, 2)[None] for t in (k, v))
    want = torch.nn.functional.scaled_dot_product_attention(q[0].view(1, hq, 1, d), kk, vv)
    torch.testing.assert_close(o[0].view(hq, d), want[0, :, 0], atol=1e-5, rtol=1e-5)
    assert torch.equal(o[2], torch.zeros_like(o[2]))


def test_cpu_path_refuses():
    c = make_cache(3, 2, 64)
    bt, kl = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv8_decode_attention(torch.zeros(1, 3 * 64), c, bt, kl, 3, 2, 64)
    with pytest.raises(ValueError):
        ops.kv8_decode_attention(torch.zeros(1, 4 * 128), c, bt, kl, 4, 2, 128)
    with pytest.raises(ValueError):
        ops.kv8_decode_attention(torch.zeros(1, 4 * 64), c, bt, kl, 4, 2, 64, window=-1)


# ------------------------------------------------------------------ write and read
@pytest.mark.gpu
@pytest.mark.parametrize("d,hq,hkv,rope,norm", [
    (128, 32, 4, "mrope", True), (128, 5, 1, "pair", False), (128, 8, 8, "half", True), (128, 6, 2, "none", False),
    (64, 16, 8, "neox", True), (64, 3, 1, "odd", False), (128, 4, 2, "odd", True), (64, 4, 4, "sections", True)])
@pytest.mark.parametrize("tokens", [1, 3, 65])
def test_store(d, hq, hkv, rope, norm, tokens):
    g = torch.Generator().manual_seed(tokens)
    width = (hq + 2 * hkv) * d
    wide = (torch.randn(tokens, width + 64, generator=g) * torch.exp(torch.randn(tokens, 1, generator=g))).bfloat16()
    wide[0, :width // 2] *= 1000
    qkv = wide.cuda()[:, :width]                              # rows of a wider tensor
    rot = {"none": 0, "half": d // 2, "odd": 24}.get(rope, d)
    cos, sin = rope_tables(max(rot, 2), 1e4, 500)
    three = rope in ("mrope", "sections")
    section = [24, 20, 20] if rope == "mrope" else ([8, 12, 12] if rope == "sections" else None)
    pos = torch.randint(0, 500, (3, tokens) if three else (tokens,), generator=g, dtype=torch.int32)
    qn, kn = ((1 + 0.3 * torch.randn(2, d, generator=g)).bfloat16().cuda()) if norm else (None, None)
    pages = 4
    slots = (torch.randperm((pages - 1) * 64, generator=g)[:tokens] + 64).int()
    if tokens > 2:
        slots[1] = -1
    cache = to(ops.KV8Cache.zeros(pages, hkv, d, "cpu"), "cuda")
    before = wide.clone()
    q = ops.kv8_store(qkv, cache, slots.cuda(), hq, hkv, d, pos.cuda(), cos.cuda(), sin.cuda(), rot_dim=rot, q_norm=qn,
                      k_norm=kn, neox=rope != "pair", mrope_section=section, interleaved=rope == "mrope")
    assert torch.equal(qkv.cpu(), before[:, :width])          # the QKV rows are left alone
    x = before[:, :width].double().view(tokens, -1, d)

    def prep(y, w):
        if w is not None:
            y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + 1e-6) * w.cpu().double()
        return apply_rope_ref(y, pos, cos.double(), sin.double(), rot, rope != "pair", section, rope == "mrope") if rot else y

    want_q = prep(x[:, :hq], qn)
    # one bf16 rounding (2^-9 relative) of values that carry fp32 errors of about 2^-22 of the row's size
    err = (q.cpu().double().view(tokens, hq, d) - want_q).abs()
    assert bool((err <= 2.0 ** -8 * want_q.abs() + 2.0 ** -19 * want_q.abs().amax(-1, keepdim=True)).all())
    live = [t for t in range(tokens) if slots[t] >= 0]
    s = slots[live].long()
    c = to(cache, "cpu")
    touched = torch.zeros(pages, PAGE, dtype=torch.bool)
    touched[s // PAGE, s % PAGE] = True
    assert int(c.k.view(torch.uint8).transpose(1, 2)[~touched].max()) == 0 and int(c.v_exp.transpose(1, 2)[~touched].abs().max()) == 0
    v, e = hold64(x[live][:, hq + hkv:])
    assert torch.equal(c.v_exp[s // PAGE, :, s % PAGE].long(), e)
    got = K._rows_ref(c, s)
    assert torch.equal(got[1].double(), v)                    # V comes in as bf16: exact
    k = prep(x[:, hq:hq + hkv], kn)[live]
    if not norm and not rot:
        assert torch.equal(got[0].double(), hold64(k)[0])
    else:
        # a value within fp32 error of a rounding boundary may take the neighbouring code: off by at
        # most one step (half a step from rounding plus the error), seldom
        want = hold64(k)[0]
        step = torch.maximum(2.0 ** -3 * k.abs(), 2.0 ** -9 * two(hold64(k)[1])[..., None])
        assert bool(((got[0].double() - want).abs() <= 1.01 * step).all())
        assert float((got[0].double() != want).double().mean()) <= 1e-3
    # the read gives back exactly what is held; slots outside the cache give zeros
    ask = torch.cat([slots[live], torch.tensor([-1, pages * 64], dtype=torch.int32)]).cuda()
    rk, rv = ops.kv8_read(cache, ask)
    assert torch.equal(rk[:-2].cpu().float(), got[0]) and torch.equal(rv[:-2].cpu().float(), got[1])
    assert int(rk[-2:].abs().max()) == 0 and int(rv[-2:].abs().max()) == 0


@pytest.mark.gpu
def test_store_marks_rows_that_are_not_finite():
    d, hq, hkv = 64, 2, 2
    qkv = torch.randn(4, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    qkv[1, hq * d + 3] = float("nan")                # key head 0
    qkv[2, (hq + hkv + 1) * d + 5] = float("inf")    # value head 1
    qkv[3, (hq + hkv) * d:(hq + hkv + 1) * d] = 0
    cache = ops.KV8Cache.zeros(2, hkv, d, "cuda")
    ops.kv8_store(qkv, cache, torch.arange(4, dtype=torch.int32, device="cuda"), hq, hkv, d)
    assert cache.k_exp[0, :, :4].tolist()[0][1] == K.EXP_BAD and cache.v_exp[0, 1, 2] == K.EXP_BAD
    assert cache.v_exp[0, 0, 3] == K.EXP_MIN
    assert (cache.k_exp == K.EXP_BAD).sum() == 1 and (cache.v_exp == K.EXP_BAD).sum() == 1
    k, v = ops.kv8_read(cache, torch.arange(4, dtype=torch.int32, device="cuda"))
    assert torch.isnan(k[1, 0]).all() and torch.isnan(v[2, 1]).all() and torch.isnan(k).sum() == d == torch.isnan(v).sum()


# ------------------------------------------------------------------ attention
HEADS = [(32, 4, 128), (16, 2, 128), (8, 8, 128), (7, 1, 128), (33, 1, 128), (6, 2, 64), (32, 8, 64), (40, 2, 64)]
MASKS = [(0, 0), (1, 0), (70, 0), (64, 3), (100, 64), (130, 100), (1000, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("window,sinks", MASKS)
def test_decode(hq, hkv, d, window, sinks):
    kv_lens = [1, 64, 0, 65, 63, 333, 700]
    cache = make_cache(24, hkv, d, "cuda")
    bt = make_table(kv_lens, 24).cuda()
    q = torch.randn(len(kv_lens), hq * d + 16, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    out = ops.kv8_decode_attention(q, cache, bt, kl, hq, hkv, d, window=window, sinks=sinks)
    assert int(out[2].abs().max()) == 0
    check_attention(out, q, cache, bt, [1] * len(kv_lens), kv_lens, hq, hkv, d, d ** -0.5, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("window,sinks", MASKS)
def test_chunk(hq, hkv, d, window, sinks):
    q_lens = [1, 0, 17, 64, 5, 130, 1]
    kv_lens = [1, 40, 17, 200, 640, 131, 500]
    cache = make_cache(40, hkv, d, "cuda", seed=1)
    bt = make_table(kv_lens, 40, seed=1).cuda()
    T = sum(q_lens)
    q = torch.randn(T, hq * d, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    out = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, window=window, sinks=sinks)
    check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,past", [([1], [5000]), ([7], [4001]), ([300], [0]), ([257, 2], [1000, 3000]), ([513], [129])])
def test_chunk_long(d, q_lens, past):
    """Contexts long enough to be split over the keys, and chunks of several row tiles."""
    hq, hkv = 16, 2
    kv_lens = [a + b for a, b in zip(q_lens, past)]
    pages = sum((n + 63) // 64 for n in kv_lens) + 2
    cache = make_cache(pages, hkv, d, "cuda", seed=2)
    bt = make_table(kv_lens, pages, seed=2, width=200).cuda()
    q = (4 * torch.randn(sum(q_lens), hq * d, generator=torch.Generator().manual_seed(5))).bfloat16().cuda()
    cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    out = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d)
    check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, 0, 0)
    if max(q_lens) == 1:
        check_attention(ops.kv8_decode_attention(q, cache, bt, kl, hq, hkv, d), q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_are_not_finite_touch_only_who_sees_them(d):
    """Marked key and value rows before, inside and after the visible range, and garbage codes past the context."""
    hq, hkv, n, new, window = 4, 2, 200, 40, 50
    cache = make_cache(6, hkv, d, "cpu", seed=3)
    bt = make_table([n], 6, seed=3)
    for j, h, exps in ((10, 0, cache.k_exp), (3, 1, cache.v_exp), (185, 0, cache.v_exp), (190, 1, cache.k_exp)):
        exps[bt[0, j // 64], h, j % 64] = K.EXP_BAD
    for j in range(n, 256):                     # never written: NaN codes and any exponent
        cache.k.view(torch.uint8)[bt[0, j // 64], :, j % 64] = 0x7F
        cache.v.view(torch.uint8)[bt[0, j // 64], :, j % 64] = 0xFF
        cache.v_exp[bt[0, j // 64], :, j % 64] = 127
    q = torch.randn(new, hq * d, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    cu, kl = torch.tensor([0, new], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    dev = to(cache, "cuda")
    out = ops.kv8_prefill_attention(q, dev, bt.cuda(), cu, kl, hq, hkv, d, window=window, sinks=2)
    assert not torch.isnan(out[:24]).any() and torch.isnan(out[25:, :2 * d]).all() and torch.isnan(out[30:, 2 * d:]).all()
    check_attention(out, q, dev, bt, [new], [n], hq, hkv, d, d ** -0.5, window, 2)
    for m in (n, 186, 185, 150):
        last = ops.kv8_decode_attention(q[:1], dev, bt.cuda(), torch.tensor([m], dtype=torch.int32).cuda(), hq, hkv, d, window=window, sinks=2)
        check_attention(last, q[:1], dev, bt, [1], [m], hq, hkv, d, d ** -0.5, window, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("v_scale", [1e-12, 1.0, 1e9])
@pytest.mark.parametrize("q_scale", [0.0, 1e-6, 30.0])
def test_sizes_of_the_values(v_scale, q_scale):
    """Values far from 1, sharp and flat softmaxes, key rows of zeros."""
    hq, hkv, d, kv_lens = 8, 2, 128, [300, 77]
    cache = make_cache(9, hkv, d, "cuda", seed=4, v_scale=v_scale)
    cache.v.view(torch.uint8)[2] = 0
    cache.v_exp[2] = K.EXP_MIN
    bt = make_table(kv_lens, 9, seed=4).cuda()
    q = (q_scale * torch.randn(2, hq * d, generator=torch.Generator().manual_seed(7))).bfloat16().cuda()
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    check_attention(ops.kv8_decode_attention(q, cache, bt, kl, hq, hkv, d, scale=0.1), q, cache, bt, [1, 1], kv_lens, hq, hkv, d, 0.1, 0, 0)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    check_attention(ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, scale=0.1), q, cache, bt, [1, 1], kv_lens, hq, hkv, d, 0.1, 0, 0)


@pytest.mark.gpu
def test_cache_past_32_bit_offsets():
    hq, hkv, d, n, pages = 8, 4, 128, 130, 66000                # codes: 2.16e9 bytes for K, as many for V
    cache = ops.KV8Cache.zeros(pages, hkv, d, "cuda")
    bt = torch.tensor([[pages - 1, 5, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn(n, (hq + 2 * hkv) * d, generator=g).bfloat16()
    j = torch.arange(n)
    slots = (bt[0].cpu()[j // 64].long() * 64 + j % 64).int()
    q = ops.kv8_store(qkv.cuda(), cache, slots.cuda(), hq, hkv, d)
    assert torch.equal(q.cpu(), qkv[:, :hq * d])
    k, v = ops.kv8_read(cache, slots.cuda())
    small = ops.KV8Cache.zeros(4, hkv, d, "cpu")
    ops.kv8_store(qkv, small, (j + 64).int(), hq, hkv, d)
    ks, vs = ops.kv8_read(small, (j + 64).int())
    assert torch.equal(k.cpu(), ks) and torch.equal(v.cpu(), vs)
    kl = torch.tensor([n], dtype=torch.int32)
    sb = torch.tensor([[1, 2, 3]], dtype=torch.int32)
    check_attention(ops.kv8_decode_attention(q[-1:], cache, bt, kl.cuda(), hq, hkv, d), q[-1:], small, sb, [1], [n], hq, hkv, d, d ** -0.5, 0, 0)
    cu = torch.tensor([0, n], dtype=torch.int32)
    check_attention(ops.kv8_prefill_attention(q, cache, bt, cu.cuda(), kl.cuda(), hq, hkv, d), q, small, sb, [n], [n], hq, hkv, d, d ** -0.5, 0, 0)


@pytest.mark.gpu
def test_other_stream_strided_output_and_repeat():
    """Results do not depend on the stream, on a strided output or table, or on the run."""
    hq, hkv, d, kv_lens = 8, 2, 128, [900, 450, 3000]
    pages = 75
    cache = make_cache(pages, hkv, d, "cuda", seed=5)
    bt = make_table(kv_lens, pages, seed=5, width=90).cuda()
    q = torch.randn(3, hq * d, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    cu = torch.arange(4, dtype=torch.int32, device="cuda")
    first = ops.kv8_decode_attention(q, cache, bt[:, :50], kl, hq, hkv, d)
    chunk = ops.kv8_prefill_attention(q, cache, bt[:, :50], cu, kl, hq, hkv, d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    wide = torch.zeros(3, hq * d + 24, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            got = ops.kv8_decode_attention(q, cache, bt[:, :50], kl, hq, hkv, d, out=wide[:, :hq * d])
            again = ops.kv8_prefill_attention(q, cache, bt[:, :50], cu, kl, hq, hkv, d)
    side.synchronize()
    assert got.data_ptr() == wide.data_ptr() and torch.equal(wide[:, :hq * d], first) and int(wide[:, hq * d:].abs().max()) == 0
    assert torch.equal(again, chunk)


@pytest.mark.gpu
def test_graph_capture():
    """The operators take part in a CUDA graph; replays follow the lengths on the device."""
    hq, hkv, d = 8, 2, 128
    cache = make_cache(30, hkv, d, "cuda", seed=6)
    bt = make_table([640, 640], 30, seed=6).cuda()
    kl = torch.tensor([640, 1], dtype=torch.int32, device="cuda")
    q = torch.randn(2, hq * d, generator=torch.Generator().manual_seed(10)).bfloat16().cuda()
    ops.kv8_decode_attention(q, cache, bt, kl, hq, hkv, d)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.kv8_decode_attention(q, cache, bt, kl, hq, hkv, d)
    for lens in ([640, 1], [0, 300], [65, 64]):
        kl.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        check_attention(out, q, cache, bt, [1, 1], lens, hq, hkv, d, d ** -0.5, 0, 0)


@pytest.mark.gpu
def test_block_table_shorter_than_the_context():
    """A request sees at most the keys that its block-table row can name, entries outside the cache read page 0."""
    hq, hkv, d = 4, 2, 64
    cache = make_cache(4, hkv, d, "cuda", seed=7)
    bt = torch.tensor([[2, 99]], dtype=torch.int32, device="cuda")
    q = torch.randn(1, hq * d, generator=torch.Generator().manual_seed(11)).bfloat16().cuda()
    out = ops.kv8_decode_attention(q, cache, bt, torch.tensor([1000], dtype=torch.int32, device="cuda"), hq, hkv, d)
    check_attention(out, q, cache, bt, [1], [128], hq, hkv, d, d ** -0.5, 0, 0)


@pytest.mark.gpu
def test_refusals():
    hq, hkv, d = 4, 2, 64
    cache = ops.KV8Cache.zeros(4, hkv, d, "cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    bt = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, hq * d, dtype=torch.bfloat16, device="cuda")
    ok = dict(num_heads=hq, num_kv_heads=hkv, head_dim=d)
    bad = [
        lambda: ops.kv8_decode_attention(q.float(), cache, bt, i32(1, 1), **ok),
        lambda: ops.kv8_decode_attention(q[:, :-8], cache, bt, i32(1, 1), **ok),
        lambda: ops.kv8_decode_attention(q[:, 1:], cache, bt, i32(1, 1), 3, 1, d),
        lambda: ops.kv8_decode_attention(q, cache, bt, i32(1, 1), 3, 2, d),
        lambda: ops.kv8_decode_attention(q, cache, bt, i32(1, 1), hq, hkv, 128),
        lambda: ops.kv8_decode_attention(q, cache, bt.long(), i32(1, 1), **ok),
        lambda: ops.kv8_decode_attention(q, cache, bt, i32(1, 1).long(), **ok),
        lambda: ops.kv8_decode_attention(q, cache, bt, i32(1, 1, 1), **ok),
        lambda: ops.kv8_decode_attention(q, cache, bt.cpu(), i32(1, 1), **ok),
        lambda: ops.kv8_decode_attention(q, cache, bt, i32(1, 1), window=-1, **ok),
        lambda: ops.kv8_decode_attention(q, cache, bt, i32(1, 1), sinks=-1, **ok),
        lambda: ops.kv8_decode_attention(q, cache, bt[:1], i32(1, 1), **ok),
        lambda: ops.kv8_decode_attention(q, cache, bt, i32(1, 1), out=q[:1], **ok),
        lambda: ops.kv8_prefill_attention(q, cache, bt, i32(0, 1), i32(1, 1), **ok),
        lambda: ops.kv8_prefill_attention(q, cache, bt, i32(0, 1, 2).cpu(), i32(1, 1), **ok),
        lambda: ops.kv8_decode_attention(q, ops.KV8Cache(cache.k.float(), cache.v, cache.k_exp, cache.v_exp), bt, i32(1, 1), **ok),
        lambda: ops.kv8_decode_attention(q, ops.KV8Cache(cache.k, cache.v, cache.k_exp[:2], cache.v_exp), bt, i32(1, 1), **ok),
        lambda: ops.kv8_read(cache, i32(1).long()),
        lambda: ops.kv8_read(cache, i32(1, 2)[None]),
        lambda: ops.kv8_store(torch.zeros(2, 8 * d, device="cuda", dtype=torch.bfloat16), cache, i32(1), **ok),
        lambda: ops.kv8_store(torch.zeros(2, 7 * d, device="cuda", dtype=torch.bfloat16), cache, i32(1, 2), **ok),
        lambda: ops.kv8_store(torch.zeros(2, 8 * d, device="cuda", dtype=torch.bfloat16), cache, i32(1, 2), positions=i32(1, 2, 3),
                              cos_tab=torch.zeros(9, d // 2, device="cuda"), sin_tab=torch.zeros(9, d // 2, device="cuda"), **ok),
        lambda: ops.kv8_store(torch.zeros(2, 8 * d, device="cuda", dtype=torch.bfloat16), cache, i32(1, 2), positions=i32(1, 2),
                              cos_tab=torch.zeros(9, d, device="cuda"), sin_tab=torch.zeros(9, d // 2, device="cuda"), **ok),
        lambda: ops.KV8Cache.zeros(2, 1, 96, "cuda") and ops.kv8_read(ops.KV8Cache.zeros(2, 1, 96, "cuda"), i32(1)),
    ]
    for n, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"case {n} was accepted")
    # nothing to do is not an error
    none = torch.zeros(0, hq * d, dtype=torch.bfloat16, device="cuda")
    assert ops.kv8_decode_attention(none, cache, bt[:0], i32(), **ok).shape == (0, hq * d)
    assert ops.kv8_prefill_attention(none, cache, bt, i32(0, 0, 0), i32(0, 5), **ok).shape == (0, hq * d)
    assert ops.kv8_read(cache, i32())[0].shape == (0, hkv, d)
    assert ops.kv8_store(torch.zeros(0, 8 * d, device="cuda", dtype=torch.bfloat16), cache, i32(), **ok).shape == (0, hq * d)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,width,top", [
    (20, 8, 300), (40, 8, 200), (80, 8, 150), (150, 8, 120),      # clusters of 4, 2, 1 CTAs a pair; shares of all tiles
    (60, 70, 300), (60, 70, 1500), (3, 300, 2500)])               # wide tables: short pairs whole; split; few and long
@pytest.mark.parametrize("d", [64, 128])
def test_decode_ways_of_sharing(batch, width, top, d):
    """Every way in which the tiles are dealt out, with empty, short and unequal contexts."""
    hq, hkv = 8, 4
    kv_lens = [0 if b % 9 == 4 else 1 + (b * 37) % top for b in range(batch)]
    pages = sum((n + 63) // 64 for n in kv_lens) + 2
    cache = make_cache(pages, hkv, d, "cuda", seed=8)
    bt = make_table(kv_lens, pages, seed=8, width=max(width, (top + 63) // 64)).cuda()
    q = torch.randn(batch, hq * d, generator=torch.Generator().manual_seed(12)).bfloat16().cuda()
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    for window, sinks in ((0, 0), (90, 5)):
        out = ops.kv8_decode_attention(q, cache, bt, kl, hq, hkv, d, window=window, sinks=sinks)
        check_attention(out, q, cache, bt, [1] * batch, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (14, 2, 128), (33, 1, 128), (2, 2, 64), (40, 8, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 64), (150, 100), (70, 3)])
def test_chunk_expanded(hq, hkv, d, window, sinks):
    """Chunks of several row tiles per request (the blocks are expanded by a launch of their own), with windows
    that begin inside, at and between blocks, and a request without new tokens."""
    q_lens = [300, 0, 257, 290]
    kv_lens = [300, 77, 700, 291]
    if hq // hkv < 4:      # more tokens to a row tile
        q_lens, kv_lens = [600, 0, 530, 520], [600, 77, 1100, 521]
    pages = sum((n + 63) // 64 for n in kv_lens) + 2
    cache = make_cache(pages, hkv, d, "cuda", seed=9)
    bt = make_table(kv_lens, pages, seed=9).cuda()
    q = torch.randn(sum(q_lens), hq * d, generator=torch.Generator().manual_seed(13)).bfloat16().cuda()
    cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    out = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, window=window, sinks=sinks)
    check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40, 300])
def test_queries_that_are_not_finite(new):
    """A query with an infinity or a NaN gives NaN, and nothing to its neighbours (decode, chunk and expanded chunk)."""
    hq, hkv, d, n = 8, 2, 128, 500
    cache = make_cache(10, hkv, d, "cuda", seed=10)
    bt = make_table([n], 10, seed=10).cuda()
    q = torch.randn(new, hq * d, generator=torch.Generator().manual_seed(14)).bfloat16()
    clean = q.clone()
    for t in {0, new // 2}:
        q[t, 3] = float("inf")                    # head 0
        q[t, 5 * d + 7] = float("nan")            # head 5
    cu, kl = torch.tensor([0, new], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    got = ops.kv8_prefill_attention(q.cuda(), cache, bt, cu, kl, hq, hkv, d).cpu().view(new, hq, d)
    want = ops.kv8_prefill_attention(clean.cuda(), cache, bt, cu, kl, hq, hkv, d).cpu().view(new, hq, d)
    hit = torch.zeros(new, hq, dtype=torch.bool)
    for t in {0, new // 2}:
        hit[t, 0] = hit[t, 5] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d", [(128, 8, 64), (128, 8, 128), (34, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (64, 64), (150, 100), (70, 3)])
def test_chunk_many_row_tiles(hq, hkv, d, window, sinks):
    """Enough row tiles and blocks that the blocks are expanded by a launch of their own (a wide block table
    counts as a long context), and few requests of few tokens, whose blocks the attention kernel expands."""
    for q_lens, kv_lens, width in (([300, 0, 257, 290], [300, 77, 700, 291], 400), ([40, 0, 33, 2], [900, 77, 1300, 300], 60)):
        pages = sum((n + 63) // 64 for n in kv_lens) + 2
        cache = make_cache(pages, hkv, d, "cuda", seed=11)
        bt = make_table(kv_lens, pages, seed=11, width=width).cuda()
        q = torch.randn(sum(q_lens), hq * d, generator=torch.Generator().manual_seed(15)).bfloat16().cuda()
        cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")
        kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        out = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, window=window, sinks=sinks)
        check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,new,top", [(16, 4, 3000), (3, 30, 5000), (5, 17, 2500)])
@pytest.mark.parametrize("d", [64, 128])
def test_chunk_ring_of_codes(batch, new, top, d):
    """Chunks whose blocks pass several times round both rings, split over the keys by unequal shares: more row
    tiles than requests of equal length would make, and requests without keys before the chunk."""
    hq, hkv = 16, 2
    q_lens = [0 if b % 7 == 3 else 1 + (b * 5) % new for b in range(batch)]
    q_lens[0] = 2 * new + 1
    kv_lens = [n + (0 if b % 4 == 1 else (b * 911 + 500) % top) for b, n in enumerate(q_lens)]
    pages = sum((n + 63) // 64 for n in kv_lens) + 2
    cache = make_cache(pages, hkv, d, "cuda", seed=12)
    bt = make_table(kv_lens, pages, seed=12).cuda()
    q = torch.randn(sum(q_lens), hq * d, generator=torch.Generator().manual_seed(16)).bfloat16().cuda()
    cu = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device="cuda")
    kl = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
    for window, sinks in ((0, 0), (700, 5)):
        out = ops.kv8_prefill_attention(q, cache, bt, cu, kl, hq, hkv, d, window=window, sinks=sinks)
        check_attention(out, q, cache, bt, q_lens, kv_lens, hq, hkv, d, d ** -0.5, window, sinks)
