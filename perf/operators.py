"""The 8-bit paged KV cache and the attention that reads it: what is measured, and the plain forms.

Four operators of one path, a decoder layer's attention over a cache in 8 bits:

* ``write``   QK RMSNorm + RoPE of a step's fused QKV rows, K and V quantised into the paged cache,
              and the written rows read back (what a stage does that hands its keys on to another);
* ``read``    rows of the cache by slot, as bf16 (a cached prefix that leaves the engine);
* ``decode``  attention of one token per request over the cache;
* ``chunk``   causal attention of a chunk of new tokens per request over the cache.

The cache of a layer: e4m3 codes ``[pages, Hkv, 64, D]`` and one power-of-two exponent (int8) for each
(token, KV head) row ``[pages, Hkv, 64]``; a row x is held as codes rne_e4m3(x * 2^-e) with the smallest e
in [-60, 60] that keeps max|x| * 2^-e <= 448, and stands for code * 2^e.  A row with an infinity or a NaN has the
exponent -128 and stands for NaN.  Attention sees keys j <= i of its request; with a window W > 0 only
the last W of them and the request's first ``sinks`` tokens.  A query that sees no key gives zeros.
"""
import math

import torch

own = False

PAGE = 64
FLAG = -128            # exponent of a row that holds an infinity or a NaN
HEADS = [(32, 4, 128), (16, 2, 128), (32, 8, 128), (16, 8, 128), (16, 8, 64), (32, 8, 64)]
EPS = 1e-6


def listed():
    return [
        # a step of 64 streams with the next token each, adjacent-pair RoPE and no norm
        dict(name="write_64", op="write", tokens=64, hq=32, hkv=8, d=128, norm=False, rope="pair"),
        # a full prefill batch
        dict(name="write_8191", op="write", tokens=8191, hq=32, hkv=4, d=128, norm=True, rope="mrope"),
        # a short prompt's rows leave the cache
        dict(name="read_517", op="read", tokens=517, hq=16, hkv=8, d=64),
        # a long shared prefix leaves the cache
        dict(name="read_130000", op="read", tokens=130000, hq=32, hkv=4, d=128),
        # one stream with a short context: latency
        dict(name="decode_1", op="decode", batch=1, ctx=517, spread=0.0, empty=0, hq=32, hkv=4, d=128, window=0, sinks=0),
        # the serving benchmark's step: 64 slots of about 1152 tokens, three of them padding
        dict(name="decode_64", op="decode", batch=64, ctx=1280, spread=0.2, empty=3, hq=32, hkv=4, d=128, window=0, sinks=0),
        # few streams with very long and unequal contexts
        dict(name="decode_long", op="decode", batch=5, ctx=130001, spread=0.6, empty=0, hq=32, hkv=8, d=128, window=0, sinks=0),
        # streams that have run past a sliding window, the first tokens kept
        dict(name="decode_window", op="decode", batch=48, ctx=20000, spread=0.5, empty=0, hq=32, hkv=8, d=64, window=4096, sinks=4),
        # a few drafted tokens of one stream to check against its context
        dict(name="chunk_8", op="chunk", batch=1, new=8, spread=0.0, ctx=3000, hq=32, hkv=4, d=128, window=0, sinks=0),
        # prompts of a batch, from an empty cache and on cached prefixes, of unequal lengths
        dict(name="chunk_ragged", op="chunk", batch=8, new=1024, spread=0.9, ctx=2500, hq=32, hkv=4, d=128, window=0, sinks=0),
        # chunks of streams that have run past a sliding window, the first tokens kept
        dict(name="chunk_window", op="chunk", batch=4, new=700, spread=0.4, ctx=9000, hq=32, hkv=8, d=64, window=1024, sinks=4),
        # one chunk of a long prompt
        dict(name="chunk_long", op="chunk", batch=1, new=2048, spread=0.0, ctx=32768, hq=32, hkv=4, d=128, window=0, sinks=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["write", "read", "decode", "decode", "chunk", "chunk"])
        hq, hkv, d = rng.choice(HEADS)
        c = dict(op=op, hq=hq, hkv=hkv, d=d)
        if op == "write":
            c |= dict(tokens=_log(rng, 1, 8192), norm=rng.random() < 0.5, rope=rng.choice(["neox", "half", "pair", "mrope", "none"]))
            if d != 128 and c["rope"] == "mrope":
                c["rope"] = "neox"
        elif op == "read":
            c |= dict(tokens=_log(rng, 1, 130000))
        else:
            window = _log(rng, 100, 8192) if rng.random() < 0.4 else 0
            c |= dict(window=window, sinks=rng.choice([0, 1, 4, 64, 100]) if window else 0)
            if op == "decode":
                c |= dict(batch=_log(rng, 1, 128), ctx=_log(rng, 1, 130001), spread=rng.uniform(0, 0.9), empty=0)
                if c["batch"] > 4 and rng.random() < 0.3:
                    c["empty"] = rng.randint(1, 3)
                if c["batch"] * c["ctx"] * hkv * d > 5 * 130001 * 8 * 128:
                    continue
            else:
                c |= dict(batch=_log(rng, 1, 12), new=_log(rng, 1, 2048), spread=rng.uniform(0, 0.9), ctx=_log(rng, 1, 32768))
                if c["batch"] * c["new"] * (c["ctx"] + c["new"]) * hq > 2048 * 34816 * 32:
                    continue
        return c


# ---------------------------------------------------------------- sizes
def _ramp(n, top, spread):
    """n lengths between top * (1 - spread) and top, in a mixed order."""
    return [max(1, int(round(top * (1.0 - spread * ((5 * i) % n) / n)))) for i in range(n)]


def _lens(case):
    """(new tokens, context length with them) of every request."""
    n = case["batch"]
    if case["op"] == "decode":
        kv = _ramp(n, case["ctx"], case["spread"])
        live = n - case["empty"]
        return [1] * n, [x if i < live else 0 for i, x in enumerate(kv)]
    new = _ramp(n, case["new"], case["spread"])
    # every fourth request of a batch starts from an empty cache
    return new, [a + (0 if n > 1 and i % 4 == 3 else max(1, int(case["ctx"] * (1.0 - case["spread"] * i / n)))) for i, a in enumerate(new)]


def _pairs(new, kv, window, sinks):
    """(query, visible key) pairs of one request, and the keys that some query sees."""
    if kv <= 0:
        return 0, 0
    if window <= 0:
        return sum(range(kv - new + 1, kv + 1)), kv
    first = max(0, kv - new + 1 - window)    # the first key of the first query's window
    return (sum(min(p, window) + min(sinks, max(0, p - window)) for p in range(kv - new + 1, kv + 1)),
            kv - first + min(sinks, first))


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "write":
        t = case["tokens"]
        # QKV rows in, rotated q out, codes and exponents out, the rows read back out
        return {"bytes": t * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * hkv * (d + 1) + 2 * hkv * d * 2),
                "flops": t * (hq + 2 * hkv) * d * 8}
    if case["op"] == "read":
        return {"bytes": case["tokens"] * 2 * hkv * (d + 1 + 2 * d), "flops": case["tokens"] * 2 * hkv * d}
    pairs = keys = 0
    new, kv = _lens(case)
    for a, b in zip(new, kv):
        p, k = _pairs(a, b, case["window"], case["sinks"])
        pairs, keys = pairs + p, keys + k
    return {"bytes": keys * 2 * hkv * (d + 1) + 2 * sum(new) * hq * d * 2, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 17)


def _hold(x):
    """Rows x [..., D] in the cache's form: (codes e4m3, exponents int8)."""
    x = x.float()
    amax = x.abs().amax(-1)
    mant, ex = torch.frexp(amax)                  # amax = mant * 2^ex, mant in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(mant <= 0.875, ex - 9, ex - 8).clamp(-60, 60)
    e = torch.where(amax == 0, torch.full_like(e, -60), e)
    bad = ~torch.isfinite(amax)
    y = (x * _pow2(-e)[..., None]).clamp(-448.0, 448.0)
    y = torch.where(bad[..., None], torch.zeros_like(y), y)
    return y.to(torch.float8_e4m3fn), torch.where(bad, torch.full_like(e, FLAG), e).to(torch.int8)


def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _values(codes, e):
    """What codes and exponents stand for, in 32 bits."""
    e = e.to(torch.int32)
    s = torch.where(e == FLAG, torch.full_like(e, 0x7FC00000).view(torch.float32), _pow2(e.clamp(-60, 60)))
    return codes.float() * s[..., None]


def _rows(g, shape, wide):
    """Key-like (channels of unequal size) or value-like rows, each token with a size of its own."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(shape[:-1], generator=g, device="cuda"))[..., None] * 0.3
    if wide:
        x *= 1.0 + 4.0 * (torch.rand(shape[-1], generator=g, device="cuda") > 0.9).float()
    return x.to(torch.bfloat16)


def _cache(g, pages, hkv, d):
    """A filled cache of one layer, made in pieces of 512 pages."""
    out = {"k": torch.empty(pages, hkv, PAGE, d, device="cuda", dtype=torch.float8_e4m3fn),
           "v": torch.empty(pages, hkv, PAGE, d, device="cuda", dtype=torch.float8_e4m3fn),
           "k_exp": torch.empty(pages, hkv, PAGE, device="cuda", dtype=torch.int8),
           "v_exp": torch.empty(pages, hkv, PAGE, device="cuda", dtype=torch.int8)}
    for a in range(0, pages, 512):
        n = min(512, pages - a)
        for name in ("k", "v"):
            codes, e = _hold(_rows(g, (n, hkv, PAGE, d), name == "k"))
            out[name][a:a + n].copy_(codes)
            out[name + "_exp"][a:a + n].copy_(e)
    return out


def prepare(case, seed):
    g = _gen(seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] in ("write", "read"):
        t = case["tokens"]
        pages = -(-t // PAGE) + 2
        slots = torch.randperm((pages - 1) * PAGE, generator=g, device="cuda")[:t] + PAGE if case["op"] == "write" else (
            (torch.randperm(pages - 1, generator=g, device="cuda")[:, None] + 1) * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:t]
        s = {"case": dict(case), "slots": slots.to(torch.int32).contiguous()}
        if case["op"] == "read":
            return s | _cache(g, pages, hkv, d)
        s |= {"k": torch.zeros(pages, hkv, PAGE, d, device="cuda").to(torch.float8_e4m3fn), "v": torch.zeros(pages, hkv, PAGE, d, device="cuda").to(torch.float8_e4m3fn),
              "k_exp": torch.zeros(pages, hkv, PAGE, device="cuda", dtype=torch.int8), "v_exp": torch.zeros(pages, hkv, PAGE, device="cuda", dtype=torch.int8)}
        s["qkv"] = _rows(g, (t, hq + 2 * hkv, d), True).reshape(t, -1).contiguous()
        if case["norm"]:
            s["q_norm"] = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
            s["k_norm"] = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
        rot = {"none": 0, "half": d // 2}.get(case["rope"], d)
        top = 16384
        first = torch.randint(0, top - t, (3,), generator=g, device="cuda") if case["rope"] == "mrope" else torch.randint(0, top - t, (1,), generator=g, device="cuda").expand(3)
        pos = first[:, None] + torch.arange(t, device="cuda")
        s["positions"] = (pos if case["rope"] == "mrope" else pos[0]).to(torch.int32).contiguous()
        f = 1e6 ** (-torch.arange(0, max(rot, 2), 2, device="cuda").float() / max(rot, 2))
        ang = torch.arange(top, device="cuda").float()[:, None] * f
        s["cos"], s["sin"] = ang.cos().contiguous(), ang.sin().contiguous()
        return s
    new, kv = _lens(case)
    need = [-(-n // PAGE) for n in kv]
    pages = sum(need) + 2
    s = {"case": dict(case)} | _cache(g, pages, hkv, d)
    ids = (torch.randperm(pages - 1, generator=g, device="cuda") + 1).tolist()
    table = [[ids[sum(need[:b]) + i] if i < n else 0 for i in range(max(need))] for b, n in enumerate(need)]
    s["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["cu_q"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["most"] = max(new)
    s["q"] = torch.randn(sum(new), hq * d, generator=g, device="cuda").to(torch.bfloat16)
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        from sglang_omni_b200 import ops

        cache = ops.KV8Cache(state["k"], state["v"], state["k_exp"], state["v_exp"])
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        if case["op"] == "write":
            rope = case["rope"]
            q = ops.kv8_store(state["qkv"], cache, state["slots"], hq, hkv, d, state["positions"], state["cos"], state["sin"],
                              rot_dim={"none": 0, "half": d // 2}.get(rope, d), q_norm=state.get("q_norm"), k_norm=state.get("k_norm"), eps=EPS,
                              neox=rope != "pair", mrope_section=[24, 20, 20] if rope == "mrope" else None, interleaved=True)
            k, v = ops.kv8_read(cache, state["slots"])
            return {"q": q, "k": k, "v": v}
        if case["op"] == "read":
            k, v = ops.kv8_read(cache, state["slots"])
            return {"k": k, "v": v}
        if case["op"] == "decode":
            return ops.kv8_decode_attention(state["q"], cache, state["table"], state["kv_lens"], hq, hkv, d, window=case["window"], sinks=case["sinks"])
        return ops.kv8_prefill_attention(state["q"], cache, state["table"], state["cu_q"], state["kv_lens"], hq, hkv, d, window=case["window"], sinks=case["sinks"])
    return {"write": _write, "read": _read, "decode": _attend, "chunk": _attend}[case["op"]](state)


def _norm(x, w):
    if w is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()


def _rotate(x, state):
    """x [T, H, D] in 32 bits, rotated by its tokens' positions."""
    rope, d = state["case"]["rope"], state["case"]["d"]
    if rope == "none":
        return x
    half = state["cos"].shape[1]
    j = torch.arange(half, device=x.device)
    pos = state["positions"].long()
    if rope == "mrope":   # pairs j = 1, 2 (mod 3) below 60 follow the height and width positions
        axis = torch.where((j % 3 == 1) & (j < 60), 1, torch.where((j % 3 == 2) & (j < 60), 2, 0))
        pos = pos[axis].t()
    else:
        pos = pos[:, None]
    cos, sin = state["cos"][pos, j][:, None], state["sin"][pos, j][:, None]
    if rope == "pair":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).reshape(x.shape)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _put(cache, exps, slots, rows):
    codes, e = _hold(rows)
    page, at = slots // PAGE, slots % PAGE
    cache.view(torch.uint8)[page, :, at] = codes.view(torch.uint8)
    exps[page, :, at] = e


def _get(cache, exps, slots):
    page, at = slots // PAGE, slots % PAGE
    return _values(cache.view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn), exps[page, :, at])


def _write(state):
    case = state["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    x = state["qkv"].float().view(-1, hq + 2 * hkv, d)
    q = _rotate(_norm(x[:, :hq], state.get("q_norm")), state)
    k = _rotate(_norm(x[:, hq:hq + hkv], state.get("k_norm")), state)
    slots = state["slots"].long()
    _put(state["k"], state["k_exp"], slots, k)
    _put(state["v"], state["v_exp"], slots, x[:, hq + hkv:])
    return {"q": q.reshape(q.shape[0], -1).to(torch.bfloat16)} | _read(state)


def _read(state):
    slots = state["slots"].long()
    return {"k": _get(state["k"], state["k_exp"], slots).to(torch.bfloat16), "v": _get(state["v"], state["v_exp"], slots).to(torch.bfloat16)}


def _attend(state):
    """Queries of all requests, padded to the longest chunk, against their gathered keys."""
    case = state["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    table, kv, cu = state["table"].long(), state["kv_lens"].long(), state["cu_q"].long()
    n, most = kv.shape[0], state["most"]
    i = torch.arange(most, device="cuda")
    new = cu[1:] - cu[:-1]
    x = state["q"].float().view(-1, hkv, hq // hkv, d)
    x = x[(cu[:-1, None] + i).clamp(max=x.shape[0] - 1)]                        # [n, most, hkv, g, d]
    x = x.permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    k = _values(state["k"].view(torch.uint8)[table].view(torch.float8_e4m3fn), state["k_exp"][table])
    k = k.transpose(1, 2).reshape(n, hkv, -1, d)
    s = torch.matmul(x, k.transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    del k
    s = s.view(n, hkv, hq // hkv, most, -1)
    j = torch.arange(s.shape[-1], device="cuda")
    p = (kv - new)[:, None] + i                                                 # positions of the queries
    see = (j <= p[..., None]) & (j < kv[:, None, None])
    if case["window"] > 0:
        see &= (j > p[..., None] - case["window"]) | (j < case["sinks"])
    s.masked_fill_(~see[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = s.sum(-1, keepdim=True)
    v = _values(state["v"].view(torch.uint8)[table].view(torch.float8_e4m3fn), state["v_exp"][table])
    v = v.transpose(1, 2).reshape(n, hkv, -1, d)
    o = torch.matmul(s.view(n, hkv, -1, s.shape[-1]), v).view(n, hkv, hq // hkv, most, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, hq * d)
    t = torch.arange(state["q"].shape[0], device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return o[r, t - cu[r]].to(torch.bfloat16)


# ---------------------------------------------------------------- 64 bits
def _two64(n):
    """2^n for whole n, exactly: a power function may be off in its last bit."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _grid64(x):
    """Rows x in 64 bits -> the values that the cache holds for them."""
    amax = x.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448.0))
    e = e - (amax * _two64(1 - e) <= 448.0).double()             # the logarithm's own rounding
    e = (e + (amax * _two64(-e) > 448.0).double()).clamp(-60.0, 60.0)
    y = (x * _two64(-e)).clamp(-448.0, 448.0)
    low = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = _two64(low - (_two64(low) > y.abs().clamp(min=2.0 ** -6)).double() - 3.0)
    return torch.round(y / step) * step * _two64(e)


def _held64(state, name, at):
    """Rows of the cache at `at` (page, offset) in 64 bits, [n, Hkv, D]."""
    c = state[name].view(torch.uint8)[at[0], :, at[1]].long()
    mant, ex = (c & 7).double(), (c >> 3) & 15
    mag = torch.where(ex > 0, (1.0 + mant / 8.0) * _two64(ex - 7), mant * 2.0 ** -9)
    return torch.where(c > 127, -mag, mag) * _two64(state[name + "_exp"][at[0], :, at[1]])[..., None]


def exact(case, seed):
    state = prepare(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "read":
        at = (state["slots"].long() // PAGE, state["slots"].long() % PAGE)
        return {"k": _held64(state, "k", at), "v": _held64(state, "v", at)}
    if case["op"] == "write":
        heads = state["qkv"].double().view(-1, hq + 2 * hkv, d)
        got = []
        for part, w in ((heads[:, :hq], state.get("q_norm")), (heads[:, hq:hq + hkv], state.get("k_norm"))):
            y = part.clone()
            if w is not None:
                y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + EPS) * w.double()
            z = y.clone()
            half = state["cos"].shape[1] if case["rope"] != "none" else 0
            for j in range(half):
                row = state["positions"]
                if case["rope"] == "mrope":
                    row = row[j % 3 if j < 60 else 0]
                c, s = state["cos"][row.long(), j].double()[:, None], state["sin"][row.long(), j].double()[:, None]
                a, b = (2 * j, 2 * j + 1) if case["rope"] == "pair" else (j, j + half)
                z[..., a] = y[..., a] * c - y[..., b] * s
                z[..., b] = y[..., a] * s + y[..., b] * c
            got.append(z)
        return {"q": got[0].reshape(got[0].shape[0], -1), "k": _grid64(got[1]), "v": _grid64(heads[:, hq + hkv:])}
    new, kv = _lens(case)
    g = hq // hkv
    out, at = torch.zeros(sum(new), hq, d, dtype=torch.float64, device="cuda"), 0
    for b, (a, n) in enumerate(zip(new, kv)):
        if n > 0:
            j = torch.arange(n, device="cuda")
            where = (state["table"][b].long()[j // PAGE], j % PAGE)
            keys, vals = _held64(state, "k", where), _held64(state, "v", where)
            i = torch.arange(n - a, n, device="cuda")[:, None]
            see = j <= i
            if case["window"] > 0:
                see = see & ((i - j < case["window"]) | (j < case["sinks"]))
            for h in range(hq):
                q = state["q"][at:at + a].double().view(a, hq, d)[:, h]
                s = (q @ keys[:, h // g].t()) / math.sqrt(d)
                s[~see] = -math.inf
                out[at:at + a, h] = torch.softmax(s, -1) @ vals[:, h // g]
        at += a
    return out.reshape(sum(new), hq * d)
