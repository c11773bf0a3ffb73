"""The 8-bit paged KV cache: quantised write, read, and the attention over it (csrc/kv8_*.cu).

Cache of one layer (:class:`KV8Cache`): e4m3 codes ``[pages, Hkv, 64, D]`` for K and for V and one
power-of-two exponent (int8) per (token, KV head) row ``[pages, Hkv, 64]``.  A row x is held as
``rne_e4m3(x * 2^-e)`` with the smallest integer e in [-60, 60] that keeps ``max|x| * 2^-e <= 448``,
and stands for ``code * 2^e``; values beyond 448 * 2^60 saturate.  A row with an infinity or a NaN is
marked (exponent -128) and stands for NaN: a query that sees it gets NaN, others are not touched.
D + 1 bytes a row instead of 2 D.  Head dims 64 and 128, up to 128 query heads per KV head.  Exponents outside the
format, which no write leaves, count as the nearest of it.

Attention is causal.  ``window`` > 0 limits a query to its last ``window`` keys plus the request's
first ``sinks`` tokens.  A query that sees no key (an empty context) gives zeros.

Reference counterparts: the kv_cache_dtype option and sliding-window layers of the SGLang runtime behind
sglang_omni/engines/ar/sglang_backend/server_args_builder.py:10-35.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _check
from ._ext import ext, status_word
from .rope import apply_rope_ref

PAGE = 64
EXP_MIN, EXP_MAX, EXP_BAD = -60, 60, -128
FORMATS = ("e4m3",)


@dataclass
class KV8Cache:
    """One layer's cache (views of the pool's tensors)."""

    k: torch.Tensor       # float8_e4m3fn [pages, Hkv, 64, D]
    v: torch.Tensor
    k_exp: torch.Tensor   # int8 [pages, Hkv, 64]
    v_exp: torch.Tensor

    @classmethod
    def zeros(cls, num_pages: int, num_kv_heads: int, head_dim: int, device) -> "KV8Cache":
        codes = torch.zeros(2, num_pages, num_kv_heads, PAGE, head_dim, dtype=torch.uint8, device=device)
        exps = torch.zeros(2, num_pages, num_kv_heads, PAGE, dtype=torch.int8, device=device)
        codes = codes.view(torch.float8_e4m3fn)
        return cls(codes[0], codes[1], exps[0], exps[1])


class KV8Layers:
    """The 8-bit caches of all layers of a pool; ``[i]`` is layer i's :class:`KV8Cache`."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, device):
        codes = torch.zeros(num_layers, 2, num_pages, num_kv_heads, PAGE, head_dim, dtype=torch.uint8, device=device)
        self.codes = codes.view(torch.float8_e4m3fn)
        self.exps = torch.zeros(num_layers, 2, num_pages, num_kv_heads, PAGE, dtype=torch.int8, device=device)
        self.layers = [KV8Cache(c[0], c[1], e[0], e[1]) for c, e in zip(self.codes, self.exps)]

    def __len__(self) -> int:
        return len(self.layers)

    def __getitem__(self, i: int) -> KV8Cache:
        return self.layers[i]


# ---------------------------------------------------------------- plain restatements (CPU path, test oracles)
def kv8_quantize_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows x [..., D] -> (codes float8_e4m3fn, exponents int8)."""
    x = x.float()
    amax = x.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    mant, ex = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))   # 448 = 0.875 * 2^9
    e = torch.where(mant <= 0.875, ex - 9, ex - 8)
    e = torch.where(amax == 0, torch.full_like(e, EXP_MIN), e.clamp(EXP_MIN, EXP_MAX))
    y = torch.ldexp(torch.where(bad[..., None], torch.zeros_like(x), x), -e[..., None]).clamp(-448.0, 448.0)
    return y.to(torch.float8_e4m3fn), torch.where(bad, torch.full_like(e, EXP_BAD), e).to(torch.int8)


def kv8_dequantize_ref(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """What codes [..., D] with exponents [...] stand for, fp32."""
    e = exps.to(torch.int32)
    y = torch.ldexp(codes.float(), e.clamp(EXP_MIN, EXP_MAX)[..., None])
    return torch.where((e == EXP_BAD)[..., None], torch.full_like(y, float("nan")), y)


def _rows_ref(cache: KV8Cache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    page, off = slots // PAGE, slots % PAGE
    return tuple(kv8_dequantize_ref(c.view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn), e[page, :, off])
                 for c, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)))


def kv8_attention_ref(q, cache: KV8Cache, block_table, q_lens, kv_lens, num_heads, num_kv_heads, head_dim, scale,
                      window=0, sinks=0):
    """q [T, Hq, D] -> [T, Hq, D] in fp32 (or in q's type where that is fp64)."""
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros(q.shape[0], num_heads, head_dim, dtype=dt, device=q.device)
    g, at = num_heads // num_kv_heads, 0
    for b, (a, n) in enumerate(zip(q_lens, kv_lens)):
        n = min(n, block_table.shape[1] * PAGE)     # a request sees at most the keys that its row can name
        if a > 0 and n > 0:
            j = torch.arange(n, device=q.device)
            pages = block_table[b, j // PAGE].long()
            k, v = _rows_ref(cache, torch.where((pages < 0) | (pages >= cache.k.shape[0]), 0, pages) * PAGE + j % PAGE)
            bad = (torch.isnan(k) | torch.isnan(v)).any(-1).t()                  # [Hkv, n]
            k, v = torch.nan_to_num(k).to(dt), torch.nan_to_num(v).to(dt)
            i = torch.arange(n - a, n, device=q.device)[:, None]
            see = j <= i
            if window > 0:
                see = see & ((j > i - window) | (j < sinks))
            s = torch.einsum("ahd,nhd->han", q[at:at + a].to(dt), k.repeat_interleave(g, 1)) * scale
            s = s.masked_fill(bad.repeat_interleave(g, 0)[:, None] & see, float("nan"))
            s = s.masked_fill(~see, float("-inf"))
            p = torch.softmax(s, -1)
            p = torch.where(see.any(-1, keepdim=True), p, torch.zeros_like(p))
            out[at:at + a] = torch.einsum("han,nhd->ahd", p, v.repeat_interleave(g, 1))
        at += a
    return out


def _check_cpu(cache: KV8Cache, num_heads: int, num_kv_heads: int, head_dim: int) -> None:
    if cache.k.dim() != 4 or cache.k.shape[1:] != (num_kv_heads, PAGE, head_dim) or cache.k.dtype != torch.float8_e4m3fn:
        raise ValueError(f"cache.k {tuple(cache.k.shape)} {cache.k.dtype} does not hold {num_kv_heads} KV heads of {head_dim} dims")
    if num_heads % num_kv_heads:
        raise ValueError(f"{num_heads} query heads are not a multiple of {num_kv_heads} KV heads")


# ---------------------------------------------------------------- operators
def kv8_store(qkv: torch.Tensor, cache: KV8Cache, slot_mapping: torch.Tensor, num_heads: int, num_kv_heads: int,
              head_dim: int, positions: torch.Tensor | None = None, cos_tab: torch.Tensor | None = None,
              sin_tab: torch.Tensor | None = None, rot_dim: int | None = None, q_norm: torch.Tensor | None = None,
              k_norm: torch.Tensor | None = None, eps: float = 1e-6, neox: bool = True,
              mrope_section: list[int] | None = None, interleaved: bool = True,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Norm + rotate q and k of the fused QKV rows [T, (Hq + 2 Hkv) * D], quantise k and v into the
    cache at ``slot_mapping`` (int32 [T]; -1 skips a token), return q [T, Hq * D] bf16.

    All arithmetic is fp32 and rounded once; ``qkv`` is not changed.  RoPE arguments as in
    ``qkv_rope_store`` (``rot_dim`` 0, or no ``cos_tab``: no rotation)."""
    rot = (head_dim if rot_dim is None else rot_dim) if cos_tab is not None else 0
    if qkv.is_cuda:
        if _check.enabled():
            if rot:
                _check.check_range("kv8_store", "positions", positions, 0, cos_tab.shape[0])
            _check.check_range("kv8_store", "slot_mapping", slot_mapping, 0, cache.k.shape[0] * PAGE, allow=-1)
        return ext().kv8_store(qkv, cache.k, cache.v, cache.k_exp, cache.v_exp, slot_mapping, num_heads, num_kv_heads,
                               head_dim, positions, cos_tab, sin_tab, rot, q_norm, k_norm, eps, neox,
                               mrope_section or [], interleaved, out)
    _check_cpu(cache, num_heads, num_kv_heads, head_dim)
    T = qkv.shape[0]
    x = qkv[:, :(num_heads + 2 * num_kv_heads) * head_dim].reshape(T, -1, head_dim).float()
    q, k, v = x[:, :num_heads], x[:, num_heads:num_heads + num_kv_heads], x[:, num_heads + num_kv_heads:]

    def prep(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.float()
        return apply_rope_ref(y, positions, cos_tab, sin_tab, rot, neox, mrope_section, interleaved) if rot else y

    q, k = prep(q, q_norm), prep(k, k_norm)
    live = ((slot_mapping >= 0) & (slot_mapping < cache.k.shape[0] * PAGE)).nonzero().squeeze(1)
    s = slot_mapping.long()[live]
    for codes, exps, rows in ((cache.k, cache.k_exp, k), (cache.v, cache.v_exp, v)):
        c, e = kv8_quantize_ref(rows[live])
        codes.view(torch.uint8)[s // PAGE, :, s % PAGE] = c.view(torch.uint8)
        exps[s // PAGE, :, s % PAGE] = e
    q = q.reshape(T, -1).to(qkv.dtype)
    if out is None:
        return q
    out.copy_(q)
    return out


def kv8_read(cache: KV8Cache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V rows of ``slots`` (int32 [n]) as bf16 [n, Hkv, D], exactly the held values; a slot
    outside the cache gives zeros."""
    if slots.is_cuda:
        return ext().kv8_read(cache.k, cache.v, cache.k_exp, cache.v_exp, slots)
    ok = (slots >= 0) & (slots < cache.k.shape[0] * PAGE)
    k, v = _rows_ref(cache, torch.where(ok, slots.long(), 0))
    return tuple(torch.where(ok[:, None, None], x, torch.zeros_like(x)).to(torch.bfloat16) for x in (k, v))


def kv8_decode_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, kv_lens: torch.Tensor,
                         num_heads: int, num_kv_heads: int, head_dim: int, scale: float | None = None,
                         window: int = 0, sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """One query token per request, the last of its ``kv_lens`` keys.  q: [B, >= Hq * D] rows."""
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    if q.is_cuda:
        if _check.enabled():
            _check.check_paged("kv8_decode_attention", block_table, kv_lens, cache.k.shape[0])
        return ext().kv8_attention(q, cache.k, cache.v, cache.k_exp, cache.v_exp, block_table, None, kv_lens,
                                   num_heads, num_kv_heads, head_dim, scale, window, sinks, out,
                                   status_word(q.device))
    return _attention_cpu(q, cache, block_table, [1] * kv_lens.shape[0], kv_lens, num_heads, num_kv_heads, head_dim,
                          scale, window, sinks, out)


def kv8_prefill_attention(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, cu_q: torch.Tensor,
                          kv_lens: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int,
                          scale: float | None = None, window: int = 0, sinks: int = 0,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each request's new tokens (rows cu_q[b] .. cu_q[b + 1] of q, the last of
    its ``kv_lens[b]`` keys).  q: [T, >= Hq * D] rows.  The new tokens' keys are in the cache already.
    Rows from cu_q[-1] on are unspecified."""
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    if q.is_cuda:
        if _check.enabled():
            _check.check_paged("kv8_prefill_attention", block_table, kv_lens, cache.k.shape[0], cu_q, q.shape[0])
        return ext().kv8_attention(q, cache.k, cache.v, cache.k_exp, cache.v_exp, block_table, cu_q, kv_lens,
                                   num_heads, num_kv_heads, head_dim, scale, window, sinks, out,
                                   status_word(q.device))
    cu = cu_q.tolist()
    return _attention_cpu(q, cache, block_table, [b - a for a, b in zip(cu, cu[1:])], kv_lens, num_heads, num_kv_heads,
                          head_dim, scale, window, sinks, out)


def _attention_cpu(q, cache, block_table, q_lens, kv_lens, hq, hkv, d, scale, window, sinks, out):
    _check_cpu(cache, hq, hkv, d)
    if window < 0 or sinks < 0:
        raise ValueError("window and sinks must not be negative")
    o = kv8_attention_ref(q[:, :hq * d].reshape(-1, hq, d), cache, block_table, q_lens, kv_lens.tolist(), hq, hkv, d,
                          scale, window, sinks)
    o = o.reshape(q.shape[0], hq * d).to(q.dtype)
    if out is None:
        return o
    out.copy_(o)
    return out
