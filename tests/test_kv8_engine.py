"""The paged engine, the decoder and the Hugging Face conversion over the 8-bit KV pool and sliding windows."""
import asyncio

import pytest
import torch

from sglang_omni_b200.engines.ar import AREngine, ARRequest, KVPool
from sglang_omni_b200.models.decoder import DecoderConfig, DecoderLM, ForwardBatch
from sglang_omni_b200.models.hf_text.convert import decoder_config_from_hf, decoder_from_hf
from sglang_omni_b200.ops import KV8Layers, prefill_tile_rows, prefill_tiles
from sglang_omni_b200.sampling_params import SamplingParams


def tiny(dtype=torch.float32, **kw):
    c = dict(vocab_size=512, hidden_size=128, num_layers=2, num_heads=8, num_kv_heads=2, head_dim=64,
             intermediate_size=256, rope_theta=10000.0, qk_norm=True, max_position=4096, dtype=dtype)
    return DecoderConfig(**(c | kw))


def logits_of(model, tokens, device, kv_format):
    """Logits of every position (fresh pool, one prefill)."""
    cfg, T = model.cfg, len(tokens)
    pool = KVPool(cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, (T + 63) // 64 + 2, device, cfg.dtype, kv_format)
    pages = pool.alloc((T + 63) // 64)
    t = torch.arange(T)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(device)  # noqa: E731
    G = cfg.num_heads // cfg.num_kv_heads
    rows = prefill_tile_rows(cfg.head_dim, G) if torch.device(device).type == "cuda" else 64
    req, tok0 = prefill_tiles([T], G, rows)
    fb = ForwardBatch(is_decode=False, positions=i32(torch.stack([t] * 3)), slot_mapping=i32(torch.tensor(pages)[t // 64] * 64 + t % 64),
                      kv_lens=i32([T]), block_table=i32([pages]), input_ids=i32(tokens), cu_q=i32([0, T]),
                      tile_req=i32(req), tile_tok0=i32(tok0), tile_rows=rows)
    return model.logits(model(fb, pool.kv)).float().cpu()


def prompts(n, length, vocab, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (length(i),), generator=g).tolist() for i in range(n)]


def run_engine(model, kv_format, ids, new, **kw):
    cfg = model.cfg
    pool = KVPool(cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, 256, model.embed.device, cfg.dtype, kv_format)
    eng = AREngine(model, pool, max_batch=8, max_context=1024, **kw)
    reqs = [ARRequest(rid=f"r{i}", prompt_ids=p, sampling=SamplingParams(temperature=0.0), max_new_tokens=new)
            for i, p in enumerate(ids)]
    eng.generate(reqs)
    return reqs


def check_greedy(model, reqs, device, tol):
    """Every token of the engine (chunked prefill, decode steps) is the teacher-forced argmax, or within tol of it."""
    for r in reqs:
        lg = logits_of(model, list(r.prompt_ids) + r.output_ids, device, "e4m3")
        for i, tok in enumerate(r.output_ids):
            row = lg[len(r.prompt_ids) - 1 + i]
            assert row[tok] >= row.max() - tol, (r.rid, i, float(row.max() - row[tok]))


def test_pool_formats():
    p = KVPool(2, 2, 64, 5, "cpu", torch.float32, "e4m3")
    assert isinstance(p.kv, KV8Layers) and len(p.kv) == 2 and p.kv[1].k.shape == (5, 2, 64, 64)
    assert p.kv[0].k_exp.dtype == torch.int8
    a = KVPool.for_memory(2, 2, 128, 1 << 20, "cpu", torch.bfloat16)
    b = KVPool.for_memory(2, 2, 128, 1 << 20, "cpu", torch.bfloat16, kv_format="e4m3")
    assert b.num_pages >= int(1.95 * a.num_pages)          # 256 bytes a row against 129
    for bad in (dict(kv_format="int4"), dict(kv_format="e4m3")):
        with pytest.raises(ValueError):
            KVPool(1, 1, 96, 3, "cpu", torch.bfloat16, **bad)


def test_eight_bit_cache_stays_near_the_native_one():
    """Codes are off by at most 2^-4 of themselves (2.6 % rms), and only the attention branch carries that
    into the logits: 5 % of their 2-norm bounds the difference."""
    model = DecoderLM(tiny(), "cpu").random_init_(seed=1, std=0.05)
    ids = prompts(1, lambda i: 150, 512, seed=2)[0]
    a, b = logits_of(model, ids, "cpu", "native"), logits_of(model, ids, "cpu", "e4m3")
    assert 0 < float((a - b).norm() / a.norm()) < 0.05


def test_window_and_sinks_bound_what_a_token_sees():
    """One layer: a last token with a window of 16 depends on the last 16 tokens (and the sinks) alone."""
    ids = prompts(2, lambda i: 100, 512, seed=3)
    x = ids[0]
    y = ids[1][:84] + x[84:]                               # other tokens before the window
    z = x[:2] + ids[1][2:84] + x[84:]                      # the first two the same
    for sinks, others, same in ((0, y, True), (2, y, False), (2, z, True)):
        model = DecoderLM(tiny(num_layers=1, sliding_window=16, sink_tokens=sinks), "cpu").random_init_(seed=4, std=0.05)
        a, b = (logits_of(model, t, "cpu", "e4m3")[-1] for t in (x, others))
        assert torch.equal(a, b) == same
    model = DecoderLM(tiny(num_layers=1, sliding_window=16, window_layers=()), "cpu").random_init_(seed=4, std=0.05)
    assert not torch.equal(logits_of(model, x, "cpu", "e4m3")[-1], logits_of(model, y, "cpu", "e4m3")[-1])
    model = DecoderLM(tiny(num_layers=1, sliding_window=16), "cpu").random_init_(seed=4)
    with pytest.raises(ValueError, match="8-bit"):
        logits_of(model, x, "cpu", "native")


def test_engine_cpu_matches_full_recompute():
    model = DecoderLM(tiny(sliding_window=24, sink_tokens=3, window_layers=(1,)), "cpu").random_init_(seed=5, std=0.05)
    reqs = run_engine(model, "e4m3", prompts(4, lambda i: 9 + 40 * i, 512, seed=6), 8, max_prefill_tokens=50, use_graphs=False)
    assert all(len(r.output_ids) == 8 for r in reqs)
    check_greedy(model, reqs, "cpu", 1e-4)


def test_sliding_window_checkpoints():
    base = {"architectures": ["MistralForCausalLM"], "vocab_size": 10, "hidden_size": 128, "num_hidden_layers": 3,
            "num_attention_heads": 2, "sliding_window": 16, "max_position_embeddings": 4096}
    c = decoder_config_from_hf(base, kv_format="e4m3")
    assert c.sliding_window == 16 and [c.window_of(i) for i in range(3)] == [(16, 0)] * 3
    q = base | {"architectures": ["Qwen2ForCausalLM"], "use_sliding_window": True, "max_window_layers": 2}
    assert [decoder_config_from_hf(q, kv_format="e4m3").window_of(i)[0] for i in range(3)] == [0, 0, 16]
    t = q | {"layer_types": ["sliding_attention", "full_attention", "sliding_attention"]}
    assert [decoder_config_from_hf(t, kv_format="e4m3").window_of(i)[0] for i in range(3)] == [16, 0, 16]
    # contexts within the window need none
    assert decoder_config_from_hf(base, max_position=16).sliding_window == 0
    transformers = pytest.importorskip("transformers")
    from sglang_omni_b200.engines.omni.factory import create_ar_engine

    cfg = transformers.MistralConfig(vocab_size=300, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
                                     num_attention_heads=4, num_key_value_heads=2, head_dim=64, sliding_window=12,
                                     max_position_embeddings=512)
    cfg.architectures = ["MistralForCausalLM"]
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    hf = transformers.AutoModelForCausalLM.from_config(cfg).float().eval()
    ids = prompts(1, lambda i: 60, 300, seed=7)[0]
    with torch.no_grad():
        ref = hf(torch.tensor([ids])).logits[0]
    got = logits_of(decoder_from_hf(hf, "cpu", kv_format="e4m3"), ids, "cpu", "e4m3")
    assert float((got - ref).norm() / ref.norm()) < 0.05
    with pytest.raises(NotImplementedError, match="e4m3"):
        create_ar_engine(hf, max_seq_len=128)
    eng = create_ar_engine(hf, max_seq_len=128, kv_format="e4m3", max_batch=2, use_graphs=False)

    async def go():
        try:
            return await eng.generate("r0", ARRequest("r0", ids, SamplingParams(temperature=0.0, ignore_eos=True), max_new_tokens=5))
        finally:
            eng.stop()

    assert len(asyncio.run(go()).output_ids) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("kw", [dict(num_heads=16, num_kv_heads=2, head_dim=128, mrope_section=[24, 20, 20]),
                                dict(num_heads=6, num_kv_heads=2, head_dim=64, sliding_window=100, sink_tokens=4, window_layers=(1,))])
def test_engine_gpu(graphs, kw):
    """Chunked prefill and CUDA-graph decode over the 8-bit pool agree with a teacher-forced prefill (the
    tolerance of the native pool's test: bf16 activations, logits of a few units)."""
    model = DecoderLM(tiny(torch.bfloat16, hidden_size=256, vocab_size=1024, **kw), "cuda").random_init_(seed=8, std=0.05)
    reqs = run_engine(model, "e4m3", prompts(11, lambda i: 3 + 31 * i, 1024, seed=9), 20, max_prefill_tokens=200, use_graphs=graphs)
    assert all(len(r.output_ids) == 20 for r in reqs)
    check_greedy(model, reqs, "cuda", 0.15)
    ids = reqs[-1].prompt_ids
    if not kw.get("sliding_window"):
        a, b = logits_of(model, ids, "cuda", "native"), logits_of(model, ids, "cuda", "e4m3")
        assert 0 < float((a - b).norm() / a.norm()) < 0.05
