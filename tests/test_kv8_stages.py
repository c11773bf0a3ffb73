"""kv_format of stages: every thinker factory takes it, and rank groups give it to each of their ranks."""
import asyncio

import pytest
import torch

from sglang_omni_b200.client import SamplingParams
from sglang_omni_b200.engines.ar import AREngine, ARRequest, KVPool
from sglang_omni_b200.models.common.ar_stage import create_ar_executor
from sglang_omni_b200.models.common.tokenizer import ByteTokenizer
from sglang_omni_b200.models.decoder import DecoderConfig, DecoderLM
from sglang_omni_b200.ops import KV8Layers


def build_windowed_rank(args, rank, world, device, group, mode):
    """The same small windowed decoder on every rank: it runs with an 8-bit pool only."""
    cfg = DecoderConfig(vocab_size=300, hidden_size=64, num_layers=2, num_heads=2, num_kv_heads=1, head_dim=64,
                        intermediate_size=128, rope_theta=10000.0, max_position=512, dtype=torch.float32,
                        sliding_window=9, window_layers=(1,), sink_tokens=2)
    return DecoderLM(cfg, device=device).random_init_(seed=3, std=0.05)


def prompts(n):
    g = torch.Generator().manual_seed(5)
    return [torch.randint(0, 300, (20 + 7 * i,), generator=g).tolist() for i in range(n)]


@pytest.mark.parametrize("mode", ["replica", "dp"])
def test_rank_groups_carry_the_format(mode):
    from sglang_omni_b200.parallel.rank_group import GroupSpec

    model = build_windowed_rank({}, 0, 1, "cpu", None, mode)
    cfg = model.cfg
    eng = AREngine(model, KVPool(cfg.num_layers, cfg.num_kv_heads, cfg.head_dim, 40, "cpu", cfg.dtype, "e4m3"),
                   max_batch=4, max_context=256, use_graphs=False)
    make = lambda: [ARRequest(rid=f"r{i}", prompt_ids=p, sampling=SamplingParams(temperature=0.0), max_new_tokens=6)  # noqa: E731
                    for i, p in enumerate(prompts(5))]
    alone = make()
    eng.generate(alone)
    spec = GroupSpec(mode=mode, world=2, builder="test_kv8_stages.build_windowed_rank", report_timeout_s=60.0)
    ex = create_ar_executor(None, "decoder", ByteTokenizer(300), max_batch=4, max_context=256, use_graphs=False,
                            rank_group=spec, kv_format="e4m3")

    async def main():
        ex.engine.start()
        try:
            return await asyncio.gather(*[ex.engine.generate(r.rid, r) for r in make()])
        finally:
            ex.engine.stop()

    outs = asyncio.run(main())
    assert [o.output_ids for o in outs] == [r.output_ids for r in alone] and all(len(o.output_ids) == 6 for o in outs)
    if mode == "dp":
        assert ex.engine.threaded.served_remote > 0 and ex.engine.threaded.served_local > 0


def test_ming_thinker_takes_the_format():
    from sglang_omni_b200.client import Client, GenerateRequest
    from sglang_omni_b200.config import PipelineRunner, compile_pipeline
    from sglang_omni_b200.models.ming_omni.config import MingOmniPipelineConfig, ming_stages
    from sglang_omni_b200.models.ming_omni.pipeline.stages import create_thinker_executor
    from test_ming import TINY

    ex = create_thinker_executor("random", "cpu", max_batch=2, max_context=256, overrides=TINY, use_graphs=False,
                                 kv_format="e4m3")
    assert isinstance(ex.engine.threaded.engine.pool.kv, KV8Layers)
    stages = ming_stages(overrides=TINY, device="cpu", max_batch=4, max_context=1024)
    next(s for s in stages if s.name == "thinker").executor.args["kv_format"] = "e4m3"

    async def main():
        coord, compiled = compile_pipeline(MingOmniPipelineConfig(model_path="random", stages=stages))
        async with PipelineRunner(coord, compiled):
            last = None
            async for ch in Client(coord).generate(GenerateRequest(prompt="Hello", max_tokens=5, stream=False,
                                                                   sampling=SamplingParams(temperature=0.0, ignore_eos=True))):
                last = ch
            return last

    assert len(asyncio.run(main()).token_ids) == 5


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_example(device):
    """Codes are off by at most 2^-4 of themselves (2.6 % rms): keys and values each bring that much, 8 % bounds both."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(__file__), "..", "examples", "kv8_cache.py")
    spec = importlib.util.spec_from_file_location("kv8_cache_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    worst, same = example.main(["--device", device, "--prompt", "150", "--chunk", "100", "--steps", "3"])
    assert 0 < worst < 0.08 and same
