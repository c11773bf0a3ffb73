"""Which layers of a Hugging Face checkpoint have a sliding window: the decoder against transformers' logits."""
import json

import pytest
import torch

from sglang_omni_b200.models.hf_text.convert import decoder_config_from_hf, decoder_from_hf
from test_kv8_engine import logits_of, prompts

transformers = pytest.importorskip("transformers")

BASE = dict(vocab_size=300, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, head_dim=64, sliding_window=12, max_position_embeddings=512)
MIXED = ["sliding_attention", "full_attention"]
QWEN = dict(use_sliding_window=True)
# every expert takes part, so that the rounding of the cache cannot change a token's experts
MOE = dict(moe_intermediate_size=64, num_experts=4, num_experts_per_tok=4, norm_topk_prob=True, decoder_sparse_step=1)
CASES = {
    "mistral": ("MistralForCausalLM", "MistralConfig", {}, (0, 1)),
    "qwen2": ("Qwen2ForCausalLM", "Qwen2Config", QWEN | {"max_window_layers": 1}, (1,)),
    "qwen2_all": ("Qwen2ForCausalLM", "Qwen2Config", QWEN | {"max_window_layers": 0}, (0, 1)),
    "qwen2_default": ("Qwen2ForCausalLM", "Qwen2Config", QWEN, ()),
    "qwen2_types": ("Qwen2ForCausalLM", "Qwen2Config", QWEN | {"layer_types": MIXED}, (0,)),
    "qwen2_unused": ("Qwen2ForCausalLM", "Qwen2Config", {"use_sliding_window": False, "max_window_layers": 0}, None),
    "qwen3": ("Qwen3ForCausalLM", "Qwen3Config", QWEN | {"max_window_layers": 1}, (1,)),
    "qwen3_types": ("Qwen3ForCausalLM", "Qwen3Config", QWEN | {"layer_types": MIXED}, (0,)),
    "qwen3_moe": ("Qwen3MoeForCausalLM", "Qwen3MoeConfig", QWEN | MOE, (0, 1)),
    "qwen3_moe_field": ("Qwen3MoeForCausalLM", "Qwen3MoeConfig", QWEN | MOE | {"max_window_layers": 28}, (0, 1)),
}


def windows(c):
    return None if c.sliding_window == 0 else tuple(i for i in range(c.num_layers) if c.window_of(i)[0])


@pytest.mark.parametrize("source", ["module", "directory", "bare"])
@pytest.mark.parametrize("name", CASES)
def test_windowed_layers_match_transformers(name, source, tmp_path):
    """The cache's codes are off by at most 2^-4 of themselves (2.6 % rms), which only the attention branch
    carries into the logits: 5 % of their 2-norm bounds the difference.  A window of 12 put into a wrong
    layer, or left out of one, at 60 tokens changes most of what that layer adds.  ``bare``: a config.json
    without the fields that transformers fills in."""
    arch, config, kw, layers = CASES[name]
    cfg = getattr(transformers, config)(**BASE, **kw)
    cfg.architectures = [arch]
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    hf = transformers.AutoModelForCausalLM.from_config(cfg).float().eval()
    ids = prompts(1, lambda i: 60, 300, seed=7)[0]
    with torch.no_grad():
        ref = hf(torch.tensor([ids])).logits[0]
    src = hf
    if source != "module":
        hf.save_pretrained(tmp_path)
        src = str(tmp_path)
        c = json.loads((tmp_path / "config.json").read_text())
        if "num_local_experts" in c:                      # published checkpoints name it num_experts
            c["num_experts"] = c.pop("num_local_experts")
        (tmp_path / "config.json").write_text(json.dumps(c))
    if source == "bare":
        for field in ("layer_types", "max_window_layers", "use_sliding_window"):
            if field not in kw:
                c.pop(field, None)
        if c.get("sliding_window") is None and kw.get("use_sliding_window") is False:
            c["sliding_window"] = 12                  # left in the file beside use_sliding_window false
        (tmp_path / "config.json").write_text(json.dumps(c))
    model = decoder_from_hf(src, "cpu", torch.float32, kv_format="e4m3")
    assert windows(model.cfg) == layers
    got = logits_of(model, ids, "cpu", "e4m3")
    assert float((got - ref).norm() / ref.norm()) < 0.05


def test_windows_that_are_not_known_are_refused():
    base = {"vocab_size": 10, "hidden_size": 128, "num_hidden_layers": 2, "num_attention_heads": 2, "sliding_window": 16,
            "max_position_embeddings": 4096}
    for bad in ({"architectures": ["LlamaForCausalLM"]}, {"model_type": "other"},
                {"architectures": ["Qwen2ForCausalLM"], "use_sliding_window": True, "layer_types": ["sliding_attention"]},
                {"architectures": ["Qwen3ForCausalLM"], "use_sliding_window": True, "layer_types": ["chunked_attention"] * 2}):
        with pytest.raises(NotImplementedError):
            decoder_config_from_hf(base | bad, kv_format="e4m3")
    # what a Mistral file does not say is transformers' default
    bare = {k: v for k, v in base.items() if k != "sliding_window"} | {"architectures": ["MistralForCausalLM"], "max_position_embeddings": 8192}
    assert windows(decoder_config_from_hf(bare, kv_format="e4m3")) == (0, 1)
    assert decoder_config_from_hf(bare, kv_format="e4m3").sliding_window == transformers.MistralConfig().sliding_window == 4096
    assert windows(decoder_config_from_hf(bare | {"sliding_window": None}, kv_format="e4m3")) is None
    # an architecture's name is enough, and so is a model type
    for named in ({"architectures": ["Qwen3MoeForCausalLM"]}, {"model_type": "qwen3_moe"}):
        assert windows(decoder_config_from_hf(base | named | {"use_sliding_window": True, "max_window_layers": 28}, kv_format="e4m3")) == (0, 1)
