"""The engine over the 8-bit key/value cache on the GPU: eager steps and decode graphs, portions, several prompts, swaps."""

import pytest
import torch

from enterprise_inference_amd.config import CacheConfig, EngineConfig, ModelConfig, SchedulerConfig
from enterprise_inference_amd.engine.llm_engine import LLMEngine
from enterprise_inference_amd.engine.sampling_params import SamplingParams
from enterprise_inference_amd.models.catalog import tiny_config

pytestmark = pytest.mark.gpu

SHAPE = dict(hidden_size=1024, intermediate_size=2048, num_attention_heads=8, num_key_value_heads=2, head_dim=128, vocab_size=1024,
             num_hidden_layers=2, max_position_embeddings=4096)


def _engine(arch="LlamaForCausalLM", eager=False, blocks=64, mbt=256, bs=128):
    extra = {"num_local_experts": 4, "num_experts_per_tok": 2} if arch.startswith("Mixtral") else {}
    cfg = EngineConfig(model=ModelConfig.from_hf_dict(tiny_config(arch, **SHAPE, **extra)),
                       cache=CacheConfig(block_size=bs, num_gpu_blocks=blocks, cache_dtype=torch.float8_e4m3fn, enable_prefix_caching=False),
                       scheduler=SchedulerConfig(max_num_seqs=16, max_num_batched_tokens=mbt, max_model_len=2048),
                       device="cuda", dtype=torch.bfloat16, load_format="dummy", enforce_eager=eager)
    return LLMEngine(cfg)


@pytest.mark.parametrize("arch,bs", [("LlamaForCausalLM", 128), ("Qwen3ForCausalLM", 64), ("MixtralForCausalLM", 16)])
def test_graphs_give_what_eager_steps_give(arch, bs):
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(3, 1000, (n,), generator=g).tolist() for n in (700, 37, 300, 5, 64, 129, 200, 90)]
    params = SamplingParams(max_tokens=24, temperature=0, ignore_eos=True)
    got = []
    for eager in (False, True):
        eng = _engine(arch, eager, blocks=64 * 128 // bs, bs=bs)
        assert bool(eng.executor.runner.graphs) != eager
        got.append([o.outputs[0].token_ids for o in eng.generate(prompt_token_ids=prompts, params=params)])
    assert all(len(t) == 24 for t in got[0])
    assert got[0] == got[1]


def test_swapped_blocks_come_back_whole():
    eng = _engine()
    r = eng.executor.runner
    if getattr(r, "swap_buf", None) is None:
        pytest.skip("no host memory for swaps")
    r.kv_buf.copy_(torch.randint(0, 127, r.kv_buf.shape, device="cuda").to(torch.uint8))
    was = r._kv_blocks()[:, :, [3, 7]].clone()
    r.swap_out([3, 7], [0, 1])
    r._kv_blocks()[:, :, [3, 7]] = 0
    r.swap_in([1, 0], [9, 5])
    torch.cuda.synchronize()
    assert torch.equal(r._kv_blocks()[:, :, [5, 9]], was)
    assert r.kv_caches[1].k[5].view(torch.uint8).eq(was[1, 0, 0, :r.kv_caches[1].k[5].numel()].view(r.kv_caches[1].k[5].shape)).all()


def test_llama4_graphs_give_what_eager_steps_give():
    """Layers with chunks of 192 tokens and layers without rotation, whose queries take a temperature; prompts and answers cross the
    chunks' borders."""
    d = tiny_config("Llama4ForCausalLM", **{**SHAPE, "num_hidden_layers": 4}, num_local_experts=4, num_experts_per_tok=1,
                    intermediate_size_mlp=2048, attention_chunk_size=192, no_rope_layers=[1, 0, 1, 0], use_qk_norm=True,
                    attn_temperature_tuning=True, floor_scale=64, attn_scale=0.1, interleave_moe_layer_step=1, moe_layers=[1, 3])
    g = torch.Generator().manual_seed(6)
    prompts = [torch.randint(3, 1000, (n,), generator=g).tolist() for n in (700, 37, 180, 5, 375, 192)]
    params = SamplingParams(max_tokens=24, temperature=0, ignore_eos=True)
    got = []
    for eager in (False, True):
        cfg = EngineConfig(model=ModelConfig.from_hf_dict(d),
                           cache=CacheConfig(block_size=64, num_gpu_blocks=64, cache_dtype=torch.float8_e4m3fn, enable_prefix_caching=False),
                           scheduler=SchedulerConfig(max_num_seqs=16, max_num_batched_tokens=256, max_model_len=2048),
                           device="cuda", dtype=torch.bfloat16, load_format="dummy", enforce_eager=eager)
        eng = LLMEngine(cfg)
        assert bool(eng.executor.runner.graphs) != eager
        assert [layer.self_attn.chunk_size for layer in eng.executor.runner.model.layers] == [192, None, 192, None]
        got.append([o.outputs[0].token_ids for o in eng.generate(prompt_token_ids=prompts, params=params)])
    assert all(len(t) == 24 for t in got[0])
    assert got[0] == got[1]
