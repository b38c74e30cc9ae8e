"""The step of a replica without requests on a GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv_dtype", [None, torch.float8_e4m3fn])
@pytest.mark.parametrize("experts", [0, 8])
def test_idle_step(kv_dtype, experts):
    from chatlearn_b200.models.nn import CausalLM, ModelArch
    from chatlearn_b200.rollout import RolloutEngine, SamplingParams
    more = dict(num_experts=experts, num_experts_per_tok=2, moe_intermediate_size=256) if experts else {}
    arch = ModelArch(model_type="qwen3_moe" if experts else "qwen3", vocab_size=2048, hidden_size=512, num_hidden_layers=2,
                     num_attention_heads=8, num_key_value_heads=2, head_dim=128, intermediate_size=1024, rope_theta=1e6, **more)
    model = CausalLM(arch, dtype=torch.bfloat16, device=torch.device("cuda", 0)).init_weights(3)
    eng = RolloutEngine(model, block_size=64, num_blocks=16, max_num_seqs=4, max_model_len=128, kv_dtype=kv_dtype)
    sp = SamplingParams(temperature=0.0, max_tokens=6, ignore_eos=True)
    want = eng.generate([[5, 6, 7]], sp)[0].output
    eng._idle_step()
    assert eng.generate([[5, 6, 7]], sp)[0].output == want
