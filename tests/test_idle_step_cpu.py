"""The step of a replica without requests, which keeps it in its peers' collectives."""
import pytest
import torch

from chatlearn_b200.models.nn import CausalLM
from chatlearn_b200.models.nn.arch import PRESETS


@pytest.mark.parametrize("kv_dtype", [None, torch.float8_e4m3fn])
@pytest.mark.parametrize("preset", ["tiny_qwen3", "tiny_moe", "tiny_qwen3_next", "tiny_llama", "tiny_mla_moe"])
def test_idle_step(preset, kv_dtype):
    """No token: every layer runs on none, and the caches stay as they are."""
    from chatlearn_b200.rollout import RolloutEngine
    if preset == "tiny_mla_moe" and kv_dtype is not None:
        return                                     # (refused when the engine is made)
    model = CausalLM(PRESETS[preset](), dtype=torch.float32).init_weights(2)
    eng = RolloutEngine(model, block_size=8, num_blocks=16, max_num_seqs=4, max_model_len=64, kv_dtype=kv_dtype)
    eng.alloc_kv_cache()
    tensors = [t for c in eng.q8_cache if c is not None for t in c] if kv_dtype is not None else eng.k_cache + eng.v_cache
    before = [t.clone() for t in tensors]
    eng._idle_step()
    assert tensors and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, tensors))
