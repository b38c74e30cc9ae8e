"""Log-probs of decode steps that read the 8-bit cache, on a GPU."""
import pytest
import torch

from chatlearn_b200 import ops
from tests.test_q8_rollout_gpu import _model

pytestmark = pytest.mark.gpu


def _steps(model, prompts, dtype, mode, tokens=4):
    """The engine's greedy tokens with 64 alternatives each."""
    from chatlearn_b200.rollout import RolloutEngine, SamplingParams
    was = ops.get_mode()
    ops.set_mode(mode)
    try:
        eng = RolloutEngine(model, block_size=64, num_blocks=64, max_num_seqs=8, max_model_len=512, kv_dtype=dtype,
                            use_cuda_graphs=mode == "native" and dtype is not None)
        return eng.generate(prompts, SamplingParams(temperature=0.0, max_tokens=tokens, ignore_eos=True, logprobs=64))
    finally:
        ops.set_mode(was)


def _apart(a, b):
    """Largest difference of the alternatives' log-probs that both name, and how many were compared, over the steps whose
    earlier tokens are the same (their prefill's own token, which reads no cached key, left out)."""
    worst, count = 0.0, 0
    for x, y in zip(a, b):
        for i in range(1, len(x.output)):
            if x.output[:i] != y.output[:i]:
                break
            other = dict(y.top_logprobs[i])
            both = [(lp, other[t]) for t, lp in x.top_logprobs[i] if t in other]
            worst, count = max([worst] + [abs(p - q) for p, q in both]), count + len(both)
    return worst, count


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_decode_steps_on_the_8_bit_cache(head_dim):
    """Against the statements on the same cache: what bf16 rounds.  Against the 16-bit cache: what e4m3 rounds.

    s is the spread of a row's logits.  A hidden state is rounded to bf16 some 14 times a layer, 28 times in all, each with
    a standard deviation of 2^-9 / sqrt 3 of itself; two runs, five deviations: 5 sqrt(2 * 28) 2^-9 / sqrt 3 = 0.042 s.
    The second layer's keys and values, apart by some 2^-7 then, fall on neighbouring codes (2^-3.5 apart) once in 2^3.5:
    sqrt(2^-3.5) 2^-3.5 = 2^-5.3 in the mean, five deviations: 0.13 s more.  e4m3 itself rounds keys and values by
    2^-5.3 in the mean, which is what an attention output is off by at most in the mean, and so a layer's share of the hidden state; two layers, five deviations: 5 sqrt 2 2^-5.3 = 0.18 s more."""
    arch, model = _model(head_dim)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, arch.vocab_size - 1, (n,), generator=g).tolist() for n in (333, 150, 90, 64)]
    from chatlearn_b200.models.nn import packed_ctx
    with torch.no_grad():
        toks = torch.tensor(prompts[0], device="cuda")
        hidden = model.hidden_states(toks, packed_ctx([toks.numel()], "cuda")[0])
        s = float(torch.nn.functional.linear(hidden, model.lm_head_weight()).float().std(1).mean())
    q8 = torch.float8_e4m3fn
    native, plain, wide = _steps(model, prompts, q8, "native"), _steps(model, prompts, q8, "library"), _steps(model, prompts, None, "native")
    worst, count = _apart(native, plain)
    assert count > 300 and worst <= (0.042 + 0.13) * s, (worst, s, count)
    worst, count = _apart(native, wide)
    assert count > 300 and worst <= (0.042 + 0.18) * s, (worst, s, count)
