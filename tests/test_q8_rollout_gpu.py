"""The 8-bit cache and the token statistics as the rollout uses them, on a GPU."""
import pytest
import torch

from chatlearn_b200 import ops
from chatlearn_b200.ops import reference as ref
from tests import q8_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("D,bs", [(128, 64), (64, 16), (256, 32)])
def test_prompts_in_chunks_then_single_tokens(D, bs):
    """Append and attend through two prompt chunks and 30 single tokens: the cache holds, code for code, what the same
    calls leave on the CPU, and every attention agrees with 64 bits on that cache."""
    nq, nkv, B = 8, 2, 3
    g = torch.Generator().manual_seed(0)
    cache, table = oracle.make_cache([220] * B, nkv, D, bs, device=DEV)
    mirror = oracle.cpu(cache)
    lens = [0] * B
    plan = [[100, 31, 1], [40, 0, 77]] + [None] * 30
    for news in plan:
        n = news or [1] * B
        lens = [a + b for a, b in zip(lens, n)]
        rows = (torch.randn(sum(n), nq + 2 * nkv, D, generator=g) * (1 + 0.2 * lens[0])).bfloat16().to(DEV)
        q, k, v = rows.split([nq, nkv, nkv], 1)
        tables = (table, _i32(lens), None if news is None else _i32(news))
        ops.kv_append_q8(k, v, cache, *tables)
        out = ops.paged_attention_q8(q, cache, *tables)
        ref.kv_append_q8(k.cpu(), v.cpu(), mirror, *(t if t is None else t.cpu() for t in tables))
        for a, b in zip(cache, mirror):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
        want, around, size = oracle.attend(q, cache, *tables)
        prob = 2.0 ** -8 if news is not None and bs % 64 else 2.0 ** -11
        assert ((out.cpu().double() - want).abs() <= oracle.attend_bound(want, around, size, max(lens), D, torch.bfloat16, prob)).all()


def _model(head_dim=128):
    from chatlearn_b200.models.nn import CausalLM, ModelArch
    arch = ModelArch(model_type="qwen3", vocab_size=2048, hidden_size=512, num_hidden_layers=2, num_attention_heads=8,
                     num_key_value_heads=2, head_dim=head_dim, intermediate_size=1024, rope_theta=1e6)
    return arch, CausalLM(arch, dtype=torch.bfloat16, device=torch.device("cuda", 0)).init_weights(3)


@pytest.mark.parametrize("head_dim", [64, 128, 256])
def test_engine_on_an_8_bit_cache(head_dim):
    """Captured and eager decode steps, chunked prompts among running sequences, shared prompts; alternatives of every
    token."""
    from chatlearn_b200.rollout import RolloutEngine, SamplingParams
    arch, model = _model(head_dim)
    g = torch.Generator().manual_seed(9)
    prompts = [torch.randint(0, arch.vocab_size - 1, (n,), generator=g).tolist() for n in (200, 333, 70, 64, 1)]
    batch = [p for p in prompts for _ in range(3)]
    sp = SamplingParams(temperature=0.0, max_tokens=24, ignore_eos=True, logprobs=5)
    outs = []
    for graphs, tokens in ((True, 32768), (False, 32768), (True, 128)):
        before = dict(ops.launch_counts)
        eng = RolloutEngine(model, block_size=64, num_blocks=256, max_num_seqs=32, max_model_len=512, use_cuda_graphs=graphs,
                            max_num_batched_tokens=tokens, kv_dtype=torch.float8_e4m3fn)
        seqs = eng.generate(batch, sp)
        for op in ("kv_append_q8", "paged_attention_q8", "token_logprob"):
            assert ops.launch_counts[op] > before.get(op, 0)
        assert all(len(s.output) == len(s.top_logprobs) == len(s.entropies) == 24 for s in seqs)
        for s in seqs:
            for tok, lp, top, ent in zip(s.output, s.logprobs, s.top_logprobs, s.entropies):
                assert top[0][0] == tok and [l for _, l in top] == sorted((l for _, l in top), reverse=True)
                # two kernels' log-probs of the same fp32 logits: 2^-20 and the logits' rounding
                assert abs(top[0][1] - lp) < 1e-4 and 0.0 <= ent <= 7.7
        outs.append([s.output for s in seqs])
        assert ops.native_ops() and "paged_attention_q8" not in ops.library_counts
    for other in outs[1:]:
        # near-ties may flip a greedy choice: the cuts between blocks go by the batch
        assert sum(a[:6] == b[:6] for a, b in zip(outs[0], other)) >= len(batch) - 3


def test_engine_refuses_on_the_gpu():
    from chatlearn_b200.rollout import RolloutEngine
    with pytest.raises(ValueError, match="8-bit KV cache"):
        RolloutEngine(_model(32)[1], kv_dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="8-bit KV cache"):
        RolloutEngine(_model()[1], kv_dtype=torch.float8_e4m3fn, block_size=8)


def test_half_the_memory_and_close_log_probs():
    """Log-probs under the 8-bit cache against the bf16 one, teacher-forced on the same tokens through both engines'
    decode steps: keys and values are off by 2^-4 at most (2^-5.3 in the mean), the first token of a response not at all."""
    from chatlearn_b200.rollout import RolloutEngine, SamplingParams
    arch, model = _model()
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, arch.vocab_size - 1, (n,), generator=g).tolist() for n in (150, 90, 64)]
    sp = SamplingParams(temperature=0.0, max_tokens=2, ignore_eos=True, logprobs=8)
    got = []
    for dt in (None, torch.float8_e4m3fn):
        eng = RolloutEngine(model, block_size=64, num_blocks=64, max_num_seqs=8, max_model_len=256, kv_dtype=dt)
        got.append((eng.kv_bytes_per_block(), eng.generate(prompts, sp)))
    assert got[1][0] < 0.51 * got[0][0]
    for a, b in zip(got[0][1], got[1][1]):
        assert a.output[0] == b.output[0] and abs(a.logprobs[0] - b.logprobs[0]) < 1e-3          # prefill: no cached key is read
