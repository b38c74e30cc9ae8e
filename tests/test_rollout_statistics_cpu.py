"""Entropies and alternatives of generated tokens on their way from the engine to a sample: partial rounds, agents."""
from types import SimpleNamespace

import pytest
import torch

from chatlearn_b200 import ops
from chatlearn_b200.models.nn import CausalLM, packed_ctx
from chatlearn_b200.models.nn.arch import PRESETS

KEYS = ("rollout_entropies", "rollout_top_ids", "rollout_top_logprobs")


def _rollout(cls, num_logprobs, **kw):
    """A rollout role on the CPU around a tiny engine, without the runtime."""
    from chatlearn_b200.rollout import RolloutEngine
    role = cls.__new__(cls)
    arch = PRESETS["tiny_qwen3"]()
    model = CausalLM(arch, dtype=torch.float32).init_weights(2)
    role.engine = RolloutEngine(model, block_size=8, num_blocks=128, max_num_seqs=16, max_model_len=128)
    role.arch, role.tokenizer = arch, None
    role._module_args = SimpleNamespace(vllm_input_ids_key="input_ids", max_response_tokens_length=8, seq_length=128, temperature=0.7,
                                        top_p=1.0, top_k=-1, min_p=0.0, presence_penalty=0.0, frequency_penalty=0.0,
                                        repetition_penalty=1.0, ignore_eos=True, num_logprobs=num_logprobs, **kw)
    return role


def _scored(role, tokens, n_prompt, n):
    """The same statistics from one pass over the whole sequence."""
    toks = torch.as_tensor(tokens)
    ctx, _ = packed_ctx([toks.numel()], "cpu")
    with torch.no_grad():
        hidden = role.engine.model.hidden_states(toks, ctx)
        z = torch.nn.functional.linear(hidden, role.engine.model.lm_head_weight()).double()[n_prompt - 1:-1]
    return ops.token_logprobs(z, toks[n_prompt:], n, 0.7)


def _check(role, r, n):
    T = int(r["response_token_length"])
    assert r["rollout_entropies"].shape == (T,) and r["rollout_top_ids"].shape == r["rollout_top_logprobs"].shape == (T, n)
    want = _scored(role, r["all_tokens"], int(r["prompt_token_length"]), n)
    # fp32 logits of a two-layer model, steps against one pass: 1e-4 is over 2^9 roundings of values near 1
    assert (r["rollout_entropies"] - want.entropy).abs().max() < 1e-4
    assert (r["rollout_top_logprobs"] - want.top_logprobs).abs().max() < 1e-4
    assert torch.equal(r["rollout_top_ids"], want.top_ids)
    return want


def _partial_rounds(role, prompts):
    """Two rounds of 4 tokens each through the manager; the samples that are handed to training."""
    from chatlearn_b200.algorithm.grpo_utils.partial_rollout_manager import PartialRolloutManager
    man = PartialRolloutManager.__new__(PartialRolloutManager)
    man._module_args = SimpleNamespace(max_rollout_round=2, rollout_ratio=[0.5, 0.5], mini_response_per_prompt=0, seed=1)
    man.global_args = SimpleNamespace(models=SimpleNamespace(policy=SimpleNamespace(max_response_tokens_length=8, num_inference_per_prompt=1)))
    man._metric_list = []
    man.setup()
    batch = [{"uid": i, "prompt_uid": str(i), "input_ids": list(p), "prompt_token_ids": list(p)} for i, p in enumerate(prompts)]
    done = []
    for _ in range(2):
        man.before_episode()
        rows = man.get_sample_for_rollout(batch)
        done += man.post_process_rollout_results(role.postprocess_func(rows, role.generate(rows)))
        batch = []
    return sorted(done, key=lambda r: r["uid"])


@pytest.mark.parametrize("n", [0, 3])
def test_statistics_of_partial_rounds(n):
    """A sample that was carried on has them for every token of its response, those of the first round in front."""
    from chatlearn_b200.models.rollout_module import RolloutModule
    role = _rollout(RolloutModule, n)
    done = _partial_rounds(role, [[5, 6, 7, 8], [9, 10, 11]])
    assert len(done) == 2
    for r in done:
        assert int(r["response_token_length"]) == 8
        if n:
            _check(role, r, n)
        else:
            assert not any(k in r for k in KEYS)


def test_statistics_of_responses_without_tokens():
    """A prompt that fills the model's length still has the keys that its batch has."""
    from chatlearn_b200.models.rollout_module import RolloutModule
    role = _rollout(RolloutModule, 2)
    rows = [{"input_ids": [3, 4, 5]}, {"input_ids": list(range(128))}]
    out = role.postprocess_func(rows, role.generate(rows))
    assert [tuple(r[k].shape) for r in out for k in KEYS] == [(8,), (8, 2), (8, 2), (0,), (0, 2), (0, 2)]


def test_log_probs_of_partial_rounds():
    """Log-probs belong to the response's tokens from its first one on: what the trainer compares them with."""
    from chatlearn_b200.models.rollout_module import RolloutModule
    role = _rollout(RolloutModule, 0)
    for r in _partial_rounds(role, [[5, 6, 7, 8], [9, 10, 11]]):
        want = _scored(role, r["all_tokens"], int(r["prompt_token_length"]), 0)
        assert r["rollout_logprobs"].shape == (8,) and (r["rollout_logprobs"] - want.logprob).abs().max() < 1e-4


def test_statistics_of_an_agents_turns():
    """Two turns with a tool's answer between them: one entry per response token, none for the tool's."""
    from chatlearn_b200.data.tokenizer import ByteTokenizer
    from chatlearn_b200.models.agent.agent_module import AgentModule
    from chatlearn_b200.models.agent.chat_model import LLMResponse
    from chatlearn_b200.models.agent.examples.math_code_agent_graph import MathCodeAgentGraph
    tok = ByteTokenizer(512)
    turns = [tok.encode('<tool_call>{"name": "execute_python", "arguments": {"code": "print(6*7)"}}</tool_call>'), tok.encode("The answer is 42")]
    role = AgentModule.__new__(AgentModule)
    role._module_args = SimpleNamespace(num_logprobs=2)
    for with_stats in ((True, True), (False, True), (True, False), (False, False)):
        gen = MathCodeAgentGraph("mathcode_agent", cfg={"max_ai_message_turn": 3}, tokenizer=tok).run(
            messages=[{"role": "user", "content": "6*7?"}], sampling_params={}, ground_truth="42")
        req, n0 = next(gen), 0
        with pytest.raises(StopIteration) as end:
            for ids, has in zip(turns, with_stats):
                n0 = n0 or len(req.token_ids)
                stats = ([0.25] * len(ids), [[(5, -0.5), (6, -1.5)]] * len(ids)) if has else (None, None)
                req = gen.send(LLMResponse(ids, [-0.5] * len(ids), "stop", *stats))
        r, = role.postprocess_func([end.value.value], [{}])
        if not any(with_stats):
            assert not any(k in r for k in KEYS)
            continue
        T = int(r["response_token_length"])
        assert r["rollout_logprobs"].shape == r["rollout_entropies"].shape == (T,)
        tool = T - len(turns[0]) - len(turns[1])
        has = torch.tensor([with_stats[0]] * len(turns[0]) + [False] * tool + [with_stats[1]] * len(turns[1]))
        assert tool > 0 and torch.equal(r["rollout_entropies"], torch.where(has, 0.25, 0.0))
        assert torch.equal(r["rollout_top_ids"], torch.where(has[:, None], torch.tensor([5, 6]), -1))
        assert torch.equal(r["rollout_top_logprobs"], torch.where(has[:, None], torch.tensor([-0.5, -1.5]), 0.0))


@pytest.mark.parametrize("schedule", ["continuous", "lockstep"])
def test_statistics_reach_the_agents(schedule):
    """Both ways of answering a graph's requests hand over what the engine has."""
    from chatlearn_b200.models.agent.agent_module import AgentModule
    from chatlearn_b200.models.agent.base_agent_graph import AgentGraphOutput, BaseAgentGraph
    from chatlearn_b200.models.agent.chat_model import LLMRequest

    class OneTurn(BaseAgentGraph):
        def run(self, sampling_params, prompt_ids=None, **query):
            a = yield LLMRequest(list(prompt_ids), {"max_new_tokens": 5}, None)
            return AgentGraphOutput("", list(prompt_ids), list(prompt_ids) + list(a.output_ids), [0] * len(prompt_ids) + [1] * 5,
                                    a.logprobs, response_entropies=a.entropies, response_top_logprobs=a.top_logprobs)

    for n in (0, 3):
        role = _rollout(AgentModule, n, agent_scheduling=schedule)
        role.tp_group = None
        role.agent_factory = {"one": OneTurn("one", llm=role)}
        data = [{"agent_name": "one", "prompt_ids": p} for p in ([5, 6, 7], [8, 9])]
        for r in role.postprocess_func(role.run_trajectories(data), data):
            if n:
                _check(role, r, n)
            else:
                assert not any(k in r for k in KEYS)
