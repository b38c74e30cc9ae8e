"""Agent graphs: user-defined multi-turn control flow around the policy model.

Parity: chatlearn/models/agent/base_agent_graph.py:37-124 (``AgentGraphOutput``,
``BaseAgentGraph.run`` / ``convert_agent_graph_output``).  The reference builds its
graphs with LangGraph; this package carries its own small ``StateGraph`` with the
same vocabulary (nodes, edges, conditional edges, entry point, ``END``).  A node is
a function ``(state, config) -> update``; a node that calls the model is a generator
(it ``yield``s ``LLMRequest``s, see ``chat_model``), which is what lets the agent
module batch the model calls of many trajectories into one engine call per turn.
"""
import inspect
from dataclasses import dataclass, field
from typing import Any, Callable, Dict, List, Optional

from .chat_model import ChatModel, as_message, find_first_ai_index, find_last_ai_index

END = "__end__"


def leading_zeros_end(mask: List[int]) -> int:
    """Index of the last element of the leading run of zeros (``-1`` if none)."""
    for i, x in enumerate(mask):
        if x != 0:
            return i - 1
    return len(mask) - 1


@dataclass
class AgentGraphOutput:
    str_output: str                      # decoded text after the prompt (model + tool tokens)
    prompt_ids: List[int]
    all_token_ids: List[int]             # prompt + generated + tool-response tokens
    loss_mask: List[int]                 # 1 = generated by the model
    response_logprobs: Optional[List[float]] = None
    reward_score: Optional[float] = None
    num_turns: int = 0
    pixel_values: Any = None
    image_grid_thw: Any = None
    visual_time_steps: Any = None        # per image / video: temporal position step (videos), None (images)
    attention_mask: Any = None
    extra_fields: Dict[str, Any] = field(default_factory=dict)
    # aligned with response_logprobs, where the sampling asks for alternatives
    response_entropies: Optional[List[float]] = None
    response_top_logprobs: Optional[List[List[tuple]]] = None


class CompiledGraph:
    def __init__(self, nodes, edges, cond, entry, max_steps):
        self.nodes, self.edges, self.cond, self.entry, self.max_steps = nodes, edges, cond, entry, max_steps

    @staticmethod
    def _merge(state: Dict[str, Any], update: Optional[Dict[str, Any]]):
        for k, v in (update or {}).items():
            if k == "messages":                      # reducer: append
                state.setdefault("messages", [])
                state["messages"] = list(state["messages"]) + [as_message(m) for m in v]
            else:
                state[k] = v

    def stream(self, state: Dict[str, Any], config: Optional[Dict[str, Any]] = None):
        """Generator running the graph; yields the ``LLMRequest``s of its nodes and
        returns the final state."""
        state = dict(state)
        state["messages"] = [as_message(m) for m in state.get("messages", [])]
        cur, steps = self.entry, 0
        while cur != END:
            steps += 1
            if steps > self.max_steps:
                raise RuntimeError(f"agent graph did not terminate within {self.max_steps} node visits")
            fn = self.nodes[cur]
            res = fn(state, config or {})
            if inspect.isgenerator(res):
                res = yield from res
            self._merge(state, res)
            if cur in self.cond:
                router, mapping = self.cond[cur]
                key = router(state)
                cur = mapping.get(key, key) if mapping else key
            else:
                cur = self.edges.get(cur, END)
        return state

    def invoke(self, state, config=None, llm: Optional[Callable] = None):
        """Run to completion with ``llm(request) -> LLMResponse`` answering each request."""
        gen = self.stream(state, config)
        try:
            req = next(gen)
            while True:
                req = gen.send(llm(req))
        except StopIteration as e:
            return e.value


class StateGraph:
    def __init__(self, state_schema=None, max_steps: int = 256):
        self._nodes: Dict[str, Callable] = {}
        self._edges: Dict[str, str] = {}
        self._cond: Dict[str, Any] = {}
        self._entry: Optional[str] = None
        self._max_steps = max_steps

    def add_node(self, name: str, fn: Callable):
        self._nodes[name] = fn

    def add_edge(self, src: str, dst: str):
        self._edges[src] = dst

    def add_conditional_edges(self, src: str, router: Callable, mapping: Optional[Dict[str, str]] = None):
        self._cond[src] = (router, mapping)

    def set_entry_point(self, name: str):
        self._entry = name

    def compile(self) -> CompiledGraph:
        assert self._entry in self._nodes, "set_entry_point must name a node"
        for s, d in self._edges.items():
            assert s in self._nodes and (d in self._nodes or d == END), f"edge {s}->{d} names an unknown node"
        return CompiledGraph(dict(self._nodes), dict(self._edges), dict(self._cond), self._entry, self._max_steps)


class BaseAgentGraph:
    """Subclass, build ``self.graph`` in ``build_graph`` and implement ``run`` as a
    generator returning an ``AgentGraphOutput`` (``default_run`` covers the common case)."""

    def __init__(self, agent_name: str, cfg=None, llm=None, tokenizer=None, processor=None,
                 model_type: str = "llm", **kwargs):
        self.agent_name, self.cfg, self.llm = agent_name, cfg, llm
        self.tokenizer, self.processor, self.model_type = tokenizer, processor, model_type
        self.chatmodel: Optional[ChatModel] = None
        self.graph: Optional[CompiledGraph] = None

    def build_graph(self):
        self.chatmodel = ChatModel(model=self.agent_name, tokenizer=self.tokenizer, processor=self.processor,
                                   model_type=self.model_type)

    def run(self, sampling_params: Dict[str, Any], **query):
        raise NotImplementedError

    def default_run(self, messages, sampling_params: Dict[str, Any], **query):
        config = {"configurable": {"chat_model": self.chatmodel, "sampling_params": sampling_params, **query}}
        state = yield from self.graph.stream({"messages": messages}, config)
        return self.convert_agent_graph_output(state)

    def convert_agent_graph_output(self, state: Dict[str, Any]) -> AgentGraphOutput:
        msgs = state["messages"]
        last, first = find_last_ai_index(msgs), find_first_ai_index(msgs)
        assert last >= 0, "the graph finished without any model turn"
        meta = msgs[last].response_metadata          # whatever follows the last model turn is dropped
        ids, mask = meta["token_ids"], meta["loss_mask"]
        pe = leading_zeros_end(mask)
        mm = msgs[first].response_metadata.get("multimodel_batch_feature") or {}
        return AgentGraphOutput(
            str_output=self.tokenizer.decode(ids[pe + 1:]), prompt_ids=ids[:pe + 1], all_token_ids=ids,
            loss_mask=mask, response_logprobs=meta.get("logprobs"), num_turns=last + 1,
            pixel_values=mm.get("pixel_values"), image_grid_thw=mm.get("image_grid_thw"),
            visual_time_steps=mm.get("visual_time_steps"),
            attention_mask=mm.get("attention_mask"),
            response_entropies=meta.get("entropies"), response_top_logprobs=meta.get("top_logprobs"))
