"""Token-in / token-out chat model for agent graphs.

Parity: chatlearn/models/agent/chat_model.py:53-254.  The reference wraps an async
SGLang engine in a LangChain ``BaseChatModel``; every conversation is its own
coroutine.  Here a conversation is a Python *generator*: ``ChatModel.invoke`` yields
an ``LLMRequest`` (the token ids to continue) and is resumed with the
``LLMResponse``; the agent module drives all conversations of a batch in lock-step
so that each turn is ONE batched call of the rollout engine.

Token bookkeeping is incremental exactly like the reference's: the ids of the whole
trajectory and a loss mask (1 = generated by the model, 0 = prompt or tool output)
ride on the last AI message; a new turn tokenizes only the messages after it.
"""
import json
import uuid
from dataclasses import dataclass, field
from typing import Any, Callable, Dict, List, Optional

from .tool_parser import ToolParser


@dataclass
class Message:
    content: str = ""
    type: str = "human"
    name: Optional[str] = None
    tool_call_id: Optional[str] = None
    tool_calls: List[Dict[str, Any]] = field(default_factory=list)
    invalid_tool_calls: List[Dict[str, Any]] = field(default_factory=list)
    response_metadata: Dict[str, Any] = field(default_factory=dict)

    def to_openai(self) -> Dict[str, Any]:
        role = {"human": "user", "ai": "assistant", "system": "system", "tool": "tool"}[self.type]
        d = {"role": role, "content": self.content}
        if self.type == "tool":
            d["name"], d["tool_call_id"] = self.name, self.tool_call_id
        if self.tool_calls:
            d["tool_calls"] = [{"type": "function", "id": c["id"],
                                "function": {"name": c["name"], "arguments": c["args"]}} for c in self.tool_calls]
        return d


def HumanMessage(content, **kw):
    return Message(content=content, type="human", **kw)


def SystemMessage(content, **kw):
    return Message(content=content, type="system", **kw)


def AIMessage(content, **kw):
    return Message(content=content, type="ai", **kw)


def ToolMessage(content, name=None, tool_call_id=None, **kw):
    return Message(content=content, type="tool", name=name, tool_call_id=tool_call_id, **kw)


def as_message(m) -> Message:
    if isinstance(m, Message):
        return m
    role = m.get("role", "user")
    typ = {"user": "human", "assistant": "ai", "system": "system", "tool": "tool"}[role]
    return Message(content=m.get("content", ""), type=typ, name=m.get("name"), tool_call_id=m.get("tool_call_id"))


def find_last_ai_index(messages) -> int:
    for i in range(len(messages) - 1, -1, -1):
        if messages[i].type == "ai":
            return i
    return -1


def find_first_ai_index(messages) -> int:
    for i, m in enumerate(messages):
        if m.type == "ai":
            return i
    return -1


@dataclass
class LLMRequest:
    token_ids: List[int]
    sampling_params: Dict[str, Any] = field(default_factory=dict)
    mm: Optional[Dict[str, Any]] = None      # vision-language requests: pixel_values + image_grid_thw of the prompt's images


@dataclass
class LLMResponse:
    output_ids: List[int]
    logprobs: Optional[List[float]] = None
    finish_reason: Optional[str] = None
    # where the sampling asks for alternatives, per generated token: entropy, likeliest (token, log-prob)
    entropies: Optional[List[float]] = None
    top_logprobs: Optional[List[List[tuple]]] = None


# statistics of the response's tokens besides their log-probs, and what stands for tokens that have none (a tool's)
_PER_TOKEN = (("entropies", 0.0), ("top_logprobs", ()))


def tool_schema(fn: Callable) -> Dict[str, Any]:
    """OpenAI function schema from a Python callable's signature and docstring."""
    import inspect
    props, req = {}, []
    for name, p in inspect.signature(fn).parameters.items():
        if name == "kwargs" or p.kind in (p.VAR_KEYWORD, p.VAR_POSITIONAL):
            continue
        typ = {int: "integer", float: "number", bool: "boolean"}.get(p.annotation, "string")
        props[name] = {"type": typ}
        if p.default is inspect.Parameter.empty:
            req.append(name)
    return {"type": "function", "function": {"name": fn.__name__, "description": (fn.__doc__ or "").strip(),
                                             "parameters": {"type": "object", "properties": props, "required": req}}}


class ChatModel:
    def __init__(self, model: str, tokenizer, processor=None, model_type: str = "llm",
                 tool_parser: str = "hermes", max_parallel_calls: int = 1):
        self.model_name = model
        self.tokenizer, self.processor, self.model_type = tokenizer, processor, model_type
        self.parser = ToolParser.get_tool_parser(tool_parser, tokenizer)
        self.max_parallel_calls = max_parallel_calls
        self.tools: Optional[List[Dict[str, Any]]] = None
        self._system_prefix: List[int] = []
        # vision-language models: {"image_token_id", "video_token_id", "merge_size"} of the engine's vision tower
        self.vision: Optional[Dict[str, int]] = None

    def bind_tools(self, tools: List[Callable]) -> "ChatModel":
        """A copy of the model that advertises ``tools`` in the chat template."""
        other = ChatModel(self.model_name, self.tokenizer, self.processor, self.model_type,
                          max_parallel_calls=self.max_parallel_calls)
        other.parser = self.parser
        other.vision = self.vision
        other.tools = [tool_schema(t) for t in tools]
        # some templates prepend a default system block to any message list; later turns strip it
        try:
            other._system_prefix = list(self._template([{}], False, True))
        except Exception:
            other._system_prefix = []
        return other

    def _template(self, openai_messages, add_generation_prompt: bool, tokenize: bool, tools=None):
        kw = dict(add_generation_prompt=add_generation_prompt, tokenize=tokenize)
        if tools:
            kw["tools"] = tools
        try:
            out = self.tokenizer.apply_chat_template(openai_messages, enable_thinking=False, **kw)
        except TypeError:
            out = self.tokenizer.apply_chat_template(openai_messages, **kw)
        if tokenize and isinstance(out, dict):
            out = out["input_ids"]
        return out

    # ---- messages -> token ids -------------------------------------------------
    def _with_images(self, ids: List[int], mm: Dict[str, Any]) -> List[int]:
        """One token per merged image patch: a single placeholder per image (what chat templates emit) is
        expanded; a template without image placeholders gets the image tokens in front of the text."""
        from chatlearn_b200.data.vision_utils import expand_image_tokens
        tok, merge = int(self.vision["image_token_id"]), int(self.vision.get("merge_size", 2))
        vtok = self.vision.get("video_token_id")
        grids = [[int(v) for v in g] for g in (mm["image_grid_thw"].tolist() if hasattr(mm["image_grid_thw"], "tolist")
                                               else mm["image_grid_thw"])]
        want = sum(t * h * w for t, h, w in grids) // (merge * merge)
        have = ids.count(tok) + (ids.count(vtok) if vtok is not None else 0)
        if have == want:
            return ids
        if have == 0:
            steps = mm.get("visual_time_steps") or [None] * len(grids)
            ids = [tok if st is None or vtok is None else vtok for st in steps] + ids      # videos carry a time step
        return expand_image_tokens(ids, grids, tok, merge, vtok)

    def preprocess(self, messages: List[Message], mm: Optional[Dict[str, Any]] = None) -> Dict[str, Any]:
        assert messages[-1].type in ("human", "tool"), \
            f"the last message must come from the user or a tool, got {messages[-1].type}"
        last_ai = find_last_ai_index(messages)
        if last_ai < 0:
            text = self._template([m.to_openai() for m in messages], True, False, self.tools)
            ids = list(self.tokenizer.encode(text))
            pre = {}
            if mm is not None and mm.get("pixel_values") is not None and self.vision is not None:
                ids = self._with_images(ids, mm)
                pre["mm"] = {"pixel_values": mm["pixel_values"], "image_grid_thw": mm["image_grid_thw"],
                             "visual_time_steps": mm.get("visual_time_steps")}
            pre.update(token_ids=ids, loss_mask=[0] * len(ids))
            return pre
        prev = messages[last_ai].response_metadata
        tail = self._template([m.to_openai() for m in messages[last_ai + 1:]], True, True)
        tail = list(tail)
        n = len(self._system_prefix)
        if n and tail[:n] == self._system_prefix:
            tail = tail[n:]
        pre = {"token_ids": list(prev["token_ids"]) + tail, "loss_mask": list(prev["loss_mask"]) + [0] * len(tail)}
        if prev.get("multimodel_batch_feature"):     # the images of the first turn stay with the conversation
            pre["mm"] = prev["multimodel_batch_feature"]
        if "logprobs" in prev:        # aligned with the response tokens; tool tokens carry 0
            pre["logprobs"] = list(prev["logprobs"]) + [0.0] * len(tail)
        for key, none in _PER_TOKEN:
            if key in prev:
                pre[key] = list(prev[key]) + [none] * len(tail)
        return pre

    # ---- generated ids -> AI message -------------------------------------------
    def postprocess(self, resp: LLMResponse, pre: Dict[str, Any]) -> Message:
        out = list(resp.output_ids)
        ids = pre["token_ids"] + out
        mask = pre["loss_mask"] + [1] * len(out)
        content, calls = self.parser.extract_tool_calls(out)
        good, bad = [], []
        for c in calls:
            err = None
            try:
                args = json.loads(c.arguments)
                if not isinstance(args, dict):
                    err = f"tool arguments must be a JSON object, got {type(args).__name__}"
            except json.JSONDecodeError as e:
                args, err = None, f"invalid JSON tool arguments: {e}"
            rec = {"name": c.name, "id": str(uuid.uuid4())}
            if err:
                bad.append({**rec, "args": c.arguments, "error": err})
            else:
                good.append({**rec, "args": args})
        meta = {"token_ids": ids, "loss_mask": mask, "finish_reason": resp.finish_reason}
        if pre.get("mm") is not None:
            meta["multimodel_batch_feature"] = pre["mm"]
        if resp.logprobs is not None:
            meta["logprobs"] = list(pre.get("logprobs", [])) + list(resp.logprobs)
            for key, none in _PER_TOKEN:
                new = getattr(resp, key)
                if new is not None or key in pre:        # (a turn without them among others)
                    meta[key] = list(pre.get(key, [none] * len(pre.get("logprobs", [])))) + (list(new) if new is not None else [none] * len(out))
        return Message(content=content, type="ai", tool_calls=good[: self.max_parallel_calls],
                       invalid_tool_calls=bad[: self.max_parallel_calls], response_metadata=meta)

    def invoke(self, messages: List[Message], sampling_params: Optional[Dict[str, Any]] = None,
               mm: Optional[Dict[str, Any]] = None):
        """Generator: ``ai_message = yield from chat_model.invoke(messages, sampling_params)``.
        ``mm``: ``pixel_values`` / ``image_grid_thw`` of the conversation's images (vision-language models)."""
        pre = self.preprocess(messages, mm)
        resp = yield LLMRequest(pre["token_ids"], dict(sampling_params or {}), pre.get("mm"))
        return self.postprocess(resp, pre)
