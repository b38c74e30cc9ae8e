"""The 8-bit key/value cache and the per-token statistics of logits on the sm_100a kernels.

append            csrc/kv_q8.cu  (page maximum, scale growth and the rows of a page in one block)
attention         csrc/paged_attention_q8.cu  (the tokens of all sequences cut evenly over the SMs)
token statistics  csrc/token_logprob.cu  (log-prob, entropy and alternatives in one pass; gradient in one more)

What the kernels do not take raises: there is no statement of another kind behind these ops.
"""
import math

import torch
from torch.autograd.function import once_differentiable

from . import q8, register_native
from . import native as _n

C = _n.C
_count = _n._count

HEAD_DIMS = (64, 128, 256)
MAX_TOP = 64


def _int32(t):
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _check_kernel(what, cache):
    if cache.k.shape[3] not in HEAD_DIMS or cache.k.shape[2] % 16 or cache.k.shape[2] == 0:
        raise ValueError(f"{what}: head dim {cache.k.shape[3]} and pages of {cache.k.shape[2]} tokens; the kernels take "
                         f"head dims {HEAD_DIMS} and pages of a multiple of 16")
    if cache.k.data_ptr() % 16 or cache.v.data_ptr() % 16:
        raise ValueError(f"{what}: codes start at a multiple of 16 bytes")


def _rows(x):
    """Heads side by side with unit stride inside a head."""
    return x if x.stride(2) == 1 else x.contiguous()


@torch.no_grad()
def kv_append_q8(k, v, cache, block_tables, seq_lens, q_lens=None):
    q8.check_append(k, v, cache, block_tables, seq_lens, q_lens)
    _check_kernel("kv_append_q8", cache)
    C.kv_append_q8(_rows(k), _rows(v), *cache, _int32(block_tables), _int32(seq_lens), None if q_lens is None else _int32(q_lens))
    _count("kv_append_q8")


@torch.no_grad()
def paged_attention_q8(q, cache, block_tables, seq_lens, q_lens=None, scale=None):
    q8.check_attend(q, cache, block_tables, seq_lens, q_lens)
    _check_kernel("paged_attention_q8", cache)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"paged_attention_q8: bf16 or fp16 queries, got {q.dtype}")
    D = q.shape[2]
    if q.stride(2) != 1 or q.stride(1) != D or q.stride(0) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
    _count("paged_attention_q8", 2)
    return C.paged_attention_q8(q, *cache, _int32(block_tables), _int32(seq_lens), None if q_lens is None else _int32(q_lens),
                                float(scale) if scale is not None else 1.0 / math.sqrt(D))


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, tokens, top_n, inv_temp):
        lp, ent, top, ids, stats = C.token_logprob_fwd(z, tokens, top_n, inv_temp)
        _count("token_logprob_fwd")
        ctx.save_for_backward(z, tokens, ent, stats, ids)
        ctx.inv_temp = inv_temp
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return lp, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, g_top, _):
        z, tokens, ent, stats, ids = ctx.saved_tensors
        g = [None if t is None else t.float().contiguous() for t in (g_lp, g_ent, g_top)]
        if all(t is None for t in g):
            return None, None, None, None
        _count("token_logprob_bwd")
        return C.token_logprob_bwd(z, tokens, ent, stats, ids, *g, ctx.inv_temp), None, None, None


def token_logprobs(logits, tokens, top_n=0, temperature=1.0):
    q8.check_token_logprobs(logits, tokens, top_n, temperature)
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"token_logprobs: fp32, bf16 or fp16 logits, got {logits.dtype}")
    if top_n > MAX_TOP:
        raise ValueError(f"token_logprobs: at most {MAX_TOP} alternatives, got {top_n}")
    if logits.shape[0] * 8 >= 2 ** 31 or logits.shape[1] >= 2 ** 30:
        raise ValueError(f"token_logprobs: logits of {tuple(logits.shape)}")
    z = logits if logits.stride(1) == 1 else logits.contiguous()
    return q8.TokenLogprobs(*_TokenLogprobs.apply(z, tokens.to(torch.int64).contiguous(), int(top_n), 1.0 / float(temperature)))


for _name, _fn in (("kv_append_q8", kv_append_q8), ("paged_attention_q8", paged_attention_q8), ("token_logprobs", token_logprobs)):
    register_native(_name, _fn)
