"""The 8-bit key/value cache and the per-token statistics of logits on the sm_100a kernels.

append            csrc/kv_q8.cu  (page maximum, scale growth and the rows of a page in one block)
attention         csrc/paged_attention_q8.cu  (single tokens: the tokens of all sequences cut evenly over the SMs)
                  csrc/attention_q8_sm100.cu  (many new tokens a sequence: tensor-core tiles of their rows)
token statistics  csrc/token_logprob.cu  (log-prob, entropy and alternatives in one pass; gradient in one more)

What the kernels do not take raises: there is no statement of another kind behind these ops.
"""
import torch

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


def _aligned(x, ok):
    """``x`` itself where it is laid out as the kernels read it, a copy otherwise."""
    return x if ok else x.clone(memory_format=torch.contiguous_format)


# The extension looks at the arguments itself (dtypes, shapes, devices, strides) and does nothing where they are not what
# its kernels read; only then the checks here run, say what is wrong, or bring the arguments into shape.
def kv_append_q8(k, v, cache, block_tables, seq_lens, q_lens=None):
    if not C.kv_append_q8(k, v, *cache, block_tables, seq_lens, q_lens):
        q8.check_append(k, v, cache, block_tables, seq_lens, q_lens)
        _check_kernel("kv_append_q8", cache)
        done = C.kv_append_q8(_aligned(k, k.stride(2) == 1), _aligned(v, v.stride(2) == 1), *cache, _int32(block_tables),
                              _int32(seq_lens), None if q_lens is None else _int32(q_lens))
        assert done, "kv_append_q8: arguments that the kernels do not take"
    _count("kv_append_q8")


def paged_attention_q8(q, cache, block_tables, seq_lens, q_lens=None, scale=None):
    scale = float(scale) if scale is not None else q.shape[-1] ** -0.5
    out = C.paged_attention_q8(q, *cache, block_tables, seq_lens, q_lens, scale)
    if out is None:
        q8.check_attend(q, cache, block_tables, seq_lens, q_lens)
        _check_kernel("paged_attention_q8", cache)
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"paged_attention_q8: bf16 or fp16 queries, got {q.dtype}")
        q = _aligned(q, q.stride(2) == 1 and q.stride(1) == q.shape[2] and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0)
        out = C.paged_attention_q8(q, *cache, _int32(block_tables), _int32(seq_lens), None if q_lens is None else _int32(q_lens), scale)
        assert out is not None, "paged_attention_q8: arguments that the kernels do not take"
    _count("paged_attention_q8", 2 if q_lens is None else 4)
    return out


def token_logprobs(logits, tokens, top_n=0, temperature=1.0):
    run = C.token_logprob_apply if logits.requires_grad and torch.is_grad_enabled() else C.token_logprob_fwd
    out = run(logits, tokens, top_n, 1.0 / temperature) if 1e-30 <= temperature <= 1e30 else ()
    if not out:
        q8.check_token_logprobs(logits, tokens, top_n, temperature)
        if torch.autograd.forward_ad.unpack_dual(logits).tangent is not None:
            raise RuntimeError("token_logprobs: no forward-mode derivative on a GPU")
        if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError(f"token_logprobs: fp32, bf16 or fp16 logits, got {logits.dtype}")
        if top_n > MAX_TOP:
            raise ValueError(f"token_logprobs: at most {MAX_TOP} alternatives, got {top_n}")
        if logits.shape[0] >= 2 ** 28 or logits.shape[1] >= 2 ** 30:
            raise ValueError(f"token_logprobs: logits of {tuple(logits.shape)}")
        z = logits if logits.stride(1) == 1 else logits.contiguous()
        out = run(z, tokens.to(torch.int64).contiguous(), int(top_n), 1.0 / float(temperature))
        assert out, "token_logprobs: arguments that the kernels do not take"
    _count("token_logprob")
    return q8.TokenLogprobs(out[0], out[1], out[2], out[3])


for _name, _fn in (("kv_append_q8", kv_append_q8), ("paged_attention_q8", paged_attention_q8), ("token_logprobs", token_logprobs)):
    register_native(_name, _fn)
