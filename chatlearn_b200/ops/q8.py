"""The paged key/value cache in 8 bits, and the argument checks that its operators share.

A cached value is an e4m3 code times a power-of-two scale; one scale per page (block of
tokens), kv head, and keys or values.  ``kv_append_q8`` writes new rows and keeps the scales,
``paged_attention_q8`` attends over the pages.  Rows are named by sequence: ``block_tables
[B, width]`` lists a sequence's pages, ``seq_lens [B]`` is its length with the new tokens,
``q_lens [B]`` how many of them are new (``None``: one row per sequence, none where its length
is 0).  The new rows of all sequences are packed one behind the other; rows behind the last
sequence are ignored.

On a GPU: head dims 64, 128 and 256, pages of a multiple of 16 tokens, any ratio of query to
kv heads; bf16 and fp16 queries, bf16, fp16 and fp32 new rows.  What the kernels do not take is
refused.  Many new tokens of a sequence go through tensor-core tiles that read its cache once where
the queries are bf16; fp16 queries go row by row, each reading what it sees: for single tokens that is
the same, for long chunks it is slow.  A page id outside the cache is skipped when appending and masked when attending.  Two
sequences of one call must not append to the same page (its contents are then undefined, no
other page is touched).  Masked places may hold anything, NaN among it, where no query of the call's
row of new tokens sees them; a NaN value that a later token of the same call sees may reach the
earlier ones (zero times NaN), as in the statements.
"""
from typing import NamedTuple

import torch

CODE_MAX = 448.0                  # largest e4m3 value
SCALE_MIN, SCALE_MAX = 2.0 ** -24, 2.0 ** 64
CODE_DTYPE = torch.float8_e4m3fn


class Q8KVCache(NamedTuple):
    """One layer's cache: codes ``k, v [pages, kv heads, page tokens, head dim]`` (e4m3) and
    power-of-two scales ``k_scale, v_scale [pages, kv heads]`` (fp32)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @staticmethod
    def empty(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, device=None) -> "Q8KVCache":
        """A cache of ``num_blocks`` pages that hold nothing yet."""
        codes = lambda: torch.zeros(num_blocks, num_kv_heads, block_size, head_dim, dtype=torch.uint8,  # noqa: E731
                                    device=device).view(CODE_DTYPE)
        scale = lambda: torch.full((num_blocks, num_kv_heads), SCALE_MIN, device=device)  # noqa: E731
        return Q8KVCache(codes(), codes(), scale(), scale())

    @staticmethod
    def bytes_per_block(block_size: int, num_kv_heads: int, head_dim: int) -> int:
        return 2 * num_kv_heads * (block_size * head_dim + 4)

    def dequantize(self):
        """Keys and values as fp32, laid out like the codes."""
        return (self.k.float() * self.k_scale[:, :, None, None], self.v.float() * self.v_scale[:, :, None, None])


def _check_tables(what, cache, block_tables, seq_lens, q_lens, rows, device):
    k, v, ks, vs = cache
    if not (k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype == CODE_DTYPE):
        raise ValueError(f"{what}: the cache holds e4m3 codes [pages, kv heads, page tokens, head dim], the same for keys and values")
    if k.shape[0] == 0:
        raise ValueError(f"{what}: a cache without pages")
    if not (ks.shape == vs.shape == k.shape[:2] and ks.dtype == vs.dtype == torch.float32):
        raise ValueError(f"{what}: one fp32 scale per page and kv head")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{what}: the cache's tensors are contiguous")
    if block_tables.dim() != 2 or seq_lens.dim() != 1 or block_tables.shape[0] != seq_lens.shape[0]:
        raise ValueError(f"{what}: block_tables [B, width] and seq_lens [B]")
    if block_tables.shape[1] * k.shape[2] >= 2 ** 30:
        raise ValueError(f"{what}: tables of {block_tables.shape[1]} pages of {k.shape[2]} tokens, 2^30 tokens and more")
    if q_lens is not None:
        if q_lens.shape != seq_lens.shape:
            raise ValueError(f"{what}: q_lens [B] like seq_lens")
    elif rows < seq_lens.shape[0]:
        raise ValueError(f"{what}: {rows} rows for {seq_lens.shape[0]} sequences (one each without q_lens)")
    for t in (k, v, ks, vs, block_tables, seq_lens) + (() if q_lens is None else (q_lens,)):
        if t.device != device:
            raise ValueError(f"{what}: all tensors on one device, got {t.device} beside {device}")
    for t in (block_tables, seq_lens) + (() if q_lens is None else (q_lens,)):
        if t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{what}: tables and lengths are int32 or int64, got {t.dtype}")


def check_append(k, v, cache, block_tables, seq_lens, q_lens):
    what = "kv_append_q8"
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"{what}: k and v [rows, kv heads, head dim], alike")
    if k.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"{what}: bf16, fp16 or fp32 rows, got {k.dtype}")
    if v.device != k.device:
        raise ValueError(f"{what}: k and v on one device")
    _check_tables(what, cache, block_tables, seq_lens, q_lens, k.shape[0], k.device)
    if (k.shape[1], k.shape[2]) != (cache.k.shape[1], cache.k.shape[3]):
        raise ValueError(f"{what}: rows of {tuple(k.shape[1:])} for a cache of {cache.k.shape[1]} heads of {cache.k.shape[3]}")


def check_attend(q, cache, block_tables, seq_lens, q_lens):
    what = "paged_attention_q8"
    if q.dim() != 3 or not q.is_floating_point():
        raise ValueError(f"{what}: q [rows, query heads, head dim]")
    _check_tables(what, cache, block_tables, seq_lens, q_lens, q.shape[0], q.device)
    if q.shape[2] != cache.k.shape[3] or cache.k.shape[1] == 0 or q.shape[1] % cache.k.shape[1] or q.shape[1] == 0:
        raise ValueError(f"{what}: {q.shape[1]} query heads of {q.shape[2]} over {cache.k.shape[1]} kv heads of {cache.k.shape[3]}")


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns, per row: the token's log-probability, the entropy, and the
    likeliest tokens with their log-probabilities, most likely first."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor
    top_ids: torch.Tensor


def check_token_logprobs(logits, tokens, top_n, temperature):
    what = "token_logprobs"
    if logits.dim() != 2 or tokens.shape != logits.shape[:1]:
        raise ValueError(f"{what}: logits [rows, vocabulary] and tokens [rows]")
    if not logits.is_floating_point() or tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: floating logits and int32 or int64 tokens, got {logits.dtype} and {tokens.dtype}")
    if tokens.device != logits.device:
        raise ValueError(f"{what}: logits and tokens on one device")
    if not 0 <= top_n <= logits.shape[1]:
        raise ValueError(f"{what}: {top_n} alternatives out of a vocabulary of {logits.shape[1]}")
    if logits.shape[1] == 0:
        raise ValueError(f"{what}: an empty vocabulary")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"{what}: the temperature is positive (1e-30 to 1e30), got {temperature}")
