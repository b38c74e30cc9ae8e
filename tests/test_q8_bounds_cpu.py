"""The bound that the attention tests hold the kernels to: it lets fp16 probabilities pass and bf16 ones not."""
import math

import pytest
import torch

from tests import q8_oracle as oracle


@pytest.mark.parametrize("dtype,passes", [(torch.float16, True), (torch.bfloat16, False)])
@pytest.mark.parametrize("D,nkv,bs", [(128, 4, 16), (64, 8, 48), (256, 2, 32)])
def test_rounded_probabilities(dtype, passes, D, nkv, bs):
    """The statement in 64 bits with its probabilities rounded once, 2^7 for a row's largest, over the first 300 tokens of
    a sequence (rows that see few keys weigh them by hand)."""
    L = 300
    cache, table = oracle.make_cache([L], nkv, D, bs)
    q = (torch.randn(L, 4 * nkv, D, generator=torch.Generator().manual_seed(1)) * 0.25).bfloat16()
    lens = torch.tensor([L], dtype=torch.int32)
    want, around, size = oracle.attend(q, cache, table, lens, lens)
    k, v = (t.double()[table[0].long()].transpose(0, 1).reshape(nkv, -1, D)[:, :L] for t in cache.dequantize())
    s = torch.einsum("nhrd,hld->hrnl", q.double().view(L, nkv, 4, D), k) / math.sqrt(D)
    s = s.masked_fill(torch.arange(L)[None] > torch.arange(L)[:, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp() * 2.0 ** 7
    out = torch.einsum("hrnl,hld->nhrd", p.to(dtype).double(), v) / p.sum(-1).permute(2, 0, 1)[..., None]
    out = out.reshape(L, 4 * nkv, D).bfloat16().double()
    assert ((out - want).abs() <= oracle.attend_bound(want, around, size, L, D, torch.bfloat16, 2.0 ** -11)).all() == passes
