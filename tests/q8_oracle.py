"""64-bit oracles and error bounds of the 8-bit cache operators and the token statistics."""
import math

import torch

from chatlearn_b200 import ops
from chatlearn_b200.ops import reference as ref

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def cpu(cache):
    return ops.Q8KVCache(*(t.cpu().clone() for t in cache))


def make_cache(lens, nkv, D, bs, seed=0, extra=3, device="cpu", width=None):
    """A cache with random contents everywhere (stale pages and slots hold NaN codes) and a block table of pages in no order."""
    g = torch.Generator().manual_seed(seed)
    lens = list(lens)
    need = [(L + bs - 1) // bs for L in lens]
    width = width or max(1, max(need, default=1))
    nb = sum(need) + extra
    perm = torch.randperm(nb, generator=g).tolist()
    table = torch.full((len(lens), width), perm[-1], dtype=torch.int32)
    codes = [(torch.randn(nb, nkv, bs, D, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    powers = torch.tensor([2.0 ** e for e in (-9, -8, -7, -6, -5)])
    scales = [powers[torch.randint(0, 5, (nb, nkv), generator=g)].contiguous() for _ in range(2)]
    used = torch.zeros(nb, bs, dtype=torch.bool)
    at = 0
    for b, (L, n) in enumerate(zip(lens, need)):
        for i in range(n):
            page = perm[at]
            table[b, i] = page
            used[page, :min(bs, L - i * bs)] = True
            at += 1
    for c in codes:
        c.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7f)
    cache = ops.Q8KVCache(codes[0].contiguous(), codes[1].contiguous(), *scales)
    return ops.Q8KVCache(*(t.to(device) for t in cache)), table.to(device)


def attend(q, cache, table, lens, news=None, scale=None):
    """(output, sum p |v| as `attend_bound` wants it, largest sum |q k| scale) in 64 bits.

    fp16 probabilities below 2^-14 are multiples of 2^-24: off by 2^-25 at most, which is 2^-28 of a row's largest (that one
    stands at 2^7 or 2^10, or at 2^-4 of it where V's scales differ).  Over all tokens that adds 2^-28 sum |v|, here as
    2^-17 of it to what is multiplied by 2^-11 or more."""
    args = (table.cpu(), lens.cpu(), None if news is None else news.cpu())
    c = cpu(cache)
    q = q.detach().cpu().double()
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[2])
    out = ref.paged_attention_q8(q, c, *args, scale)
    raw = c.v.view(torch.uint8) & 0x7f
    absolute = c._replace(v=raw.view(torch.float8_e4m3fn))
    around = ref.paged_attention_q8(q, absolute, *args, scale)
    around += 2.0 ** -17 * max(int(lens.max()), 1) * ref.paged_attention_q8(torch.zeros_like(q), absolute, *args, scale)
    k = c.dequantize()[0].nan_to_num(nan=0.0).abs().amax((0, 2))                 # [nkv, D]
    size = (q.abs() * k.double().repeat_interleave(q.shape[1] // k.shape[0], 0)[None]).sum(-1).max() * scale if q.numel() else torch.tensor(0.0)
    return out, around, float(size) * (1 if scale >= 0 else -1)


def attend_bound(out, around, size, L, D, dtype, prob=2.0 ** -11):
    """How far a result may be off.  The output is rounded once (half a step).  Probabilities are rounded to fp16 for
    the product (2^-11 of each: ``prob``; the kernel that takes long chunks rounds them to two bf16, 2^-16, where its
    tiles of 64 keys hold pages whose V scales are far apart).  A score is a sum of D exact products in fp32 (truncating adds: 2^-23 each) times
    rounded factors (4 roundings): (D + 8) 2^-23 of sum |q k|; fp16 queries lose 2^-11 of elements below 2^-24 of their
    row's largest: 2^-33 sum |q k|, inside that.  The exponential adds 2^-22, and the maximum it is relative to as much again.
    Numerator and denominator each carry the score's error.  The sums over L tokens: 2^-23 per add."""
    score = (D + 8) * 2.0 ** -23 * size + 2.0 ** -20 + 2.0 ** -22 * 1.5 * size
    rel = prob + 2 * score + 2 * (L / 16 + 32) * 2.0 ** -23
    return HALF_STEP[dtype] * out.abs() * 1.01 + rel * around + 2.0 ** -24 * HALF_STEP[dtype]


def statistics_bound(z, temp, lp):
    """Absolute error of a log-probability: x = z c - M has 3 roundings of terms up to Z = max |z| / temperature in
    bits (log2 e of it), in the numerator and in the sum; the sum has V / 512 adds in a row and 24 joins, each 2^-24; the
    exponential and the logarithm 2^-22 each; the result is rounded."""
    fin = torch.where(z.isfinite(), z, 0.0).double().abs()
    Z = fin.amax(1) / temp * 1.4427
    tol = 2.0 ** -20 + 16 * 2.0 ** -24 * Z + (z.shape[1] / 512 + 24) * 2.0 ** -24
    return tol if lp is None else tol + 2.0 ** -22 * torch.where(lp.isfinite(), lp.abs(), 0.0)
