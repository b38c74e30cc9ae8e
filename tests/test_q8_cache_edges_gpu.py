"""The 8-bit cache on a GPU: what the operators owe the kernels after them, and scales far apart."""
import pytest
import torch

from chatlearn_b200 import ops
from tests import q8_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("lens,news,width", [
    ([20] * 3, None, 60),                  # every unit is one tile: no cut divides any
    ([100], None, 8),
    ([1024] * 37, None, 16),               # as many units as shares, all alike
    ([4000] * 12, [24] * 12, 63),          # every sequence goes by tiles: the list of rows is empty
    ([2000, 7], None, 32),
])
def test_the_next_kernel_sees_the_output(lens, news, width):
    """A product that may start before its predecessor ends, right behind the attention: the same as after a pause."""
    nq, nkv, D = 32, 8, 128
    cache, table = oracle.make_cache(lens, nkv, D, 64, device=DEV, width=width)
    lens_t, news_t = _i32(lens), None if news is None else _i32(news)
    T = len(lens) if news is None else sum(news)
    g = torch.Generator(DEV).manual_seed(0)
    q = torch.randn(T, nq, D, device=DEV, dtype=torch.bfloat16, generator=g)
    w = torch.randn(1024, nq * D, device=DEV, dtype=torch.bfloat16, generator=g) * 0.02

    def attend():
        return ops.paged_attention_q8(q, cache, table, lens_t, news_t).view(T, nq * D)
    with torch.no_grad():
        out = attend()
        torch.cuda.synchronize()
        want = ops.linear(out, w)
        before = dict(ops.launch_counts)
        for _ in range(50):
            out.fill_(float("nan"))          # what stands where the next output will be
            del out
            out = attend()
            got = ops.linear(out, w)
            assert torch.equal(got, want)
    assert ops.launch_counts["gemm_bf16_nt"] == before["gemm_bf16_nt"] + 50


@pytest.mark.parametrize("D,nkv,bs", [(128, 4, 16), (64, 8, 48), (256, 2, 32)])
@pytest.mark.parametrize("apart", [14, 26, 40])
def test_small_keys_beside_a_large_page(D, nkv, bs, apart):
    """Pages inside a tile of 64 keys whose K scales are far apart, the large one behind the earlier rows: those see
    their own keys as if it were not there.  Queries as large as their keys are small."""
    L, n, big = 300, 280, 160                      # the page of token `big` is large: rows of earlier tokens do not see it
    cache, table = oracle.make_cache([L], nkv, D, bs, device=DEV)
    at = big // bs * bs
    plain = [t.clone() for t in cache]
    cache.k_scale[table[0, big // bs].long()] = 2.0 ** (apart - 7)
    q = (torch.randn(n, 4 * nkv, D, generator=torch.Generator().manual_seed(0)) * 0.5).bfloat16().to(DEV)
    got = ops.paged_attention_q8(q, cache, table, _i32([L]), _i32([n]))
    rows = at - (L - n)                            # new tokens in front of the page
    want, around, size = oracle.attend(q[:rows], ops.Q8KVCache(*plain), table, _i32([at]), _i32([rows]))
    off, tol = (got[:rows].cpu().double() - want).abs(), oracle.attend_bound(want, around, size, L, D, torch.bfloat16)
    assert rows > 64 and (off <= tol).all(), f"worst {(off / tol.clamp_min(1e-30)).max():.3g} times the bound"


@pytest.mark.parametrize("nq,nkv,D,bs", [(32, 8, 128, 64), (16, 4, 128, 16), (32, 4, 64, 64), (16, 2, 256, 32), (64, 8, 64, 48), (32, 2, 128, 64)])
@pytest.mark.parametrize("power", [18, 24, 30, 45, 70])
@pytest.mark.parametrize("chunk", [False, True])
def test_scores_far_from_zero(nq, nkv, D, bs, power, chunk):
    """Scores of 2^18 to 2^70 whose largest is twice the next: all weight is on that key, whose value comes back as it is.
    (One element of q and of each key: the scores are exact, but for the softmax scale.)"""
    L = 200
    cache, table = oracle.make_cache([L], nkv, D, bs, device=DEV)
    # token 0 is the one: every row of new tokens sees it
    cache.k.view(torch.uint8).zero_()
    codes = torch.full((cache.k.shape[0], nkv, bs), 8.0)
    codes[int(table[0, 0]), :, 0] = 16.0
    cache.k[..., 5] = codes.to(DEV).to(cache.k.dtype)
    cache.k_scale.fill_(2.0 ** (power // 2))
    n = 180 if chunk else 1
    q = torch.zeros(n, nq, D, device=DEV, dtype=torch.bfloat16)
    q[..., 5] = 1.5 * 2.0 ** (power - power // 2)
    got = ops.paged_attention_q8(q, cache, table, _i32([L]), _i32([n]) if chunk else None)
    v = cache.dequantize()[1][int(table[0, 0]), :, 0]                          # [nkv, D], exact in bf16
    assert torch.equal(got.float(), v.repeat_interleave(nq // nkv, 0)[None].expand(n, -1, -1))
    # all but that key at the same score: where it is out of sight, the mean
    cache.k[..., 5] = torch.full_like(codes, 8.0).to(DEV).to(cache.k.dtype)
    got = ops.paged_attention_q8(q, cache, table, _i32([L]), _i32([n]) if chunk else None).cpu().double()
    want, around, _ = oracle.attend(q, cache, table, _i32([L]), _i32([n]) if chunk else None)
    assert ((got - want).abs() <= oracle.attend_bound(want, around, 0.0, L, D, torch.bfloat16)).all()


@pytest.mark.parametrize("D,nkv,bs", [(128, 4, 16), (64, 8, 48), (256, 2, 32), (64, 8, 16)])
@pytest.mark.parametrize("apart", [0, 8, 9, 30])
@pytest.mark.parametrize("lens,news", [([300], [300]), ([130, 400, 77], [130, 100, 70])])
def test_probabilities_on_small_pages(D, nkv, bs, apart, lens, news):
    """Tiles of several pages hold probabilities to 2^-11 or better, whatever their V scales are (2^8 apart: the last
    that fp16 takes; 2^9: the first that it does not)."""
    cache, table = oracle.make_cache(lens, nkv, D, bs, device=DEV)
    if apart:
        cache.v_scale.fill_(2.0 ** -7)
        cache.v_scale[table[:, 1::2].long()] = 2.0 ** (apart - 7)
    g = torch.Generator().manual_seed(1)
    q = (torch.randn(sum(news), 4 * nkv, D, generator=g) * 0.25).bfloat16().to(DEV)
    lens_t, news_t = _i32(lens), _i32(news)
    got = ops.paged_attention_q8(q, cache, table, lens_t, news_t).cpu().double()
    want, around, size = oracle.attend(q, cache, table, lens_t, news_t)
    off, tol = (got - want).abs(), oracle.attend_bound(want, around, size, max(lens), D, torch.bfloat16, 2.0 ** -11)
    assert (off <= tol).all(), f"worst {(off / tol.clamp_min(1e-30)).max():.3g} times the bound"
