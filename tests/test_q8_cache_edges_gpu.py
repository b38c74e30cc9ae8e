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
