"""Token statistics on a GPU at the places where blocks, vectors and lists of candidates end."""
import pytest
import torch

from chatlearn_b200 import ops
from tests.test_token_logprobs_gpu import _check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [4097, 4098, 8193, 8195, 8199, 32769, 49153, 49155])
@pytest.mark.parametrize("pad", [0, 1, 3, 6])
def test_gradient_of_the_last_columns(dtype, V, pad):
    """Vocabularies a little longer than a whole number of a block's stretches (4,096 fp32 or 8,192 16-bit logits), rows that
    begin anywhere inside 16 bytes: the tokens and their alternatives are the last columns, behind the last whole vector."""
    R = 17
    g = torch.Generator().manual_seed(V + pad)
    z = (torch.randn(R, V + pad, generator=g) * 2).to(dtype)
    z[:, V - 9:V] += 6
    tok = V - 1 - torch.arange(R) % 9
    rows, tok = z.to(DEV)[:, :V], tok.to(DEV)
    _check(rows, tok, 6, 1.0)
    leaf = rows.detach().requires_grad_(True)
    first = None
    for _ in range(20):
        out = ops.token_logprobs(leaf, tok, 6)
        dz, = torch.autograd.grad(out.logprob.sum() + out.top_logprobs.sum(), leaf)
        first = dz if first is None else first
        assert torch.equal(dz, first)
