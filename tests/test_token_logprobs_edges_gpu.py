"""Token statistics on a GPU at the places where blocks, vectors and lists of candidates end."""
import math

import pytest
import torch

from chatlearn_b200 import ops
from chatlearn_b200.ops import reference as ref
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V", [(1, 151936), (3, 40001), (3, 997), (400, 4099), (310, 100003)])
@pytest.mark.parametrize("n", [1, 8, 64])
def test_nan_ranks_as_minus_infinity(dtype, R, V, n):
    """Rows of nothing but NaN, and rows with fewer other logits than alternatives: ids as the statement has them, with
    a cluster to a row and with one block."""
    g = torch.Generator().manual_seed(R + V)
    z = (torch.randn(R, V, generator=g) * 2).to(dtype)
    rows = [z[r] for r in (0, R // 2, R - 1)]
    rows[0].fill_(math.nan)
    if R > 1:
        rows[1][3:].fill_(math.nan)                                  # three ordinary logits, at the front
        rows[2].fill_(math.nan)
        rows[2][[V // 3, V - 1]] = torch.tensor([1.0, 2.0], dtype=dtype)
    if R > 3:
        z[1, :V // 2] = math.nan                                     # half a row
        z[2, ::2] = math.nan                                         # every other one
        z[3] = -math.inf
        z[3, V // 2:] = math.nan                                     # equal ranks: by index
    tok = torch.randint(0, V, (R,), generator=g)
    got = ops.token_logprobs(z.to(DEV), tok.to(DEV), n)
    want = ref.token_logprobs(z, tok, n)
    assert torch.equal(got.top_ids.cpu(), want.top_ids)
    nan = z.isnan().any(1)
    assert got.logprob.cpu()[nan].isnan().all() and got.entropy.cpu()[nan].isnan().all() and got.top_logprobs.cpu()[nan].isnan().all()
    assert torch.isfinite(got.logprob.cpu()[~nan]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V", [(400, 8000), (4, 8000), (4, 60001), (400, 60001)])
def test_equal_logits_beside_nan(dtype, R, V):
    """Thousands of logits reach the n-th largest, and whole stretches between them are NaN."""
    z = torch.zeros(R, V, dtype=dtype)
    z[0, :V // 4] = math.nan
    z[1, 600:2700] = math.nan
    z[1, V - 5] = 3.0
    z[2, 1:] = math.nan
    z[3] = math.nan
    tok = torch.zeros(R, dtype=torch.long)
    for n in (2, 64):
        got, want = ops.token_logprobs(z.to(DEV), tok.to(DEV), n), ref.token_logprobs(z, tok, n)
        assert torch.equal(got.top_ids.cpu(), want.top_ids)


@pytest.mark.parametrize("which", ["logprob", "entropy", "top_logprobs"])
def test_second_derivatives_are_refused(which):
    """A gradient whose graph is asked for is no constant, with constant incoming gradients either."""
    z = torch.randn(3, 500, device=DEV, requires_grad=True)
    w = torch.randn(3, 500, device=DEV, requires_grad=True)
    tok = torch.tensor([1, 2, 3], device=DEV)
    plain, = torch.autograd.grad(getattr(ops.token_logprobs(z, tok, 4), which).sum(), z)
    dz, = torch.autograd.grad(getattr(ops.token_logprobs(z, tok, 4), which).sum(), z, create_graph=True)
    assert torch.equal(dz, plain) and dz.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        (dz.square().sum() + w.sum()).backward()
    # incoming gradients that need one themselves
    weight = torch.ones(3, device=DEV, requires_grad=True)
    dz, = torch.autograd.grad((ops.token_logprobs(z, tok, 4).logprob * weight).sum(), z, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dz.sum().backward()
    # a graph of what lies in front of the operator stays open
    loss = ops.token_logprobs(w * w, tok, 4).logprob.sum()
    first, = torch.autograd.grad(loss, w, create_graph=True)
    assert first.shape == w.shape


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """A tangent on the logits is not dropped."""
    import torch.autograd.forward_ad as fwad
    z, tok = torch.randn(3, 500, device=DEV), torch.tensor([1, 2, 3], device=DEV)
    with fwad.dual_level():
        dual = fwad.make_dual(z.requires_grad_(grad), torch.ones_like(z))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.token_logprobs(dual, tok, 4)
        with pytest.raises(RuntimeError, match="forward-mode"), torch.no_grad():
            ops.token_logprobs(dual, tok, 4)
        ops.token_logprobs(z.detach(), tok, 4)
    assert ops.token_logprobs(z, tok, 4).logprob.requires_grad == grad
