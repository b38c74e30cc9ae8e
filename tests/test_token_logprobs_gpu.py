"""Token log-probabilities, entropies and alternatives on a GPU against their 64-bit statement."""
import math

import pytest
import torch

from chatlearn_b200 import ops
from chatlearn_b200.ops import reference as ref
from tests import q8_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _close(got, want, tol):
    got, want = got.detach().cpu().double(), want.detach().double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    worst = float((off / tol).detach().max()) if off.numel() else 0.0
    assert not worst > 1, f"worst {worst:.3g} times the bound"


def _check(z, tok, n, temp, grad=True, which=(0, 1, 2)):
    """Forward and gradient of logits `z` (a view on the GPU) against 64 bits."""
    leaf = z.detach().requires_grad_(grad)
    got = ops.token_logprobs(leaf, tok, n, temp)
    wide = z.detach().cpu().double().requires_grad_(grad)
    want = ref.token_logprobs(wide, tok.cpu(), n, temp)
    tol = oracle.statistics_bound(z.cpu(), temp, None)
    lp_tol = oracle.statistics_bound(z.cpu(), temp, want.logprob.detach())
    assert torch.equal(got.top_ids.cpu(), want.top_ids)
    _close(got.logprob, want.logprob, lp_tol)
    _close(got.top_logprobs, want.top_logprobs, tol[:, None] + 2.0 ** -22 * torch.where(want.top_logprobs.isfinite(), want.top_logprobs.abs(), 0.0))
    _close(got.entropy, want.entropy, 2 * tol * (1 + want.entropy.detach()))
    if not grad:
        return
    g = torch.Generator().manual_seed(5)
    R = z.shape[0]
    gs = [torch.randn(R, generator=g), torch.randn(R, generator=g), torch.randn(R, n, generator=g)]
    pick = [i for i in which if i < 2 or n > 0]
    dz, = torch.autograd.grad([got[i] for i in pick], leaf, [gs[i].to(DEV) for i in pick])
    ref_dz, = torch.autograd.grad([want[i] for i in pick], wide, [gs[i].double() for i in pick])
    assert dz.shape == z.shape and dz.dtype == z.dtype
    # p has the relative error of a log-probability; p (ln p + H) both
    with torch.no_grad():
        empty = (wide == -math.inf).all(1)
        zz = torch.where(empty[:, None], torch.zeros_like(wide), wide) / temp
        logp = torch.log_softmax(zz, -1)
        p = logp.exp()
        G = sum(gs[i].double().abs() if i == 0 else gs[i].double().abs().sum(-1) for i in pick if i != 1) + torch.zeros(R, dtype=torch.float64)
        ge = gs[1].double().abs() if 1 in pick else torch.zeros(R, dtype=torch.float64)
        factor = G[:, None] + ge[:, None] * (logp.clamp_min(-800).abs() + want.entropy[:, None] + 2)
        # a probability below 2^-126 is no normal fp32 number and flushed to 0: all of it is lost, times the same factor
        # (at temperature 0.01 that is 2^-126 * 200 * 100 = 2e-34, far above the smallest bf16)
        lost = torch.where(p < 2.0 ** -125, p, 0.0)
        bound = ((4 * tol[:, None] + 2.0 ** -22) * p + lost) * factor / temp + 2.0 ** -22 * ref_dz.abs() + 1e-36
    half = oracle.HALF_STEP[z.dtype]
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[z.dtype]
    _close(dz, ref_dz, bound * (1 + half) + half * ref_dz.abs() + tiny)


def _tokens(R, V, seed=0):
    return torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V,n,temp", [(1, 1, 1, 1.0), (3, 7, 7, 0.5), (5, 1000, 0, 1.0), (2, 32001, 20, 0.8), (130, 4099, 5, 1.0),
                                        (300, 2048, 64, 1.7), (1, 151936, 64, 1.0), (40, 50000, 8, 0.01)])
def test_matches(dtype, R, V, n, temp):
    g = torch.Generator().manual_seed(R * 31 + V)
    z = (torch.randn(R, V, generator=g) * 3).to(dtype).to(DEV)
    _check(z, _tokens(R, V), n, temp)


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2)])
def test_partial_gradients(which):
    z = torch.randn(9, 3001, device=DEV) * 2
    _check(z, _tokens(9, 3001), 6, 1.1, which=which)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off,pad", [(0, 63), (1, 0), (3, 6), (0, 1)])
def test_strided_rows(dtype, off, pad):
    V = 5003
    base = (torch.randn(17, off + V + pad, generator=torch.Generator().manual_seed(1)) * 3).to(dtype).to(DEV)
    _check(base[:, off:off + V], _tokens(17, V), 9, 1.0)


def test_expanded_and_transposed_logits():
    row = torch.randn(1, 777, device=DEV)
    _check(row.expand(5, 777), _tokens(5, 777), 4, 1.0)
    _check(torch.randn(777, 6, device=DEV).t(), _tokens(6, 777), 4, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 8, 33, 64])
def test_ties_go_to_the_lowest_index(dtype, n):
    V = 40001
    g = torch.Generator().manual_seed(2)
    z = torch.randint(-3, 4, (6, V), generator=g).to(dtype)
    z[1] = 0.0                                                   # all equal
    z[2] = torch.arange(V).flip(0).to(dtype)                     # falling
    z[3] = torch.arange(V).to(dtype)                             # rising (bf16: long stretches of equal values)
    z[4, ::2] = -0.0
    z[5] = torch.randn(V, generator=g).sort().values.to(dtype) * 1e-3
    _check(z.to(DEV), _tokens(6, V), n, 1.0, grad=False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n", [0, 3, 64])
def test_masked_rows(dtype, n):
    V = 9001
    g = torch.Generator().manual_seed(4)
    z = (torch.randn(8, V, generator=g) * 3).to(dtype)
    z[0] = -math.inf
    z[1, 1:] = -math.inf
    z[2, :-1] = -math.inf
    z[3, torch.rand(V, generator=g) < 0.999] = -math.inf
    z[4] = torch.finfo(dtype).min
    z[5, 5:] = torch.finfo(dtype).min
    tok = torch.tensor([3, 0, 5, 7, 9, 2, -1, V + 5], device=DEV)
    _check(z.to(DEV), tok, n, 1.0, grad=False)
    keep = [0, 1, 2, 3, 6, 7]
    _check(z[keep].to(DEV), tok[keep], n, 0.9)


def test_nan_and_infinite_logits_stay_in_their_rows():
    z = torch.randn(4, 3000, device=DEV)
    z[1, 17] = math.nan
    z[2, 18] = math.inf
    out = ops.token_logprobs(z, _tokens(4, 3000), 5)
    for t in (out.logprob, out.entropy, out.top_logprobs.sum(-1)):
        assert t.isnan().tolist() == [False, True, True, False]
    assert 17 not in out.top_ids[1].tolist() and out.top_ids[2, 0] == 18


def test_peaked_rows_keep_their_precision():
    """Entropy and log-probability near 0 are not differences of large numbers."""
    z = torch.zeros(3, 50000, device=DEV)
    z[0, 7] = 40.0
    z[1, 7] = 25.0
    z[2] += 1000.0
    z[2, 9] = 1030.0
    tok = torch.tensor([7, 7, 9], device=DEV)
    got = ops.token_logprobs(z, tok, 2)
    want = ref.token_logprobs(z.cpu().double(), tok.cpu(), 2)
    # S is near 1 and rounded at every join on its way (5 of a warp, 15 of a block, 3 of a cluster, 1 for the logarithm):
    # 24 times 2^-24; a sum of logits near 1000 taken as it is would be off by 2^-15
    for a, b in ((got.logprob, want.logprob), (got.entropy, want.entropy)):
        assert ((a.cpu() - b).abs() <= 24 * 2.0 ** -24 * (1 + b.abs())).all()


def test_deterministic_and_captured():
    """Equal on every run, inside a graph too, forward and gradient.  (Nothing of an eager pass over the same leaf is alive
    while its gradient is captured: autograd would join the capture with the eager pass's stream.)"""
    z = (torch.randn(33, 20011, device=DEV) * 3).requires_grad_(True)
    tok = _tokens(33, 20011)
    g = torch.randn(33, device=DEV)

    def step():
        out = ops.token_logprobs(z, tok, 7)
        dz, = torch.autograd.grad((out.logprob * g + out.entropy).sum() + out.top_logprobs.sum(), z)
        return [t.detach() for t in out] + [dz]
    a = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = step()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_gradient_against_differences():
    z = (torch.randn(2, 50, device=DEV, generator=torch.Generator(DEV).manual_seed(0)) * 2).requires_grad_(True)
    tok = torch.tensor([3, 44], device=DEV)
    w = torch.tensor([0.3, -1.2, 0.7, 0.2], device=DEV)

    def f(x):
        o = ops.token_logprobs(x, tok, 4, 0.9)
        return (o.logprob.sum() + 0.5 * o.entropy.sum() + (o.top_logprobs * w).sum())
    dz, = torch.autograd.grad(f(z), z)
    step = 2.0 ** -6
    for r, c in ((0, 3), (0, 10), (1, 44), (1, 7)):
        d = torch.zeros_like(z)
        d[r, c] = step
        with torch.no_grad():
            slope = (f(z + d) - f(z - d)) / (2 * step)
        # central difference: third derivative (below 8 / temperature^3 for these sums) step^2 / 6, and fp32 noise of f over the step
        assert abs(float(slope - dz[r, c])) <= 8 / 0.9 ** 3 * step ** 2 / 6 + 64 * 2.0 ** -23 * abs(float(f(z))) / step


def test_refusals_on_the_gpu():
    z = torch.randn(2, 100, device=DEV)
    tok = _tokens(2, 100)
    with pytest.raises(ValueError, match="at most 64"):
        ops.token_logprobs(z, tok, 65)
    with pytest.raises(TypeError, match="logits"):
        ops.token_logprobs(z.double(), tok)
    with pytest.raises(ValueError, match="one device"):
        ops.token_logprobs(z, tok.cpu())
    out = ops.token_logprobs(z[:0], tok[:0], 3)
    assert out.logprob.shape == (0,) and out.top_ids.shape == (0, 3)
