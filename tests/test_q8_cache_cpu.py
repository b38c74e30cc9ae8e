"""The paged 8-bit key/value cache and the token statistics on the CPU: their statements against plain 64-bit code, what
they refuse, and the rollout engine on top of them."""
import math

import pytest
import torch

from chatlearn_b200 import ops
from chatlearn_b200.models.nn import CausalLM
from chatlearn_b200.models.nn.arch import PRESETS
from chatlearn_b200.ops import q8
from tests import q8_oracle as oracle


def _i(x):
    return torch.tensor(x, dtype=torch.int32)


# ------------------------------------------------------------------ append
def test_scale_is_the_smallest_power_of_two():
    from chatlearn_b200.ops.reference import q8_scale
    amax = torch.tensor([448.0, 448.5, 449.0, 1.0, 0.875, 1.75, 1.7501, 3.4e38, 1e-30, 0.0])
    s = q8_scale(amax).double()
    assert (torch.frexp(s)[0] == 0.5).all()                              # powers of two
    inside = (amax > 448 * q8.SCALE_MIN) & (amax <= 448 * q8.SCALE_MAX)
    assert (amax.double() <= 448 * s)[inside].all() and (amax.double() > 224 * s)[inside].all()
    assert s[-1] == s[-2] == q8.SCALE_MIN and s[-3] == q8.SCALE_MAX


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,news", [([1, 0, 9, 16], None), ([5, 33, 0, 16], [5, 20, 0, 1])])
def test_append_rounds_once_to_nearest(dtype, lens, news):
    """What stands in the cache afterwards is within half a step of e4m3 (2^-4 of a value, or half of the scale's
    smallest step) of the rows, per page and head; pages that the call does not touch stay as they were."""
    nkv, D, bs = 2, 12, 8
    cache, table = oracle.make_cache(lens, nkv, D, bs, seed=1)
    n = news or [min(1, L) for L in lens]
    rows = len(lens) if news is None else sum(n)
    g = torch.Generator().manual_seed(3)
    k, v = ((torch.randn(rows, nkv, D, generator=g) * 40).to(dtype) for _ in range(2))
    before = [t.clone() for t in cache]
    ops.kv_append_q8(k, v, cache, table, _i(lens), None if news is None else _i(news))
    kk, vv = cache.dequantize()
    touched, at = set(), 0
    for b, (L, m) in enumerate(zip(lens, n)):
        for i in range(m):
            pos = L - m + i
            page = int(table[b, pos // bs])
            touched.add(page)
            row = b if news is None else at + i
            for x, got, s in ((k, kk, cache.k_scale), (v, vv, cache.v_scale)):
                want = x[row].double()
                err = (got[page, :, pos % bs].double() - want).abs()
                assert (err <= torch.maximum(want.abs() * 2.0 ** -4, s[page, :, None].double() * 2.0 ** -10)).all()
        at += m
    for page in range(cache.k.shape[0]):
        if page not in touched:
            for a, b in zip(before, cache):
                assert torch.equal(a[page].view(torch.uint8), b[page].view(torch.uint8))


def test_append_in_one_call_or_token_by_token():
    """A page's scale ends up the same; codes differ only where an intermediate scale rounded them once more."""
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(20, 2, 16, generator=g) * torch.exp2(torch.arange(20.0) / 2)[:, None, None] for _ in range(2))
    table = torch.tensor([[2, 0, 1]])
    once, steps = ops.Q8KVCache.empty(3, 8, 2, 16), ops.Q8KVCache.empty(3, 8, 2, 16)
    ops.kv_append_q8(k, v, once, table, _i([20]), _i([20]))
    for i in range(20):
        ops.kv_append_q8(k[i:i + 1], v[i:i + 1], steps, table, _i([i + 1]))
    assert torch.equal(once.k_scale, steps.k_scale) and torch.equal(once.v_scale, steps.v_scale)
    a, b = once.dequantize()[0], steps.dequantize()[0]
    step = once.k_scale[:, :, None, None] * 2.0 ** -9                    # of the smallest codes under the final scale
    assert ((a - b).abs() <= torch.maximum(a.abs() * 2.0 ** -3, step)).all()


def test_append_starts_over_with_a_page():
    """A page that is handed to another sequence keeps nothing of its old scale."""
    cache = ops.Q8KVCache.empty(1, 8, 1, 4)
    table = torch.tensor([[0]])
    ops.kv_append_q8(torch.full((1, 1, 4), 4e4), torch.full((1, 1, 4), 4e4), cache, table, _i([1]))
    assert float(cache.k_scale) == 128.0
    ops.kv_append_q8(torch.full((1, 1, 4), 0.5), torch.full((1, 1, 4), 0.5), cache, table, _i([1]))
    assert float(cache.k_scale) == 2.0 ** -9 and float(cache.dequantize()[0][0, 0, 0, 0]) == 0.5


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("lens,news", [([1, 0, 9, 30], None), ([5, 33, 0, 16], [5, 20, 0, 1])])
def test_attend_matches_softmax(lens, news):
    nkv, rep, D, bs = 2, 3, 16, 8
    cache, table = oracle.make_cache(lens, nkv, D, bs, seed=2)
    n = news or [min(1, L) for L in lens]
    rows = len(lens) if news is None else sum(n)
    q = torch.randn(rows + 2, nkv * rep, D, dtype=torch.float64)
    got = ops.paged_attention_q8(q, cache, table, _i(lens), None if news is None else _i(news))
    kk, vv = (t.double() for t in cache.dequantize())
    want, at = torch.zeros_like(q), 0
    for b, (L, m) in enumerate(zip(lens, n)):
        ids = table[b, :(L + bs - 1) // bs].long()
        for i in range(m):
            seen = L - m + i + 1
            row = b if news is None else at + i
            for h in range(nkv * rep):
                k = kk[ids, h // rep].reshape(-1, D)[:seen]
                v = vv[ids, h // rep].reshape(-1, D)[:seen]
                want[row, h] = torch.softmax(k @ q[row, h] / math.sqrt(D), 0) @ v
        at += m
    assert (got - want).abs().max() <= 1e-12 * want.abs().max().clamp_min(1)
    assert not got[rows:].any()


def test_bad_pages_are_masked_and_skipped():
    cache, table = oracle.make_cache([20, 20], 1, 8, 8, seed=3)
    q = torch.randn(2, 2, 8, dtype=torch.float64)
    part = table.clone()
    part[0, 1] = -7
    part[1] = 10 ** 6
    got = ops.paged_attention_q8(q, cache, part, _i([20, 20]))
    keep = torch.cat([table[0, :1], table[0, 2:]])[None]
    kk, vv = (t.double() for t in cache.dequantize())
    k = kk[keep[0].long(), 0].reshape(-1, 8)[:12]
    v = vv[keep[0].long(), 0].reshape(-1, 8)[:12]
    want = torch.stack([torch.softmax(k @ q[0, h] / math.sqrt(8), 0) @ v for h in range(2)])
    assert (got[0] - want).abs().max() <= 1e-12 * want.abs().max() and not got[1].any()
    before = [t.clone() for t in cache]
    x = torch.randn(2, 1, 8)
    ops.kv_append_q8(x, x, cache, torch.full_like(table, 10 ** 6), _i([20, 20]))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, cache))


# ------------------------------------------------------------------ token statistics
def test_token_logprobs_statement():
    g = torch.Generator().manual_seed(0)
    z = torch.randn(6, 40, generator=g, dtype=torch.float64)
    z[1] = -math.inf
    z[2, 3:] = -math.inf
    z[3, ::2] = z[3, 0]
    tok = torch.tensor([4, 5, 2, 0, -1, 77])
    out = ops.token_logprobs(z, tok, 5, 0.7)
    for r in range(6):
        if r == 1:
            assert out.logprob[r] == -math.inf and out.entropy[r] == 0 and out.top_ids[r].tolist() == [0, 1, 2, 3, 4]
            continue
        p = torch.softmax(z[r] / 0.7, 0)
        want = sorted(range(40), key=lambda i: (-float(z[r, i]), i))[:5]
        assert out.top_ids[r].tolist() == want
        # a sum of 40 terms of at most 1 in 64 bits
        assert abs(float(out.entropy[r] + (p * p.log().nan_to_num(neginf=0.0)).sum())) < 1e-13
        assert (out.top_logprobs[r] - p.log()[want]).nan_to_num().abs().max() < 1e-13
        assert float(out.logprob[r]) == 0 if r > 3 else abs(float(out.logprob[r] - p.log()[tok[r]])) < 1e-13


def test_token_logprobs_gradient():
    z = torch.randn(4, 9, dtype=torch.float64, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
    tok = torch.tensor([0, 3, -1, 8])
    assert torch.autograd.gradcheck(lambda x: ops.token_logprobs(x, tok, 3, 0.7)[:3], z)
    y = z.detach().clone()
    y[1] = -math.inf
    y[2, 2:] = -math.inf
    y.requires_grad_(True)
    out = ops.token_logprobs(y, tok, 2)
    (out.logprob[[0, 2, 3]].sum() + out.entropy.sum()).backward()
    assert torch.isfinite(y.grad).all() and not y.grad[1].any()


# ------------------------------------------------------------------ refusals
def test_refusals():
    cache, table = oracle.make_cache([20], 2, 8, 8)
    x = torch.randn(1, 2, 8)
    lens = _i([20])
    ok = lambda **kw: {**dict(k=x, v=x, cache=cache, block_tables=table, seq_lens=lens, q_lens=None), **kw}  # noqa: E731
    ops.kv_append_q8(**ok())
    bad = [dict(v=x[:, :1]), dict(k=x[..., :4], v=x[..., :4]), dict(block_tables=table[0]), dict(seq_lens=_i([20, 3])),
           dict(q_lens=_i([1, 1])), dict(k=x[:0], v=x[:0]), dict(cache=cache._replace(k=cache.k[:, :1])),
           dict(cache=cache._replace(k_scale=cache.k_scale.double())), dict(cache=cache._replace(v=cache.v.transpose(2, 3)))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.kv_append_q8(*ok(**kw).values())
    for kw in (dict(k=x.double(), v=x.double()), dict(seq_lens=lens.float())):
        with pytest.raises(TypeError):
            ops.kv_append_q8(*ok(**kw).values())
    q = torch.randn(1, 4, 8)
    for args in ((q[0], cache, table, lens), (q[:, :3], cache, table, lens), (q[..., :4], cache, table, lens),
                 (q, cache, table, _i([1, 2])), (q[:0], cache, table, lens)):
        with pytest.raises(ValueError):
            ops.paged_attention_q8(*args)
    z, tok = torch.randn(3, 10), torch.tensor([1, 2, 3])
    for args in ((z, tok[:2]), (z[0], tok), (z, tok, 11), (z, tok, -1), (z, tok, 2, 0.0), (z, tok, 2, -1.0), (z, tok, 2, math.nan),
                 (z[:, :0], tok)):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args)
    for args in ((z.long(), tok), (z, tok.float())):
        with pytest.raises(TypeError):
            ops.token_logprobs(*args)


# ------------------------------------------------------------------ rollout engine
def _engine(preset="tiny_qwen3", seed=2, **kw):
    from chatlearn_b200.rollout import RolloutEngine
    arch = PRESETS[preset]()
    model = CausalLM(arch, dtype=torch.float32).init_weights(seed)
    args = dict(block_size=8, num_blocks=128, max_num_seqs=16, max_model_len=128)
    return arch, RolloutEngine(model, **{**args, **kw})


def _prompts(arch, lens, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, arch.vocab_size - 1, (n,), generator=g).tolist() for n in lens]


def test_engine_on_an_8_bit_cache():
    """Steps with and without the captured step's host side (padded rows, tables kept on the device), with preemptions and
    shared prompts: the same greedy tokens, and half of the cache's memory."""
    from chatlearn_b200.rollout import SamplingParams
    sp = SamplingParams(temperature=0.0, max_tokens=14, ignore_eos=True, logprobs=3)
    outs = []
    for graphs, blocks in ((False, 128), ("emulate", 128), ("emulate", 20)):
        arch, eng = _engine(use_cuda_graphs=graphs, num_blocks=blocks, kv_dtype=torch.float8_e4m3fn)
        prompts = _prompts(arch, (37, 16, 9))
        seqs = eng.generate([p for p in prompts for _ in range(2)], sp)
        outs.append([s.output for s in seqs])
        if blocks == 128:
            assert all(len(s.top_logprobs) == len(s.entropies) == 14 and len(s.top_logprobs[0]) == 3 for s in seqs)
            assert all(t[0][0] == tok for s in seqs for tok, t in zip(s.output, s.top_logprobs))        # greedy
            assert eng.q8_cache and all(c.k.dtype == torch.float8_e4m3fn for c in eng.q8_cache)
        wide = _engine(num_blocks=blocks)[1]
        assert eng.kv_bytes_per_block() * 3.5 < wide.kv_bytes_per_block()          # fp32 model: a quarter, and the scales
    assert outs[0] == outs[1]
    # a sequence that was preempted comes back through prefill, whose attention sees its keys unrounded
    assert sum(a[:4] == b[:4] for a, b in zip(outs[0], outs[2])) >= 4


def test_engine_hands_back_alternatives():
    """Alternatives and entropies of an exact cache against scoring the whole sequence."""
    from chatlearn_b200.models.nn import packed_ctx
    from chatlearn_b200.rollout import SamplingParams
    for graphs in (False, "emulate"):
        arch, eng = _engine(use_cuda_graphs=graphs)
        prompts = _prompts(arch, (11, 30))
        sps = [SamplingParams(temperature=0.7, max_tokens=6, ignore_eos=True, logprobs=n) for n in (4, 0)]
        got = eng.generate(prompts, sps)
        assert not got[1].top_logprobs and not got[1].entropies and len(got[1].logprobs) == 6
        s = got[0]
        toks = torch.tensor(s.prompt + s.output)
        ctx, _ = packed_ctx([toks.numel()], "cpu")
        with torch.no_grad():
            hidden = eng.model.hidden_states(toks, ctx)
            z = torch.nn.functional.linear(hidden, eng.model.lm_head_weight()).double()[len(s.prompt) - 1:-1]
        want = ops.token_logprobs(z, toks[len(s.prompt):], 4, 0.7)
        # fp32 logits of a two-layer model, steps against one pass: 1e-4 is over 2^9 roundings of values near 1
        assert (torch.tensor(s.logprobs) - want.logprob).abs().max() < 1e-4
        assert (torch.tensor(s.entropies) - want.entropy).abs().max() < 1e-4
        assert [[i for i, _ in t] for t in s.top_logprobs] == want.top_ids.tolist()
        assert (torch.tensor([[l for _, l in t] for t in s.top_logprobs]) - want.top_logprobs).abs().max() < 1e-4


def test_refuses_empty_caches_wide_tables_and_far_temperatures():
    x, lens = torch.randn(1, 2, 16), _i([20])
    with pytest.raises(ValueError, match="without pages"):
        ops.paged_attention_q8(x, ops.Q8KVCache.empty(0, 16, 2, 16), _i([[0, 1]]), lens)
    with pytest.raises(ValueError, match="tokens and more"):
        ops.paged_attention_q8(x, ops.Q8KVCache.empty(1, 1024, 2, 16), _i([[0]]).expand(1, 2 ** 20), lens)
    for t in (0.0, -1.0, 1e-31, 1e31, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_logprobs(torch.randn(2, 5), torch.tensor([0, 1]), 2, t)


def test_engine_refuses():
    from chatlearn_b200.rollout import RolloutEngine, SamplingParams
    with pytest.raises(ValueError, match="latent"):
        RolloutEngine(CausalLM(PRESETS["tiny_mla_moe"](), dtype=torch.float32), kv_dtype=torch.float8_e4m3fn)
    _, eng = _engine()
    with pytest.raises(ValueError, match="logprobs"):
        eng.generate([[1, 2, 3]], SamplingParams(logprobs=65))


def test_config_keys():
    from chatlearn_b200.configs.policy_config import PolicyConfig
    c = PolicyConfig()
    assert c.kv_cache_dtype == "auto" and c.num_logprobs == 0
    c.kv_cache_dtype, c.num_gpu = "int4", 1
    with pytest.raises(AssertionError, match="kv_cache_dtype"):
        c._validate_impl()
