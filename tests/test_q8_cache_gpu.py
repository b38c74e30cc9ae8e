"""The paged 8-bit key/value cache on a GPU against its 64-bit statements."""
import pytest
import torch

from chatlearn_b200 import ops
from chatlearn_b200.ops import reference as ref
from tests import q8_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _check_append(dtype, lens, news, nkv, D, bs, seed=0, tweak=None, rows=None, layout="qkv", gain=1.0):
    new = news if news is not None else [min(1, L) for L in lens]
    cache, table = oracle.make_cache(lens, nkv, D, bs, seed, device=DEV)
    T = (sum(new) if news is not None else len(lens)) if rows is None else rows
    g = torch.Generator().manual_seed(seed + 1)
    if layout == "qkv":                       # views of the projection's rows: keys and values beside the queries
        base = (torch.randn(T, 4 * nkv, D, generator=g) * gain).to(dtype).to(DEV)
        k, v = base[:, 2 * nkv:3 * nkv], base[:, 3 * nkv:]
    elif layout == "heads":                   # head-major storage
        k, v = ((torch.randn(nkv, T, D, generator=g) * gain).to(dtype).to(DEV).transpose(0, 1) for _ in range(2))
    else:                                     # odd strides: rows do not start at 16 bytes
        base = (torch.randn(T, 2 * nkv * D + 3, generator=g) * gain).to(dtype).to(DEV)
        k, v = (base[:, 1 + i * nkv * D:1 + (i + 1) * nkv * D].unflatten(1, (nkv, D)) for i in range(2))
    if tweak is not None:
        k, v = tweak(k), tweak(v)
    want = oracle.cpu(cache)
    ref.kv_append_q8(k.cpu(), v.cpu(), want, table.cpu(), torch.tensor(lens), None if news is None else torch.tensor(news))
    ops.kv_append_q8(k, v, cache, table, _i32(lens), None if news is None else _i32(news))
    got = oracle.cpu(cache)
    for name in ("k_scale", "v_scale"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    for name in ("k", "v"):
        a, b = getattr(got, name).float(), getattr(want, name).float()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0), b.nan_to_num(nan=0.0)), name
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,news,nkv,D,bs", [
    ([1], None, 1, 64, 16),
    ([1, 0, 64, 65, 128, 2000], None, 8, 128, 64),
    ([17, 33, 16], None, 2, 256, 32),
    ([5], [5], 1, 128, 64),
    ([64, 65, 1, 0, 130], [64, 1, 1, 0, 130], 4, 128, 64),
    ([40, 333, 7, 100, 31], [37, 0, 7, 12, 1], 3, 64, 16),
    ([300, 129], [200, 3], 2, 256, 128),
])
def test_append_matches(dtype, lens, news, nkv, D, bs):
    _check_append(dtype, lens, news, nkv, D, bs)


@pytest.mark.parametrize("layout", ["heads", "odd"])
@pytest.mark.parametrize("news", [None, [3, 20, 1]])
def test_append_strides(layout, news):
    _check_append(torch.bfloat16, [5, 70, 64], news, 2, 128, 64, layout=layout)


@pytest.mark.parametrize("gain", [1e-12, 1e-4, 300.0, 1e9])
@pytest.mark.parametrize("news", [None, [9, 30, 2]])
def test_append_grows_the_scale(gain, news):
    """Rows far larger or smaller than what the page holds: older codes are rounded again under the grown scale."""
    _check_append(torch.float32, [20, 60, 130], news, 2, 64, 32, gain=gain)


def test_append_zeros_infinities_and_nan():
    def tweak(x):
        x = x.clone()
        x[0] = 0.0
        x[1, 0, 3] = float("inf")
        x[1, 1, 5] = -float("inf")
        x[2, 0, 7] = float("nan")
        return x
    _check_append(torch.bfloat16, [16, 20, 3], None, 2, 64, 16, tweak=tweak)
    _check_append(torch.bfloat16, [16, 20, 3], [16, 1, 3], 2, 64, 16, tweak=tweak)


def test_append_ignores_rows_behind_the_last_sequence_and_bad_pages():
    _check_append(torch.bfloat16, [5, 70], [5, 9], 2, 64, 16, rows=40)
    _check_append(torch.bfloat16, [5, 70], None, 2, 64, 16, rows=9)
    for news in (None, [3, 4]):
        cache, table = oracle.make_cache([20, 20], 2, 64, 16, device=DEV)
        table[0] = -1
        table[1] = cache.k.shape[0]
        before = [t.clone() for t in cache]
        x = torch.randn(7, 2, 64, device=DEV, dtype=torch.bfloat16)
        ops.kv_append_q8(x, x, cache, table, _i32([20, 20]), None if news is None else _i32(news))
        for a, b in zip(before, cache):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def _check_attend(dtype, lens, news, nq, nkv, D, bs, seed=0, scale=None, gain=1.0, tweak=None, rows=None, width=None):
    cache, table = oracle.make_cache(lens, nkv, D, bs, seed, device=DEV, width=width)
    if tweak is not None:
        tweak(cache, table)
    T = rows or (len(lens) if news is None else sum(news))
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(T, nq, D, generator=g) * gain).to(dtype).to(DEV)
    lens_t, news_t = _i32(lens), None if news is None else _i32(news)
    got = ops.paged_attention_q8(q, cache, table, lens_t, news_t, scale).cpu().double()
    want, around, size = oracle.attend(q, cache, table, lens_t, news_t, scale)
    wide = news is not None and dtype == torch.bfloat16 and max(news) >= 8 and bs % 64 != 0
    tol = oracle.attend_bound(want, around, size, max(lens), D, dtype, 2.0 ** -8 if wide else 2.0 ** -11)
    bad = (got - want).abs() > tol
    assert not bad.any() and torch.isfinite(got).all(), \
        f"{int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol.clamp_min(1e-30)).max():.3g} times the bound"
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq,nkv,D,bs", [(32, 8, 128, 64), (4, 4, 64, 16), (16, 2, 256, 32), (7, 1, 128, 128), (40, 1, 64, 48), (34, 2, 128, 16)])
@pytest.mark.parametrize("lens", [[1], [16, 0, 17, 63, 64, 65, 128, 1], [1500, 3, 777]])
def test_attend_one_token(dtype, nq, nkv, D, bs, lens):
    _check_attend(dtype, lens, None, nq, nkv, D, bs)


def test_attend_many_sequences():
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 400, (700,), generator=g).tolist()
    _check_attend(torch.bfloat16, lens, None, 8, 2, 128, 64)


def test_attend_long_context():
    _check_attend(torch.bfloat16, [40000, 1], None, 8, 2, 128, 64)


@pytest.mark.parametrize("nq,nkv,D,bs", [(32, 8, 128, 64), (4, 4, 64, 16), (16, 2, 256, 32), (40, 1, 64, 48)])
@pytest.mark.parametrize("lens,news", [([100, 33, 7, 64, 90], [10, 0, 7, 1, 64]), ([300], [130]), ([70, 0, 1], [70, 0, 1]), ([3, 80], [5, 2])])
def test_attend_chunks(nq, nkv, D, bs, lens, news):
    _check_attend(torch.bfloat16, lens, news, nq, nkv, D, bs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nq,nkv,D,bs", [(8, 2, 128, 64), (7, 1, 64, 48), (4, 4, 128, 16), (16, 1, 256, 128), (34, 1, 64, 64), (6, 2, 256, 80)])
@pytest.mark.parametrize("lens,news", [([700, 8, 9, 129, 64], [300, 8, 7, 128, 33]), ([1000], [1000]), ([2000, 40], [65, 40])])
def test_attend_long_chunks(dtype, nq, nkv, D, bs, lens, news):
    """Sequences on both sides of the length from which tiles of tokens are taken, and of the tiles' own bounds."""
    _check_attend(dtype, lens, news, nq, nkv, D, bs)
    from chatlearn_b200.ops import native
    assert native.C.paged_attention_q8_last_status() == 0


@pytest.mark.parametrize("bs", [32, 64])
def test_attend_chunks_far_apart_scales_and_bad_pages(bs):
    def tweak(cache, table):
        cache.v_scale[table[:, 0].long()] = 2.0 ** 12
        cache.v_scale[table[:, 1].long()] = 2.0 ** -20
        cache.v_scale[table[:, 2].long()] = 0.0
        cache.k_scale[table[:, 3].long()] = 2.0 ** -24
        table[0, 4] = -1
        table[1, 5] = cache.k.shape[0]
    _check_attend(torch.bfloat16, [64 * 6 + 3, 64 * 6], [200, 64 * 6], 8, 2, 128, bs, tweak=tweak, gain=4.0)
    _check_attend(torch.bfloat16, [64 * 6 + 3, 64 * 6], [200, 64 * 6], 8, 2, 128, bs, tweak=tweak, gain=0.0)
    _check_attend(torch.bfloat16, [64 * 6 + 3, 64 * 6], [200, 64 * 6], 8, 2, 128, bs, tweak=tweak, scale=-0.05)


def test_attend_chunks_short_tables_and_rows():
    """More new tokens than the sequence has, than the table has pages for, and than there are rows."""
    got = _check_attend(torch.bfloat16, [30, 100], [60, 20], 4, 2, 64, 16)
    assert not got[:30].any()
    _check_attend(torch.bfloat16, [100, 40], [90, 40], 4, 2, 64, 16, rows=70)
    cache, table = oracle.make_cache([200, 90], 2, 64, 16, device=DEV)
    q = torch.randn(290, 4, 64, device=DEV, dtype=torch.bfloat16)
    lens = _i32([200, 90])
    got = ops.paged_attention_q8(q, cache, table[:, :4].contiguous(), lens, lens).cpu().double()
    want, around, size = oracle.attend(q, cache, table[:, :4].contiguous(), lens, lens)
    assert ((got - want).abs() <= oracle.attend_bound(want, around, size, 200, 64, torch.bfloat16, 2.0 ** -8)).all()


@pytest.mark.parametrize("nq,nkv,D,bs", [(32, 8, 128, 64), (8, 8, 64, 64), (16, 8, 256, 64), (200, 2, 64, 64), (128, 1, 128, 128), (130, 2, 256, 64)])
@pytest.mark.parametrize("most", [3, 7, 40, 150])
def test_attend_many_chunks(nq, nkv, D, bs, most):
    """New tokens from none to `most` in each of 60 sequences: rows, tiles of one group of rows and of two side by side."""
    g = torch.Generator().manual_seed(most)
    news = torch.randint(0, most + 1, (60,), generator=g).tolist()
    news[7], news[31] = most, 0
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 190, (60,), generator=g))]
    _check_attend(torch.bfloat16, lens, news, nq, nkv, D, bs)
    from chatlearn_b200.ops import native
    assert native.C.paged_attention_q8_last_status() == 0


@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("D,nkv", [(128, 4), (64, 8), (256, 2)])
def test_attend_chunks_at_their_bounds(bs, D, nkv):
    """Tiles whose sequence is shorter than its new tokens, has no key, no page, or fewer rows than tokens."""
    got = _check_attend(torch.bfloat16, [30, 0, 100, 300], [160, 20, 20, 130], 4 * nkv, nkv, D, bs)
    assert not got[:130].any() and not got[160:180].any()
    _check_attend(torch.bfloat16, [300, 140], [290, 140], 4 * nkv, nkv, D, bs, rows=270)
    got = _check_attend(torch.bfloat16, [300, 140], [20, 140], 4 * nkv, nkv, D, bs, rows=400)
    assert not got[160:].any()

    def tweak(cache, table):
        table[0] = -1
        table[1, 0] = cache.k.shape[0]
        table[1, -1] = 1 << 30
    got = _check_attend(torch.bfloat16, [200, 333], [150, 230], 4 * nkv, nkv, D, bs, tweak=tweak)
    assert not got[:150].any()


def test_attend_rows_behind_the_last_sequence_are_zero():
    got = _check_attend(torch.bfloat16, [30, 50], None, 4, 2, 64, 16, rows=9)
    assert not got[2:].any()
    got = _check_attend(torch.bfloat16, [30, 50], [3, 4], 4, 2, 64, 16, rows=20)
    assert not got[7:].any()


def test_attend_masks_bad_pages():
    def tweak(cache, table):
        table[0, 1] = -5
        table[1, 0] = cache.k.shape[0]
        table[2] = 1 << 30
    for news in (None, [2, 3, 4]):
        got = _check_attend(torch.bfloat16, [60, 40, 33], news, 4, 2, 64, 16, tweak=tweak)
        assert not got[-1].any()


def test_attend_far_apart_scales():
    """Pages whose values differ by powers of two of 20 and more, with queries that pick either."""
    def tweak(cache, table):
        cache.v_scale[table[:, 0].long()] = 2.0 ** 12
        cache.v_scale[table[:, 1].long()] = 2.0 ** -20
        cache.v_scale[table[:, 2].long()] = 0.0
        cache.k_scale[table[:, 3].long()] = 2.0 ** -24
    _check_attend(torch.bfloat16, [64 * 5 + 3, 64 * 4], None, 8, 2, 128, 64, tweak=tweak, gain=4.0)


@pytest.mark.parametrize("gain,scale", [(1e-6, None), (1e6, 1e-6), (3e4, 1e-5), (0.0, None), (1.0, 0.0)])
def test_attend_query_ranges(gain, scale):
    _check_attend(torch.bfloat16, [300, 5], None, 8, 2, 128, 64, gain=gain, scale=scale)


def test_attend_nan_key_reaches_only_its_rows():
    cache, table = oracle.make_cache([80, 80], 2, 64, 16, device=DEV)
    cache.k.view(torch.uint8)[int(table[0, 1]), 0, 3, 5] = 0x7f
    q = torch.randn(2, 4, 64, device=DEV, dtype=torch.bfloat16)
    got = ops.paged_attention_q8(q, cache, table, _i32([80, 80]))
    assert got[0, :2].isnan().all() and not got[0, 2:].isnan().any() and not got[1].isnan().any()


@pytest.mark.parametrize("nq,nkv,D,bs", [(32, 8, 128, 64), (8, 4, 64, 16), (16, 4, 256, 32), (32, 4, 64, 128), (16, 4, 128, 48)])
@pytest.mark.parametrize("news", [None, [5, 0, 130, 64, 2], [300, 9, 1, 40, 3]])
def test_attend_never_reads_what_no_row_sees(nq, nkv, D, bs, news):
    """NaN codes in every slot behind the lengths and in every page without tokens, NaN scales where there are no tokens."""
    lens = [321, 9, 130, 64, 3]

    def tweak(cache, table):
        used = torch.zeros(cache.k.shape[0], bs, dtype=torch.bool)
        for b, L in enumerate(lens):
            for t in range(L):
                used[int(table[b, t // bs]), t % bs] = True
        for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            codes.view(torch.uint8).masked_fill_(~used[:, None, :, None].to(DEV), 0x7f)
            scale.masked_fill_(~used.any(1)[:, None].to(DEV), float("nan"))
    _check_attend(torch.bfloat16, lens, news, nq, nkv, D, bs, tweak=tweak, width=-(-321 // bs) + 2)


def test_attend_two_streams_and_a_graph():
    """Two calls at once on two streams, and a captured call beside an eager one: nothing is shared between them."""
    cache, table = oracle.make_cache([500, 300], 4, 128, 64, device=DEV)
    lens, news = _i32([500, 300]), _i32([200, 100])
    q = torch.randn(300, 16, 128, device=DEV, dtype=torch.bfloat16)
    want_rows, want = ops.paged_attention_q8(q[:2], cache, table, lens), ops.paged_attention_q8(q, cache, table, lens, news)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for s, out, n in zip(streams, got, (None, news)):
            with torch.cuda.stream(s):
                out.append(ops.paged_attention_q8(q[:2] if n is None else q, cache, table, lens, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want_rows) for x in got[0]) and all(torch.equal(x, want) for x in got[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = ops.paged_attention_q8(q[:2], cache, table, lens), ops.paged_attention_q8(q, cache, table, lens, news)
    for _ in range(3):
        a.fill_(7), b.fill_(7)
        graph.replay()
        assert torch.equal(ops.paged_attention_q8(q, cache, table, lens, news), want)
        torch.cuda.synchronize()
        assert torch.equal(a, want_rows) and torch.equal(b, want)


def test_attend_is_deterministic_and_takes_strided_queries():
    cache, table = oracle.make_cache([3000, 10, 900], 2, 128, 64, device=DEV)
    base = torch.randn(3, 3, 8, 128, device=DEV, dtype=torch.bfloat16)
    lens = _i32([3000, 10, 900])
    a = ops.paged_attention_q8(base[:, 1], cache, table, lens)
    for _ in range(5):
        assert torch.equal(a, ops.paged_attention_q8(base[:, 1].contiguous(), cache, table.long(), lens.long()))


def test_graphs_and_streams():
    """Two captured graphs of the pair replay with new lengths and rows, in turn and on streams of their own."""
    lens0 = [5, 100, 64, 0]
    cache, table = oracle.make_cache([260] * 4, 2, 128, 64, device=DEV)
    rows = torch.randn(4, 2 + 2 * 2, 128, device=DEV, dtype=torch.bfloat16)
    lens = _i32(lens0)

    def step():
        q, k, v = rows.split([2, 2, 2], 1)
        ops.kv_append_q8(k, v, cache, table, lens)
        return ops.paged_attention_q8(q, cache, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for i in range(4):
        lens.copy_(_i32([5 + i, 100 + i, 64 + i, i]))
        rows.copy_(torch.randn_like(rows))
        want = oracle.cpu(cache)
        ref.kv_append_q8(rows[:, 2:4].cpu(), rows[:, 4:].cpu(), want, table.cpu(), lens.cpu())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[i % 2].replay()
        torch.cuda.synchronize()
        out, around, size = oracle.attend(rows[:, :2], cache, table, lens)
        assert torch.equal(cache.k.cpu().view(torch.uint8), want.k.view(torch.uint8))
        assert ((outs[i % 2].cpu().double() - out).abs() <= oracle.attend_bound(out, around, size, 260, 128, torch.bfloat16)).all()


def test_refusals_on_the_gpu():
    cache, table = oracle.make_cache([20], 2, 96, 16, device=DEV)
    x = torch.randn(1, 2, 96, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="head dim"):
        ops.kv_append_q8(x, x, cache, table, _i32([20]))
    with pytest.raises(ValueError, match="head dim"):
        ops.paged_attention_q8(x, cache, table, _i32([20]))
    cache, table = oracle.make_cache([20], 2, 64, 24, device=DEV)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.paged_attention_q8(x[..., :64], cache, table, _i32([20]))
    cache, table = oracle.make_cache([20], 2, 64, 16, device=DEV)
    with pytest.raises(TypeError, match="queries"):
        ops.paged_attention_q8(x[..., :64].float(), cache, table, _i32([20]))
    with pytest.raises(ValueError, match="one device"):
        ops.paged_attention_q8(x[..., :64], cache, table.cpu(), _i32([20]))
