"""Paged attention where numbers are large, small, unequal or none at all; both attention kernels."""
import pytest
import torch

from sunshape_b200 import paged
from sunshape_b200.codec import SunShapeBlockCodec
from sunshape_b200.paged import SunShapePagedCache
from tests.paged_bounds import attention_bounds
from tests.paged_reference import make_paged_codec

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def no_error_left():
    paged.paged_error(DEV)
    yield
    assert paged.paged_error(DEV) is None


def _randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def _cache(codec, H, lens, prefix, page, dtype, seed=0):
    """A cache with a page table for ``lens``, a prefix, and a page more than both."""
    cols, first = max(1, -(-max(lens) // page)), -(-prefix // page)
    pages = len(lens) * cols + first + 1
    cache = SunShapePagedCache.allocate(codec, pages, H, page_size=page, dtype=dtype)
    g = torch.Generator().manual_seed(seed)
    cache.indices.copy_(torch.randint(0, codec.n_centroids, cache.indices.shape, generator=g))
    cache.values.copy_(_randn(*cache.values.shape, seed=seed + 1))
    if cache.heavy is not None:
        cache.heavy.copy_(_randn(*cache.heavy.shape, seed=seed + 2))
    order = torch.randperm(pages, generator=g).to(DEV, torch.int32)
    table = order[first:first + len(lens) * cols].view(len(lens), cols).contiguous()
    return cache, table, torch.tensor(lens, dtype=torch.int32, device=DEV), order[:first].contiguous()


def _near(got, cache, q, table, n, pt=None, prefix=0, rows=None, **kw):
    ref, bound, worst = attention_bounds(cache, q, table, n, pt, prefix, **kw)
    bad = ~((got.double().cpu() - ref).abs() <= bound)
    if rows is not None:
        bad = bad & rows[:, :, None, None]
    assert not bool(bad.any())
    return worst


# rows of a KV head: 8 go to the memory-bound kernel, 24 and more to the tensor-core one (one and two groups of 128 rows,
# the second one not full; more than 256)
ROWS = [(1, 8), (3, 8), (20, 8), (33, 8)]


@pytest.mark.parametrize("B,G", ROWS)
@pytest.mark.parametrize("value", ["pool", -1, 2 ** 31 - 1])
def test_bad_prefix_page(B, G, value):
    codec, _ = make_paged_codec(64, 8, 2, seed=1)
    cache, table, n, pt = _cache(codec, 2, [5] * B, 600, 16, BF16)
    q = _randn(B, 2 * G, 1, 64, seed=3, dtype=BF16)
    bad = pt.clone()
    bad[20] = cache.num_pages if value == "pool" else value
    got = cache.attention(q, table, n, prefix_table=bad, prefix_len=600)
    assert "page number" in paged.paged_error(DEV) and bool(got.isnan().all())
    _near(cache.attention(q, table, n, prefix_table=pt, prefix_len=600), cache, q, table, n, pt, 600)
    # entries behind the prefix's end are not read
    bad = torch.cat((pt, torch.full((3,), -7, dtype=torch.int32, device=DEV)))
    _near(cache.attention(q, table, n, prefix_table=bad, prefix_len=600), cache, q, table, n, pt, 600)


@pytest.mark.parametrize("B,G", ROWS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_of_every_kind_behind_a_prefix(B, G, dtype):
    """Zero, tiny, huge, infinite and NaN queries: each row is its own affair."""
    codec, _ = make_paged_codec(64, 8, 2, heavy=2, seed=2)
    cache, table, n, pt = _cache(codec, 2, [5, 0, 17] * (B // 3) + [1] * (B % 3), 300, 16, dtype)
    q = _randn(B, 2 * G, 1, 64, seed=3, dtype=dtype)
    q[0, 0] = 0
    q[0, 1] *= 1e-4 if dtype == F16 else 1e-30
    q[-1, 2] *= 1e3 if dtype == F16 else 1e30
    q[-1, 3, 0, 5] = float("nan")
    q[0, 4, 0, 7] = float("inf")
    got = cache.attention(q, table, n, prefix_table=pt, prefix_len=300)
    rows = torch.ones(B, 2 * G, dtype=torch.bool)
    rows[-1, 2] = rows[-1, 3] = rows[0, 4] = False
    _near(got, cache, q.nan_to_num(0, 0, 0), table, n, pt, 300, rows=rows)
    assert bool(got[-1, 3].isnan().all()) and bool(got[-1, 2].isfinite().all())


@pytest.mark.parametrize("B,G", ROWS)
@pytest.mark.parametrize("scale", [0.0, -0.7, 3.0])
def test_scales_behind_a_prefix(B, G, scale):
    codec, _ = make_paged_codec(64, 8, 2, seed=4)
    cache, table, n, pt = _cache(codec, 2, [5] * B, 300, 16, BF16)
    q = (0.1 * _randn(B, 2 * G, 1, 64, seed=3)).to(BF16)
    got = cache.attention(q, table, n, prefix_table=pt, prefix_len=300, scale=scale)
    _near(got, cache, q, table, n, pt, 300, scale=scale)


def _ramp(H, dtype, pages, page):
    """A codec whose key is one number, its codeword's index / 4, and a cache of them."""
    codec = SunShapeBlockCodec(64, 8, 256, device=torch.device(DEV), kv_heads=H)
    codec.centroids.zero_()
    codec.centroids[:, 0, :, 0] = torch.arange(256, device=DEV) / 4
    codec.invalidate()
    cache = SunShapePagedCache.allocate(codec, pages, H, page_size=page, dtype=dtype)
    cache.values.copy_(_randn(*cache.values.shape, seed=1))
    return cache


@pytest.mark.parametrize("B,G", ROWS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("order", ["up", "down", "steps", "last"])
def test_maximum_that_moves(B, G, dtype, order):
    """Scores that grow by more than the slack from tile to tile, fall, jump, or have one large one at the very end; some
    rows see the opposite."""
    T, page = 1500, 32
    cache = _ramp(1, dtype, -(-T // page) + B, page)
    t = torch.arange(T)
    level = {"up": t * 255 // (T - 1), "down": 255 - t * 255 // (T - 1), "steps": (t // 128 * 37) % 256, "last": t // (T - 1) * 255}[order]
    first = -(-T // page)
    cache.indices[:first, 0, :, 0].view(-1)[:T] = level.to(DEV, torch.uint8)
    pt = torch.arange(first, dtype=torch.int32, device=DEV)
    table = first + torch.arange(B, dtype=torch.int32, device=DEV)[:, None]
    n = torch.full((B,), 3, dtype=torch.int32, device=DEV)
    q = torch.zeros(B, G, 1, 64, dtype=dtype, device=DEV)
    q[..., 0] = torch.tensor([1.0, -1.0, 4.0, -4.0, 0.25, 0.0, 2.0, -0.5], device=DEV)[:G, None].to(dtype)
    got = cache.attention(q, table, n, prefix_table=pt, prefix_len=T, scale=1.0)
    _near(got, cache, q, table, n, pt, T, scale=1.0, exact_scores=True)


@pytest.mark.parametrize("B,G", ROWS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_blocks_far_smaller_than_the_largest(B, G, dtype):
    """Blocks at 1e-5 and 1e-8 of the codebook's largest codewords, and queries that look at these blocks alone."""
    codec, _ = make_paged_codec(64, 8, 2, seed=5)
    codec.centroids[:, 1] *= 1e-5
    codec.centroids[:, 2] *= 1e-8
    codec.invalidate()
    cache, table, n, pt = _cache(codec, 2, [40] * B, 300, 16, dtype)
    looks = torch.zeros(4, 64, device=DEV)
    for i, blocks in enumerate(([1], [2], [1, 2], [0, 1, 2, 3, 4, 5, 6, 7])):
        for b in blocks:
            looks[i, codec.permutation[8 * b:8 * b + 8]] = 4e3 if len(blocks) < 8 else 1.0
    q = (_randn(B, 2 * G, 1, 64, seed=3) * looks[torch.arange(2 * G, device=DEV) % 4, None]).to(dtype)
    got = cache.attention(q, table, n, prefix_table=pt, prefix_len=300)
    worst = _near(got, cache, q, table, n, pt, 300)
    assert worst < 0.3                                                   # the bound says something


@pytest.mark.parametrize("B,G,prefix", [(1200, 1, False), (296, 128, True)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_small_weights_beside_a_large_one(B, G, prefix, dtype):
    """20000 tokens whose weights are 2^-25.5 of the first one's and that carry the result.  All sequences read the same
    pages, and are so many that a warp or thread block walks a whole one beside that first maximum."""
    T, page = 20000, 128
    first = -(-T // page)
    cache = _ramp(1, dtype, first, page)
    cache.values.fill_(1)
    cache.values[0, :, 0] = 0
    cache.indices[0, 0, 0, 0] = 68                                       # key 17, the others 0
    pages = torch.arange(first, dtype=torch.int32, device=DEV)
    q = torch.zeros(B, G, 1, 64, dtype=dtype, device=DEV)
    q[..., 0] = 1
    scale = 25.5 * 0.6931471805599453 / 17
    own = torch.full((B,), 0 if prefix else T, dtype=torch.int32, device=DEV)
    got = cache.attention(q, pages.expand(B, -1), own, prefix_table=pages if prefix else None, prefix_len=T if prefix else 0,
                          scale=scale)
    ref, bound, _ = attention_bounds(cache, q[:1, :1], pages[None], [T], scale=scale, exact_scores=True)
    # the scores' fp32 roundings: 2^-23 of 17.7 each
    assert bool(((got.double().cpu() - ref).abs() <= bound + 2.0 ** -18 * ref.abs()).all())


@pytest.mark.parametrize("B,G,L,bd", [(1, 8, 1, 8), (2, 2, 2, 4), (1, 2, 3, 2), (20, 8, 1, 8), (9, 2, 2, 4), (20, 1, 1, 2)])
@pytest.mark.parametrize("dtype,unit", [(BF16, 1.0), (BF16, 1024.0), (F16, 1.0)])
def test_dense_blocks_beyond_fp16(B, G, L, bd, dtype, unit):
    """A dense key that fp16 can not hold is recorded and makes the rows NaN that see it; one at the limit is exact, and
    neither NaN queries nor what lies behind a sequence's end count.  Codewords far smaller than dense keys do not narrow
    the range, larger ones widen it."""
    codec, _ = make_paged_codec(64, bd, 1, heavy=3, seed=6)
    codec.centroids.mul_((0.75 * 2.0 ** -8 if unit == 1 else 0.75 * unit) / codec.centroids.norm(dim=-1).max())
    codec.invalidate()
    cache, table, n, pt = _cache(codec, 1, [33] * B, 300, 16, dtype)
    q = (0.25 / unit * _randn(B, G, L, 64, seed=3)).to(dtype)
    dense = codec.permutation.view(-1, bd)[codec.mixed_high_precision_blocks].flatten()
    q[..., dense[0]] = 2.0 ** -10 / unit                                    # of the element that grows
    run = lambda: cache.attention(q, table, n, prefix_table=pt, prefix_len=300)
    at_prefix, own_last = (int(pt[7]), 0, 3, 0, 0), (int(table[0, 2]), 0, 0, 0, 0)
    behind = (int(table[0, 2]), 0, 1, 0, 0)
    limit, beyond = (65504.0, None) if dtype == F16 else (65280.0 * unit, 65536.0 * unit)
    for place in (at_prefix, own_last):
        was = cache.heavy[place].item()
        for sign in (1, -1):
            cache.heavy[place] = sign * limit
            _near(run(), cache, q, table, n, pt, 300)
            assert paged.paged_error(DEV) is None
            if beyond is None:
                continue
            cache.heavy[place] = sign * beyond
            got = run()
            assert "dense key block" in paged.paged_error(DEV)
            if place is at_prefix:
                assert bool(got.isnan().all())
            else:                                                           # the last token: of the last query alone
                assert bool(got[0, :, -1].isnan().all()) and not bool(got[1:].isnan().any())
                assert not bool(got[0, :, :-1].isnan().any())
        cache.heavy[place] = was
    for value in (limit if beyond is None else beyond, float("inf"), float("nan")):
        cache.heavy[behind] = value
        _near(run(), cache, q, table, n, pt, 300)
    q[0, 0, 0, 0] = float("nan")                                            # the query's doing: not recorded
    assert bool(run()[0, 0, 0].isnan().all())


def test_norm_rotate_outputs_over_other_inputs():
    """An output over another tensor's input, over the other output or over itself would be written while it is read."""
    q = torch.randn(2, 4, 3, 64, device=DEV).to(BF16)
    k, other = q.clone(), q.clone()
    for out in ((k, other), (other, q), (other, other), (k, q), (other[:, :1].expand(-1, 4, -1, -1), k)):
        before = [t.clone() for t in (q, k)]
        with pytest.raises(RuntimeError, match="out must not"):
            paged.norm_rotate(q, k, out=out)
        assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    paged.norm_rotate(q, k, q_weight=torch.ones(64, device=DEV), out=(q, k))
    e = q[:0]
    paged.norm_rotate(e, e, out=(e, e))


def test_prefix_of_millions_of_tokens():
    """A prefix of 14 million tokens, one page over and over, behind 37888 rows: a third of a second in which the sequences'
    own tokens must not wait with full rings.  The result is that page's."""
    B, G, page, repeats = 4736, 8, 128, 110000
    codec, _ = make_paged_codec(64, 8, 1, seed=12)
    cache, _, _, _ = _cache(codec, 1, [0], 0, page, BF16)
    q = _randn(B, G, 1, 64, seed=3, dtype=BF16)
    table = torch.zeros(B, 1, dtype=torch.int32, device=DEV)
    none = torch.zeros(B, dtype=torch.int32, device=DEV)
    got = cache.attention(q, table, none, prefix_table=torch.zeros(repeats, dtype=torch.int32, device=DEV),
                          prefix_len=repeats * page)
    want = cache.attention(q, table, none + page)
    assert paged.paged_error(DEV) is None
    # both within half a step of the output and of each weight; sums of 1.4e7 weights in fp32 in pieces of 1e5 tiles: 1e5 2^-24
    assert float((got.float() - want.float()).abs().max()) <= (2.0 ** -7 + 2.0 ** -7 + 0.006) * float(cache.values.abs().max())
    _near(want[:3], cache, q[:3], table[:3], none[:3] + page)
