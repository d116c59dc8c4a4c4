"""Paged-serving operators against their plain 64-bit forms: sizes, layouts and masks where they can go wrong."""
import pytest
import torch

from sunshape_b200 import paged
from sunshape_b200.paged import SunShapePagedCache
from tests.paged_reference import (HALF_STEP, attention64, encode64, make_paged_codec, norm64, rotate64)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def _positions(B, L, n, seed):
    return torch.randint(0, n - L + 1, (B, 1), generator=torch.Generator().manual_seed(seed)).to(DEV) + torch.arange(L, device=DEV)


@pytest.fixture(autouse=True)
def no_error_left():
    paged.paged_error(DEV)
    yield
    assert paged.paged_error(DEV) is None


# ------------------------------------------------------------------------------------------------ norm_rotate
def _check_norm_rotate(got, x, w, eps, cos, sin, pos, inter):
    y = norm64(x, w, eps)
    ref = rotate64(y, cos, sin, pos, inter)
    # fp32: the mean's sum and root (D + 8 roundings of 2^-24 of the norm factor), three products, one sum of a pair
    size = rotate64(y.abs(), None if cos is None else cos.abs(), None if sin is None else -sin.abs(), pos, inter).abs()
    size = torch.maximum(size, y.abs())
    bound = HALF_STEP[x.dtype] * ref.abs() + (x.shape[-1] + 16) * 2.0 ** -24 * 2 * size + 1e-30
    if x.dtype == torch.float16:
        bound += 2.0 ** -25          # half a step below fp16's normal range
    assert got.shape == x.shape and got.dtype == x.dtype
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,Hq,Hk,D,R,inter,norm", [
    (1, 1, 14, 2, 64, 64, False, True), (8, 1, 64, 8, 128, 128, False, True), (3, 37, 5, 1, 128, 64, True, True),
    (2, 9, 4, 4, 96, 96, False, True), (2, 5, 3, 1, 96, 32, False, False), (1, 33, 2, 2, 256, 128, True, True),
    (2, 3, 2, 1, 10, 6, False, True), (2, 3, 2, 1, 65, 64, False, True), (1, 4, 3, 3, 24, 24, True, True),
    (5, 700, 32, 8, 128, 128, False, True), (4, 3, 2, 2, 128, 0, False, True)])
def test_norm_rotate(dtype, B, L, Hq, Hk, D, R, inter, norm):
    q = _randn(B, L, Hq, D, seed=1, dtype=dtype).transpose(1, 2)
    k = _randn(B, Hk, L, D, seed=2, dtype=dtype)
    qw = (1 + 0.3 * _randn(D, seed=3)).to(dtype) if norm else None
    kw = (1 + 0.3 * _randn(D, seed=4)).to(dtype) if norm else None
    cos, sin = paged.rotary_table(40000, R, device=DEV) if R else (None, None)
    pos = _positions(B, L, 40000, 5) if R else None
    gq, gk = paged.norm_rotate(q, k, q_weight=qw, k_weight=kw, eps=1e-5, cos=cos, sin=sin, positions=pos,
                               interleaved=inter)
    assert gq.stride() == q.stride()
    _check_norm_rotate(gq, q, qw, 1e-5, cos, sin, pos, inter)
    _check_norm_rotate(gk, k, kw, 1e-5, cos, sin, pos, inter)


def test_norm_rotate_layouts_in_place_and_only_query():
    """A view of a fused projection, misaligned by one element; in place; int32 and broadcast positions; fp32 weights on
    16-bit rows; zero and huge rows."""
    B, L, D = 2, 7, 64
    fused = _randn(B, L, 6 * D + 1, seed=1, dtype=torch.bfloat16)
    cos, sin = paged.rotary_table(512, D, device=DEV)
    pos = torch.arange(100, 100 + L, device=DEV, dtype=torch.int32)
    w = 1 + 0.1 * _randn(D, seed=3)
    for off in (0, 1):
        q = fused[..., off:off + 4 * D].unflatten(-1, (4, D)).transpose(1, 2)
        got, none = paged.norm_rotate(q, q_weight=w, eps=0.0, cos=cos, sin=sin, positions=pos)
        assert none is None
        _check_norm_rotate(got, q, w, 0.0, cos, sin, pos.expand(B, L), False)
    for D2 in (64, 62):              # the vector kernel and the general one
        x = _randn(B, 3, L, 64, seed=6, dtype=torch.bfloat16)[..., :D2].contiguous()
        x[0, 0, 0] = 0
        x[0, 1, 0] *= 1e15
        c2, s2 = paged.rotary_table(512, D2, device=DEV)
        before = x.clone()
        w2 = w[:D2].contiguous()
        got, _ = paged.norm_rotate(x, q_weight=w2, cos=c2, sin=s2, positions=pos, out=(x, None))
        assert got is x
        _check_norm_rotate(x, before, w2, 1e-6, c2, s2, pos.expand(B, L), False)


def test_norm_rotate_empty_and_bad_positions():
    cos, sin = paged.rotary_table(16, 64, device=DEV)
    q = _randn(2, 3, 4, 64, seed=1, dtype=torch.bfloat16)
    pos = torch.tensor([[0, 15, 16, -1], [1, 2, 3, 4]], device=DEV)
    for x in (q, q[..., :62].contiguous()):
        c, s = cos[:, :x.shape[-1] // 2].contiguous(), sin[:, :x.shape[-1] // 2].contiguous()
        got, _ = paged.norm_rotate(x, cos=c, sin=s, positions=pos)
        assert "position" in paged.paged_error(DEV)
        assert bool(got[0, :, 2:].isnan().all()) and not bool(got[0, :, :2].isnan().any()) and not bool(got[1].isnan().any())
    e = q[:, :, :0]
    assert paged.norm_rotate(e, cos=cos, sin=sin, positions=pos[:, :0])[0].shape == e.shape


# ------------------------------------------------------------------------------------------------------ append
def _append_case(codec, H, B, L, *, page, dtype, R, inter=False, seed=0, scale=None, spare=3):
    D = codec.head_dim
    k = _randn(B, L, H, D, seed=seed + 1)
    k = (k * scale.to(DEV) if scale is not None else k).to(dtype).transpose(1, 2)
    v = _randn(B, L, H, D, seed=seed + 2, dtype=dtype).transpose(1, 2)
    each = -(-L // page) + 1
    cache = SunShapePagedCache.allocate(codec, B * each + spare, H, page_size=page, dtype=dtype)
    g = torch.Generator().manual_seed(seed)
    cache.indices.copy_(torch.randint(0, 256, cache.indices.shape, generator=g))
    cache.values.copy_(_randn(*cache.values.shape, seed=seed + 4))
    if cache.heavy is not None:
        cache.heavy.copy_(_randn(*cache.heavy.shape, seed=seed + 5))
    table = torch.randperm(B * each + spare, generator=g)[:B * each].view(B, each).to(DEV)
    at = torch.randint(0, page, (B, 1), generator=g).to(DEV) + torch.arange(L, device=DEV)
    slots = cache.slots(table, at)
    slots[torch.rand(B, L, generator=g).to(DEV) < 0.2] = -1
    rot = {}
    if R:
        cos, sin = paged.rotary_table(5000, R, device=DEV)
        rot = dict(cos=cos, sin=sin, positions=_positions(B, L, 5000, seed + 3), interleaved=inter)
    return cache, k, v, slots, rot


def _check_append(cache, k, v, slots, rot, before):
    codec, ps = cache.codec, cache.page_size
    z = rotate64(k, rot.get("cos"), rot.get("sin"), rot.get("positions"), rot.get("interleaved", False))
    idx, blocks = encode64(codec, z)
    want = [t if t is None else t.clone() for t in before]
    s = slots.cpu()
    keep = s >= 0
    page, row = s[keep] // ps, s[keep] % ps
    want[0][page, :, row] = idx.transpose(1, 2)[keep].to(torch.uint8)
    want[1][page, :, row] = v.cpu().transpose(1, 2)[keep]
    assert torch.equal(cache.indices.cpu(), want[0])
    assert torch.equal(cache.values.cpu(), want[1])
    if want[2] is not None:
        mask = codec.mixed_high_precision_blocks.cpu()
        want[2][page, :, row] = blocks[..., mask, :].transpose(1, 2)[keep].float().to(cache.dtype)
        assert torch.equal(cache.heavy.cpu(), want[2])


def _state(cache):
    return [cache.indices.cpu(), cache.values.cpu(), None if cache.heavy is None else cache.heavy.cpu()]


@pytest.mark.parametrize("B,L,H,D,bd,C,heavy,R,inter,page,dtype,shared", [
    (1, 1, 1, 64, 8, 256, 0, 64, False, 16, torch.bfloat16, False),
    (7, 1, 8, 128, 8, 256, 0, 128, False, 64, torch.bfloat16, False),
    (3, 77, 2, 128, 8, 256, 4, 128, False, 48, torch.bfloat16, False),
    (2, 130, 2, 128, 4, 256, 0, 64, True, 32, torch.float16, False),
    (2, 65, 2, 64, 2, 256, 3, 64, False, 16, torch.float16, True),
    (1, 300, 3, 128, 8, 256, 0, 0, False, 128, torch.bfloat16, True),
    (2, 9, 2, 96, 8, 100, 1, 96, False, 16, torch.bfloat16, False),
    (1, 40, 1, 256, 8, 16, 0, 256, False, 16, torch.bfloat16, False),
    (1, 70, 2, 64, 8, 1, 0, 64, False, 16, torch.float16, False),
    (1, 1000, 2, 128, 8, 256, 16, 128, False, 64, torch.bfloat16, False)])
def test_append(B, L, H, D, bd, C, heavy, R, inter, page, dtype, shared):
    codec, scale = make_paged_codec(D, bd, H, heavy=heavy, C=C, shared=shared, seed=D + bd)
    cache, k, v, slots, rot = _append_case(codec, H, B, L, page=page, dtype=dtype, R=R, inter=inter, scale=scale, seed=7)
    before = _state(cache)
    paged.append_paged(cache, k, v, slots, **rot)
    _check_append(cache, k, v, slots, rot, before)


@pytest.mark.parametrize("L", [5, 600])
def test_append_ties_and_borders(L):
    """Codewords twice, codewords that differ in the last fp32 bit, keys halfway between codewords, zero keys,
    infinite, NaN and huge keys: the lowest index of the 64-bit minimum, 0 where no distance is finite."""
    D, bd, H = 64, 8, 2
    codec, _ = make_paged_codec(D, bd, H, seed=1)
    c = codec.centroids
    c[:, :, 128:] = c[:, :, :128].flip(2)                                       # every codeword twice
    c[:, 1, 64:128] = torch.nextafter(c[:, 1, :64], torch.full_like(c[:, 1, :64], 9.0))
    c[:, 2, 1] = -c[:, 2, 0]
    c[:, 3] *= 1e-20
    c[:, 4] *= 1e15
    codec.invalidate()
    cache, k, v, slots, rot = _append_case(codec, H, 1, L, page=16, dtype=torch.bfloat16, R=0, seed=3)
    perm = codec.permutation
    kp = torch.empty_like(k)
    kp[..., perm] = k
    k = kp.contiguous()
    k[0, :, 0] = 0
    k[0, 0, 1] = float("inf")
    k[0, 1, 1] = float("nan")
    k[0, :, 2] = 3e38
    k[0, 0, 3, 5] = -float("inf")
    near = c[:, :, :L].to(torch.bfloat16).float()                                # rounded codewords, block by block
    n = min(L - 4, near.shape[2])
    k[0][:, 4:4 + n][..., perm] = near.permute(0, 2, 1, 3).reshape(H, -1, D)[:, :n].to(torch.bfloat16)
    slots = torch.arange(L, device=DEV)[None].clamp(max=cache.num_pages * 16 - 1)
    before = _state(cache)
    paged.append_paged(cache, k, v, slots, **rot)
    # numpy's argmin takes the first NaN as the smallest, which is index 0 as documented: all of a block's are NaN
    _check_append(cache, k, v, slots, rot, before)


def test_append_out_of_range_is_left_out():
    codec, scale = make_paged_codec(64, 8, 2, seed=2)
    cache, k, v, slots, rot = _append_case(codec, 2, 1, 6, page=16, dtype=torch.bfloat16, R=64, scale=scale)
    total = cache.num_pages * 16
    before = _state(cache)
    bad = torch.tensor([[0, total, 5, -2, 2 ** 40, 7]], device=DEV)
    paged.append_paged(cache, k, v, bad, **rot)
    assert "slot" in paged.paged_error(DEV)
    kept = torch.where((bad >= 0) & (bad < total), bad, -1)
    _check_append(cache, k, v, kept, rot, before)
    before = _state(cache)
    rot["positions"] = torch.tensor([[1, 5000, 2, -1, 3, 4]], device=DEV)
    good = torch.arange(20, 26, device=DEV)[None]
    paged.append_paged(cache, k, v, good, **rot)
    assert "position" in paged.paged_error(DEV)
    kept = torch.where((rot["positions"] >= 0) & (rot["positions"] < 5000), good, -1)
    _check_append(cache, k, v, kept, dict(rot, positions=rot["positions"].clamp(0, 4999)), before)


# --------------------------------------------------------------------------------------------------- attention
def _filled(codec, H, pages, page, dtype, Dv=None, seed=0, scale=None):
    cache = SunShapePagedCache.allocate(codec, pages, H, page_size=page, value_dim=Dv, dtype=dtype)
    g = torch.Generator().manual_seed(seed)
    cache.indices.copy_(torch.randint(0, codec.n_centroids, cache.indices.shape, generator=g))
    cache.values.copy_(_randn(*cache.values.shape, seed=seed + 1))
    if cache.heavy is not None:
        cache.heavy.copy_(_randn(*cache.heavy.shape, seed=seed + 2) * 2)
    return cache


def _attention_case(codec, H, G, B, L, lens, prefix, page, dtype, Dv=None, seed=0):
    cols = max(1, -(-max(lens, default=0) // page)) + 1
    first = -(-prefix // page)
    cache = _filled(codec, H, B * cols + first + 1, page, dtype, Dv, seed)
    order = torch.randperm(B * cols + first + 1, generator=torch.Generator().manual_seed(seed)).to(DEV, torch.int32)
    # what lies behind a sequence's end is garbage of every kind
    table = order[first:first + B * cols].view(B, cols).contiguous()
    for b, n in enumerate(lens):
        page_of = table[b].long()
        rest = n % page
        if n // page < cols:
            cache.values[page_of[n // page], :, rest:] = float("nan")
            if cache.heavy is not None:
                cache.heavy[page_of[n // page], :, rest:] = float("inf")
            cache.indices[page_of[n // page], :, rest:] = 255
        for j in range(n // page + 1, cols):
            cache.values[page_of[j]] = float("nan")
    if prefix % page:
        cache.values[order[first - 1].long(), :, prefix % page:] = float("nan")
        if cache.heavy is not None:
            cache.heavy[order[first - 1].long(), :, prefix % page:] = float("nan")
    q = _randn(B, H * G, L, codec.head_dim, seed=seed + 9, dtype=dtype)
    return cache, q, table, torch.tensor(lens, dtype=torch.int32, device=DEV), order[:first].contiguous() if first else None


def _check_attention(got, cache, q, table, lens, pt, prefix, **kw):
    ref, bound = attention64(cache, q, table, lens, pt, prefix, **kw)
    assert got.dtype == cache.dtype and got.shape == ref.shape
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} of the bound"


@pytest.mark.parametrize("D,Dv,bd,C,heavy,H,G,L,page,lens,prefix,dtype", [
    (64, 64, 8, 256, 0, 2, 7, 1, 16, [517], 0, torch.float16),
    (128, 128, 8, 256, 0, 2, 4, 1, 64, [1, 64, 65, 0, 200, 63], 0, torch.bfloat16),
    (128, 128, 8, 256, 4, 2, 8, 1, 16, [130, 1, 77], 0, torch.bfloat16),
    (128, 128, 4, 256, 0, 2, 4, 4, 32, [3, 500, 4, 1], 0, torch.bfloat16),
    (128, 128, 4, 256, 5, 1, 8, 5, 48, [31, 800], 0, torch.float16),
    (64, 128, 2, 256, 2, 2, 3, 1, 16, [333, 20], 0, torch.bfloat16),
    (128, 64, 2, 256, 0, 1, 1, 1, 128, [1000, 129], 0, torch.float16),
    (64, 64, 4, 100, 0, 1, 16, 2, 16, [90, 15], 0, torch.bfloat16),
    (64, 64, 8, 1, 0, 1, 2, 1, 16, [40], 0, torch.bfloat16),
    (64, 64, 8, 256, 8, 1, 8, 1, 16, [100, 5], 0, torch.bfloat16),
    (128, 128, 8, 256, 0, 2, 8, 1, 64, [5, 0, 130, 64], 300, torch.bfloat16),
    (128, 128, 8, 256, 4, 2, 4, 1, 16, [17] * 9, 1000, torch.bfloat16),
    (64, 64, 8, 256, 0, 2, 7, 3, 16, [0, 2, 33], 129, torch.float16),
    (128, 128, 4, 256, 0, 1, 8, 1, 32, [1, 2, 3] * 7, 1, torch.bfloat16),
    (128, 64, 8, 256, 2, 1, 24, 2, 64, [70, 10], 700, torch.float16),
    (64, 128, 2, 64, 0, 2, 4, 1, 48, [50, 51], 257, torch.bfloat16),
    (128, 128, 8, 256, 3, 2, 8, 1, 16, [1, 0, 5, 17] * 10, 2000, torch.bfloat16),
    (64, 64, 4, 256, 0, 3, 8, 1, 32, [3] * 50, 383, torch.float16),
    (128, 64, 4, 256, 2, 1, 4, 2, 48, [9] * 17, 128, torch.bfloat16),
    (64, 64, 2, 256, 5, 2, 16, 1, 64, [2, 70], 1025, torch.bfloat16),
    (128, 128, 2, 256, 0, 1, 8, 1, 128, [1] * 33, 1500, torch.float16)])
def test_paged_attention(D, Dv, bd, C, heavy, H, G, L, page, lens, prefix, dtype):
    codec, _ = make_paged_codec(D, bd, H, heavy=heavy, C=C, seed=D + bd + G, shared=(G == 7))
    cache, q, table, n, pt = _attention_case(codec, H, G, len(lens), L, lens, prefix, page, dtype, Dv, seed=G)
    got = paged.paged_attention(cache, q, table, n, prefix_table=pt, prefix_len=prefix)
    _check_attention(got, cache, q, table, n, pt, prefix)
    if L > 1:
        got = paged.paged_attention(cache, q, table, n, prefix_table=pt, prefix_len=prefix, causal=False, scale=-0.3)
        _check_attention(got, cache, q, table, n, pt, prefix, causal=False, scale=-0.3)


def test_paged_attention_long_and_ragged():
    """Runs of one row joined from many thread blocks, next to sequences of a few tokens."""
    codec, _ = make_paged_codec(128, 8, 2, seed=5)
    lens = [9000, 3, 0, 4111, 64, 1]
    cache, q, table, n, _ = _attention_case(codec, 2, 4, len(lens), 1, lens, 0, 64, torch.bfloat16, seed=2)
    got = paged.paged_attention(cache, q, table, n)
    _check_attention(got, cache, q, table, n, None, 0)
    again = paged.paged_attention(cache, q, table, n)
    assert torch.equal(got, again)


def test_paged_attention_extreme_logits():
    """Logits of thousands, all equal logits, zero and infinite queries."""
    codec, _ = make_paged_codec(64, 8, 1, seed=6)
    cache, q, table, n, _ = _attention_case(codec, 1, 4, 2, 1, [300, 40], 0, 16, torch.bfloat16, seed=3)
    q[0, 0] = 0
    q[0, 1] *= 1e30
    q[0, 2] *= 1e-30
    got = paged.paged_attention(cache, q, table, n, scale=0.125)
    ref, bound = attention64(cache, q, table, n, scale=0.125)
    rows = torch.tensor([True, False, True, True])
    assert bool(((got.double().cpu() - ref).abs() <= bound)[0, rows].all())
    assert bool(got[0, 1].isfinite().all())
    q[1, 3, 0, 0] = float("nan")
    got = paged.paged_attention(cache, q, table, n, scale=0.125)
    assert bool(got[1, 3].isnan().all()) and not bool(got[1, :3].isnan().any())


def test_paged_attention_bad_pages_and_lengths():
    codec, _ = make_paged_codec(64, 8, 2, seed=7)
    cache, q, table, n, pt = _attention_case(codec, 2, 2, 4, 1, [40, 50, 60, 0], 20, 16, torch.bfloat16, seed=4)
    for value in (cache.num_pages, -1, 2 ** 31 - 1):
        t = table.clone()
        t[1, 2] = value
        got = paged.paged_attention(cache, q, t, n, prefix_table=pt, prefix_len=20)
        assert "page number" in paged.paged_error(DEV)
        assert bool(got[1].isnan().all())
        ref, bound = attention64(cache, q, table, n, pt, 20)
        rest = [0, 2, 3]
        assert bool(((got.double().cpu() - ref).abs() <= bound)[rest].all())
    for value in (-1, table.shape[1] * 16 + 1, 2 ** 31 - 1):
        m = n.clone()
        m[2] = value
        got = paged.paged_attention(cache, q, table, m, prefix_table=pt, prefix_len=20)
        assert "longer than its page table" in paged.paged_error(DEV)
        assert bool(got[2].isnan().all()) and not bool(got[[0, 1, 3]].isnan().any())
    bad = pt.clone()
    bad[1] = cache.num_pages
    got = paged.paged_attention(cache, q, table, n, prefix_table=bad, prefix_len=20)
    assert "page number" in paged.paged_error(DEV) and bool(got.isnan().all())


def test_paged_attention_empty_calls():
    codec, _ = make_paged_codec(64, 8, 2, seed=7)
    cache = SunShapePagedCache.allocate(codec, 4, 2, page_size=16)
    table, n = torch.zeros(3, 2, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    q = _randn(3, 4, 1, 64, seed=1, dtype=torch.bfloat16)
    assert bool((paged.paged_attention(cache, q, table, n) == 0).all())
    assert bool((paged.paged_attention(cache, q, table[:, :0], n) == 0).all())
    assert paged.paged_attention(cache, q[:0], table[:0], n[:0]).shape == (0, 4, 1, 64)
    assert paged.paged_attention(cache, q[:, :, :0], table, n).shape == (3, 4, 0, 64)


@pytest.mark.parametrize("B,H,G,L,prefix,shared", [(300, 2, 2, 1, 0, False), (700, 1, 1, 2, 0, True), (300, 1, 2, 1, 70, True)])
def test_paged_attention_many_sequences(B, H, G, L, prefix, shared):
    """More sequences than the plan's chunks, many of them empty, and one codebook for all heads."""
    codec, _ = make_paged_codec(64, 8, H, seed=B, shared=shared)
    lens = [(i * 37) % 41 if i % 3 else 0 for i in range(B)]
    cache, q, table, n, pt = _attention_case(codec, H, G, B, L, lens, prefix, 16, torch.bfloat16, seed=1)
    got = paged.paged_attention(cache, q, table, n, prefix_table=pt, prefix_len=prefix)
    _check_attention(got, cache, q, table, n, pt, prefix)


@pytest.mark.parametrize("H,G,L,n,prefix,shared", [(1, 8, 1, 30000, 0, False), (3, 2, 1, 5000, 0, True), (1, 4, 1, 1, 20000, False),
                                                   (2, 16, 2, 7, 20000, False)])
def test_paged_attention_one_sequence_over_all_blocks(H, G, L, n, prefix, shared):
    """One sequence whose runs are spread over the whole device and joined in order."""
    codec, _ = make_paged_codec(128, 8, H, seed=n, shared=shared)
    cache, q, table, lens, pt = _attention_case(codec, H, G, 1, L, [n], prefix, 128, torch.bfloat16, seed=3)
    got = paged.paged_attention(cache, q, table, lens, prefix_table=pt, prefix_len=prefix)
    _check_attention(got, cache, q, table, lens, pt, prefix)
    assert torch.equal(got, paged.paged_attention(cache, q, table, lens, prefix_table=pt, prefix_len=prefix))


def test_paged_attention_views_and_out():
    """Queries as a view of a fused projection's output, a sliced page table, a given output, and pages that two
    sequences share."""
    codec, _ = make_paged_codec(64, 4, 2, seed=4)
    cache, q, table, n, _ = _attention_case(codec, 2, 3, 4, 1, [40, 33, 5, 64], 0, 16, torch.float16, seed=6)
    wide = torch.zeros(4, table.shape[1] + 5, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + table.shape[1]] = table
    wide[3] = wide[0]
    t = wide[:, 2:2 + table.shape[1]]
    n = torch.tensor([40, 33, 5, 40], dtype=torch.int32, device=DEV)
    fused = _randn(4, 1, 10, 64, seed=5, dtype=torch.float16)
    q = fused[:, :, 2:8].transpose(1, 2)
    out = torch.full((4, 6, 1, 64), 7.0, dtype=torch.float16, device=DEV)
    got = paged.paged_attention(cache, q, t, n, out=out)
    assert got is out
    _check_attention(got, cache, q, t, n, None, 0)


def test_codebook_edited_in_place():
    """``invalidate`` renews what the paged kernels derived from the codebooks."""
    codec, scale = make_paged_codec(64, 8, 2, seed=8)
    cache, k, v, slots, rot = _append_case(codec, 2, 1, 30, page=16, dtype=torch.bfloat16, R=64, scale=scale)
    for _ in range(2):
        before = _state(cache)
        cache.append(k, v, slots, **rot)
        _check_append(cache, k, v, slots, rot, before)
        codec.centroids.mul_(0.5).add_(0.1)
        codec.invalidate()
    q = _randn(1, 4, 1, 64, seed=3, dtype=torch.bfloat16)
    table, n = torch.arange(2, dtype=torch.int32, device=DEV)[None], torch.tensor([20], dtype=torch.int32, device=DEV)
    _check_attention(cache.attention(q, table, n), cache, q, table, n, None, 0)


def test_positions_beyond_the_table_are_recorded():
    codec, scale = make_paged_codec(64, 8, 2, seed=9)
    cache, k, v, _, _ = _append_case(codec, 2, 1, 4, page=16, dtype=torch.bfloat16, R=0, scale=scale)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    slots = cache.slots(table, torch.tensor([[31, 32, 1000000, -5]], device=DEV))
    before = _state(cache)
    cache.append(k, v, slots)
    assert "slot" in paged.paged_error(DEV)
    _check_append(cache, k, v, torch.tensor([[15, -1, -1, -1]]), {}, before)


def test_codec_that_no_longer_fits_its_pools():
    codec, _ = make_paged_codec(64, 8, 2, heavy=2, seed=9)
    cache = SunShapePagedCache.allocate(codec, 6, 2, page_size=16)
    k = _randn(1, 2, 3, 64, seed=1, dtype=torch.bfloat16)
    codec.mixed_high_precision_blocks.fill_(True)
    codec.invalidate()
    with pytest.raises(RuntimeError, match="dense blocks or device"):
        cache.append(k, k, torch.arange(3, device=DEV)[None])
    with pytest.raises(RuntimeError, match="dense blocks or device"):
        cache.attention(k, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV))


def test_append_strided_and_misaligned_rows():
    """Values and keys that begin off a 16-byte boundary, a flat ragged batch, positions that broadcast."""
    codec, scale = make_paged_codec(64, 8, 2, seed=9)
    cache = SunShapePagedCache.allocate(codec, 6, 2, page_size=16)
    fused = _randn(37, 2 * 2 * 64 + 3, seed=2, dtype=torch.bfloat16)
    kv = fused[:, 1:1 + 256].unflatten(1, (4, 64)).transpose(0, 1).unsqueeze(0)      # [1, 4, 37, 64]
    k, v = kv[:, :2], kv[:, 2:]
    cos, sin = paged.rotary_table(64, 32, device=DEV)
    rot = dict(cos=cos, sin=sin, positions=torch.arange(37, device=DEV, dtype=torch.int32))
    slots = torch.randperm(96, generator=torch.Generator().manual_seed(1))[:37][None].to(DEV)
    before = _state(cache)
    cache.append(k, v, slots, **rot)
    _check_append(cache, k, v, slots, dict(rot, positions=rot["positions"][None]), before)


def test_calls_on_a_stream_of_their_own():
    """A chain of calls on a side stream, without any synchronisation in between."""
    codec, scale = make_paged_codec(128, 8, 2, seed=10)
    cache, q, table, n, pt = _attention_case(codec, 2, 8, 3, 1, [300, 64, 7], 130, 64, torch.bfloat16, seed=5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            q2, _ = paged.norm_rotate(q, q_weight=torch.ones(128, device=DEV))
            got = paged.paged_attention(cache, q2, table, n, prefix_table=pt, prefix_len=130)
    side.synchronize()
    _check_attention(got, cache, q2, table, n, pt, 130)


# ---------------------------------------------------------------------------------------------- used together
def test_decode_steps_together_match_contiguous_cache():
    """A prompt and three decode steps as an engine runs them -- norms and rotation, append, attention behind a shared
    prompt -- against the contiguous path on the same tokens."""
    from sunshape_b200.vllm_attn_backend import _apply_quantized_attention, quantize_codec_keys

    D, H, G, page, B, prompt = 64, 2, 4, 16, 3, 37
    codec, _ = make_paged_codec(D, 8, H, heavy=2, seed=11)
    cache = SunShapePagedCache.allocate(codec, 32, H, page_size=page)
    cos, sin = paged.rotary_table(256, D, device=DEV)
    w = (1 + 0.1 * _randn(D, seed=8)).to(torch.bfloat16)
    pt = torch.tensor([3, 1, 7], dtype=torch.int32, device=DEV)
    table = torch.tensor([[10, 11], [2, 4], [20, 30]], dtype=torch.int32, device=DEV)

    def tokens(b, n, seed):
        return _randn(b, n, H, D, seed=seed, dtype=torch.bfloat16).transpose(1, 2)

    k0, v0 = tokens(1, prompt, 1), tokens(1, prompt, 2)
    pos = torch.arange(prompt, device=DEV)[None]
    k0 = paged.norm_rotate(k0, q_weight=w, cos=cos, sin=sin, positions=pos)[0]
    paged.append_paged(cache, k0, v0, cache.slots(pt[None], pos))
    keys, vals = [k0.expand(B, -1, -1, -1)], [v0.expand(B, -1, -1, -1)]
    for step in range(3):
        q, k, v = tokens(B, 1, 10 + step), tokens(B, 1, 20 + step), tokens(B, 1, 30 + step)
        q = q.repeat_interleave(G, 1)
        at = torch.full((B, 1), step, device=DEV)
        q, k = paged.norm_rotate(q, k, q_weight=w, k_weight=w, cos=cos, sin=sin, positions=at + prompt)
        cache.append(k, v, cache.slots(table, at))
        lens = torch.full((B,), step + 1, dtype=torch.int32, device=DEV)
        got = cache.attention(q, table, lens, prefix_table=pt, prefix_len=prompt)
        _check_attention(got, cache, q, table, lens, pt, prompt)
        keys.append(k)
        vals.append(v)
        full = quantize_codec_keys(codec, torch.cat(keys, 2).contiguous())
        ref = _apply_quantized_attention(codec=codec, query=q, key=full, value=torch.cat(vals, 2).contiguous(),
                                         attn_mask=None, scale=D ** -0.5)
        assert float((got.float() - ref.float()).abs().max()) <= 2e-2 * float(ref.float().abs().max())


def test_graph_replay_streams_and_two_graphs():
    """One decode step captured twice, the graphs replayed on two streams at once with changed inputs."""
    D, H, G, page = 128, 2, 4, 64
    codec, scale = make_paged_codec(D, 8, H, seed=12)
    cos, sin = paged.rotary_table(4096, D, device=DEV)
    sides = []
    for side in range(2):
        cache, q, table, n, pt = _attention_case(codec, H, G, 3, 1, [700, 5, 64], 200, page, torch.bfloat16, seed=side)
        k, v = _randn(3, H, 1, D, seed=side + 40, dtype=torch.bfloat16), _randn(3, H, 1, D, seed=side + 50, dtype=torch.bfloat16)
        pos = n.long()[:, None] - 1

        def step(cache=cache, q=q, table=table, n=n, pt=pt, k=k, v=v, pos=pos):
            qr, kr = paged.norm_rotate(q, k, cos=cos, sin=sin, positions=pos + 200)
            paged.append_paged(cache, kr, v, cache.slots(table, pos))
            return paged.paged_attention(cache, qr, table, n, prefix_table=pt, prefix_len=200), qr

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, qr = step()
        sides.append((g, out, qr, cache, q, k, table, n, pt, step))       # step holds the graph's other inputs
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(3):
        for g, out, qr, cache, q, k, *_ in sides:
            q.copy_(_randn(*q.shape, seed=100 + round_))
            k.copy_(_randn(*k.shape, seed=200 + round_))
        torch.cuda.synchronize()
        for s, side in zip(streams, sides):
            with torch.cuda.stream(s):
                side[0].replay()
        torch.cuda.synchronize()
        for g, out, qr, cache, q, k, table, n, pt, _ in sides:
            _check_attention(out, cache, qr, table, n, pt, 200)


def test_pool_offsets_beyond_32_bits():
    """A value pool of more than 2^32 bytes (and 2^31 elements): its last page is appended to and read."""
    D, H, page = 128, 8, 128
    codec, scale = make_paged_codec(D, 8, H, seed=13)
    pages = 2 ** 31 // (H * page * D) + 8
    cache = SunShapePagedCache(codec, torch.zeros(pages, H, page, 16, dtype=torch.uint8, device=DEV),
                               torch.empty(pages, H, page, D, dtype=torch.bfloat16, device=DEV))
    k, v = _randn(1, H, 5, D, seed=1, dtype=torch.bfloat16), _randn(1, H, 5, D, seed=2, dtype=torch.bfloat16)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV)
    paged.append_paged(cache, k, v, cache.slots(table, torch.arange(5, device=DEV)[None]))
    small = SunShapePagedCache(codec, cache.indices[-1:].contiguous(), cache.values[-1:].contiguous())
    idx, _ = encode64(codec, k.double().cpu())
    assert torch.equal(small.indices[0, :, :5].cpu(), idx[0].to(torch.uint8))
    assert torch.equal(small.values[0, :, :5].cpu(), v[0].cpu())
    q = _randn(1, H * 2, 1, D, seed=3, dtype=torch.bfloat16)
    n = torch.tensor([5], dtype=torch.int32, device=DEV)
    got = paged.paged_attention(cache, q, table, n)
    _check_attention(got, small, q, torch.zeros_like(table), n, None, 0)


# --------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    codec, _ = make_paged_codec(64, 8, 2, seed=1)
    cache = SunShapePagedCache.allocate(codec, 4, 2, page_size=16)
    q = _randn(2, 4, 1, 64, seed=1, dtype=torch.bfloat16)
    k = _randn(2, 2, 1, 64, seed=1, dtype=torch.bfloat16)
    table, n = torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    slots = torch.arange(2, device=DEV)[:, None]
    cos, sin = paged.rotary_table(8, 64, device=DEV)
    pos = torch.zeros(2, 1, dtype=torch.long, device=DEV)

    def no(match, f, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            f(*a, **kw)

    no("needs cos, sin and positions", paged.norm_rotate, q, cos=cos)
    no("fp32 tables", paged.norm_rotate, q, cos=cos.half(), sin=sin.half(), positions=pos)
    no("rotate 64 elements", paged.norm_rotate, q[..., :32], cos=cos, sin=sin, positions=pos)
    no("int32 or int64", paged.norm_rotate, q, cos=cos, sin=sin, positions=pos.float())
    no("positions must have shape", paged.norm_rotate, q, cos=cos, sin=sin, positions=pos[:, :0])
    no("unit stride", paged.norm_rotate, q.transpose(1, 3))
    no("norm weights", paged.norm_rotate, q, q_weight=cos[0])
    no("agree in dtype", paged.norm_rotate, q, k.float())
    no("CUDA", paged.norm_rotate, q.cpu())
    no("kv_heads and value_dim", paged.append_paged, cache, k, k[..., :32], slots)
    no("cache's dtype", paged.append_paged, cache, k.half(), k.half(), slots)
    no("slots must be", paged.append_paged, cache, k, k, slots.int())
    no("head_dim", paged.append_paged, cache, k[..., :32], k, slots)
    no("divisible by kv-head", paged.paged_attention, cache, q[:, :3], table, n)
    no("page_table must be", paged.paged_attention, cache, q, table.long(), n)
    no("seq_lens must be", paged.paged_attention, cache, q, table, n[:1])
    no("needs a prefix_table", paged.paged_attention, cache, q, table, n, prefix_len=3)
    no("hold prefix_len tokens", paged.paged_attention, cache, q, table, n, prefix_len=17, prefix_table=n[:1])
    no("cache's dtype", paged.paged_attention, cache, q.half(), table, n)
    no("out must be", paged.paged_attention, cache, q, table, n, out=q[:1])
    no("page_size", SunShapePagedCache.allocate, codec, 4, 2, page_size=8)
    no("bf16 or f16", SunShapePagedCache.allocate, codec, 4, 2, dtype=torch.float32)
    no("codebooks for", SunShapePagedCache.allocate, codec, 4, 3)
    odd, _ = make_paged_codec(96, 8, 2, seed=1)
    wide = SunShapePagedCache.allocate(odd, 4, 2, page_size=16)
    no("head_dim 64 or 128", paged.paged_attention, wide, _randn(2, 4, 1, 96, seed=1, dtype=torch.bfloat16), table, n)
