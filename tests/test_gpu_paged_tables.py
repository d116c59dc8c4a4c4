"""Order and lifetime of what the paged kernels read of a codec: several streams, captured graphs, edits in between."""
import pytest
import torch

from sunshape_b200 import paged
from sunshape_b200.paged import SunShapePagedCache
from tests.paged_reference import attention64, encode64, make_paged_codec

pytestmark = pytest.mark.gpu
DEV = "cuda"
D, H, PAGE = 64, 2, 16


def _randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, torch.bfloat16)


def _cache(codec, seed):
    cache = SunShapePagedCache.allocate(codec, 6, H, page_size=PAGE)
    cache.indices.copy_(torch.randint(0, 256, cache.indices.shape, generator=torch.Generator().manual_seed(seed)))
    cache.values.copy_(_randn(*cache.values.shape, seed=seed))
    if cache.heavy is not None:
        cache.heavy.copy_(_randn(*cache.heavy.shape, seed=seed + 1))
    return cache


def _inputs(seed):
    table = torch.tensor([[0, 1], [3, 2]], dtype=torch.int32, device=DEV)
    return _randn(2, 2 * H, 1, D, seed=seed), table, torch.tensor([30, 17], dtype=torch.int32, device=DEV)


def _check_attention(got, cache, q, table, n):
    ref, bound = attention64(cache, q, table, n)
    assert bool(((got.double().cpu() - ref).abs() <= bound).all())


def _edit(codec):
    codec.centroids.mul_(-0.5).add_(0.25)
    codec.permutation.copy_(codec.permutation.flip(0))
    codec.inv_permutation[codec.permutation] = torch.arange(D, device=DEV)


def test_two_caches_on_two_streams():
    """Right after the caches are made, and after edits on one stream that the other one's work is ordered behind."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    codec, _ = make_paged_codec(D, 8, H, heavy=2, seed=1)
    torch.cuda.synchronize()
    caches = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            torch.cuda._sleep(20_000_000 if i == 0 else 0)
            caches.append(_cache(codec, 10 * i))
    inputs = [_inputs(5 + i) for i in range(2)]
    torch.cuda.synchronize()
    for turn in range(3):
        if turn:
            with torch.cuda.stream(streams[0]):
                torch.cuda._sleep(20_000_000)
                _edit(codec)
                edited = torch.cuda.Event()
                edited.record()
            streams[1].wait_event(edited)
            codec.invalidate()
        got = []
        for s, cache, (q, table, n) in zip(streams, caches, inputs):
            with torch.cuda.stream(s):
                got.append(cache.attention(q, table, n))
        torch.cuda.synchronize()
        for out, cache, (q, table, n) in zip(got, caches, inputs):
            _check_attention(out, cache, q, table, n)


@pytest.mark.parametrize("another_call", [False, True])
def test_graph_captured_before_an_edit(another_call):
    """A graph that was captured before ``invalidate`` replays with the edited codebooks, permutation and dense blocks,
    whatever the allocator has handed out since."""
    codec, _ = make_paged_codec(D, 8, H, heavy=2, seed=2)
    cache = _cache(codec, 3)
    q, table, n = _inputs(4)
    k = _randn(1, H, 7, D, seed=6)
    slots = 4 * PAGE + torch.arange(7, device=DEV)[None]

    def step():
        cache.append(k, k, slots)
        return cache.attention(q, table, n)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        if turn:
            _edit(codec)
            codec.mixed_high_precision_blocks.copy_(codec.mixed_high_precision_blocks.roll(1))
            codec.invalidate()
        if another_call:
            cache.attention(q, table, n)
        size = codec._paged_tables.buffer.numel()
        other = [torch.full((size,), 255, dtype=torch.uint8, device=DEV) for _ in range(8)]
        other += [torch.full((m,), 255, dtype=torch.uint8, device=DEV) for m in (8, 512, 1024) for _ in range(20)]
        graph.replay()
        torch.cuda.synchronize()
        _check_attention(out, cache, q, table, n)
        idx, _ = encode64(codec, k.double().cpu())
        assert torch.equal(cache.indices[4, :, :7].cpu(), idx[0].to(torch.uint8))
        del other


def test_graph_of_another_number_of_dense_blocks():
    """A graph captured with two dense blocks goes on with two, and its memory, when the codec gets four."""
    codec, _ = make_paged_codec(D, 8, H, heavy=2, seed=7)
    cache = _cache(codec, 3)
    q, table, n = _inputs(4)
    cache.attention(q, table, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(q, table, n)
    graph.replay()
    want = out.clone()
    codec.mixed_high_precision_blocks[(~codec.mixed_high_precision_blocks).nonzero()[:2]] = True
    codec.centroids.mul_(2)
    codec.invalidate()
    with pytest.raises(RuntimeError, match="dense blocks"):
        cache.attention(q, table, n)
    other = [torch.full((codec._paged_tables.buffer.numel(),), 255, dtype=torch.uint8, device=DEV) for _ in range(8)]
    graph.replay()
    assert torch.equal(out, want) and len(other) == 8


def test_not_derived_during_a_capture():
    """An edit during a capture is refused there, and the capture's earlier calls hold."""
    codec, _ = make_paged_codec(D, 8, H, seed=8)
    cache = _cache(codec, 3)
    q, table, n = _inputs(4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(q, table, n)
        codec.invalidate()
        with pytest.raises(RuntimeError, match="captured"):
            cache.attention(q, table, n)
    graph.replay()
    _check_attention(out, cache, q, table, n)
    _check_attention(cache.attention(q, table, n), cache, q, table, n)


def test_codec_loaded_again_and_inference_mode():
    """``load_state_dict`` renews the tables, and so does an edit outside the inference mode that they were made in."""
    with torch.inference_mode():
        codec, _ = make_paged_codec(D, 8, H, seed=9)
    codec = type(codec)(D, 8, 256, device=torch.device(DEV), kv_heads=H)
    first, _ = make_paged_codec(D, 8, H, seed=9)
    second, _ = make_paged_codec(D, 8, H, seed=10)
    codec.load_state_dict(first.state_dict())
    with torch.inference_mode():
        cache = _cache(codec, 3)
        q, table, n = _inputs(4)
        _check_attention(cache.attention(q, table, n), cache, q, table, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(q, table, n)
    codec.load_state_dict(second.state_dict())
    graph.replay()
    _check_attention(out, cache, q, table, n)
    _edit(codec)
    codec.invalidate()
    _check_attention(cache.attention(q, table, n), cache, q, table, n)
    assert paged.paged_error(DEV) is None


def test_shared_prefix_in_two_graphs():
    """The tensor-core prefix kernel, its join and the sequences' own tokens beside it, captured twice and replayed on two
    streams at once, over and over."""
    codec, _ = make_paged_codec(D, 8, H, heavy=2, seed=11)
    B, n, prefix = 20, 50, 700
    sides = []
    for side in range(2):
        cache = SunShapePagedCache.allocate(codec, 44 + 4 * B, H, page_size=PAGE)
        cache.indices.copy_(torch.randint(0, 256, cache.indices.shape, generator=torch.Generator().manual_seed(side)))
        cache.values.copy_(_randn(*cache.values.shape, seed=side))
        cache.heavy.copy_(_randn(*cache.heavy.shape, seed=side + 1))
        pt = torch.arange(44, dtype=torch.int32, device=DEV)
        table = 44 + torch.arange(4 * B, dtype=torch.int32, device=DEV).view(B, 4)
        lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
        q = _randn(B, 2 * H, 1, D, seed=side + 2)
        want = cache.attention(q, table, lens, prefix_table=pt, prefix_len=prefix)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [cache.attention(q, table, lens, prefix_table=pt, prefix_len=prefix) for _ in range(3)]
        sides.append((graph, outs, want, torch.cuda.Stream(), (cache, pt, table, lens, q)))
        ref, bound = attention64(cache, q, table, lens, pt, prefix)
        assert bool(((want.double().cpu() - ref).abs() <= bound).all())
    for _ in range(20):
        for graph, *_, stream, _ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, outs, want, _, _ in sides:
        assert all(torch.equal(out, want) for out in outs)
