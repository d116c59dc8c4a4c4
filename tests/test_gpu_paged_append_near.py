"""Keys whose two nearest codewords are almost equally far, at every margin that the search's steps have to tell apart."""
import pytest
import torch

from sunshape_b200 import paged
from sunshape_b200.codec import SunShapeBlockCodec
from sunshape_b200.paged import SunShapePagedCache
from tests.paged_reference import encode64

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bd", [2, 4, 8])
@pytest.mark.parametrize("size", [1e-3, 1.0, 300.0])
def test_two_nearest_codewords(bd, dtype, size):
    """128 keys a block and, for each, two codewords at random places that are the nearest by far, their distances apart
    by 2^-6 to 2^-30 of themselves: the index is that of the 64-bit minimum."""
    H, D = 4, 128
    nb, L = D // bd, 128
    g = torch.Generator().manual_seed(bd)
    key = (size * torch.randn(H, nb, L, bd, generator=g)).to(dtype)
    z = key.double()
    # distinct keys, and codewords closer to theirs than to any other one
    apart = torch.cdist(z, z) + torch.eye(L) * 1e9
    radius = (0.3 * apart.amin(-1, keepdim=True)).clamp(min=1e-6 * size)

    def direction():
        u = torch.randn(H, nb, L, bd, generator=g, dtype=torch.float64)
        return u / u.norm(dim=-1, keepdim=True)

    margin = torch.exp2(-6 - 24 * torch.rand(H, nb, L, 1, generator=g, dtype=torch.float64))
    margin *= torch.randn(H, nb, L, 1, generator=g, dtype=torch.float64).sign()
    pair = torch.stack((z + radius * direction(), z + radius * (1 + margin) * direction()), 3)     # [H, nb, L, 2, bd]
    where = torch.rand(H, nb, 256, generator=g).argsort(-1)[..., None].expand(-1, -1, -1, bd)
    cents = torch.empty(H, nb, 256, bd).scatter_(2, where, pair.flatten(2, 3).float())
    codec = SunShapeBlockCodec(D, bd, 256, device=torch.device(DEV), kv_heads=H)
    codec.centroids.copy_(cents)
    codec.invalidate()
    cache = SunShapePagedCache.allocate(codec, L // 16, H, page_size=16, dtype=dtype)
    k = key.transpose(1, 2).reshape(1, H, L, D).to(DEV)
    cache.append(k, k, torch.arange(L, device=DEV)[None])
    want, _ = encode64(codec, k.double().cpu())
    got = cache.indices.cpu().transpose(0, 1).flatten(1, 2)
    assert torch.equal(got, want[0].to(torch.uint8))
    # both codewords of a pair occur, at all margins
    first = where[..., 0].reshape(H, nb, L, 2)[..., 0].transpose(1, 2)
    share = (got.long() == first).float().mean()
    assert 0.3 < float(share) < 0.7 and paged.paged_error(DEV) is None


@pytest.mark.parametrize("bd", [2, 4, 8])
@pytest.mark.parametrize("C", [1, 70, 255])
def test_keys_where_missing_codewords_are_kept(bd, C):
    """Codebooks of fewer than 256 codewords, keys and codewords around 1e18, where the search keeps the missing ones."""
    H, D, L = 2, 64, 48
    g = torch.Generator().manual_seed(C)
    codec = SunShapeBlockCodec(D, bd, C, device=torch.device(DEV), kv_heads=H)
    codec.centroids.copy_(1e18 * (1 + 0.5 * torch.randn(codec.centroids.shape, generator=g)))
    codec.invalidate()
    cache = SunShapePagedCache.allocate(codec, L // 16, H, page_size=16)
    k = (1e18 * (1 + 0.1 * torch.randn(1, H, L, D, generator=g))).to(torch.bfloat16).to(DEV)
    k[:, :, :4] = 1e18
    cache.append(k, k, torch.arange(L, device=DEV)[None])
    want, _ = encode64(codec, k.double().cpu())
    assert torch.equal(cache.indices.cpu().transpose(0, 1).flatten(1, 2), want[0].to(torch.uint8))
