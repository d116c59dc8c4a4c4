"""Plain 64-bit implementations of the paged-serving operators, row by row, and the error bounds that the kernels'
roundings allow."""
import math

import numpy as np
import torch

from tests.helpers import make_codec

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rotate64(x, cos, sin, pos, interleaved):
    """x [B, H, L, D] (any dtype), pos [B, L] -> the rotated rows in 64 bits."""
    x = x.double().cpu()
    if cos is None:
        return x
    half = cos.shape[1]
    c, s = cos.double().cpu()[pos.cpu().long()][:, None], sin.double().cpu()[pos.cpu().long()][:, None]
    out = x.clone()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def norm64(x, w, eps):
    x = x.double().cpu()
    if w is None:
        return x
    return x * w.double().cpu() / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def make_paged_codec(D, bd, H, *, heavy=0, C=256, shared=False, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    nb = D // bd
    mask = torch.zeros(nb, dtype=torch.bool)
    mask[torch.randperm(nb, generator=g)[:heavy]] = True
    scale = torch.exp(0.75 * torch.randn(D, generator=g))
    perm = torch.randperm(D, generator=g)
    cents = (torch.randn(1 if shared else H, C, D, generator=g) * scale)[..., perm].view(-1, C, nb, bd).transpose(1, 2)
    cents = cents.contiguous()
    cents[:, mask] = 0
    codec = make_codec(perm, cents[0] if shared else cents, mask, D, bd, C, device)
    return codec, scale


def encode64(codec, z):
    """Nearest codewords of rotated keys z [B, H, L, D] (64 bits): [B, H, L, nb], lowest index on ties."""
    B, H, L, D = z.shape
    cents = codec.centroids.double().cpu()
    cents = cents.expand(H, *cents.shape) if cents.ndim == 3 else cents
    zp = z[..., codec.permutation.cpu()].view(B, H, L, codec.n_blocks, 1, codec.block_dim)
    d = (zp - cents[:, None]).square().sum(-1)
    idx = torch.from_numpy(np.argmin(d.numpy(), -1))
    return idx.masked_fill(codec.mixed_high_precision_blocks.cpu(), 0), zp[..., 0, :]


def dense_tokens(cache, pages, n, h):
    """Keys (model basis) and values of one head's first n tokens in 64 bits."""
    c = cache.codec
    p = pages.cpu().long()[: -(-n // cache.page_size)]
    idx = cache.indices.cpu()[p, h].reshape(-1, c.n_blocks)[:n].long()
    cents = c.centroids.double().cpu()
    cents = cents if cents.ndim == 3 else cents[h]
    k = cents[torch.arange(c.n_blocks), idx]
    if cache.heavy is not None:
        mask = c.mixed_high_precision_blocks.cpu()
        k[:, mask] = cache.heavy.cpu()[p, h].reshape(-1, int(mask.sum()), c.block_dim)[:n].double()
    return k.reshape(n, c.head_dim)[:, c.inv_permutation.cpu()], cache.values.cpu()[p, h].reshape(-1, cache.value_dim)[:n].double()


def attention64(cache, q, table, lens, prefix_table=None, prefix_len=0, scale=None, causal=True):
    """(output, bound) in 64 bits.  bound: what the roundings that paged_attention documents allow, element by element.

    Keys and queries in fp16: |ds| <= 2 * 2^-11 * scale * sum |q_d k_d| =: e (one half step each; fp32 sums are below
    2^-14 of that).  A weight is then off by a factor within exp(2 e) of its share (its own error and the normaliser's), times
    a half step of the cache's dtype for the rounded weight and 2^-20 for the exponential; the output rounds once more."""
    B, Hq, L, D = q.shape
    H = cache.kv_heads
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, L, cache.value_dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    half = HALF_STEP[cache.dtype]
    for h in range(H):
        shared = dense_tokens(cache, prefix_table, prefix_len, h) if prefix_len else None
        for b in range(B):
            n = int(lens[b])
            k, v = dense_tokens(cache, table[b], n, h)
            if shared is not None:
                k, v = torch.cat((shared[0], k)), torch.cat((shared[1], v))
            for l in range(L):
                m = prefix_len + (max(0, n - (L - 1 - l)) if causal else n)
                if m == 0:
                    continue
                qq = q[b, h * G:(h + 1) * G, l].double().cpu()
                w = torch.softmax(scale * (qq @ k[:m].T), -1)
                e = (2 * 2.0 ** -11 * abs(scale) * (qq.abs() @ k[:m].abs().T)).amax(-1, keepdim=True)
                o, a = w @ v[:m], w @ v[:m].abs()
                out[b, h * G:(h + 1) * G, l] = o
                bound[b, h * G:(h + 1) * G, l] = (torch.expm1(2 * e) + half + 2.0 ** -20) * a + half * o.abs() + 1e-30
    return out, bound
