"""Paged attention in 64 bits with the error that its roundings allow, down to the subnormal range of fp16."""
import math

import torch

from tests.paged_reference import HALF_STEP, dense_tokens


def attention_bounds(cache, q, table, lens, prefix_table=None, prefix_len=0, scale=None, causal=True, exact_scores=False):
    """(output, bound, largest error of a score) in 64 bits.

    A key element is off by half a step of fp16, 2^-11 of itself or, below 2^-14 of the scaled codebook's largest norm,
    2^-25 of the scale's unit, which is at most twice the largest codeword norm C: 2^-24 C (C is 1/2 at least where the codec
    has dense blocks, whose scale is at most 1).  A query element (fp16 and bf16
    have no more bits than fp16) is off by 2^-25 of the row's unit where it is below 2^-14 of it: 2^-25 max |q|.  So
        |ds| <= scale * sum_d (2^-11 |q_d k_d| + 2^-24 C |q_d| + 2^-25 max|q| |k_d|) =: e
    (and 2^-10 of that for terms of second order and fp32 sums).  A weight is then off by a factor within exp(2 e), by
    half a step of the cache's dtype, 2^-20 for the exponential, and in fp16 by 2^-25 of 2^-7 of the largest weight:
    2^-32 each.  ``exact_scores``: all elements and products are fp16 and fp32 numbers, e is 0."""
    B, Hq, L, D = q.shape
    H = cache.kv_heads
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, Hq, L, cache.value_dim, dtype=torch.float64)
    bound, worst = torch.zeros_like(out), 0.0
    half = HALF_STEP[cache.dtype]
    cents = cache.codec.centroids.double().cpu()
    cents = cents if cents.ndim == 4 else cents[None]
    for h in range(H):
        C = max(float(cents[h % cents.shape[0]].norm(dim=-1).max()), 0.0 if cache.heavy is None else 0.5)
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
                ak, aq = k[:m].abs(), qq.abs()
                e = 2.0 ** -11 * (aq @ ak.T) + 2.0 ** -24 * C * aq.sum(-1, keepdim=True)
                e = e + 2.0 ** -25 * aq.amax(-1, keepdim=True) * ak.sum(-1)
                e = 0 * e if exact_scores else (1 + 2.0 ** -10) * abs(scale) * e
                e = e.amax(-1, keepdim=True)
                worst = max(worst, float(e.max()))
                o, a = w @ v[:m], w @ v[:m].abs()
                low = m * 2.0 ** -32 * v[:m].abs().amax(0) + 2.0 ** -25 if cache.dtype == torch.float16 else 1e-30
                out[b, h * G:(h + 1) * G, l] = o
                bound[b, h * G:(h + 1) * G, l] = (torch.expm1(2 * e) + half + 2.0 ** -20) * a + half * o.abs() + low
    return out, bound, worst
