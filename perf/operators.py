"""Cases of the paged-serving operators: head norms with rotation, appending to the paged compressed cache, and
attention over it, with or without a prefix that the whole batch shares.

``run`` computes each operator in elementary torch operations where ``own`` is false, and through
``sunshape_b200.paged`` where it is true.  Both write or return the same tensors.  Shapes follow the decode
configurations of ``sunshape_b200.workloads`` (14/2, 32/8 and 64/8 heads, head_dim 64 and 128, block_dim 8 and 4,
four dense blocks in the mixed codec) with batch and lengths varied around them.

Formulas (x a query or key row of one head, pairs (i, j) = (i, i + R/2), or (2i, 2i + 1) where ``interleaved``,
of its first R elements, c = cos[pos, i], s = sin[pos, i], w the norm's weight):

* norm:      y = x * w / sqrt(mean(x^2) + eps)
* rotation:  z_i = y_i c - y_j s,  z_j = y_j c + y_i s
* append:    index[slot, b] = argmin_k |z[perm]_b - C_b[k]|^2 (lowest k on ties); a dense block of the mixed codec
             keeps z[perm]_b itself and index 0; value[slot] = v;  slots of -1 are left out
* attention: o = sum_t softmax_t(scale <q, khat_t>) v_t,  khat_t[perm] = the codewords (or dense blocks) of token t;
             tokens are the shared prefix's and then the sequence's own; query l of L sees all but the last
             L - 1 - l of them; a row that sees none is zero
"""
import math

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


# ----------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of 8 sequences, 64/8 heads: latency
        dict(name="norm_rotate_step", op="norm_rotate", batch=8, length=1, q_heads=64, kv_heads=8, dim=128, rot=128,
             norm=True, interleaved=False, dtype="bf16"),
        # prompts of two sequences, 32/8 heads: bandwidth
        dict(name="norm_rotate_prompt", op="norm_rotate", batch=2, length=8192, q_heads=32, kv_heads=8, dim=128,
             rot=128, norm=True, interleaved=False, dtype="bf16"),
        # a model without head norms that rotates half of each head in neighbouring pairs; an odd length
        dict(name="rotate_partial_odd", op="norm_rotate", batch=3, length=1777, q_heads=14, kv_heads=2, dim=64,
             rot=32, norm=False, interleaved=True, dtype="f16"),
        # one decode step of 64 sequences: 64 new tokens of 8 heads
        dict(name="append_step", op="append", batch=64, length=1, kv_heads=8, dim=128, block=8, heavy=0, rot=128,
             interleaved=False, page=64, dtype="bf16"),
        # a prompt of 4096 tokens, block_dim 4 (32 blocks a head)
        dict(name="append_prompt", op="append", batch=1, length=4096, kv_heads=8, dim=128, block=4, heavy=0, rot=128,
             interleaved=False, page=64, dtype="bf16"),
        # five prompts of unequal length in one padded batch, mixed codec with four dense blocks, pages of 16
        dict(name="append_ragged_mixed", op="append", batch=5, length=1111, kv_heads=8, dim=128, block=8, heavy=4,
             rot=128, interleaved=False, page=16, dtype="bf16"),
        # one short sequence of a small model: latency
        dict(name="attention_small", op="attention", batch=1, length=1, q_heads=14, kv_heads=2, dim=64, block=8,
             heavy=0, page=16, prefix=0, longest=517, shortest=517, dtype="f16"),
        # an ordinary serving batch: 64 sequences of 1k to 8k tokens
        dict(name="attention_batch", op="attention", batch=64, length=1, q_heads=32, kv_heads=8, dim=128, block=8,
             heavy=0, page=64, prefix=0, longest=8192, shortest=1000, dtype="bf16"),
        # the long-context step: 8 sequences of 128k tokens
        dict(name="attention_long", op="attention", batch=8, length=1, q_heads=64, kv_heads=8, dim=128, block=8,
             heavy=0, page=64, prefix=0, longest=131072, shortest=130001, dtype="bf16"),
        # four query tokens a step (drafted tokens being checked), block_dim 4, pages of 32
        dict(name="attention_drafted", op="attention", batch=16, length=4, q_heads=32, kv_heads=8, dim=128, block=4,
             heavy=0, page=32, prefix=0, longest=6000, shortest=3, dtype="bf16"),
        # 64 requests behind one document of 32k tokens, 8 queries a KV head
        dict(name="attention_shared", op="attention", batch=64, length=1, q_heads=64, kv_heads=8, dim=128, block=8,
             heavy=0, page=64, prefix=32768, longest=700, shortest=1, dtype="bf16"),
        # 32 requests behind a prompt of 10k tokens, mixed codec; the prefix ends inside a page
        dict(name="attention_shared_mixed", op="attention", batch=32, length=1, q_heads=32, kv_heads=8, dim=128,
             block=8, heavy=4, page=64, prefix=10007, longest=1500, shortest=0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rotate", "append", "attention", "attention"])
    dim = rng.choice([64, 128, 128])
    q_heads, kv_heads = rng.choice([(14, 2), (32, 8), (64, 8), (16, 16), (8, 1), (24, 4)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "norm_rotate":
        tokens = _log(rng, 1, 16384)
        batch = rng.choice([1, 2, 3, 8])
        return dict(op=op, batch=batch, length=max(1, min(8192, tokens // batch)), q_heads=q_heads,
                    kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2]), norm=rng.random() < 0.7,
                    interleaved=rng.random() < 0.3, dtype=dtype)
    block = rng.choice([8, 8, 4])
    heavy = rng.choice([0, 0, 2, 4])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        tokens = _log(rng, 1, 4096)
        batch = rng.choice([1, 3, 5, 16])
        return dict(op=op, batch=batch, length=max(1, tokens // batch), kv_heads=min(kv_heads, 8), dim=dim,
                    block=block, heavy=heavy, rot=rng.choice([dim, dim, dim // 2, 0]),
                    interleaved=rng.random() < 0.3, page=page, dtype=dtype)
    batch, length = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5])
    prefix = rng.choice([0, 0, 1]) * _log(rng, 100, min(40000, 120_000_000 // (batch * length * q_heads)))
    longest = _log(rng, 1, max(2, min(100000, (2 if prefix else 40) * 100000 // (batch * kv_heads))))
    return dict(op=op, batch=batch, length=length, q_heads=q_heads, kv_heads=kv_heads, dim=dim,
                block=block, heavy=heavy, page=page, prefix=prefix, longest=longest,
                shortest=rng.randint(0, longest), dtype=dtype)


def _lengths(case):
    """The sequences' own token counts: spread between the case's shortest and longest, in a fixed order."""
    lo, hi, n = case["shortest"], case["longest"], case["batch"]
    return [hi - (i * 7919 % max(1, n)) * (hi - lo) // max(1, n - 1) for i in range(n)]


def _new_tokens(case):
    """How many of the padded batch's rows each sequence appends."""
    n = case["length"]
    return [max(1, n - i * 13 % max(1, n)) for i in range(case["batch"])]


def work(case):
    e = 2
    if case["op"] == "norm_rotate":
        rows = case["batch"] * case["length"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * rows * case["dim"] * e + case["batch"] * case["length"] * (8 + 4 * case["rot"]),
                "flops": rows * (4 * case["dim"] * case["norm"] + 3 * case["rot"])}
    nb, D, H = case["dim"] // case["block"], case["dim"], case["kv_heads"]
    codebooks = H * (nb - case["heavy"]) * 256 * case["block"] * 4
    if case["op"] == "append":
        rows = sum(_new_tokens(case)) * H
        return {"bytes": rows * (D * e + 2 * D * e + nb + case["heavy"] * case["block"] * e) + codebooks
                + case["batch"] * case["length"] * 16 + sum(_new_tokens(case)) * 4 * case["rot"],
                "flops": rows * (3 * case["rot"] + (nb - case["heavy"]) * 256 * 2 * case["block"])}
    tokens = sum(_lengths(case))
    rows = case["length"] * case["q_heads"]
    return {"bytes": (tokens + case["prefix"]) * H * (nb + case["heavy"] * case["block"] * e + D * e) + codebooks
            + 2 * case["batch"] * rows * D * e + 4 * (tokens + case["prefix"]) // case["page"],
            "flops": 4 * D * rows * (tokens + case["batch"] * case["prefix"])}


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _table(n, rot):
    """cos and sin [n, rot/2] of n positions, angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / max(rot, 1))
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _codec_tensors(case, g, scale):
    """Permutation, per-head codebooks of keys' blocks (channels of unequal scale) and the dense blocks' mask."""
    D, bd, H = case["dim"], case["block"], case["kv_heads"]
    nb = D // bd
    perm = torch.randperm(D, generator=g, device=DEV)
    cents = (_normal(g, H, 256, D) * scale)[..., perm].view(H, 256, nb, bd).transpose(1, 2).contiguous()
    mask = torch.zeros(nb, dtype=torch.bool, device=DEV)
    if case["heavy"]:
        mass = (scale[perm] ** 2).view(nb, bd).sum(1)
        mask[torch.argsort(mass, descending=True)[:case["heavy"]]] = True
        cents[:, mask] = 0
    return perm, cents, mask


def _pools(case, g, pages, scale, perm, mask):
    """Pages that hold tokens already: indices, values and dense key blocks."""
    H, D, bd, ps, dt = case["kv_heads"], case["dim"], case["block"], case["page"], _DT[case["dtype"]]
    nb = D // bd
    idx = torch.randint(0, 256, (pages, H, ps, nb), generator=g, device=DEV, dtype=torch.uint8)
    val = torch.empty(pages, H, ps, D, device=DEV, dtype=dt).normal_(generator=g)
    heavy = None
    if case["heavy"]:
        idx[..., mask] = 0
        heavy = torch.empty(pages, H, ps, case["heavy"], bd, device=DEV, dtype=dt).normal_(generator=g)
        heavy *= scale[perm].view(nb, bd)[mask].to(dt)
    return idx, val, heavy


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    B, L, D, dt = case["batch"], case["length"], case["dim"], _DT[case["dtype"]]
    H = case["kv_heads"]
    scale = torch.exp(0.75 * _normal(g, D))
    s = dict(case=case)
    if case["op"] in ("norm_rotate", "append"):
        s["cos"], s["sin"] = _table(32768, case["rot"])
        start = torch.randint(0, 32768 - L + 1, (B, 1), generator=g, device=DEV)
        s["positions"] = start + torch.arange(L, device=DEV)
    if case["op"] == "norm_rotate":
        # a fused projection's output [B, L, heads, D], seen as [B, heads, L, D]
        s["q"] = (_normal(g, B, L, case["q_heads"], D)).to(dt).transpose(1, 2)
        s["k"] = (_normal(g, B, L, H, D) * scale).to(dt).transpose(1, 2)
        s["qw"] = (1 + 0.2 * _normal(g, D)).to(dt) if case["norm"] else None
        s["kw"] = (1 + 0.2 * _normal(g, D)).to(dt) if case["norm"] else None
        return s
    s["perm"], s["cents"], s["mask"] = _codec_tensors(case, g, scale)
    ps = case["page"]
    if case["op"] == "append":
        s["k"] = (_normal(g, B, L, H, D) * scale).to(dt).transpose(1, 2)
        s["v"] = (_normal(g, B, L, H, D)).to(dt).transpose(1, 2)
        each = -(-L // ps) + 1
        s["indices"], s["values"], s["heavy"] = _pools(case, g, B * each + 2, scale, s["perm"], s["mask"])
        table = torch.randperm(B * each + 2, generator=g, device=DEV)[:B * each].view(B, each)
        at = torch.randint(0, ps, (B, 1), generator=g, device=DEV) + torch.arange(L, device=DEV)   # mid-page starts
        slots = table.gather(1, at // ps) * ps + at % ps
        new = torch.tensor(_new_tokens(case), device=DEV)[:, None]
        s["slots"] = torch.where(torch.arange(L, device=DEV) < new, slots, slots.new_full((), -1))
    else:
        lens = _lengths(case)
        each = max(1, -(-max(lens) // ps))
        first = -(-case["prefix"] // ps)
        total = B * each + first + 1
        s["indices"], s["values"], s["heavy"] = _pools(case, g, total, scale, s["perm"], s["mask"])
        order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        s["prefix_table"] = order[:first].contiguous() if first else None
        s["page_table"] = order[first:first + B * each].view(B, each).contiguous()
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["q"] = _normal(g, B, case["q_heads"], L, D).to(dt)
    if own:
        from sunshape_b200 import SunShapeBlockCodec
        from sunshape_b200.paged import SunShapePagedCache

        codec = SunShapeBlockCodec(D, case["block"], 256, device=torch.device(DEV), kv_heads=H,
                                   mode="profileperm_mixed_precision" if case["heavy"] else "profileperm_baseline")
        codec.permutation.copy_(s["perm"])
        codec.inv_permutation[s["perm"]] = torch.arange(D, device=DEV)
        codec.centroids.copy_(s["cents"])
        codec.mixed_high_precision_blocks.copy_(s["mask"])
        codec.invalidate()
        s["cache"] = SunShapePagedCache.from_pools(codec, s["indices"], s["values"], s["heavy"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _rotated(x, cos, sin, rot, interleaved):
    """Rows [..., L, D] with their first ``rot`` elements rotated; cos, sin [B, 1, L, rot/2]."""
    if not rot:
        return x
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, rest), -1)


def _plain_norm_rotate(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]

    def one(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        return _rotated(y, cos, sin, c["rot"], c["interleaved"]).to(x.dtype)

    return one(s["q"], s["qw"]), one(s["k"], s["kw"])


def _plain_append(s):
    c = s["case"]
    H, D, bd = c["kv_heads"], c["dim"], c["block"]
    nb = D // bd
    keep = s["slots"] >= 0
    slot = s["slots"][keep]
    page, row = slot // c["page"], slot % c["page"]
    # rotated in 64 bits: the nearest codeword is decided next to borders between codewords
    cos, sin = s["cos"][s["positions"]][:, None].double(), s["sin"][s["positions"]][:, None].double()
    z = _rotated(s["k"].double(), cos, sin, c["rot"], c["interleaved"])
    z = z.transpose(1, 2)[keep][..., s["perm"]].view(-1, H, nb, 1, bd)
    dist = (z - s["cents"].double()).square_().sum(-1)                      # [tokens, H, nb, 256]
    idx = dist.argmin(-1).masked_fill(s["mask"], 0)
    s["indices"][page, :, row] = idx.to(torch.uint8)
    s["values"][page, :, row] = s["v"].transpose(1, 2)[keep]
    if s["heavy"] is not None:
        s["heavy"][page, :, row] = z[..., 0, :][:, :, s["mask"]].to(s["heavy"].dtype)
    return {"indices": s["indices"], "values": s["values"]} | ({} if s["heavy"] is None else {"heavy": s["heavy"]})


def _plain_tokens(s, table):
    """Keys (in the permuted basis) and values [..., H, T, D] in 32 bits of the pages that ``table`` names."""
    c = s["case"]
    H, D, bd = c["kv_heads"], c["dim"], c["block"]
    nb = D // bd
    idx = s["indices"][table.long()].transpose(-4, -3).flatten(-3, -2).long()     # [..., H, T, nb]
    head, block = torch.arange(H, device=DEV)[:, None, None], torch.arange(nb, device=DEV)
    k = s["cents"][head, block, idx]                                              # [..., H, T, nb, bd]
    if s["heavy"] is not None:
        k[..., s["mask"], :] = s["heavy"][table.long()].transpose(-5, -4).flatten(-4, -3).float()
    v = s["values"][table.long()].transpose(-4, -3).flatten(-3, -2).float()
    return k.flatten(-2), v


def _plain_attention(s):
    c = s["case"]
    B, L, Hq, H, D = c["batch"], c["length"], c["q_heads"], c["kv_heads"], c["dim"]
    G = Hq // H
    q = s["q"].float()[..., s["perm"]].view(B, H, G, L, D) / math.sqrt(D)
    k, v = _plain_tokens(s, s["page_table"])
    T = k.shape[-2]
    sc = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).view(B, H, G, L, T)
    # query l sees the sequence's tokens but the last L - 1 - l
    seen = s["seq_lens"].long()[:, None] - torch.arange(L - 1, -1, -1, device=DEV)
    sc = sc.masked_fill(torch.arange(T, device=DEV) >= seen[:, None, None, :, None], -math.inf)
    v = v.masked_fill((torch.arange(T, device=DEV) >= s["seq_lens"].long()[:, None])[:, None, :, None], 0.0)
    top = sc.amax(-1, keepdim=True)
    if c["prefix"]:
        pk, pv = (x[:, :c["prefix"]] for x in _plain_tokens(s, s["prefix_table"]))
        ps = torch.matmul(q.permute(1, 0, 2, 3, 4).reshape(H, B * G * L, D), pk.transpose(-1, -2))
        ps = ps.view(H, B, G, L, -1).transpose(0, 1)
        top = torch.maximum(top, ps.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)
    e = torch.exp(sc - top)
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.flatten(2, 3), v).view(B, H, G, L, D)
    if c["prefix"]:
        e = torch.exp(ps - top)
        total = total + e.sum(-1, keepdim=True)
        o = o + torch.matmul(e.transpose(0, 1).reshape(H, B * G * L, -1), pv).view(H, B, G, L, D).transpose(0, 1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.view(B, Hq, L, D).to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        from sunshape_b200 import paged

        if c["op"] == "norm_rotate":
            return paged.norm_rotate(s["q"], s["k"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS, cos=s["cos"],
                                     sin=s["sin"], positions=s["positions"], interleaved=c["interleaved"])
        if c["op"] == "append":
            rotation = dict(cos=s["cos"], sin=s["sin"], positions=s["positions"]) if c["rot"] else {}
            paged.append_paged(s["cache"], s["k"], s["v"], s["slots"], interleaved=c["interleaved"], **rotation)
            return ({"indices": s["indices"], "values": s["values"]}
                    | ({} if s["heavy"] is None else {"heavy": s["heavy"]}))
        return paged.paged_attention(s["cache"], s["q"], s["page_table"], s["seq_lens"],
                                     prefix_table=s["prefix_table"], prefix_len=c["prefix"],
                                     scale=1.0 / math.sqrt(c["dim"]))
    return {"norm_rotate": _plain_norm_rotate, "append": _plain_append, "attention": _plain_attention}[c["op"]](s)


# ------------------------------------------------------------------------------------------ values in 64 bits
def _exact_rotation(x, s, c):
    """x [B, H, L, D] in 64 bits: each pair as a complex number times e^(i angle)."""
    R = c["rot"]
    if not R:
        return x
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]
    z = x.clone()
    if c["interleaved"]:
        z[..., :R] = torch.view_as_real(torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], R // 2, 2).contiguous())
                                        * turn).reshape(*x.shape[:-1], R)
    else:
        w = torch.complex(x[..., :R // 2], x[..., R // 2:R].contiguous()) * turn
        z[..., :R // 2], z[..., R // 2:R] = w.real, w.imag
    return z


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "norm_rotate":
        def one(x, w):
            y = x.double()
            if w is not None:
                y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / c["dim"] + EPS) * w.double()
            return _exact_rotation(y, s, c)
        return one(s["q"], s["qw"]), one(s["k"], s["kw"])
    D, H, ps = c["dim"], c["kv_heads"], c["page"]
    nb, bd = D // c["block"], c["block"]
    if c["op"] == "append":
        values = s["values"].double()
        heavy = None if s["heavy"] is None else s["heavy"].double()
        z = _exact_rotation(s["k"].double(), s, c)
        for b in range(c["batch"]):
            n = _new_tokens(c)[b]
            page, row = s["slots"][b, :n] // ps, s["slots"][b, :n] % ps
            for h in range(H):
                values[page, h, row] = s["v"][b, h, :n].double()
                if heavy is not None:
                    blocks = z[b, h, :n].index_select(-1, s["perm"]).view(n, nb, bd)
                    heavy[page, h, row] = blocks[:, s["mask"].nonzero().flatten()]
        return {"indices": None, "values": values} | ({} if heavy is None else {"heavy": heavy})
    B, L, G = c["batch"], c["length"], c["q_heads"] // H
    inv = torch.empty_like(s["perm"])
    inv[s["perm"]] = torch.arange(D, device=DEV)
    out = torch.zeros(B, c["q_heads"], L, D, device=DEV, dtype=torch.float64)

    def tokens(table, n, h):
        """Keys in the model's basis and values of one head's first n tokens."""
        p = table.long()[:-(-n // ps)]
        idx = s["indices"][p, h].reshape(-1, nb)[:n].long()
        k = torch.stack([s["cents"][h, b].double()[idx[:, b]] for b in range(nb)], 1)
        if s["heavy"] is not None:
            k[:, s["mask"]] = s["heavy"][p, h].reshape(-1, c["heavy"], bd)[:n].double()
        return k.reshape(n, D)[:, inv], s["values"][p, h].reshape(-1, D)[:n].double()

    for h in range(H):
        shared = tokens(s["prefix_table"], c["prefix"], h) if c["prefix"] else None
        for b, n in enumerate(_lengths(c)):
            k, v = tokens(s["page_table"][b], n, h)
            if shared is not None:
                k, v = torch.cat((shared[0], k)), torch.cat((shared[1], v))
            for l in range(L):
                m = c["prefix"] + max(0, n - (L - 1 - l))
                if m:
                    logits = s["q"][b, h * G:(h + 1) * G, l].double() @ k[:m].T / math.sqrt(D)
                    out[b, h * G:(h + 1) * G, l] = torch.softmax(logits, -1) @ v[:m]
    return out
