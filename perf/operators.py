"""Cases of the low-bit serving operators, and their plain form in elementary torch operations.

Four operators: the block tables and slot map of a paged cache built from request lengths, the
append to (and read back from) a key/value cache held in 4 bits, the attention over that cache, and
the linear layer in 8-bit integers with a scale for each token and each output channel.

The 4-bit pool is ``uint8 [pages, kv_heads, page bytes]``; a page is a run of 16-token blocks of
``20 * head_dim`` bytes (``G = head_dim / 32`` groups of 32 channels, each with an fp16 scale and an
fp16 minimum):

  K codes   16 x head_dim/2   token row: chunk t (4 of them): for group j: channels 32j+8t .. +7
  K scales  16 x 4G           token row: for group j: (scale, minimum)
  V codes   16 x head_dim/2   token row: chunk g (8 of them): for group j: channels 32j+4g .. +3
  V scales  16 x 4G           for group j, for t (4): scales of tokens t, t+4, t+8, t+12, then minima
"""
import math

import torch

own = False

DEV = "cuda"


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a full server: one more token for each of 256 requests
        dict(name="tables_decode", op="tables", batch=256, min_cached=1, max_cached=8192, min_new=1, max_new=1, page=64),
        # prefill of a long-context batch: the slots of half a million tokens
        dict(name="tables_prefill", op="tables", batch=8, min_cached=0, max_cached=0, min_new=8192, max_new=131072,
             page=64),
        # the new keys and values of a decode step of 64 requests
        dict(name="append_decode", op="append", tokens=64, padding=0, heads_k=8, dim=128, page=64),
        # the keys and values of a prefill of 8 x 4096 tokens
        dict(name="append_prefill", op="append", tokens=32768, padding=0, heads_k=8, dim=128, page=64),
        # a handful of short requests: latency
        dict(name="attn_short", op="attn", batch=4, heads_q=28, heads_k=4, dim=128, min_q=1, max_q=1, min_kv=37,
             max_kv=1000, page=16, masked=False),
        # one request with a long context
        dict(name="attn_long", op="attn", batch=1, heads_q=32, heads_k=8, dim=128, min_q=1, max_q=1, min_kv=131072,
             max_kv=131072, page=64, masked=False),
        # a full server: 64 requests of mixed lengths
        dict(name="attn_server", op="attn", batch=64, heads_q=24, heads_k=8, dim=128, min_q=1, max_q=1, min_kv=512,
             max_kv=8192, page=64, masked=False),
        # several new tokens a request (drafted tokens to verify, a short prompt), with masked keys
        dict(name="attn_several", op="attn", batch=8, heads_q=16, heads_k=4, dim=64, min_q=1, max_q=15, min_kv=1024,
             max_kv=16384, page=32, masked=True),
        # one token through a square projection: latency and the weights' bytes
        dict(name="linear_one", op="linear", tokens=1, in_features=4096, out_features=4096, bias=False, dtype="float16"),
        # the down projection of a decode step
        dict(name="linear_decode", op="linear", tokens=64, in_features=18944, out_features=3584, bias=False,
             dtype="bfloat16"),
        # an odd number of tokens through a biased projection
        dict(name="linear_ragged", op="linear", tokens=777, in_features=3584, out_features=4608, bias=True,
             dtype="float16"),
        # the up projection of a prefill
        dict(name="linear_prefill", op="linear", tokens=8192, in_features=4096, out_features=14336, bias=False,
             dtype="float16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attn", "attn", "linear", "linear"])
    if op == "tables":
        batch = _log_int(rng, 1, 1024)
        if rng.random() < 0.5:
            return dict(op=op, batch=batch, min_cached=0, max_cached=_log_int(rng, 1, 16384), min_new=0,
                        max_new=_log_int(rng, 1, 15), page=rng.choice([16, 32, 64, 128]))
        most = _log_int(rng, 16, max(16, min(131072, 1048576 // batch)))
        return dict(op=op, batch=batch, min_cached=0, max_cached=0, min_new=rng.randint(0, most), max_new=most,
                    page=rng.choice([16, 32, 64, 128]))
    if op == "append":
        return dict(op=op, tokens=_log_int(rng, 1, 16384), padding=rng.choice([0, 0, 5, 33]),
                    heads_k=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]))
    if op == "attn":
        heads_k, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
        batch = _log_int(rng, 1, 128)
        max_kv = _log_int(rng, 16, max(16, min(131072, 262144 // batch)))
        several = rng.random() < 0.4
        max_q = rng.randint(2, 15) if several else 1
        min_kv = rng.randint(max_q, max(max_q, max_kv))
        return dict(op=op, batch=batch, heads_q=heads_k * group, heads_k=heads_k, dim=rng.choice([64, 128]),
                    min_q=rng.randint(0, 1) if several else 1, max_q=max_q, min_kv=min_kv, max_kv=max(max_kv, min_kv),
                    page=rng.choice([16, 32, 64, 128]), masked=rng.random() < 0.3)
    tokens = _log_int(rng, 1, 8192)
    k = _log_int(rng, 64, 16384)
    return dict(op=op, tokens=tokens, in_features=k, out_features=_log_int(rng, 33, 14336), bias=rng.random() < 0.5,
                dtype=rng.choice(["float16", "bfloat16"]))


def _lengths(case, held, new, seed):
    """Two lengths for each request, ``held`` and ``new`` naming their ranges: those of the case, in the seed's order."""
    of_case = torch.Generator().manual_seed(sum(case[key] * prime for key, prime in (
        ("batch", 7919), ("min_" + held, 31), ("max_" + held, 37), ("min_" + new, 41), ("max_" + new, 43))))
    ranges = [(case["min_" + name], case["max_" + name] + 1) for name in (held, new)]
    lengths = [torch.randint(lo, hi, (case["batch"],), generator=of_case) for lo, hi in ranges]
    order = torch.randperm(case["batch"], generator=torch.Generator().manual_seed(seed))
    return lengths[0][order], lengths[1][order]


def work(case):
    if case["op"] == "tables":
        cached, new = _lengths(case, "cached", "new", 0)
        page, tokens = case["page"], int(new.sum())
        taken = int(((cached + new + page - 1) // page - (cached + page - 1) // page).sum())
        return {"bytes": tokens * 12 + taken * 8 + case["batch"] * 16, "flops": 0}
    if case["op"] == "append":
        values = 2 * case["tokens"] * case["heads_k"] * case["dim"]
        # fp16 values read and 5 bits a value written; the same 5 bits read back and fp16 written
        return {"bytes": values * (2 + 0.625 + 0.625 + 2) + case["tokens"] * 16, "flops": values * 6}
    if case["op"] == "attn":
        kv, new = _lengths(case, "kv", "q", 0)
        new = torch.minimum(new, kv)
        keys, rows, pairs = int(kv.sum()), int(new.sum()), int((kv * new - new * (new - 1) // 2).sum())
        return {"bytes": keys * (case["heads_k"] * 1.25 * case["dim"] + case["masked"]) + 4 * rows * case["heads_q"] * case["dim"],
                "flops": 4.0 * case["dim"] * case["heads_q"] * pairs}
    m, k, n = case["tokens"], case["in_features"], case["out_features"]
    return {"bytes": 2 * m * k + n * k + 2 * m * n + 4 * n, "flops": 2.0 * m * n * k}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _keys_and_values(tokens, heads, dim, g):
    """Values ~ N(0, 1); two channels of every key head carry outliers, as key caches have them."""
    k = torch.randn(tokens, heads, dim, generator=g, device=DEV)
    v = torch.randn(tokens, heads, dim, generator=g, device=DEV)
    for h in range(heads):
        k[:, h, (5 * h + 3) % dim] *= 12
        k[:, h, (11 * h + 40) % dim] *= 12
    return k.half(), v.half()


def _new_pool(pages, page, heads, dim):
    return torch.zeros(pages, heads, page * dim * 5 // 4, dtype=torch.uint8, device=DEV)


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "tables":
        cached, new = _lengths(case, "cached", "new", seed)
        page = case["page"]
        held = (cached + page - 1) // page
        need = (cached + new + page - 1) // page - held
        pages = int((held + need).sum()) + 64
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
        table = torch.full((case["batch"], int((held + need).max()) + 2), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(held.tolist()):
            table[b, :n] = order[at:at + n].int()
            at += n
        # the ring of free pages: those not held, starting in the ring's middle
        free = order[at:].int()
        head = int(torch.randint(0, pages, (1,), generator=torch.Generator().manual_seed(seed + 2)))
        ring = torch.zeros(pages, dtype=torch.int32)
        ring[(head + torch.arange(free.numel())) % pages] = free
        return dict(op="tables", cached=cached.int().to(DEV), new=new.int().to(DEV), table=table.to(DEV),
                    ring=ring.to(DEV), span=torch.tensor([head, head + free.numel()], device=DEV), page=page,
                    total=max(1, int(new.sum())))
    if case["op"] == "append":
        n, page = case["tokens"], case["page"]
        pages = (n + page - 1) // page + 3
        k, v = _keys_and_values(n + case["padding"], case["heads_k"], case["dim"], g)
        # whole pages in a mixed order, as a prefill fills them; the rows behind the last sequence have no slot
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(n, device=DEV)
        slots = torch.full((n + case["padding"],), -1, dtype=torch.int64, device=DEV)
        slots[:n] = order[at // page] * page + at % page
        return dict(op="append", k=k, v=v, slots=slots, pool=_new_pool(pages, page, case["heads_k"], case["dim"]))
    if case["op"] == "attn":
        page, heads, dim = case["page"], case["heads_k"], case["dim"]
        kv, new = _lengths(case, "kv", "q", seed)
        new = torch.minimum(new, kv)
        if int(new.sum()) == 0:
            new[0] = 1
        held = (kv + page - 1) // page
        pages = int(held.sum()) + 3
        pool = _new_pool(pages, page, heads, dim)
        step = max(1, 16777216 // (page * heads * dim))
        for p in range(0, pages, step):
            n = min(step, pages - p) * page
            k, v = _keys_and_values(n, heads, dim, g)
            _plain_append(k, v, torch.arange(n, device=DEV) + p * page, pool)
        order = torch.randperm(pages, generator=g, device=DEV)
        table = torch.full((case["batch"], int(held.max())), -1, dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(held.tolist()):
            table[b, :n] = order[at:at + n].int()
            at += n
        cu = torch.zeros(case["batch"] + 1, dtype=torch.int32)
        cu[1:] = new.cumsum(0)
        q = torch.randn(int(new.sum()), case["heads_q"], dim, generator=g, device=DEV).half()
        mask = None
        if case["masked"]:  # left padding, and keys dropped here and there
            mask = torch.rand(case["batch"], int(kv.max()), generator=g, device=DEV) > 0.1
            start = (torch.rand(case["batch"], 1, generator=g, device=DEV) * 0.2 * kv.max()).long()
            mask &= torch.arange(mask.shape[1], device=DEV)[None] >= start
        return dict(op="attn", q=q, pool=pool, table=table, kv=kv.int().to(DEV), cu=cu.to(DEV),
                    max_q=int(new.max()), max_kv=int(kv.max()), mask=mask)
    dtype = getattr(torch, case["dtype"])
    m, k, n = case["tokens"], case["in_features"], case["out_features"]
    x = torch.randn(m, k, generator=g, device=DEV)
    x[:, torch.randint(0, k, (4,), generator=g, device=DEV)] *= 20
    w = torch.randn(n, k, generator=g, device=DEV) * 0.02
    amax = w.abs().amax(1)
    w8 = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=DEV)  # rows of whole 16 bytes, laid out once
    w8[:, :k] = (w * (127.0 / amax)[:, None]).round().to(torch.int8)
    bias = torch.randn(n, generator=g, device=DEV).to(dtype) if case["bias"] else None
    return dict(op="linear", x=x.to(dtype), w8=w8[:, :k], w_scale=amax / 127, bias=bias)


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _plain_tables(cached, new, table, ring, span, page, total):
    cached64, new64 = cached.long(), new.long()
    held = (cached64 + page - 1) // page
    need = (cached64 + new64 + page - 1) // page - held
    first = need.cumsum(0) - need
    width = torch.arange(table.shape[1], device=table.device)[None]
    mine = (width >= held[:, None]) & (width < (held + need)[:, None])
    taken = ring[(span[0] + first[:, None] + (width - held[:, None])) % ring.numel()]
    table = torch.where(mine, taken, table)
    cu = torch.zeros(new.numel() + 1, dtype=torch.int64, device=new.device)
    cu[1:] = new64.cumsum(0)
    token = torch.arange(total, device=new.device)
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=new.device), new64)[:total]
    if seq.numel() < total:  # no token at all
        return (torch.full_like(token, -1), torch.zeros_like(token, dtype=torch.int32), cu.int(), cached + new, span,
                table)
    pos = cached64[seq] + token - cu[seq]
    slots = table[seq, pos // page].long() * page + pos % page
    return slots, pos.int(), cu.int(), cached + new, torch.stack((span[0] + need.sum(), span[1])), table


def _plain_codes(x):
    """(codes, scales, minima) of [tokens, heads, dim]: groups of 32 channels."""
    x = x.float().unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    step = (hi - lo) / torch.full_like(hi, 15)  # by a tensor: a division, not a product with 1/15
    scale = step.half()  # rounded down, so that scale * 15 + lo is never beyond the type's range
    scale = (scale.view(torch.int16) - (scale.float() > step).short()).view(torch.float16)
    wide = scale.float()[..., None]
    codes = torch.where(wide > 0, (x - lo[..., None]) / wide, 0.0).round().clamp(0, 15)
    return codes.to(torch.uint8), scale, lo.half()


def _plain_append(k, v, slots, pool):
    heads, dim = k.shape[1], k.shape[2]
    groups, half = dim // 32, dim // 2
    page = pool.shape[2] * 4 // (5 * dim)
    blocks = pool.view(pool.shape[0], heads, page // 16, 20 * dim)
    p, sub, tok = slots // page, slots % page // 16, slots % 16
    head = torch.arange(heads, device=k.device)

    def put(offset, values):  # values [tokens, heads, bytes] at byte `offset` [tokens, bytes] of each block
        blocks[p[:, None, None], head[None, :, None], sub[:, None, None], offset[:, None, :]] = values

    codes, scale, low = _plain_codes(k)
    codes = codes.view(-1, heads, groups, 4, 4, 2)
    packed = (codes[..., 0] | codes[..., 1] << 4).transpose(2, 3).reshape(-1, heads, half)
    put(tok[:, None] * half + torch.arange(half, device=k.device), packed)
    pair = torch.stack((scale, low), -1).view(torch.uint8).reshape(-1, heads, 4 * groups)
    put(16 * half + tok[:, None] * 4 * groups + torch.arange(4 * groups, device=k.device), pair)

    codes, scale, low = _plain_codes(v)
    codes = codes.view(-1, heads, groups, 8, 2, 2)
    packed = (codes[..., 0] | codes[..., 1] << 4).transpose(2, 3).reshape(-1, heads, half)
    base = 10 * dim
    put(base + tok[:, None] * half + torch.arange(half, device=k.device), packed)
    where = (torch.arange(groups, device=k.device) * 64)[None] + (tok % 4 * 16 + tok // 4 * 2)[:, None]
    where = base + 16 * half + where
    both = torch.arange(2, device=k.device)
    put((where[..., None] + both).flatten(1), scale.view(torch.uint8).reshape(-1, heads, 2 * groups))
    put((where[..., None] + 8 + both).flatten(1), low.view(torch.uint8).reshape(-1, heads, 2 * groups))


def _plain_blocks(blocks, dim):
    """16-token blocks [..., 20 * dim] of bytes -> fp32 (keys, values) [..., 16, dim]."""
    lead, groups, half = blocks.shape[:-1], dim // 32, dim // 2

    def nibbles(b):
        return torch.stack((b & 15, b >> 4), -1).flatten(-2)

    kc = nibbles(blocks[..., :8 * dim].unflatten(-1, (16, 4, groups, 4))).transpose(-3, -2).float()
    ks = blocks[..., 8 * dim:10 * dim].contiguous().view(torch.float16).unflatten(-1, (16, groups, 2)).float()
    k = kc.reshape(*lead, 16, groups, 32) * ks[..., :1] + ks[..., 1:]
    vc = nibbles(blocks[..., 10 * dim:18 * dim].unflatten(-1, (16, 8, groups, 2))).transpose(-3, -2).float()
    vs = blocks[..., 18 * dim:].contiguous().view(torch.float16).unflatten(-1, (groups, 4, 2, 4)).float()
    # [group, t, scale or minimum, quarter] -> [quarter, t, group]: token = 4 * quarter + t
    sv = vs.movedim(-1, -4).movedim(-3, -2).reshape(*lead, 16, groups, 2)
    v = vc.reshape(*lead, 16, groups, 32) * sv[..., :1] + sv[..., 1:]
    return k.flatten(-2), v.flatten(-2)


def _plain_read(pool, slots, dim):
    page = pool.shape[2] * 4 // (5 * dim)
    blocks = pool.view(pool.shape[0], pool.shape[1], page // 16, 20 * dim)
    there, at = slots >= 0, slots.clamp(min=0)
    k, v = _plain_blocks(blocks[at // page, :, at % page // 16], dim)
    tok = (at % 16)[:, None, None, None].expand(-1, k.shape[1], 1, dim)
    k, v = k.gather(2, tok)[:, :, 0], v.gather(2, tok)[:, :, 0]
    return torch.where(there[:, None, None], k, 0.0).half(), torch.where(there[:, None, None], v, 0.0).half()


def _plain_attention(q, pool, table, kv, cu, max_q, max_kv, mask):
    rows, heads_q, dim = q.shape
    heads = pool.shape[1]
    page, batch = pool.shape[2] * 4 // (5 * dim), table.shape[0]
    used = (max_kv + page - 1) // page
    blocks = pool.view(pool.shape[0], heads, page // 16, 20 * dim)[table[:, :used].long().clamp(min=0)]
    blocks = blocks.transpose(1, 2)  # [batch, heads, pages, blocks, bytes]
    k, v = _plain_blocks(blocks, dim)
    k, v = k.reshape(batch, heads, -1, dim)[:, :, :max_kv], v.reshape(batch, heads, -1, dim)[:, :, :max_kv]
    new = (cu[1:] - cu[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(batch, device=q.device), new)
    inside = torch.arange(rows, device=q.device) - cu[seq].long()
    dense = torch.zeros(batch, max_q, heads, heads_q // heads, dim, device=q.device)
    dense[seq, inside] = q.float().view(rows, heads, -1, dim)
    key = torch.arange(max_kv, device=q.device)
    last = kv.long()[:, None] - new[:, None] + torch.arange(max_q, device=q.device)[None]
    seen = (key[None, None] <= last[:, :, None]) & (key[None, None] < kv[:, None, None])
    if mask is not None:
        seen = seen & mask[:, None, :max_kv]
    seen = seen[:, None, :, None]  # [batch, 1, max_q, 1, keys]
    s = (dense.permute(0, 2, 1, 3, 4).flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, (max_q, -1)) * dim ** -0.5
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ torch.where((key[None] < kv[:, None])[:, None, :, None], v, 0.0)).unflatten(2, (max_q, -1))
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4)
    return o[seq, inside].reshape(rows, heads_q, dim).half()


def _plain_linear(x, w8, w_scale, bias):
    wide = x.float()
    amax = wide.abs().amax(1, keepdim=True)
    y = torch.where(amax > 0, wide * 127 / amax, 0.0)
    codes = torch.sign(y) * torch.floor(y.abs() + 0.5)
    out = (codes @ w8.float().t()) * (amax / 127) * w_scale
    if bias is not None:
        out = out + bias.float()
    return out.to(x.dtype)


def run(state):
    s = state
    if s["op"] == "tables":
        if own:
            from tilemix_b200.attention.kv4 import build_block_tables

            t = build_block_tables(s["cached"], s["new"], s["table"], s["ring"], s["span"], page_size=s["page"],
                                   max_new_tokens=s["total"])
            return t.slots, t.positions, t.cu_seqlens_q, t.kv_lens, t.free_span, s["table"]
        return _plain_tables(s["cached"], s["new"], s["table"], s["ring"], s["span"], s["page"], s["total"])
    if s["op"] == "append":
        if own:
            from tilemix_b200.attention.kv4 import kv4_append, kv4_read

            kv4_append(s["k"], s["v"], s["pool"], s["slots"])
            return kv4_read(s["pool"], s["slots"], s["k"].shape[2])
        there = s["slots"] >= 0
        _plain_append(s["k"][there], s["v"][there], s["slots"][there], s["pool"])
        return _plain_read(s["pool"], s["slots"], s["k"].shape[2])
    if s["op"] == "attn":
        if own:
            from tilemix_b200.attention.kv4 import kv4_attention

            return kv4_attention(s["q"], s["pool"], s["table"], s["kv"], s["cu"], s["max_q"], key_mask=s["mask"],
                                 max_kv_len=s["max_kv"])
        return _plain_attention(s["q"], s["pool"], s["table"], s["kv"], s["cu"], s["max_q"], s["max_kv"], s["mask"])
    if own:
        from tilemix_b200.linear.int8_linear import int8_linear

        return int8_linear(s["x"], s["w8"], s["w_scale"], s["bias"])
    return _plain_linear(s["x"], s["w8"], s["w_scale"], s["bias"])


# ------------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_quantised(x):
    """The values that the 4-bit codes of x stand for."""
    d = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    low = d.min(-1, keepdim=True).values
    wide = (d.max(-1, keepdim=True).values - low) / 15
    step = wide.half()
    step = torch.where(step.double() > wide, (step.view(torch.int16) - 1).view(torch.float16), step).double()
    n = torch.where(step > 0, torch.round((d - low) / step), torch.zeros_like(d))
    return (n.clamp(max=15) * step + low).reshape(x.shape)


def _exact_tokens(pool, page_numbers, dim, length):
    """Keys and values [heads, length, dim] of a sequence, each channel's byte found by its address."""
    page = pool.shape[2] * 4 // (5 * dim)
    groups = dim // 32
    token = torch.arange(length, device=pool.device)
    rows = pool[page_numbers[token // page]].permute(1, 0, 2)  # [heads, length, page bytes]
    base, tok = token % page // 16 * (20 * dim), token % 16
    c = torch.arange(dim, device=pool.device)
    group, inside = c // 32, c % 32

    def nibble(at, shift):
        got = rows.gather(2, (base[:, None] + at)[None].expand(rows.shape[0], -1, -1))
        return (got >> shift.to(torch.uint8)) & 15

    def half(at):
        at = (base[:, None] + at)[None].expand(rows.shape[0], -1, -1)
        low, high = rows.gather(2, at).int(), rows.gather(2, at + 1).int()
        return (low | high << 8).to(torch.int16).view(torch.float16).double()

    k_at = tok[:, None] * (dim // 2) + (inside // 8 * groups + group) * 4 + inside % 8 // 2
    ks_at = 8 * dim + tok[:, None] * 4 * groups + group * 4
    v_at = 10 * dim + tok[:, None] * (dim // 2) + (inside // 4 * groups + group) * 2 + inside % 4 // 2
    vs_at = 18 * dim + (group * 4 + tok[:, None] % 4) * 16 + tok[:, None] // 4 * 2
    shift = (c % 2 * 4).expand_as(k_at)
    k = nibble(k_at, shift).double() * half(ks_at) + half(ks_at + 2)
    v = nibble(v_at, shift).double() * half(vs_at) + half(vs_at + 8)
    return k, v


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "tables":
        return None
    if s["op"] == "append":
        there = (s["slots"] >= 0).double()[:, None, None]
        return _exact_quantised(s["k"]) * there, _exact_quantised(s["v"]) * there
    if s["op"] == "attn":
        q, cu, kv = s["q"].double(), s["cu"].tolist(), s["kv"].tolist()
        heads_q, dim = q.shape[1], q.shape[2]
        out = torch.zeros_like(q)
        for b, length in enumerate(kv):
            n = cu[b + 1] - cu[b]
            if n == 0:
                continue
            k, v = _exact_tokens(s["pool"], s["table"][b].long(), dim, length)
            group = heads_q // k.shape[0]
            for i in range(n):
                seen = length - n + i + 1
                keep = torch.ones(seen, dtype=torch.bool, device=q.device)
                if s["mask"] is not None:
                    keep = s["mask"][b, :seen]
                if not bool(keep.any()):
                    continue
                rows = q[cu[b] + i].reshape(k.shape[0], group, dim)
                score = torch.einsum("hgd,hkd->hgk", rows, k[:, :seen][:, keep]) / math.sqrt(dim)
                out[cu[b] + i] = torch.einsum("hgk,hkd->hgd", score.softmax(-1), v[:, :seen][:, keep]).reshape(heads_q, dim)
        return out
    x, w = s["x"].double(), s["w8"].double()
    top = x.abs().max(1, keepdim=True).values
    scaled = torch.where(top > 0, x * 127 / top, torch.zeros_like(x))
    codes = torch.trunc(scaled + 0.5 * torch.sign(scaled))
    out = torch.einsum("mk,nk->mn", codes, w) * (top / 127) * s["w_scale"].double()
    return out if s["bias"] is None else out + s["bias"].double()
