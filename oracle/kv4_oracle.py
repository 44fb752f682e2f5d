"""Paged 4-bit key/value cache in numpy: block tables, quantiser, byte layout and attention.

Restates the operators' definitions: integers exactly, the quantiser in the fp32 steps that define
it, the attention in 64 bits on the values that the cache stands for.
"""
from __future__ import annotations

import numpy as np

GROUP = 32


def build_block_tables(cached, new, table, ring, span, page, n_slots):
    """(slots, positions, cu, kv_lens, span, table, served) for one step, request by request."""
    cached, new, table = [int(c) for c in cached], [int(n) for n in new], np.array(table, dtype=np.int32)
    head, tail = int(span[0]), int(span[1])
    pages = lambda tokens: -(-tokens // page)  # noqa: E731
    negative = any(c < 0 or n < 0 for c, n in zip(cached, new))
    need = 0 if negative else sum(pages(c + n) - pages(c) for c, n in zip(cached, new))
    served = (not negative and need <= tail - head and sum(new) <= n_slots
              and all(c + n <= table.shape[1] * page for c, n in zip(cached, new)))
    slots, positions = np.full(n_slots, -1, dtype=np.int64), np.zeros(n_slots, dtype=np.int32)
    cu = np.zeros(len(cached) + 1, dtype=np.int32)
    if not served:
        return slots, positions, cu, np.array(cached, np.int32), np.array([head, tail], np.int64), table, False
    row = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        for col in range(pages(c), pages(c + n)):
            table[b, col] = ring[head % len(ring)]
            head += 1
        for pos in range(c, c + n):
            slots[row] = int(table[b, pos // page]) * page + pos % page
            positions[row] = pos
            row += 1
        cu[b + 1] = row
    return (slots, positions, cu, np.array([c + n for c, n in zip(cached, new)], np.int32),
            np.array([head, tail], np.int64), table, True)


def quantise(x):
    """fp16 [..., dim] -> (codes uint8 [..., groups, 32], scale fp16 [..., groups], minimum fp16 [..., groups])."""
    x = np.asarray(x, dtype=np.float16).astype(np.float32)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        lo, hi = x.min(-1), x.max(-1)
        step = (hi - lo) / np.float32(15)
        scale = step.astype(np.float16)  # rounded down
        scale = np.where(scale.astype(np.float32) > step, np.nextafter(scale, np.float16(0)), scale)
        wide = scale.astype(np.float32)[..., None]
        q = np.where((wide > 0) & np.isfinite(wide), (x - lo[..., None]) / wide, np.float32(0))
    return np.minimum(np.rint(q), 15).astype(np.uint8), scale, lo.astype(np.float16)


def dequantise(codes, scale, low):
    """64-bit values [..., dim] that codes, scales and minima stand for."""
    v = codes.astype(np.float64) * scale.astype(np.float64)[..., None] + low.astype(np.float64)[..., None]
    return v.reshape(*v.shape[:-2], v.shape[-2] * GROUP)


def block_offsets(dim, tok):
    """Byte offsets inside a 16-token block of 20 dim bytes, for token ``tok`` of it: (K code byte, V code byte) [dim]
    (the nibble is the channel's parity) and (K scale, V scale) [groups]; minima follow 2 and 8 bytes on."""
    c, groups = np.arange(dim), dim // GROUP
    j, i = c // GROUP, c % GROUP
    kc = tok * (dim // 2) + (i // 8 * groups + j) * 4 + i % 8 // 2
    vc = 10 * dim + tok * (dim // 2) + (i // 4 * groups + j) * 2 + i % 4 // 2
    g = np.arange(groups)
    return kc, vc, 8 * dim + tok * 4 * groups + g * 4, 18 * dim + (g * 4 + tok % 4) * 16 + tok // 4 * 2


def append(pool, k, v, slots):
    """Store quantised k / v [n, heads, dim] in ``pool`` (uint8 [pages, heads, page bytes]), in place."""
    dim = k.shape[2]
    page = pool.shape[2] // (20 * dim) * 16
    both = [(quantise(x), at) for x, at in ((k, 0), (v, 1))]
    for i, slot in enumerate(np.asarray(slots)):
        if slot < 0:
            continue
        rows = pool[slot // page]
        base, tok = slot % page // 16 * (20 * dim), int(slot % 16)
        offsets = block_offsets(dim, tok)
        for (codes, scale, low), which in both:
            n = codes[i].reshape(rows.shape[0], dim)
            at = base + offsets[which]
            rows[:, at[0::2]] = n[:, 0::2] | n[:, 1::2] << 4
            for value, more in ((scale[i], 0), (low[i], 2 if which == 0 else 8)):
                raw = np.ascontiguousarray(value).view(np.uint8).reshape(rows.shape[0], -1, 2)
                for byte in range(2):
                    rows[:, base + offsets[2 + which] + more + byte] = raw[:, :, byte]


def read(pool, slots, dim):
    """64-bit (k, v) [n, heads, dim] at ``slots``; zeros for slot -1."""
    heads, page = pool.shape[1], pool.shape[2] // (20 * dim) * 16
    out = np.zeros((2, len(slots), heads, dim))
    shift = (np.arange(dim) % 2 * 4).astype(np.uint8)
    for i, slot in enumerate(np.asarray(slots)):
        if slot < 0:
            continue
        rows = pool[slot // page]
        base = slot % page // 16 * (20 * dim)
        offsets = block_offsets(dim, int(slot % 16))
        for which, more in ((0, 2), (1, 8)):
            codes = (rows[:, base + offsets[which]] >> shift) & 15
            half = lambda at: np.ascontiguousarray(np.stack([rows[:, at], rows[:, at + 1]], -1)).view(np.float16)[..., 0]  # noqa: E731
            out[which, i] = dequantise(codes.reshape(heads, -1, GROUP), half(base + offsets[2 + which]),
                                       half(base + offsets[2 + which] + more))
    return out[0], out[1]


def attention(q, keys, values, kv_len, sm_scale, causal, key_mask=None):
    """64-bit attention of one request's n query tokens [n, heads_q, dim] over keys / values [kv_len, heads_k, dim],
    and a bound on what fp16 operands may change.

    Bound: scores come from the codes, s (q . n) + m sum q: products of two fp16 numbers are exact, their fp32 sums are
    rounded (or cut) a few times at 2^-22 of sum |q| 15 s + |m| sum |q|, and the sum of q over a group is held to 2^-22
    of it: with |m| at most 100 s, as it is for these inputs, under 2^-12 s sum |q| together; 2^-10 is allowed. The fp32
    steps that follow add 2^-21 sum |q| |k|. With d the sum of both, times sm_scale, a weight changes by the factor
    e^(2 d) (numerator and sum). v and p are rounded to fp16 (2^-11 each; a p under 2^-14 by at most 2^-25 of the largest weight), the result
    once more; 2^-18 covers the fp32 sums and exponentials.
    """
    n, heads_q, dim = q.shape
    group = heads_q // keys.shape[1]
    out, bound = np.zeros((n, heads_q, dim)), np.full((n, heads_q, dim), 2.0 ** -25)
    q = q.astype(np.float64)
    for i in range(n):
        seen = np.arange(kv_len) < (kv_len - n + i + 1 if causal else kv_len)
        if key_mask is not None:
            padded = np.zeros(kv_len, dtype=bool)
            m = key_mask[:kv_len]
            padded[:len(m)] = m
            seen &= padded
        if not seen.any():
            continue
        for h in range(heads_q):
            k, v = keys[seen, h // group], values[seen, h // group]
            s = k @ q[i, h] * sm_scale
            p = np.exp(s - s.max())
            groups = k.reshape(len(k), -1, GROUP)
            step = (groups.max(-1) - groups.min(-1)) / 15
            d = sm_scale * (2.0 ** -10 * step @ np.abs(q[i, h]).reshape(-1, GROUP).sum(-1)
                            + 2.0 ** -21 * np.abs(k) @ np.abs(q[i, h])).max()
            total = p.sum()
            out[i, h] = p @ v / total
            near = p @ np.abs(v) / total
            bound[i, h] += (near * (np.expm1(2 * d) + 3 * 2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25 * np.abs(v).sum(0) / total
                            + 2.0 ** -11 * np.abs(out[i, h]))
    return out, bound
