"""Batches over a paged cache for the tests, with everything that a call must not look at filled with what would show, and the formulas in
64 bits.  The batches live on whatever device is asked for; the formulas are numpy."""
from fractions import Fraction
from types import SimpleNamespace

import numpy as np
import torch


def make(sequences, heads, kv_heads, dim, page, dtype=torch.bfloat16, heads_first=False, seed=0, device="cuda", spare_rows=0, scale=1.0,
         with_first=True, spare_width=1):
    """`sequences`: (new tokens, length) of each.  Places behind a sequence's length hold NaN, entries of the page table behind its pages
    numbers that no cache has, and `spare_rows` rows stand behind the last sequence."""
    rng = np.random.default_rng(seed)
    need = [-(-max(length, 0) // page) for _, length in sequences]
    pages, width = sum(need) + 2, max(max(need), 1) + spare_width
    order = rng.permutation(pages)
    table = rng.choice(np.array([-1, pages, 2 ** 31 - 1, -2 ** 31], np.int64), size=(len(sequences), width)).astype(np.int32)
    k, v = (torch.full((pages, page, kv_heads, dim), float("nan"), dtype=dtype) for _ in range(2))
    stored, at = [], 0
    for s, (n, length) in enumerate(sequences):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
        ks, vs = (torch.from_numpy(rng.standard_normal((length, kv_heads, dim)) * scale).to(dtype) for _ in range(2))
        t = np.arange(length)
        k[table[s, t // page], t % page] = ks
        v[table[s, t // page], t % page] = vs
        stored.append((ks.double().numpy(), vs.double().numpy()))
    first = np.concatenate([[0], np.cumsum([n for n, _ in sequences])]).astype(np.int32)
    tokens = int(first[-1]) + spare_rows
    q = torch.from_numpy(rng.standard_normal((tokens, heads * dim)) * scale).to(dtype)

    def placed(x):
        if not heads_first:
            return x.to(device)
        return x.transpose(1, 2).contiguous().to(device).transpose(1, 2)

    b = SimpleNamespace(sequences=sequences, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, stored=stored, table=table,
                        first=first, tokens=tokens, used=int(first[-1]))
    b.k_pages, b.v_pages, b.q = placed(k), placed(v), q.to(device)
    b.page_table = torch.from_numpy(table).to(device)
    b.lengths = torch.tensor([length for _, length in sequences], dtype=torch.int32, device=device)
    b.first_dev = torch.from_numpy(first).to(device) if with_first else None
    b.max_new = max(1, max(n for n, _ in sequences))
    return b


def attention(b, scale=None):
    """(out, lse, bound of out's error, bound of lse's error) in 64 bits, rows behind the last sequence left out.

    The bounds count roundings, u = 2^-24 in f32: a score of D products is off by (D + 4) u sum |q k| at most, an exponential by that, 2^-21 of
    its own and the rounding of its argument (u |score|, twice), a sum over the keys by u a key; in bf16 P and the result are rounded once,
    2^-8 each.  P is formed against a maximum up to 2^8 away, which costs its argument another 16 u."""
    u, group = 2.0 ** -24, b.heads // b.kv_heads
    scale = b.dim ** -0.5 if scale is None else scale
    q = b.q.double().cpu().numpy().reshape(-1, b.kv_heads, group, b.dim)
    out, lse = np.zeros((b.used, b.kv_heads, group, b.dim)), np.full((b.used, b.kv_heads, group), -np.inf)
    out_bound, lse_bound = np.zeros_like(out), np.zeros_like(lse)
    half = 2.0 ** -8 if b.dtype == torch.bfloat16 else u
    for s, (n, length) in enumerate(b.sequences):
        k, v = b.stored[s]
        for i in range(n):
            sees, row = length - n + i + 1, b.first[s] + i
            if sees <= 0:
                continue
            z = np.einsum("hgd,lhd->hgl", q[row], k[:sees]) * scale
            size = np.einsum("hgd,lhd->hgl", np.abs(q[row]), np.abs(k[:sees])).max(-1) * scale
            m = z.max(-1, keepdims=True)
            p = np.exp(z - m)
            total = p.sum(-1)
            p /= total[..., None]
            off = (b.dim + 4) * u * size + 2 * u * np.abs(z).max(-1) + 2.0 ** -21 + 16 * u + sees * u
            out[row] = np.einsum("hgl,lhd->hgd", p, v[:sees])
            reach = np.einsum("hgl,lhd->hgd", p, np.abs(v[:sees]))
            lse[row] = m[..., 0] + np.log(total)
            lse_bound[row] = 2 * off + 8 * u * np.abs(lse[row]) + 2.0 ** -21
            out_bound[row] = reach * (2 * off[..., None] + (half if b.dtype == torch.bfloat16 else 0)) * 1.01 + half * np.abs(out[row]) + 1e-30
    shape = (b.used, b.heads)
    return out.reshape(b.used, -1), lse.reshape(shape), out_bound.reshape(b.used, -1), lse_bound.reshape(shape)


def rotate(x, positions, frequencies, interleaved):
    """x [tokens, heads, channels] in 64 bits, turned by positions * frequencies."""
    dims = 2 * len(frequencies)
    if dims == 0:
        return x
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(frequencies, np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    y = x.copy()
    a, b = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, dims // 2), slice(dims // 2, dims))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def sample(logits, draw, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row in 64 bits; the controls as the f32 values that they are."""
    x = np.asarray(logits, np.float64)
    finite = np.flatnonzero(np.isfinite(x))
    if len(finite) == 0:
        return -1, 0.0
    if not temperature > 0:
        return int(finite[np.argmax(x[finite])]), 1.0
    top = x[finite].max()
    ranked = finite[np.lexsort((finite, -x[finite]))]
    weight = lambda i: np.exp((x[i] - top) / np.float64(temperature))  # noqa: E731
    if 0 < top_k < len(ranked):
        ranked = ranked[:top_k]
    if 0 < top_p < 1:
        reached = np.cumsum(weight(ranked))
        ranked = ranked[:1 + int(np.searchsorted(reached, top_p * reached[-1], side="left"))]
    ranked = ranked[weight(ranked) >= min(1.0, min_p)]
    stays = np.sort(ranked)
    reached = np.cumsum(weight(stays))
    # the first whose sum is above the product, which is not rounded: a draw may fall on a border (0.7 of 49500 equal tokens is below 34650)
    border = Fraction(min(max(draw, 0.0), 1.0)) * Fraction(reached[-1])
    at = min(int(np.searchsorted(reached, float(border), side="right")), len(stays) - 1)
    while at > 0 and Fraction(reached[at - 1]) > border:
        at -= 1
    while at < len(stays) - 1 and Fraction(reached[at]) <= border:
        at += 1
    return int(stays[at]), float(weight(stays[at]) / reached[-1])
