"""Plain 64-bit forms of the paged serving ops: tables, commit, attention.

Tables are worked out request by request in Python integers; attention row by
row of the definition in float64, with the size of the terms that make up each
result beside it (what a bound of the rounding errors is made of).
"""
from __future__ import annotations

import math

import torch


def paged_tables(ctx_lens, new_lens, block_table, free_pages, num_free, page_size, num_pages,
                 max_tokens):
    """(cu_q, kv_lens, slots, free_left, block_table) as lists; block_table [R][W] is copied."""
    table = [list(row) for row in block_table]
    width = len(table[0]) if table else 0
    available = min(max(num_free, 0), len(free_pages))
    cu, kv, slots, taken = [0], [], [], 0
    for r, (ctx, new) in enumerate(zip(ctx_lens, new_lens)):
        ctx, new = max(ctx, 0), max(new, 0)
        end = min(cu[-1] + new, max_tokens)
        new = end - cu[-1]
        cu.append(end)
        kv.append(min(ctx + new, 2 ** 31 - 1))
        for j in range(-(-ctx // page_size), min(width, -(-(ctx + new) // page_size))):
            at = available - 1 - taken
            taken += 1
            page = free_pages[at] if at >= 0 else -1
            table[r][j] = page if 0 <= page < num_pages else -1
        for pos in range(ctx, ctx + new):
            page = table[r][pos // page_size] if pos // page_size < width else -1
            held = 0 <= page < num_pages
            slots.append(page * page_size + pos % page_size if held else -1)
    return cu, kv, slots + [-1] * (max_tokens - len(slots)), available - taken, table


def kv_commit_rope_paged(src_k, src_v, pages_k, pages_v, slots, cos, sin):
    """New (pages_k, pages_v): src [L, T, H, D], pages [L, N, P, H, D]. The rotation as torch
    evaluates it in fp32, one rounding to the element type."""
    L, N, P, H, D = pages_k.shape
    out_k, out_v = pages_k.clone(), pages_v.clone()
    x = src_k.float()
    if cos is not None:
        turned = torch.stack((-x[..., 1::2], x[..., 0::2]), -1).flatten(-2)
        x = x * cos[None, :, None, :] + turned * sin[None, :, None, :]
    x = x.to(src_k.dtype)
    for n, s in enumerate(slots.tolist()):
        if 0 <= s < N * P:
            out_k[:, s // P, s % P] = x[:, n]
            out_v[:, s // P, s % P] = src_v[:, n]
    return out_k, out_v


def attention(q, k, v, seen, scale):
    """One request: q [n, Hq, D], k, v [m, Hkv, D], seen bool [n, m]. Float64 (out, size,
    score): out [n, Hq, D]; size = sum_j p_j |v_j|; score [n, Hq] = the largest
    scale * sum_d |q_d k_d| of a key that the row sees. Rows that see nothing are zeros, and
    what a row does not see takes no part (a NaN there stays out)."""
    n, Hq, D = q.shape
    m, Hkv, _ = k.shape
    group = Hq // Hkv
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    size, score = torch.zeros_like(out), torch.zeros(n, Hq, dtype=torch.float64)
    if n == 0 or m == 0:
        return out, size, score
    for h in range(Hq):
        qh, kh, vh = (t.double() for t in (q[:, h], k[:, h // group], v[:, h // group]))
        s = (qh @ kh.t() * scale).masked_fill(~seen, -math.inf)
        top = s.amax(1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        p = torch.where(seen, p, 0.0)
        total = p.sum(1, keepdim=True)
        p = p / torch.where(total == 0, 1.0, total)
        hidden_bad = ~torch.isfinite(vh).all(1)[None, :] & ~seen
        if bool(hidden_bad.any()):  # rows that must not meet these values one by one
            for i in range(n):
                out[i, h] = p[i, seen[i]] @ vh[seen[i]]
                size[i, h] = p[i, seen[i]] @ vh[seen[i]].abs()
        else:
            out[:, h], size[:, h] = p @ vh, p @ vh.abs()
        a = (qh.abs() @ kh.abs().t() * scale).masked_fill(~seen, 0.0)
        score[:, h] = a.amax(1)
    return out, size, score


def attention_bound(dtype, out, size, score, n_keys, v_max):
    """Element-wise bound of |kernel - out| for results of `dtype`.

    u = half a step of dtype. The result is rounded once (u |out|) and each
    probability once before it meets v (u size). In fp32: a score is a sum of D
    products and its scaling, off by at most (D + 4) 2^-24 score; the power of
    two adds 2^-22 relative; both act on the weights and again on their sum
    (twice); the sums over the keys add (n_keys + 64) 2^-24 size. fp16
    probabilities below 2^-14 are rounded to a multiple of 2^-24 instead: at
    most 2^-25 v_max a key over a sum of weights of at least one.
    """
    u = torch.finfo(dtype).eps / 2
    D = out.shape[-1]
    e32 = 2 * ((D + 4) * 2.0 ** -24 * score + 2.0 ** -22) + (n_keys + 64) * 2.0 ** -24
    bound = u * out.abs() + (u + e32[..., None]) * (1 + u) * size
    if dtype == torch.float16:
        bound = bound + n_keys * 2.0 ** -25 * v_max + 2.0 ** -25
    return bound + 1e-30
