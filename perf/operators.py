"""The serving attention path as timed cases: paged KV tables, the paged commit, attention.

A server that runs many streams on one GPU keeps their K and V in pages of one pool. A step
of it makes four kinds of calls: the block tables and slot maps of the step from the request
lengths (paged_tables), the step's K rotated and V copied into their pages
(kv_commit_rope_paged), attention of the new tokens over the pages (attention_paged), and
attention over whole prompts that are packed one behind the other (attention_varlen). The
heads are the package's own (32 heads of 128 and a cache of 1560 tokens a latent frame, in
pages of one latent row of 52) and grouped forms of them; lengths run from single tokens to
whole contexts.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

_root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _ops():
    path = os.path.join(_root, "joyai-video-edit_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import joyomni_ops
    return joyomni_ops


def listed() -> list:
    return [
        # Tables of a step of single tokens: 32 running requests, one token each.
        dict(name="tables_decode", kind="tables", R=32, P=16, W=1024, ctx_lo=16, ctx_hi=16000,
             new_lo=1, new_hi=1,
             pad=0, lens=1),
        # Tables of a step that admits many prompts, in a padded step of fixed size.
        dict(name="tables_admit", kind="tables", R=500, P=64, W=512, ctx_lo=1, ctx_hi=16000,
             new_lo=1, new_hi=128,
             pad=777, lens=2),
        # Commit of one token of each of 30 requests in a step padded to 32, one layer.
        dict(name="commit_decode", kind="commit", layers=1, T=30, pad=2, H=8, D=128, P=16,
             rope=True, dtype="bf16"),
        # Commit of one latent frame for all 40 layers, a page for each latent row.
        dict(name="commit_frame", kind="commit", layers=40, T=1560, pad=0, H=32, D=128, P=52,
             rope=True, dtype="bf16"),
        # Single tokens of a few short requests: latency.
        dict(name="decode_few", kind="paged", R=4, Hkv=8, G=4, D=128, P=16, ctx_lo=300, ctx_hi=2000,
             new_lo=1, new_hi=1, causal=True, lens=3, dtype="bf16"),
        # Single tokens of a full batch with contexts of very different lengths.
        dict(name="decode_batch", kind="paged", R=64, Hkv=8, G=4, D=128, P=16, ctx_lo=100,
             ctx_hi=16384,
             new_lo=1, new_hi=1, causal=True, lens=4, dtype="bf16"),
        # Single tokens of two very long contexts: the keys have to be split.
        dict(name="decode_long", kind="paged", R=2, Hkv=4, G=8, D=128, P=64, ctx_lo=90000,
             ctx_hi=131071,
             new_lo=1, new_hi=1, causal=True, lens=5, dtype="fp16"),
        # Chunks of prompts beside single tokens, as a scheduler mixes them.
        dict(name="chunk_mixed", kind="paged", R=20, Hkv=8, G=4, D=128, P=32, ctx_lo=40,
             ctx_hi=8000,
             new_lo=1, new_hi=512, causal=True, lens=6, dtype="bf16"),
        # Two latent frames over three cached ones and themselves, every token seen.
        dict(name="frames_over_cache", kind="paged", R=1, Hkv=32, G=1, D=128, P=52,
             ctx_lo=4680, ctx_hi=4680, new_lo=3120, new_hi=3120, causal=False, lens=7, dtype="bf16"),
        # Three short prompts: the smallest call of whole prompts.
        dict(name="prompts_short", kind="varlen", R=3, Hkv=32, G=1, D=128, lq_lo=12, lq_hi=77,
             causal=True, lens=8, dtype="bf16"),
        # Prompts of different lengths packed into one call, small heads.
        dict(name="prompts_packed", kind="varlen", R=8, Hkv=4, G=4, D=64, lq_lo=200, lq_hi=3500,
             causal=True, lens=9, dtype="fp16"),
        # One long prompt with grouped heads: the largest call.
        dict(name="prompt_long", kind="varlen", R=1, Hkv=8, G=4, D=128, lq_lo=16384, lq_hi=16384,
             causal=True, lens=10, dtype="bf16"),
    ]


# ---------------------------------------------------------------------------
# Drawn cases.
# ---------------------------------------------------------------------------
def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_once(rng) -> dict:
    kind = rng.choice(("tables", "commit", "paged", "paged", "paged", "varlen", "varlen"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    D = rng.choice((64, 128, 128, 128, 256))
    P = rng.choice((1, 8, 16, 16, 32, 52, 64, 128, rng.randint(2, 200)))
    lens = rng.randint(100, 10 ** 6)
    if kind == "tables":
        new = _log(rng, 1, 512)
        ctx = _log(rng, 1, 30000)
        return dict(kind=kind, R=_log(rng, 1, 2000), P=max(P, 8), W=(ctx + new) // max(P, 8) + 1,
                    ctx_lo=rng.choice((0, 1, ctx)), ctx_hi=ctx, new_lo=rng.choice((0, 1, new)),
                    new_hi=new,
                    pad=rng.choice((0, 1, 100)), lens=lens)
    if kind == "commit":
        return dict(kind=kind, layers=_log(rng, 1, 40), T=_log(rng, 1, 1560),
                    pad=rng.choice((0, 1, 40)),
                    H=rng.choice((1, 4, 8, 8, 24, 32, rng.randint(2, 32))),
                    D=D, P=P, rope=rng.random() < 0.75, dtype=dtype)
    Hkv = rng.choice((1, 2, 4, 8, 8, 32, rng.randint(3, 24)))
    G = rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 16)) if Hkv <= 8 else rng.choice((1, 1, 2))
    causal = rng.random() < 0.75
    if kind == "varlen":
        hi = _log(rng, 1, 16384)
        return dict(kind=kind, R=_log(rng, 1, 48), Hkv=Hkv, G=G, D=D,
                    lq_lo=rng.choice((1, hi, hi // 4 + 1)),
                    lq_hi=hi,
                    causal=causal, lens=lens, dtype=dtype)
    new = rng.choice((1, 1, _log(rng, 1, 16), _log(rng, 1, 3120)))
    ctx = _log(rng, 1, 100000)
    return dict(kind=kind, R=_log(rng, 1, 128), Hkv=Hkv, G=G, D=D, P=P,
                ctx_lo=rng.choice((0, 1, ctx, ctx // 8)), ctx_hi=ctx, new_lo=rng.choice((1, new)),
                new_hi=new,
                causal=causal, lens=lens, dtype=dtype)


def draw(rng) -> dict:
    """A call of the ranges above that costs no more than the largest listed ones and whose
    plain form (which pads every request to the longest) stays in memory."""
    c = _draw_once(rng)
    while not _fits(c):
        c = _draw_once(rng)
    return c


def _fits(c: dict) -> bool:
    w = work(c)
    if w["flops"] > 2.2e12 or w["bytes"] > 2.1e9:
        return False
    if c["kind"] not in ("paged", "varlen"):
        return True
    nq, nk = _lengths(c)
    lq, lk = max(nq), max(nk)
    heads = c["Hkv"] * c["G"]
    return c["R"] * heads * lq * lk * 4 <= 36e9 and c["R"] * lk * c["Hkv"] * c["D"] * 8 <= 12e9


# ---------------------------------------------------------------------------
# Lengths (from the case alone) and inputs (from the seed).
# ---------------------------------------------------------------------------
def _spread(rng, lo: int, hi: int) -> int:
    if lo < 1:  # a range from nothing: some of its requests have nothing
        return 0 if rng.random() < 0.2 else _log(rng, 1, max(hi, 1))
    return _log(rng, lo, hi)


def _lengths(c: dict) -> tuple:
    """(new tokens, keys) of each request. In a mix of chunks and single tokens one
    request in five brings a chunk."""
    rng = random.Random(c["lens"])
    nq, nk = [], []
    for i in range(c["R"]):
        if c["kind"] == "varlen":
            n = _spread(rng, c["lq_lo"], c["lq_hi"])
            nq.append(n)
            nk.append(n)
            continue
        lo, hi = c["new_lo"], c["new_hi"]
        if c["kind"] == "paged" and lo < hi:
            n = hi - rng.randint(0, (hi - lo) // 4) if i % 5 == 0 else lo
        else:
            n = _spread(rng, lo, hi)
        nq.append(n)
        nk.append(n + _spread(rng, c["ctx_lo"], c["ctx_hi"]))
    return nq, nk


def _cu(lens: list) -> list:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _gen(seed: int):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, mul=1.0, dtype=torch.bfloat16):
        # In parts: 32-bit numbers of a whole pool need not be held at once.
        out = torch.empty(shape, dtype=dtype, device="cuda")
        for part in out.view(-1).split(1 << 28):
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(mul))
        return out

    def perm(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32)

    return rand, perm


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case: dict, seed: int) -> dict:
    c, kind = case, case["kind"]
    rand, perm = _gen(seed)
    t = {"case": c}
    if kind == "tables":
        nq, nk = _lengths(c)
        R, P, W = c["R"], c["P"], c["W"]
        ctx = [k - n for n, k in zip(nq, nk)]
        have = torch.tensor([-(-x // P) for x in ctx], device="cuda").clamp(max=W)
        total = R * W + 8
        ids = perm(total)
        table = ids[:R * W].view(R, W).clone()
        held = torch.arange(W, device="cuda")[None, :] < have[:, None]
        t["table"] = torch.where(held, table, torch.full_like(table, -1))
        t["free"] = torch.cat((ids[:R * W].view(R, W)[~held], ids[R * W:]))
        t["num_free"] = _i32([t["free"].numel() - 3])
        t["ctx"], t["new"] = _i32(ctx), _i32(nq)
        t["num_pages"], t["max_tokens"] = total, sum(nq) + c["pad"]
        return t
    if kind == "commit":
        L, T, H, D, P = c["layers"], c["T"], c["H"], c["D"], c["P"]
        dt, all_tokens = DTYPES[c["dtype"]], T + c["pad"]
        N = -(-T // P) + 3
        t["k"], t["v"] = (rand(L, all_tokens, H, D, dtype=dt) for _ in range(2))
        t["pages_k"], t["pages_v"] = (rand(L, N, P, H, D, dtype=dt) for _ in range(2))
        # A frame fills pages in order; single tokens land anywhere.
        t["slots"] = torch.full((all_tokens,), -1, dtype=torch.int64, device="cuda")
        n = torch.arange(T, device="cuda")
        t["slots"][:T] = (perm(N)[n // P] * P + n % P if T >= P else perm(N * P)[:T]).long()
        t["real"] = T
        if c["rope"]:
            pos = torch.arange(all_tokens, device="cuda") + 1000 * (seed % 7)
            freq = 10000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
            ang = (pos[:, None] * freq[None, :]).repeat_interleave(2, 1)
            t["cos"], t["sin"] = ang.cos().float(), ang.sin().float()
        return t
    dt, D, Hkv = DTYPES[c["dtype"]], c["D"], c["Hkv"]
    Hq = Hkv * c["G"]
    nq, nk = _lengths(c)
    t["cu_q"], t["max_q"], t["max_k"] = _i32(_cu(nq)), max(nq), max(nk)
    T = sum(nq)
    if kind == "varlen":
        # q, k and v are slices of one packed projection, as a model has them.
        qkv = rand(T, (Hq + 2 * Hkv) * D, mul=1.3, dtype=dt)
        t["q"] = qkv[:, :Hq * D].view(T, Hq, D)
        t["k"] = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
        t["v"] = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
        return t
    P, R = c["P"], c["R"]
    need = [-(-k // P) for k in nk]
    N, W = sum(need) + 5, max(max(need), 1)
    t["q"] = rand(T, Hq, D, mul=1.3, dtype=dt)
    t["pages_k"], t["pages_v"] = rand(N, P, Hkv, D, mul=1.3, dtype=dt), rand(N, P, Hkv, D, dtype=dt)
    first = torch.tensor(_cu(need)[:-1], device="cuda")[:, None]
    col = torch.arange(W, device="cuda")[None, :]
    held = col < torch.tensor(need, device="cuda")[:, None]
    ids = perm(N)[torch.where(held, first + col, 0)]
    t["table"] = torch.where(held, ids, torch.full_like(ids, -1))
    t["kv_lens"] = _i32(nk)
    return t


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------
def run(t: dict):
    c = t["case"]
    kind = c["kind"]
    if own:
        jo = _ops()
        if kind == "tables":
            made = jo.paged_tables(t["ctx"], t["new"], t["table"], t["free"], t["num_free"], c["P"],
                                   t["num_pages"], t["max_tokens"])
            return (*made, t["table"])
        if kind == "commit":
            jo.kv_commit_rope_paged(t["k"], t["pages_k"], t["slots"], t.get("cos"), t.get("sin"),
                                    src_v=t["v"], pages_v=t["pages_v"])
            return t["pages_k"], t["pages_v"]
        if kind == "paged":
            return jo.attention_paged(t["q"], t["pages_k"], t["pages_v"], t["table"], t["cu_q"],
                                      t["kv_lens"], causal=c["causal"])
        return jo.attention_varlen(t["q"], t["k"], t["v"], t["cu_q"], causal=c["causal"])
    if kind == "tables":
        return _plain_tables(t)
    if kind == "commit":
        return _plain_commit(t)
    if kind == "paged":
        R, W, P = c["R"], t["table"].shape[1], c["P"]
        ids = t["table"].clamp(min=0).long()
        k = t["pages_k"][ids].view(R, W * P, c["Hkv"], c["D"])[:, :t["max_k"]]
        v = t["pages_v"][ids].view(R, W * P, c["Hkv"], c["D"])[:, :t["max_k"]]
        return _plain_attention(t["q"], k, v, t["cu_q"], t["kv_lens"], t["max_q"], c["causal"])
    nk = t["cu_q"][1:] - t["cu_q"][:-1]
    rows = t["cu_q"][:-1, None] + torch.arange(t["max_k"], device="cuda")
    rows = rows.clamp(max=t["k"].shape[0] - 1)
    return _plain_attention(t["q"], t["k"][rows], t["v"][rows], t["cu_q"], nk, t["max_q"],
                            c["causal"])


def _plain_tables(t: dict):
    c, table, free, max_tokens = t["case"], t["table"], t["free"], t["max_tokens"]
    P, W, num_pages = c["P"], c["W"], t["num_pages"]
    ctx, new = t["ctx"].long().clamp(min=0), t["new"].long().clamp(min=0)
    cu = torch.cat((new.new_zeros(1), new.cumsum(0).clamp(max=max_tokens)))
    kv = ctx + cu[1:] - cu[:-1]
    have, need = ((ctx + P - 1) // P).clamp(max=W), ((kv + P - 1) // P).clamp(max=W)
    fresh = (need - have).clamp(min=0)
    base = fresh.cumsum(0) - fresh
    col = torch.arange(W, device="cuda")[None, :]
    at = t["num_free"].long() - 1 - base[:, None] - (col - have[:, None])
    ids = free[at.clamp(0, free.numel() - 1)]
    ids = torch.where((at >= 0) & (ids >= 0) & (ids < num_pages), ids, -1)
    table.copy_(torch.where((col >= have[:, None]) & (col < need[:, None]), ids, table))
    tok = torch.arange(max_tokens, device="cuda")
    r = torch.searchsorted(cu[1:], tok, right=True).clamp(max=c["R"] - 1)
    pos = ctx[r] + tok - cu[r]
    page = table[r, (pos // P).clamp(0, W - 1)].long()
    held = (tok < cu[-1]) & (pos // P < W) & (page >= 0) & (page < num_pages)
    slots = torch.where(held, page * P + pos % P, -1)
    left = t["num_free"] - fresh.sum().int()
    return cu.int(), kv.int(), slots, left, table


def _plain_commit(t: dict):
    c, n = t["case"], t["real"]
    L, H, D = c["layers"], c["H"], c["D"]
    where = t["slots"][:n]
    k = t["k"][:, :n]
    if c["rope"]:
        x = k.float()
        turned = torch.stack((-x[..., 1::2], x[..., 0::2]), -1).flatten(-2)
        k = (x * t["cos"][:n, None, :] + turned * t["sin"][:n, None, :]).to(k.dtype)
    t["pages_k"].view(L, -1, H, D).index_copy_(1, where, k)
    t["pages_v"].view(L, -1, H, D).index_copy_(1, where, t["v"][:, :n])
    return t["pages_k"], t["pages_v"]


def _plain_attention(q, k, v, cu_q, kv_lens, max_q, causal):
    """Attention of packed q [T, Hq, D] over padded k, v [R, Lk, Hkv, D], all heads and requests
    at once, every request padded to the longest."""
    T, Hq, D = q.shape
    R, Lk, Hkv, _ = k.shape
    G = Hq // Hkv
    dev = q.device
    n_new = (cu_q[1:] - cu_q[:-1]).long()
    rows = (cu_q[:-1, None].long() + torch.arange(max_q, device=dev)).clamp(max=T - 1)
    qp = q[rows].float().view(R, max_q, Hkv, G, D).permute(0, 2, 3, 1, 4)
    qp = qp.reshape(R, Hkv, G * max_q, D)
    kp = k.float().permute(0, 2, 3, 1)
    s = torch.matmul(qp, kp).view(R, Hkv, G, max_q, Lk).mul_(D ** -0.5)
    key = torch.arange(Lk, device=dev)
    hidden = (key[None, :] >= kv_lens[:, None])[:, None, None, None, :]
    if causal:
        last = (kv_lens.long() - n_new)[:, None] + torch.arange(max_q, device=dev)[None, :]
        hidden = hidden | (key[None, None, :] > last[:, :, None])[:, None, None]
    s.masked_fill_(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    # A request's keys end before the padding: rows of the padding weigh nothing.
    o = torch.matmul(s.view(R, Hkv, G * max_q, Lk), v.float().permute(0, 2, 1, 3))
    o = o.view(R, Hkv, G, max_q, D) / torch.where(total == 0, torch.ones_like(total), total)
    tok = torch.arange(T, device=dev)
    r = torch.searchsorted(cu_q[1:].long(), tok, right=True).clamp(max=R - 1)
    return o.permute(0, 3, 1, 2, 4)[r, tok - cu_q[r]].reshape(T, Hq, D).to(q.dtype)


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(c: dict) -> dict:
    kind = c["kind"]
    if kind == "commit":
        rows = c["layers"] * c["T"] * c["H"] * c["D"]
        tables = 2 * c["T"] * c["D"] // 2 * 4 if c["rope"] else 0
        return {"bytes": 8 * rows + tables + 8 * c["T"], "flops": 3.0 * rows if c["rope"] else 0.0}
    nq, nk = _lengths(c)
    if kind == "tables":
        P, W = c["P"], c["W"]
        fresh = sum(max(0, min(W, -(-k // P)) - min(W, -(-(k - n) // P))) for n, k in zip(nq, nk))
        return {"bytes": 16 * c["R"] + 8 * fresh + 8 * (sum(nq) + c["pad"]) + 12,
                "flops": 4.0 * (c["R"] + sum(nq))}
    D, Hkv = c["D"], c["Hkv"]
    Hq = Hkv * c["G"]
    pairs = sum(n * k - (n * (n - 1) // 2 if c["causal"] else 0) for n, k in zip(nq, nk))
    n_bytes = 2 * D * (2 * Hq * sum(nq) + 2 * Hkv * sum(nk))
    if kind == "paged":
        n_bytes += 4 * sum(-(-k // c["P"]) for k in nk)
    return {"bytes": n_bytes, "flops": 4.0 * D * Hq * pairs}


# ---------------------------------------------------------------------------
# The same in 64 bits, request by request.
# ---------------------------------------------------------------------------
def exact(case: dict, seed: int):
    t, kind = prepare(case, seed), case["kind"]
    if kind == "tables":
        return None  # whole numbers
    if kind == "commit":
        L, H, D = case["layers"], case["H"], case["D"]
        out = []
        for pages, src, turn in ((t["pages_k"], t["k"], case["rope"]),
                                 (t["pages_v"], t["v"], False)):
            flat = pages.double().view(L, -1, H, D)
            for i in range(L):
                x = src[i, :t["real"]].double()
                if turn:
                    a, b = x[..., 0::2], x[..., 1::2]
                    cs = t["cos"][:t["real"], None, ::2].double()
                    sn = t["sin"][:t["real"], None, ::2].double()
                    x = torch.stack((a * cs - b * sn, b * cs + a * sn), -1).flatten(-2)
                flat[i, t["slots"][:t["real"]]] = x
            out.append(flat.view(pages.shape))
        return tuple(out)
    nq, nk = _lengths(case)
    cu, G, P = _cu(nq), case["G"], case.get("P")
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for r, (n, m) in enumerate(zip(nq, nk)):
        if n == 0 or m == 0:
            continue
        if kind == "paged":
            ids = t["table"][r, :-(-m // P)].long()
            k, v = (t[x][ids].flatten(0, 1)[:m] for x in ("pages_k", "pages_v"))
        else:
            k, v = t["k"][cu[r]:cu[r + 1]], t["v"][cu[r]:cu[r + 1]]
        for h in range(t["q"].shape[1]):
            kh, vh = k[:, h // G].double(), v[:, h // G].double()
            qh = t["q"][cu[r]:cu[r + 1], h].double()
            for i in range(0, n, 4096):
                s = qh[i:i + 4096] @ kh.t().contiguous() / math.sqrt(case["D"])
                if case["causal"]:
                    last = m - n + torch.arange(i, min(i + 4096, n), device="cuda")
                    key = torch.arange(m, device="cuda")
                    s.masked_fill_(key[None, :] > last[:, None], -math.inf)
                p = torch.softmax(s, -1)
                out[cu[r] + i:cu[r] + i + p.shape[0], h] = p @ vh
    return out
