"""paged_tables and kv_commit_rope_paged against their plain forms, exactly, and a serving loop
of all four paged calls against attention over the whole sequences."""
from __future__ import annotations

import random

import pytest
import torch

import joyomni_ops as jo
from oracle import serving

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def tables_case(dev, ctx, new, W, P, free, num_free, num_pages, max_tokens, table=None):
    R = len(ctx)
    if table is None:
        table = [[(r * W + j) % max(num_pages, 1) for j in range(W)] for r in range(R)]
    want = serving.paged_tables(ctx, new, table, free, num_free, P, num_pages, max_tokens)
    t = torch.tensor(table, dtype=torch.int32, device=dev).view(R, W)
    got = jo.paged_tables(i32(ctx, dev), i32(new, dev), t, i32(free, dev), i32([num_free], dev), P,
                          num_pages, max_tokens)
    names = ("cu_q", "kv_lens", "slots", "free_left", "block_table")
    for name, g, w in zip(names, (*got, t), (*want[:3], [want[3]], want[4])):
        assert g.tolist() == w, name


@pytest.mark.parametrize("P", (1, 3, 16, 64))
@pytest.mark.parametrize("R", (1, 2, 63, 64, 65, 300, 1023, 1025, 2500))
def test_tables(dev, R, P):
    rng = random.Random(R * 100 + P)
    ctx = [rng.choice((0, 1, P, P - 1, rng.randint(0, 200))) for _ in range(R)]
    new = [rng.choice((0, 1, 1, rng.randint(0, 3 * P))) for _ in range(R)]
    W = max(-(-(c + n) // P) for c, n in zip(ctx, new)) or 1
    pages = sum(-(-(c + n) // P) - -(-c // P) for c, n in zip(ctx, new))
    free = list(range(pages + 5))
    rng.shuffle(free)
    tables_case(dev, ctx, new, W, P, free, pages + 2, R * W + pages + 5, sum(new) + 9)


def test_tables_many_tokens(dev):
    """More tokens than the launch's threads."""
    tables_case(dev, [5, 0, 70], [70000, 1, 3000], 9000, 16, list(range(5000)), 5000, 30000, 73005)


def test_tables_out_of_room(dev):
    """Pages, table columns and tokens that run out: -1, and the count of what is missing."""
    ctx, new = [5, 0, 17, 3], [20, 9, 40, 1]
    tables_case(dev, ctx, new, 10, 4, list(range(40, 47)), 7, 60, 80)   # pages
    tables_case(dev, ctx, new, 10, 4, list(range(40, 47)), 99, 60, 80)  # a count past the stack
    tables_case(dev, ctx, new, 10, 4, list(range(40, 47)), -3, 60, 80)
    tables_case(dev, ctx, new, 10, 4, [], 0, 60, 80)
    tables_case(dev, ctx, new, 6, 4, list(range(60)), 60, 60, 80)       # columns
    for most in (0, 1, 20, 29, 33, 69, 70):
        tables_case(dev, ctx, new, 10, 4, list(range(60)), 60, 60, most)  # tokens


def test_tables_ids_that_name_no_page(dev):
    table = [[9, -1, 3], [99, 2, 2], [-7, 1, 1]]
    tables_case(dev, [3, 2, 4], [6, 3, 1], 3, 4, [1, 50, -2, 7], 4, 10, 12, table=table)


def test_tables_strange_lengths(dev):
    big = 2 ** 31 - 1
    ctx, new, W, P = [big, -5, big, 4], [big, 3, -1, big], 3, 16
    # (The plain form walks every token: max_tokens keeps it short.)
    table = [[0, 1, 2] for _ in ctx]
    t = torch.tensor(table, dtype=torch.int32, device=dev)
    cu, kv, slots, left = jo.paged_tables(i32(ctx, dev), i32(new, dev), t, i32([5, 6], dev),
                                          i32([2], dev), P, 10, 40)
    assert cu.tolist() == [0, 40, 40, 40, 40] and kv.tolist() == [big, 0, big, 4]
    assert slots.tolist() == [-1] * 40 and left.tolist() == [2] and t.tolist() == table
    ctx, new = [0, 0], [big, big]
    cu, kv, slots, left = jo.paged_tables(i32(ctx, dev), i32(new, dev), t[:2], i32([5, 6], dev),
                                          i32([2], dev), P, 10, 20)
    assert cu.tolist() == [0, 20, 20] and slots.tolist() == [6 * 16 + i for i in range(16)] + [
        5 * 16 + i for i in range(4)]


def test_tables_nothing(dev):
    e = i32([], dev)
    cu, kv, slots, left = jo.paged_tables(e, e, e.view(0, 4), i32([3], dev), i32([1], dev), 16, 4, 3)
    assert cu.tolist() == [0] and kv.tolist() == [] and slots.tolist() == [-1] * 3
    assert left.tolist() == [1]
    tables_case(dev, [3], [0], 2, 4, [1], 1, 9, 0)


def test_tables_row_stride(dev):
    big = torch.full((4, 10), -9, dtype=torch.int32, device=dev)
    t = big[:, 2:6]
    jo.paged_tables(i32([0, 0, 0, 0], dev), i32([5, 0, 9, 1], dev), t, i32([0, 1, 2, 3, 4, 5, 6], dev),
                    i32([7], dev), 4, 7, 20)
    assert t.tolist() == [[6, 5, -9, -9], [-9] * 4, [4, 3, 2, -9], [1, -9, -9, -9]]
    assert bool((big[:, :2] == -9).all()) and bool((big[:, 6:] == -9).all())


# ---------------------------------------------------------------------------
# The commit.
# ---------------------------------------------------------------------------
def commit_case(dev, L, T, H, D, N, P, dtype, rope=True, seed=0, skip=(), layers_dim=True,
                packed=False):
    g = torch.Generator().manual_seed(seed)

    def rand(*s):
        return torch.randn(s, generator=g).to(dtype)

    if packed:  # slices of one projection of all layers
        kv = rand(L, T, 2, H, D)
        k, v = kv[:, :, 0], kv[:, :, 1]
        dkv = kv.to(dev)
        dk, dv = dkv[:, :, 0], dkv[:, :, 1]
    else:
        k, v = rand(L, T, H, D), rand(L, T, H, D)
        dk, dv = k.to(dev), v.to(dev)
    pk, pv = rand(L, N, P, H, D), rand(L, N, P, H, D)
    slots = torch.randperm(N * P, generator=g)[:T]
    for i, s in skip:
        slots[i] = s
    cos = sin = None
    if rope:
        ang = torch.rand(T, D, generator=g) * 100
        cos, sin = ang.cos(), ang.sin()
    want = serving.kv_commit_rope_paged(k, v, pk, pv, slots, cos, sin)
    gk, gv = pk.to(dev), pv.to(dev)
    one = (lambda t: t) if layers_dim else (lambda t: t[0])  # noqa: E731
    to = (lambda t: None if t is None else t.to(dev))  # noqa: E731
    jo.kv_commit_rope_paged(one(dk), one(gk), slots.to(dev), to(cos), to(sin), src_v=one(dv),
                            pages_v=one(gv))
    assert torch.equal(gk.cpu(), want[0]) and torch.equal(gv.cpu(), want[1])
    k_only = pk.to(dev)
    jo.kv_commit_rope_paged(one(dk), one(k_only), slots.to(dev), to(cos), to(sin))
    assert torch.equal(k_only.cpu(), want[0])


@pytest.mark.parametrize("rope", (True, False))
@pytest.mark.parametrize("dtype", (BF16, FP16))
@pytest.mark.parametrize("L,T,H,D,N,P", ((1, 1, 1, 64, 1, 1), (1, 30, 8, 128, 4, 16),
                                         (3, 77, 2, 64, 3, 52), (2, 9, 4, 256, 5, 7),
                                         (2, 100, 32, 128, 9, 16), (1, 5, 3, 96, 2, 4),
                                         (2, 6, 5, 2, 2, 4), (1, 4, 24, 128, 3, 3),
                                         (1, 3, 33, 128, 2, 2)))
def test_commit(dev, L, T, H, D, N, P, dtype, rope):
    commit_case(dev, L, T, H, D, N, P, dtype, rope)


def test_commit_leaves_out_slots_outside_the_pool(dev):
    skip = ((0, -1), (5, -(2 ** 40)), (7, 64), (9, 2 ** 31), (11, 2 ** 32), (12, 2 ** 62))
    commit_case(dev, 2, 40, 4, 128, 4, 16, BF16, skip=skip)
    commit_case(dev, 2, 40, 3, 6, 4, 16, BF16, skip=skip)  # element-wise kernel


def test_commit_forms(dev):
    commit_case(dev, 1, 20, 4, 128, 4, 16, BF16, layers_dim=False)
    commit_case(dev, 3, 20, 4, 128, 4, 16, BF16, packed=True)
    commit_case(dev, 1, 1, 4, 128, 4, 16, BF16, packed=True, layers_dim=False)


def test_commit_matches_the_contiguous_commit(dev):
    """The same rows through kv_commit_rope into a contiguous pool: equal bits."""
    L, T, H, D, P = 2, 104, 8, 128, 52
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(L, T, H, D, generator=g).to(BF16).to(dev) for _ in range(2))
    ang = torch.rand(T, D, generator=g) * 100
    cos, sin = ang.cos().to(dev), ang.sin().to(dev)
    a = [torch.zeros(L, 1, T, H, D, dtype=BF16, device=dev) for _ in range(2)]
    jo.kv_commit_rope(k[:, None], a[0], 0, cos, sin, src_v=v[:, None], dst_v=a[1])
    b = [torch.zeros(L, 2, P, H, D, dtype=BF16, device=dev) for _ in range(2)]
    jo.kv_commit_rope_paged(k, b[0], torch.arange(T, device=dev), cos, sin, src_v=v, pages_v=b[1])
    for x, y in zip(a, b):
        assert torch.equal(x.view(L, T, H, D), y.view(L, T, H, D))


def test_commit_pool_past_32_bits(dev):
    """Rows of a pool of more than 2^31 elements."""
    H, D, P = 32, 128, 64
    N = 2 ** 31 // (P * H * D) + 3
    pk = torch.empty(N, P, H, D, dtype=BF16, device=dev)
    k = torch.randn(4, H, D, device=dev).to(BF16)
    at = [(N - 1, 63), (N - 2, 0), (0, 5), (N - 1, 0)]
    jo.kv_commit_rope_paged(k, pk, torch.tensor([p * P + o for p, o in at], device=dev))
    for i, (p, o) in enumerate(at):
        assert torch.equal(pk[p, o], k[i])


# ---------------------------------------------------------------------------
# All four together: prompts in chunks, then single tokens, captured and replayed.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("captured", (False, True))
def test_serving_loop(dev, captured):
    """Three requests: prompts admitted in chunks beside single tokens of the others, in a
    padded step of fixed size, each step's tables, commit and attention from its lengths alone.
    Every step's rows equal attention over the request's whole sequence so far (packed), up to
    the roundings of the two results."""
    R, Hq, Hkv, D, P, step = 3, 8, 2, 128, 16, 64
    totals = [150, 37, 90]
    plan = [[40, 0, 20], [60, 3, 1], [49, 0, 1], [1, 20, 1], [0, 1, 40], [0, 13, 27]]
    assert [sum(p[r] for p in plan) for r in range(R)] == totals
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(sum(totals), h, D, generator=g).to(BF16).to(dev) for h in (Hq, Hkv, Hkv))
    ang = torch.rand(max(totals), D // 2, generator=g).repeat_interleave(2, 1) * 50
    cos_all, sin_all = ang.cos().to(dev), ang.sin().to(dev)
    start = [0, 150, 187]
    W, N = 12, 30
    table = torch.full((R, W), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(N, generator=g).to(torch.int32).to(dev)
    num_free, ctx, new = i32([N], dev), i32([0] * R, dev), i32([0] * R, dev)
    pk, pv = (torch.full((N, P, Hkv, D), float("nan"), dtype=BF16, device=dev) for _ in range(2))
    sq, sk, sv = (torch.zeros(step * 2, h, D, dtype=BF16, device=dev) for h in (Hq, Hkv, Hkv))
    cos, sin = (torch.zeros(step * 2, D, device=dev) for _ in range(2))

    def serve():
        cu, kv, slots, left = jo.paged_tables(ctx, new, table, free, num_free, P, N, step * 2)
        jo.kv_commit_rope_paged(sk, pk, slots, cos, sin, src_v=sv, pages_v=pv)
        return jo.attention_paged(sq, pk, pv, table, cu, kv), left, kv

    graph = None
    if captured:
        serve()  # no request has tokens: nothing is written
        torch.cuda.synchronize(dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = serve()
    done = [0] * R
    for lens in plan:
        at = 0
        for r, n in enumerate(lens):
            rows, pos = slice(start[r] + done[r], start[r] + done[r] + n), slice(done[r], done[r] + n)
            for dst, src in ((sq, q), (sk, k), (sv, v)):
                dst[at:at + n] = src[rows]
            cos[at:at + n], sin[at:at + n] = cos_all[pos], sin_all[pos]
            at += n
        ctx.copy_(i32(done, dev))
        new.copy_(i32(lens, dev))
        if captured:
            graph.replay()
            out, left, kv = held
        else:
            out, left, kv = serve()
        num_free.copy_(left)
        done = [d + n for d, n in zip(done, lens)]
        assert kv.tolist() == done
        at = 0
        for r, n in enumerate(lens):
            if n:
                m = done[r]
                rows = slice(start[r], start[r] + m)
                turned = jo.apply_rotary_emb(k[None, rows], (cos_all[:m], sin_all[:m]))[0]
                want = jo.attention_varlen(q[rows].contiguous(), turned, v[rows].contiguous(),
                                           i32([0, m], dev))[m - n:]
                diff = (out[at:at + n].float() - want.float()).abs()
                assert float(diff.max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())
            at += n
        assert bool((out[at:] == 0).all())
    held_pages = sum(-(-t // P) for t in totals)
    assert num_free.item() == N - held_pages
