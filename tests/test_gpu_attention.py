"""attention_varlen and attention_paged against the definition in 64 bits, with bounds made of
the roundings they are allowed (oracle.serving.attention_bound)."""
from __future__ import annotations

import math

import pytest
import torch

import joyomni_ops as jo
from oracle import serving

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def cu_of(lens):
    return [0] + torch.tensor(lens, dtype=torch.int64).cumsum(0).tolist() if lens else [0]


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def randn(shape, dtype, seed, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * mul).to(dtype)


def seen_mask(n, m, causal, hidden=None):
    """bool [n, m]: what the i-th of n new tokens sees of m keys; hidden: keys that have no
    place (bool [m])."""
    j = torch.arange(m)[None, :]
    seen = (j <= m - n + torch.arange(n)[:, None]) if causal else torch.ones(n, m, dtype=torch.bool)
    return seen if hidden is None else seen & ~hidden[None, :]


def check(out, q, requests, scale, dtype):
    """requests: [(q0, q1, k, v, seen)] of the rows that belong to a request."""
    out = out.cpu()
    rest = torch.ones(q.shape[0], dtype=torch.bool)
    for q0, q1, k, v, seen in requests:
        rest[q0:q1] = False
        if q1 == q0:
            continue
        want, size, score = serving.attention(q[q0:q1], k, v, seen, scale)
        fin = torch.isfinite(want)
        got = out[q0:q1].double()
        v_max = float(v.double().nan_to_num(0, 0, 0).abs().max()) if v.numel() else 0.0
        bound = serving.attention_bound(dtype, want.nan_to_num(), size.nan_to_num(), score.nan_to_num(),
                                        int(seen.sum(1).max()) if seen.numel() else 0, v_max)
        assert bool((torch.isfinite(got) == fin).all()), "finite where the definition is not, or not"
        err = (got - want).abs()[fin]
        over = err > bound[fin]
        assert not bool(over.any()), (
            f"{int(over.sum())} of {err.numel()} beyond the bound; worst "
            f"{float((err / bound[fin]).max()):.3f} of it")
        empty = ~seen.any(1)
        assert bool((out[q0:q1][empty] == 0).all()), "a row that sees nothing must be zeros"
    return rest


# ---------------------------------------------------------------------------
# Packed sequences.
# ---------------------------------------------------------------------------
def varlen_case(dev, lq, lk, Hq, Hkv, D, dtype, causal, seed=0, pad=0, mul=1.3, packed=False,
                scale=None, out=None):
    T, Tk = sum(lq) + pad, sum(lk) + pad
    if packed:
        qkv = randn((T, Hq + 2 * Hkv, D), dtype, seed, mul)
        q, k, v = qkv.split((Hq, Hkv, Hkv), 1)
        dq = qkv.to(dev)
        gq, gk, gv = dq.split((Hq, Hkv, Hkv), 1)
    else:
        q, k, v = (randn((t, h, D), dtype, seed + i, m)
                   for i, (t, h, m) in enumerate(((T, Hq, mul), (Tk, Hkv, mul), (Tk, Hkv, 1.0))))
        gq, gk, gv = q.to(dev), k.to(dev), v.to(dev)
    cq, ck = cu_of(lq), cu_of(lk)
    got = jo.attention_varlen(gq, gk, gv, i32(cq, dev), None if lq is lk else i32(ck, dev),
                              causal=causal, scale=scale, out=out)
    reqs = [(cq[r], cq[r + 1], k[ck[r]:ck[r + 1]], v[ck[r]:ck[r + 1]],
             seen_mask(lq[r], lk[r], causal)) for r in range(len(lq))]
    rest = check(got, q, reqs, scale or D ** -0.5, dtype)
    if out is None:
        assert bool((got.cpu()[rest] == 0).all())
    return got


LENS = [[1], [2, 1, 1], [0, 5, 0, 64, 65, 1, 0], [127, 128, 129], [300], [17] * 9, [31, 33, 16, 15],
        [255, 1, 257]]


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("dtype", (BF16, FP16))
def test_varlen_lengths(dev, dtype, lens, causal):
    varlen_case(dev, lens, lens, 4, 2, 128, dtype, causal)


@pytest.mark.parametrize("D", (64, 128, 256))
@pytest.mark.parametrize("heads", ((1, 1), (3, 3), (6, 2), (5, 1), (7, 1), (16, 1), (20, 1), (40, 2), (8, 8)),
                         ids=lambda x: f"{x[0]}over{x[1]}")
def test_varlen_heads(dev, heads, D):
    lens = [3, 70, 1, 130]
    varlen_case(dev, lens, lens, *heads, D, BF16, True, seed=1)
    varlen_case(dev, lens, lens, *heads, D, FP16, False, seed=2)


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("lq,lk", (([5, 9], [0, 3]), ([1, 1, 1], [500, 0, 1]), ([40], [1700]),
                                   ([100, 3], [20, 64]), ([0, 7], [9, 7]), ([64, 0], [0, 0]),
                                   ([200], [64]), ([33], [2100])))
def test_varlen_cross_lengths(dev, lq, lk, causal):
    """Fewer keys than tokens leave the first tokens with nothing to see (causal)."""
    for D in (64, 128, 256):
        varlen_case(dev, lq, lk, 4, 2, D, BF16, causal, seed=3)


@pytest.mark.parametrize("D", (64, 128, 256))
@pytest.mark.parametrize("heads", ((4, 4), (8, 2)))
def test_varlen_packed_projection(dev, heads, D):
    lens = [77, 12, 140]
    varlen_case(dev, lens, lens, *heads, D, BF16, True, seed=4, packed=True)


def test_varlen_scale_and_peaked_scores(dev):
    lens = [90, 200]
    varlen_case(dev, lens, lens, 4, 2, 128, BF16, True, seed=5, scale=0.5)
    varlen_case(dev, lens, lens, 4, 2, 64, FP16, False, seed=6, mul=6.0)
    varlen_case(dev, lens, lens, 4, 2, 128, BF16, True, seed=7, scale=1e-3)


def test_rows_behind_the_last_sequence(dev):
    lens = [60, 9]
    varlen_case(dev, lens, lens, 4, 2, 128, BF16, True, seed=8, pad=201)  # zeros in a new tensor
    out = torch.full((270, 4, 128), 7.0, dtype=BF16, device=dev)
    got = varlen_case(dev, lens, lens, 4, 2, 128, BF16, True, seed=8, pad=201, out=out)
    assert got is out
    assert bool((out[69:] == 7).all())


def test_strided_out_keeps_its_gaps(dev):
    lens = [60, 9, 130]
    big = torch.full((199, 6, 200), 3.0, dtype=BF16, device=dev)
    out = big[:, 1:5, 8:136]
    varlen_case(dev, lens, lens, 4, 2, 128, BF16, True, seed=9, out=out)
    keep = big.clone()
    keep[:, 1:5, 8:136] = 3.0
    assert bool((keep == 3).all())


def test_no_requests_and_no_tokens(dev):
    q = torch.ones(5, 2, 64, dtype=BF16, device=dev)
    assert bool((jo.attention_varlen(q, q, q, i32([0], dev)) == 0).all())
    e = q[:0]
    assert jo.attention_varlen(e, e, e, i32([0, 0], dev)).shape == (0, 2, 64)
    assert bool((jo.attention_varlen(q, e, e, i32([0, 5], dev), i32([0, 0], dev)) == 0).all())


@pytest.mark.parametrize("bad", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("D", (64, 128, 256))
def test_later_tokens_do_not_reach_earlier_ones(dev, D, bad):
    """NaN and infinities in k and v of the token at place 100: the tokens before it, and every
    other sequence, are as if it were not there."""
    lens, Hq, Hkv = [150, 120, 40], 4, 2
    cu = cu_of(lens)
    q, k, v = (randn((sum(lens), h, D), BF16, 10 + i) for i, h in enumerate((Hq, Hkv, Hkv)))
    clean = jo.attention_varlen(q.to(dev), k.to(dev), v.to(dev), i32(cu, dev)).cpu()
    at = cu[1] + 100
    v[at, :, ::3] = bad
    k[at, :, ::5] = math.nan
    got = jo.attention_varlen(q.to(dev), k.to(dev), v.to(dev), i32(cu, dev)).cpu()
    before = torch.ones(sum(lens), dtype=torch.bool)
    before[at:cu[2]] = False
    assert bool(torch.isfinite(got[before]).all())
    reqs = [(cu[r], cu[r + 1], k[cu[r]:cu[r + 1]], v[cu[r]:cu[r + 1]],
             seen_mask(lens[r], lens[r], True)) for r in (0, 2)]
    n = 100
    reqs.append((cu[1], cu[1] + n, k[cu[1]:cu[1] + n], v[cu[1]:cu[1] + n], seen_mask(n, n, True)))
    check(got, q, reqs, D ** -0.5, BF16)
    assert bool(torch.isnan(got[at:cu[2]]).all())  # who sees a NaN score has no result
    assert bool((clean[:cu[1]] == got[:cu[1]]).all())


def test_seen_infinities_are_the_definition_s(dev):
    """An infinite v that is seen gives infinities in its own columns alone."""
    lens, D = [70], 128
    q, k, v = (randn((70, 1, D), BF16, 20 + i) for i in range(3))
    v[30, 0, 5] = math.inf
    got = jo.attention_varlen(q.to(dev), k.to(dev), v.to(dev), i32([0, 70], dev)).cpu()
    assert bool(torch.isinf(got[30:, 0, 5]).all()) and bool(torch.isfinite(got[:30]).all())
    other = torch.arange(D) != 5
    assert bool(torch.isfinite(got[:, :, other]).all())


def test_lengths_outside_the_tensors_are_cut(dev):
    """cu_q past the tokens: the sequences end with the tensor."""
    q, k, v = (randn((50, 2, 64), BF16, 30 + i) for i in range(3))
    got = jo.attention_varlen(q.to(dev), k.to(dev), v.to(dev), i32([0, 20, 1000], dev))
    want = jo.attention_varlen(q.to(dev), k.to(dev), v.to(dev), i32([0, 20, 50], dev))
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# Paged keys.
# ---------------------------------------------------------------------------
def paged_case(dev, new, ctx, P, Hq, Hkv, D, dtype, causal, seed=0, holes=(), fill=math.nan,
               head_major=False, extra_width=2, pad=0, scale=None, mul=1.3):
    """Requests of new[r] tokens over ctx[r] cached ones and their own. Every place of the pool
    that holds no key of a request is `fill`; holes: (request, column) entries without a page."""
    R = len(new)
    keys = [n + c for n, c in zip(new, ctx)]
    need = [-(-m // P) for m in keys]
    W, N = max(need + [1]) + extra_width, sum(need) + 3
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(N, generator=g).tolist()
    q = randn((sum(new) + pad, Hq, D), dtype, seed + 1, mul)
    shape = (N, Hkv, P, D) if head_major else (N, P, Hkv, D)
    pk, pv = (torch.full(shape, fill, dtype=dtype) for _ in range(2))
    vk, vv = (x.transpose(1, 2) if head_major else x for x in (pk, pv))
    table = torch.full((R, W), -1, dtype=torch.int32)
    cq, reqs = cu_of(new), []
    for r in range(R):
        pages = [order.pop() for _ in range(need[r])]
        table[r, :need[r]] = torch.tensor(pages, dtype=torch.int32)
        table[r, need[r]:] = 10 ** 6 if r % 2 else -1  # never looked at
        k, v = (randn((keys[r], Hkv, D), dtype, seed + 10 * r + 2 + i, m)
                for i, m in enumerate((mul, 1.0)))
        hidden = torch.zeros(keys[r], dtype=torch.bool)
        for j in range(keys[r]):
            vk[pages[j // P], j % P], vv[pages[j // P], j % P] = k[j], v[j]
        for hr, col in holes:
            if hr == r and col < need[r]:
                table[r, col] = -1 if col % 2 else N + col
                hidden[col * P:(col + 1) * P] = True
        reqs.append((cq[r], cq[r + 1], k, v, seen_mask(new[r], keys[r], causal, hidden)))
    dk, dv = pk.to(dev), pv.to(dev)
    if head_major:
        dk, dv = dk.transpose(1, 2), dv.transpose(1, 2)
    got = jo.attention_paged(q.to(dev), dk, dv, table.to(dev), i32(cq, dev), i32(keys, dev),
                             causal=causal, scale=scale)
    rest = check(got, q, reqs, scale or D ** -0.5, dtype)
    assert bool((got.cpu()[rest] == 0).all())
    return got


@pytest.mark.parametrize("P", (1, 7, 16, 52, 64, 128))
@pytest.mark.parametrize("D,dtype", ((64, BF16), (128, BF16), (256, BF16), (128, FP16)))
def test_paged_single_tokens(dev, D, dtype, P):
    paged_case(dev, [1] * 6, [0, 1, 15, 64, 130, 333], P, 8, 2, D, dtype, True)


@pytest.mark.parametrize("P", (1, 16, 52, 64))
@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("D", (64, 128, 256))
def test_paged_chunks(dev, D, causal, P):
    paged_case(dev, [5, 0, 1, 70, 33, 128], [40, 9, 200, 0, 64, 31], P, 4, 2, D, BF16, causal, seed=1)


@pytest.mark.parametrize("heads", ((1, 1), (3, 3), (6, 2), (5, 1), (16, 1), (20, 1), (33, 1), (12, 4)),
                         ids=lambda x: f"{x[0]}over{x[1]}")
def test_paged_heads(dev, heads):
    for D in (64, 128, 256):
        paged_case(dev, [1, 2, 1, 9], [70, 3, 0, 100], 16, *heads, D, BF16, True, seed=2)


@pytest.mark.parametrize("new,ctx", (([1], [5000]), ([1, 1], [4000, 3]), ([3], [3000]), ([70], [2500]),
                                     ([1] * 40, [37 * i % 900 for i in range(40)]),
                                     ([1, 200, 1, 1], [2000, 700, 1, 0])))
@pytest.mark.parametrize("D", (64, 128, 256))
def test_paged_long_keys_are_split(dev, D, new, ctx):
    paged_case(dev, new, ctx, 16, 4, 1, D, BF16, True, seed=3)
    paged_case(dev, new, ctx, 52, 2, 2, D, FP16, False, seed=4)


@pytest.mark.parametrize("fill", (math.nan, math.inf, 0.0))
def test_paged_entries_without_a_page(dev, fill):
    """Table entries that name no page: their keys are not there, whatever page 0 holds."""
    holes = ((0, 0), (1, 1), (1, 2), (2, 0), (2, 1), (3, 5))
    for D in (64, 128):
        for new in ([1, 1, 1, 1], [40, 3, 70, 20]):
            paged_case(dev, new, [100, 200, 10, 333], 32, 4, 2, D, BF16, True, seed=5, holes=holes,
                       fill=fill)


def test_paged_head_major_pages(dev):
    paged_case(dev, [1, 40, 1], [77, 100, 0], 16, 8, 2, 128, BF16, True, seed=6, head_major=True)


def test_paged_padded_step(dev):
    paged_case(dev, [1, 1, 30], [77, 100, 0], 16, 8, 2, 128, BF16, True, seed=7, pad=97)


def test_paged_more_new_tokens_than_keys(dev):
    """kv_lens below a request's tokens: the first ones see nothing."""
    D, dtype = 128, BF16
    q, pk, pv = randn((9, 2, D), dtype, 1), randn((2, 4, 2, D), dtype, 2), randn((2, 4, 2, D), dtype, 3)
    got = jo.attention_paged(q.to(dev), pk.to(dev), pv.to(dev), i32([[1, 0]], dev), i32([0, 9], dev),
                             i32([5], dev))
    k, v = (x[[1, 0]].flatten(0, 1)[:5] for x in (pk, pv))
    check(got, q, [(0, 9, k, v, seen_mask(9, 5, True))], D ** -0.5, dtype)


def test_paged_lengths_past_the_table(dev):
    """kv_lens past what the table's rows can place: keys end with the table, positions do not."""
    D, dtype = 128, BF16
    q, pk, pv = randn((1, 2, D), dtype, 1), randn((3, 4, 2, D), dtype, 2), randn((3, 4, 2, D), dtype, 3)
    got = jo.attention_paged(q.to(dev), pk.to(dev), pv.to(dev), i32([[2, 0]], dev), i32([0, 1], dev),
                             i32([2 ** 31 - 1], dev))
    k, v = (x[[2, 0]].flatten(0, 1) for x in (pk, pv))
    check(got, q, [(0, 1, k, v, torch.ones(1, 8, dtype=torch.bool))], D ** -0.5, dtype)
    none = jo.attention_paged(q.to(dev), pk[:0].to(dev), pv[:0].to(dev), i32([[2, 0]], dev),
                              i32([0, 1], dev), i32([4], dev))
    assert bool((none == 0).all())


@pytest.mark.parametrize("new", (1, 40))
def test_paged_pool_past_32_bits(dev, new):
    """A pool of 2^31 elements and more (4.3 GB each of K and V): its last pages."""
    P, Hkv, D, ctx = 64, 8, 128, 300
    N = 2 ** 31 // (P * Hkv * D) + 9
    pk, pv = (torch.empty((N, P, Hkv, D), dtype=BF16, device=dev) for _ in range(2))
    m = ctx + new
    need = -(-m // P)
    q, k, v = randn((new, 16, D), BF16, 1), randn((m, Hkv, D), BF16, 2), randn((m, Hkv, D), BF16, 3)
    pages = [N - 1 - i for i in range(need)]
    for i, p in enumerate(pages):
        part = slice(i * P, min(m, (i + 1) * P))
        n = part.stop - part.start
        pk[p, :n], pv[p, :n] = k[part].to(dev), v[part].to(dev)
    got = jo.attention_paged(q.to(dev), pk, pv, i32([pages], dev), i32([0, new], dev), i32([m], dev))
    check(got, q, [(0, new, k, v, seen_mask(new, m, True))], D ** -0.5, BF16)


# ---------------------------------------------------------------------------
# Streams, graphs, repeats.
# ---------------------------------------------------------------------------
def step_inputs(dev, seed=0, new=(1, 1, 40, 1), ctx=(700, 20, 100, 3000), P=16):
    keys = [n + c for n, c in zip(new, ctx)]
    need = [-(-m // P) for m in keys]
    N, W = sum(need), max(need)
    table = torch.full((len(new), W), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = torch.arange(at, at + n)
        at += n
    q = randn((sum(new), 8, 128), BF16, seed, 1.3).to(dev)
    pk, pv = (randn((N, P, 2, 128), BF16, seed + i).to(dev) for i in (1, 2))
    return q, pk, pv, table.to(dev), i32(cu_of(list(new)), dev), i32(keys, dev)


def test_same_call_same_bits(dev):
    args = step_inputs(dev)
    first = jo.attention_paged(*args)
    for _ in range(3):
        assert torch.equal(jo.attention_paged(*args), first)


def test_side_stream(dev):
    args = step_inputs(dev)
    want = jo.attention_paged(*args)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        got = jo.attention_paged(*args)
    s.synchronize()
    assert torch.equal(got, want)


def test_two_captured_graphs_with_new_lengths(dev):
    """Two graphs of different steps, replayed in turn with eager work between, lengths and
    inputs changed in place: every replay equals the eager call."""
    a, b = step_inputs(dev, 1), step_inputs(dev, 2, new=(1, 1, 1, 1), ctx=(5000, 20, 9, 0))
    graphs, outs = [], []
    for args in (a, b):
        jo.attention_paged(*args)
        torch.cuda.synchronize(dev)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = jo.attention_paged(*args)
        graphs.append(g)
        outs.append(o)
    for k in range(4):
        for args, g, o in ((a, graphs[0], outs[0]), (b, graphs[1], outs[1])):
            args[0].copy_(randn(tuple(args[0].shape), BF16, 50 + k, 1.3))
            args[5].sub_(3 if k % 2 else 0).clamp_(min=0)
            want = jo.attention_paged(*args)
            g.replay()
            torch.cuda.synchronize(dev)
            assert torch.equal(o, want), k


def test_paged_equals_packed(dev):
    """The same keys in pages and packed: whole prompts through both entry points."""
    lens, Hq, Hkv, D, P = [130, 7, 64], 8, 2, 128, 16
    q, k, v = (randn((sum(lens), h, D), BF16, 60 + i).to(dev) for i, h in enumerate((Hq, Hkv, Hkv)))
    cu = i32(cu_of(lens), dev)
    packed = jo.attention_varlen(q, k, v, cu)
    need = [-(-n // P) for n in lens]
    pk, pv = (torch.zeros(sum(need), P, Hkv, D, dtype=BF16, device=dev) for _ in range(2))
    table, at = torch.full((3, max(need)), -1, dtype=torch.int32), 0
    for r, n in enumerate(lens):
        for j in range(need[r]):
            rows = slice(cu_of(lens)[r] + j * P, min(cu_of(lens)[r + 1], cu_of(lens)[r] + (j + 1) * P))
            m = rows.stop - rows.start
            pk[at, :m], pv[at, :m], table[r, j] = k[rows], v[rows], at
            at += 1
    paged = jo.attention_paged(q, pk, pv, table.to(dev), cu, i32(lens, dev))
    diff = (paged.float() - packed.float()).abs()
    # Both within their bound of the same value: together twice a step of bf16 of the terms' size.
    assert float(diff.max()) <= 4 * 2.0 ** -8 * float(v.float().abs().max())


# ---------------------------------------------------------------------------
# Many requests, strides, sizes at random.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("R", (64, 65, 129, 256, 257, 700))
def test_many_requests(dev, R):
    """Past 64 requests a wave looks after four each, past 256 the keys are not split."""
    g = torch.Generator().manual_seed(R)

    def ints(hi):
        return torch.randint(0, hi, (R,), generator=g).tolist()
    paged_case(dev, [1] * R, [c if r % 7 else 0 for r, c in enumerate(ints(90))], 16, 4, 2, 64, BF16,
               True, seed=R)
    new = [n if n < 4 else 0 for n in ints(7)]
    new[R // 2], new[-1] = 70, 41
    paged_case(dev, new, ints(50), 7, 6, 2, 64, FP16, True, seed=R + 1, pad=5)
    lens = [n if n < 9 else 0 for n in ints(12)]
    lens[3], lens[R - 2] = 150, 33
    varlen_case(dev, lens, lens, 4, 1, 128, BF16, True, seed=R + 2, pad=3)


def test_long_context_beside_many_short_ones(dev):
    for R in (66, 258):
        ctx = [3] * R
        ctx[R - 1], ctx[10] = 4000, 1500
        paged_case(dev, [1] * R, ctx, 16, 8, 1, 128, BF16, True, seed=70)
        paged_case(dev, [1] * (R - 1) + [90], ctx, 16, 8, 1, 128, BF16, True, seed=71)


def test_strides(dev):
    """Head-major q and out, K and V of different strides, one key head seen as many."""
    T, Hq, D = 150, 4, 128
    cu, lens = [0, 100, 150], [100, 50]
    q, k, v = (randn((T, Hq, D), BF16, 80 + i) for i in range(3))
    reqs = [(cu[r], cu[r + 1], k[cu[r]:cu[r + 1]], v[cu[r]:cu[r + 1]],
             seen_mask(lens[r], lens[r], True)) for r in range(2)]

    def major(x):  # the same values, heads outermost
        return x.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
    wide = torch.zeros(T, Hq, D + 24, dtype=BF16, device=dev)
    wide[:, :, 8:D + 8] = v.to(dev)
    out = major(torch.zeros(T, Hq, D, dtype=BF16))
    got = jo.attention_varlen(major(q), k.to(dev), wide[:, :, 8:D + 8], i32(cu, dev), out=out)
    assert got is out
    check(got, q, reqs, D ** -0.5, BF16)
    one = jo.attention_varlen(q.to(dev), k[:, :1].to(dev).expand(T, 2, D),
                              major(v[:, :1]).expand(T, 2, D), i32(cu, dev))
    reqs = [(a, b, k[a:b, :1], v[a:b, :1], s) for a, b, _, _, s in reqs]
    check(one, q, reqs, D ** -0.5, BF16)


def test_paged_out_keeps_other_rows(dev):
    q, pk, pv, table, cu, kv = step_inputs(dev, 4)
    want = jo.attention_paged(q, pk, pv, table, cu, kv)
    more = torch.cat((q, q[:20]))
    out = torch.full_like(more, 5.0)
    assert jo.attention_paged(more, pk, pv, table, cu, kv, out=out) is out
    assert torch.equal(out[:q.shape[0]], want) and bool((out[q.shape[0]:] == 5).all())


@pytest.mark.parametrize("seed", range(24))
def test_sizes_at_random(dev, seed):
    g = torch.Generator().manual_seed(1000 + seed)

    def pick(*of):
        return of[int(torch.randint(0, len(of), (1,), generator=g))]

    def ints(n, hi):
        return torch.randint(0, hi + 1, (n,), generator=g).tolist()
    R, Hkv, G = pick(1, 2, 3, 5, 17), pick(1, 2, 3), pick(1, 2, 3, 5, 8)
    D, dtype, causal = pick(64, 128, 256), pick(BF16, FP16), pick(True, True, False)
    top = pick(1, 3, 20, 150)
    new, ctx = ints(R, top), ints(R, pick(0, 5, 90, 1500))
    paged_case(dev, new, ctx, pick(1, 5, 16, 24, 52, 64, 100, 128), Hkv * G, Hkv, D, dtype, causal,
               seed=2000 + seed, pad=pick(0, 3), head_major=pick(True, False))
    varlen_case(dev, new, pick(new, ints(R, 300)), Hkv * G, Hkv, D, dtype, causal, seed=3000 + seed,
                pad=pick(0, 3))


# ---------------------------------------------------------------------------
# The C entry points, and what is refused.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("short", (None, 16, -16))
def test_workspace_of_the_c_entry_point(dev, abi, short):
    """None, or less than the plan's: the keys are not split, and the result is as good."""
    q, pk, pv, table, cu, kv = step_inputs(dev, 5, new=(1, 1), ctx=(3000, 40))
    T, Hq, D = q.shape
    N, P, Hkv, _ = pk.shape
    need = abi.lib().jo_attention_workspace_bytes(T, 2, Hq, Hkv, D, table.shape[1] * P, 1)
    assert need > 16
    size = 0 if short is None else short % need if short > 0 else need + short
    ws = torch.empty(max(size, 16) + 64, dtype=torch.uint8, device=dev).fill_(7)
    out = torch.empty_like(q)
    st = abi.lib().jo_attention_paged(
        q.data_ptr(), pk.data_ptr(), pv.data_ptr(), out.data_ptr(), T, 2, Hq, Hkv, D, N, P,
        Hq * D, D, P * Hkv * D, Hkv * D, D, P * Hkv * D, Hkv * D, D, Hq * D, D, table.data_ptr(),
        table.shape[1], table.shape[1], cu.data_ptr(), kv.data_ptr(), D ** -0.5, 1, 1, 2,
        ws.data_ptr() if short is not None else None, size,
        torch.cuda.current_stream(dev).cuda_stream)
    assert st == abi.JO_OK, abi.last_error()
    reqs = []
    for r in range(2):
        m = int(kv[r])
        k, v = (x.cpu()[table[r].cpu().clamp(min=0).long()].flatten(0, 1)[:m] for x in (pk, pv))
        reqs.append((r, r + 1, k, v, seen_mask(1, m, True)))
    check(out, q.cpu(), reqs, D ** -0.5, BF16)
    assert bool((ws == 7).all())


def test_refused_tensors(dev):
    q, pk, pv, table, cu, kv = step_inputs(dev, 6)
    k = torch.zeros(q.shape[0], 2, 128, dtype=BF16, device=dev)
    vl, pg = jo.attention_varlen, jo.attention_paged

    def no(msg, call, *a, **kw):
        with pytest.raises((RuntimeError, ValueError, TypeError), match=msg):
            call(*a, **kw)
    no("bf16 or fp16", vl, q.float(), k.float(), k.float(), cu)
    no("q's dtype", vl, q, k.half(), k, cu)
    no("q's dtype", vl, q, k, k, cu, out=torch.empty_like(q).half())
    no("must be on", vl, q, k.cpu(), k, cu)
    no("cu_q", vl, q, k, k, cu.cpu())
    no("cu_q", vl, q, k, k, cu.long())
    no("cu_k", vl, q, k, k, cu, cu[:-1])
    no("kv_lens", pg, q, pk, pv, table, cu, kv[:-1])
    no("kv_lens", pg, q, pk, pv, table, cu, kv.long())
    no("block_table", pg, q, pk, pv, table.long(), cu, kv)
    no("block_table", pg, q, pk, pv, table.t(), cu, kv)
    no("q's tokens", vl, q, k[:5], k[:5], cu)
    no("key tensor's shape", vl, q, k, k[:, :1], cu)
    no("key tensor's shape", pg, q, pk, pv[:3], table, cu, kv)
    no("multiple of the key heads", vl, q[:, :7], k, k, cu)
    no("head_dim", vl, q[:, :, :96], k[:, :, :96], k[:, :, :96], cu)
    no("tokens, heads, head_dim", vl, q[0], k, k, cu)
    no("pages, page_size", pg, q, k, k, table, cu, kv)
    no("contiguous head_dim", vl, q[:, :, ::2], k[:, :, :64], k[:, :, :64], cu)
    no("multiples of 8", vl, torch.zeros(q.shape[0], 8, 132, dtype=BF16, device=dev)[:, :, :128], k, k, cu)
    flat = torch.zeros(q.numel() + 8, dtype=BF16, device=dev)
    no("16-byte aligned", vl, flat[4:-4].view(q.shape), k, k, cu)
    no("out must have q's shape", vl, q, k, k, cu, out=torch.empty_like(q)[:-1])
    no("overlap an input", vl, q, k, k, cu, out=q)
    no("overlap an input", vl, q, k, k, cu, out=q.view(-1)[:].view(q.shape))
    no("must not overlap", vl, q, k, k, cu, out=torch.empty_like(q[:1]).expand_as(q))
    rows = torch.empty(q.shape[0] * 256 + 1024, dtype=BF16, device=dev)
    no("must not overlap", vl, q, k, k, cu, out=rows.as_strided(q.shape, (256, 128, 1)))
    no("scale", vl, q, k, k, cu, scale=0.0)
    no("scale", vl, q, k, k, cu, scale=math.nan)


def test_refused_tables_and_commits(dev):
    ctx, new, n = i32([3, 9], dev), i32([1, 1], dev), i32([4], dev)
    table, free = torch.full((2, 4), -1, dtype=torch.int32, device=dev), i32(list(range(9)), dev)

    def no(msg, call, *a, **kw):
        with pytest.raises((RuntimeError, ValueError, TypeError), match=msg):
            call(*a, **kw)
    no("same length", jo.paged_tables, ctx, new[:1], table, free, n, 4, 9, 8)
    no("new_lens", jo.paged_tables, ctx, new.long(), table, free, n, 4, 9, 8)
    no("num_free", jo.paged_tables, ctx, new, table, free, ctx, 4, 9, 8)
    no("block_table", jo.paged_tables, ctx, new, table[:1], free, n, 4, 9, 8)
    no("block_table", jo.paged_tables, ctx, new, table.t(), free, n, 4, 9, 8)
    no("free_pages", jo.paged_tables, ctx, new, table, free.cpu(), n, 4, 9, 8)
    no("max_tokens", jo.paged_tables, ctx, new, table, free, n, 4, 9, -1)
    no("page_size", jo.paged_tables, ctx, new, table, free, n, 0, 9, 8)
    no("table stride", jo.paged_tables, ctx, new, table[:1].expand(2, 4), free, n, 4, 9, 8)
    src, pages = (torch.zeros(s, dtype=BF16, device=dev) for s in ((2, 2, 64), (3, 4, 2, 64)))
    slots, cos = torch.zeros(2, dtype=torch.int64, device=dev), torch.ones(2, 64, device=dev)
    c = jo.kv_commit_rope_paged
    no("slots", c, src, pages, slots.int())
    no("slots", c, src, pages, slots[:1])
    no("dtype", c, src, pages.half(), slots)
    no("bf16 or fp16", c, src.float(), pages.float(), slots)
    no("src_k's heads", c, src, pages[:, :, :1], slots)
    no("go together", c, src, pages, slots, cos)
    no("go together", c, src, pages, slots, src_v=src)
    no("cos and sin", c, src, pages, slots, cos, cos[:1])
    no("contiguous heads", c, src, pages.transpose(1, 2).contiguous().transpose(1, 2), slots)


def test_two_streams_at_once(dev):
    """Calls of two streams side by side: each has a workspace of its own."""
    a, b = step_inputs(dev, 7), step_inputs(dev, 8, new=(1, 1, 1), ctx=(6000, 100, 9))
    want = [jo.attention_paged(*x) for x in (a, b)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(dev))
    for _ in range(8):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(jo.attention_paged(*x))
    torch.cuda.synchronize(dev)
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_ops_keep_to_their_schemas(dev):
    """What the schemas and the shape functions say of results, changed inputs and aliases."""
    q, pk, pv, table, cu, kv = step_inputs(dev, 9)
    tests = ("test_schema", "test_faketensor")
    ops = torch.ops.joyomni_ops
    k = torch.zeros(q.shape[0], 2, 128, dtype=BF16, device=dev)
    torch.library.opcheck(ops.attention_varlen.default, (q, k, k, cu, None, None, True), test_utils=tests)
    torch.library.opcheck(ops.attention_paged.default, (q, pk, pv, table, cu, kv, None, True),
                          test_utils=tests)
    torch.library.opcheck(ops.attention_paged_out.default,
                          (q, pk, pv, table, cu, kv, None, True, torch.empty_like(q)), test_utils=tests)
    torch.library.opcheck(ops.paged_tables.default,
                          (kv, torch.ones_like(kv), table, torch.arange(9, device=dev, dtype=torch.int32),
                           i32([9], dev), 16, pk.shape[0], 8), test_utils=tests)
    torch.library.opcheck(ops.kv_commit_rope_paged.default,
                          (k, k, pk, pv, torch.arange(k.shape[0], device=dev), None, None),
                          test_utils=tests)


@pytest.mark.parametrize("lq,lk", (([3100], [5000]), ([1100, 1090, 1100], [4200, 4200, 4100]),
                                   ([2500, 400, 400], [4300, 90, 4200]), ([2100, 0, 1], [4200, 0, 4200])),
                         ids=("one", "alike", "not-alike", "nearly-one"))
@pytest.mark.parametrize("D", (64, 128))
def test_last_round_split(dev, D, lq, lk):
    """Tokens that see every key, more tiles than the GPU runs at once and not a multiple: the last
    round's tiles have their keys split. A few heads against the definition."""
    H, heads = 32, [0, 17, 31]
    q = randn((sum(lq), H, D), BF16, 90, 1.3)
    k, v = (randn((sum(lk), H, D), BF16, 91 + i, 1.3 - 0.3 * i) for i in range(2))
    cq, ck = cu_of(lq), cu_of(lk)
    got = jo.attention_varlen(q.to(dev), k.to(dev), v.to(dev), i32(cq, dev), i32(ck, dev), causal=False)
    reqs = [(cq[r], cq[r + 1], k[ck[r]:ck[r + 1], heads], v[ck[r]:ck[r + 1], heads],
             seen_mask(lq[r], lk[r], False)) for r in range(len(lq))]
    check(got[:, heads], q[:, heads], reqs, D ** -0.5, BF16)
    again = jo.attention_varlen(q.to(dev), k.to(dev), v.to(dev), i32(cq, dev), i32(ck, dev), causal=False)
    assert torch.equal(got, again)


def test_compiled_without_a_graph_break(dev):
    """A step's four calls, traced: the block table and the pages are changed in place."""
    g = torch.Generator().manual_seed(5)
    P, N, D, T = 16, 20, 64, 8

    def step(q, k, v, pk, pv, ctx, new, table, free, n):
        cu, kv, slots, left = jo.paged_tables(ctx, new, table, free, n, P, N, T)
        jo.kv_commit_rope_paged(k, pk, slots, src_v=v, pages_v=pv)
        o = jo.attention_paged(q, pk, pv, table, cu, kv)
        into = torch.zeros_like(o)
        jo.attention_varlen(q, k, v, cu, out=into)
        return o, into, left, jo.attention_varlen(q, k, v, cu, causal=False)

    def inputs():
        g.manual_seed(5)
        rnd = lambda *s: torch.randn(*s, generator=g).to(BF16).to(dev)  # noqa: E731
        table = torch.full((2, 6), -1, dtype=torch.int32, device=dev)
        table[0, :3] = i32([4, 9, 2], dev)
        return [rnd(T, 4, D), rnd(T, 2, D), rnd(T, 2, D), rnd(N, P, 2, D), rnd(N, P, 2, D),
                i32([40, 0], dev), i32([1, 5], dev), table, i32(list(range(10, 19)), dev), i32([9], dev)]
    a, b = inputs(), inputs()
    want = step(*a)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(*b)
    for x, y in zip(list(got) + b, list(want) + a):
        assert torch.equal(x, y)


@pytest.mark.filterwarnings("ignore::UserWarning")
def test_forward_only(dev):
    """No gradient reaches the inputs: the result warns when it is differentiated."""
    q = randn((5, 2, 64), BF16, 1).to(dev).requires_grad_()
    k = randn((5, 2, 64), BF16, 2).to(dev)
    out = jo.attention_varlen(q, k, k, i32([0, 5], dev))
    assert torch.equal(out.detach(), jo.attention_varlen(q.detach(), k, k, i32([0, 5], dev)))
    with pytest.warns(UserWarning, match="autograd kernel was not registered"):
        out.sum().backward()
    assert q.grad is None


@pytest.mark.parametrize("causal", (True, False))
@pytest.mark.parametrize("R,top,cached", ((2, 700, 0), (9, 300, 900), (40, 1, 1500), (64, 1, 300),
                                          (64, 40, 500), (30, 200, 20)))
@pytest.mark.parametrize("D", (64, 256))
def test_longest_items_first(dev, D, R, top, cached, causal):
    """More items than the GPU runs at once, of up to 64 requests of all lengths, nothing among
    them: every row is written, by the item it belongs to."""
    H, heads = 64, [0, 40]
    g = torch.Generator().manual_seed(R + top)
    new = torch.randint(0 if R > 2 else 1, top + 1, (R,), generator=g).tolist()
    ctx = (torch.rand(R, generator=g) ** 3 * cached).int().tolist()
    if cached:
        ctx[R // 2] = cached
    if top == 1:
        new = [1] * R
    new[0] = top
    P, keys = 16, [n + c for n, c in zip(new, ctx)]
    need = [-(-m // P) for m in keys]
    table, at = torch.full((R, max(need)), -1, dtype=torch.int32), 0
    for r, n in enumerate(need):
        table[r, :n] = torch.arange(at, at + n)
        at += n
    q = randn((sum(new), H, D), BF16, R, 1.3)
    pk, pv = randn((at, P, H, D), BF16, R + 1, 1.3), randn((at, P, H, D), BF16, R + 2)
    cu = cu_of(new)
    out = torch.full(q.shape, math.nan, dtype=BF16, device=dev)
    jo.attention_paged(q.to(dev), pk.to(dev), pv.to(dev), table.to(dev), i32(cu, dev), i32(keys, dev),
                       causal=causal, out=out)
    reqs = []
    for r in range(R):
        k, v = (x[table[r, :need[r]].long()].flatten(0, 1)[:keys[r], heads] for x in (pk, pv))
        reqs.append((cu[r], cu[r + 1], k, v, seen_mask(new[r], keys[r], causal)))
    assert bool(torch.isfinite(out).all())
    check(out[:, heads], q[:, heads], reqs, D ** -0.5, BF16)
    if cached == 0:
        cut = randn((sum(new), H, D), BF16, 5), randn((sum(new), H, D), BF16, 6)
        out.fill_(math.nan)
        jo.attention_varlen(q.to(dev), cut[0].to(dev), cut[1].to(dev), i32(cu, dev), causal=causal, out=out)
        reqs = [(cu[r], cu[r + 1], cut[0][cu[r]:cu[r + 1], heads], cut[1][cu[r]:cu[r + 1], heads],
                 seen_mask(new[r], new[r], causal)) for r in range(R)]
        assert bool(torch.isfinite(out).all())
        check(out[:, heads], q[:, heads], reqs, D ** -0.5, BF16)


def test_sequences_that_overlap_stay_inside(dev):
    """cu_q that is not sorted gives more rows than tokens: no result is promised for them, but
    nothing outside the call's tensors changes."""
    T, H, D, P = 200, 16, 128, 16
    q = randn((T, H, D), BF16, 1).to(dev)
    pk = randn((64, P, H, D), BF16, 2).to(dev)
    table = torch.arange(64, dtype=torch.int32, device=dev).view(8, 8)
    big = torch.full((T + 64, H, D), 5.0, dtype=BF16, device=dev)
    for cu in ([0, 200, 0, 200, 0, 200, 0, 200, 0], [0, -5, 300, 10, 2 ** 31 - 1, 7, 200, 3, 200],
               [200, 0, 0, 0, 0, 0, 0, 0, 200]):
        for causal in (True, False):
            jo.attention_paged(q, pk, pk, table, i32(cu, dev), i32([128] * 8, dev), causal=causal,
                               out=big[32:T + 32])
            jo.attention_varlen(q, q, q, i32(cu, dev), causal=causal, out=big[32:T + 32])
            torch.cuda.synchronize(dev)
            assert bool((big[:32] == 5).all()) and bool((big[T + 32:] == 5).all())
