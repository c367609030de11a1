"""CPU tests of the paged serving entry points: refused arguments come back as status codes
without touching a GPU, the ops are registered for device tensors only, and the plain forms in
oracle.serving say what they should."""
from __future__ import annotations

import pytest
import torch

import joyomni_ops as jo
from oracle import serving

P = 0x1000  # an aligned address that is never read


def varlen(**kw):
    a = dict(q=P, k=P, v=P, out=P, T=4, Tk=4, R=1, Hq=4, Hkv=2, D=128, qt=512, qh=128, kt=256, kh=128,
             vt=256, vh=128, ot=512, oh=128, cu_q=P, cu_k=P, scale=0.1, causal=1, fill=1, dtype=2,
             ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return "jo_attention_varlen", list(a.values())


def paged(**kw):
    a = dict(q=P, k=P, v=P, out=P, T=4, R=1, Hq=4, Hkv=2, D=128, N=8, P=16, qt=512, qh=128, kp=4096,
             kt=256, kh=128, vp=4096, vt=256, vh=128, ot=512, oh=128, table=P, ts=4, W=4, cu_q=P,
             kv_lens=P, scale=0.1, causal=1, fill=1, dtype=2, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return "jo_attention_paged", list(a.values())


def tables(**kw):
    a = dict(ctx=P, new=P, R=2, table=P, ts=4, W=4, free=P, cap=4, num=P, P=16, N=8, most=8, cu=P,
             kv=P, slots=P, left=P + 64, stream=None)
    a.update(kw)
    return "jo_paged_tables", list(a.values())


def commit(**kw):
    a = dict(sk=P, sv=P, pk=P, pv=P, L=1, T=4, H=2, D=128, sl=0, st=256, pl=0, pp=4096, pt=256, N=8,
             P=16, slots=P, cos=P, sin=P, tab=128, dtype=2, stream=None)
    a.update(kw)
    return "jo_kv_commit_rope_paged", list(a.values())


BIG = 2 ** 31
REFUSED = [
    (varlen(dtype=0), "bf16 or fp16"), (varlen(dtype=9), "bf16 or fp16"),
    (varlen(D=96), "unsupported head_dim"), (varlen(Hq=5), "no multiple"),
    (varlen(Hkv=0), "bad shape"), (varlen(T=-1), "bad shape"), (varlen(Tk=-1), "bad shape"),
    (varlen(Tk=BIG), "bad shape"), (varlen(T=BIG), "too large"), (varlen(Hq=1 << 20, Hkv=2), "too large"),
    (varlen(R=BIG), "too large"), (varlen(scale=0.0), "scale"), (varlen(scale=-1.0), "scale"),
    (varlen(scale=float("nan")), "scale"), (varlen(scale=float("inf")), "scale"),
    (varlen(q=None), "null"), (varlen(k=None), "null"), (varlen(out=None), "null"),
    (varlen(cu_q=None), "null"), (varlen(cu_k=None), "null"), (varlen(q=P + 8), "aligned"),
    (varlen(out=P + 2), "aligned"), (varlen(qt=516), "multiples of 8"), (varlen(vh=4), "multiples of 8"),
    (varlen(kt=-256), "multiples of 8"), (varlen(ot=64), "overlap"), (varlen(oh=0), "overlap"),
    (paged(P=0), "bad shape"), (paged(P=BIG), "bad shape"), (paged(N=-1), "bad shape"),
    (paged(N=BIG), "bad shape"), (paged(W=-1), "bad shape"), (paged(R=2, ts=3), "table stride"),
    (paged(kv_lens=None), "null"), (paged(table=None), "null"), (paged(v=None), "null"),
    (paged(kp=4100), "multiples of 8"), (paged(Hq=3), "no multiple"), (paged(D=32), "head_dim"),
    (tables(R=4097), "too many requests"), (tables(R=-1), "bad shape"), (tables(P=0), "page_size"),
    (tables(P=BIG), "page_size"), (tables(W=BIG), "too large"), (tables(N=BIG), "too large"),
    (tables(most=BIG), "too large"), (tables(cap=BIG), "too large"), (tables(most=-1), "bad shape"),
    (tables(ts=3), "table stride"), (tables(cu=None), "null"), (tables(ctx=None), "null"),
    (tables(kv=None), "null"), (tables(slots=None), "null"), (tables(free=None), "null"),
    (tables(num=None), "null"), (tables(table=None), "null"), (tables(left=P), "num_free itself"),
    (commit(dtype=0), "bf16 or fp16"), (commit(H=0), "bad shape"), (commit(L=-1), "bad shape"),
    (commit(P=0), "page_size"), (commit(N=2 ** 28), "page_size"), (commit(D=127), "even"),
    (commit(H=2 ** 30), "row too long"), (commit(cos=None), "go together"), (commit(st=255), "stride"),
    (commit(pt=8), "stride"), (commit(pp=-1), "stride"), (commit(tab=64), "stride"),
    (commit(sv=None), "source and a destination"), (commit(T=2 ** 30), "too many rows"),
    (commit(T=2 ** 62, L=4), "too many rows"), (commit(sk=None), "null"), (commit(slots=None), "null"),
]


REFUSED += [
    # Rows of out that share elements without being too close one by one.
    (varlen(ot=256, oh=128), "overlap"), (varlen(ot=128, oh=256), "overlap"),
    (paged(ot=392, oh=128), "overlap"), (varlen(ot=128, oh=504), "overlap"),
    # Rows of K and V that 32 bits do not reach.
    (varlen(kt=2 ** 24), "stride"), (paged(vp=2 ** 36, N=8), "64 GiB"),
    # Rows of the pool that share elements: pages, layers, places.
    (commit(pp=0), "overlap"), (commit(pp=3900), "overlap"), (commit(L=3, pl=4096), "overlap"),
    (commit(L=3, pl=0), "overlap"), (commit(pp=256, pt=256), "overlap"), (commit(pp=2 ** 62), "too large"),
    # Results in the place of what other workgroups still read.
    (tables(kv=P, cu=P + 2 ** 16, slots=P + 2 ** 17, table=P + 2 ** 18), "overlaps an input"),
    (tables(kv=P + 2 ** 15, cu=P + 2 ** 16, slots=P + 2 ** 17, table=P + 8), "overlaps an input"),
]


@pytest.mark.parametrize("call,msg", REFUSED, ids=lambda x: x if isinstance(x, str) else None)
def test_refused(abi, call, msg):
    name, args = call
    assert getattr(abi.lib(), name)(*args) == abi.JO_ERR_INVALID
    assert msg in abi.last_error(), abi.last_error()


@pytest.mark.parametrize("call", (varlen(T=0), paged(T=0), commit(T=0), commit(L=0), commit(N=0)),
                         ids=lambda c: c[0])
def test_nothing_to_do(abi, call):
    name, args = call
    assert getattr(abi.lib(), name)(*args) == abi.JO_OK


def test_ops_have_no_cpu_kernel():
    q = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        jo.attention_varlen(q, q, q, i)
    with pytest.raises((RuntimeError, NotImplementedError)):
        jo.attention_paged(q, q[None], q[None], i[None], i, i[:1])
    with pytest.raises((RuntimeError, NotImplementedError)):
        jo.paged_tables(i, i, i.view(2, 1), i, i[:1], 16, 4, 8)
    with pytest.raises((RuntimeError, NotImplementedError)):
        jo.kv_commit_rope_paged(q, q[None], torch.zeros(2, dtype=torch.int64))


def test_shapes_under_tracing():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty(7, 4, 128, dtype=torch.bfloat16, device="cuda")
        i = torch.empty(3, dtype=torch.int32, device="cuda")
        o = jo.attention_varlen(q, q, q, i)
        assert o.shape == q.shape and o.dtype == q.dtype
        pages = torch.empty(5, 16, 2, 128, dtype=torch.bfloat16, device="cuda")
        assert jo.attention_paged(q, pages, pages, i.view(3, 1), i, i).shape == q.shape
        cu, kv, slots, left = jo.paged_tables(i, i, i.view(3, 1), i, i[:1], 16, 5, 40)
        assert (cu.shape, kv.shape, slots.shape, left.shape) == ((4,), (3,), (40,), (1,))
        assert slots.dtype == torch.int64


def test_plain_tables():
    """A step by hand: pages of 4, two requests."""
    cu, kv, slots, left, table = serving.paged_tables([3, 0], [2, 5], [[7, -1, -1], [-1, -1, -1]],
                                                      [1, 2, 9, 4], 4, 4, 9, 10)
    assert cu == [0, 2, 7] and kv == [5, 5] and left == 1
    assert table == [[7, 4, -1], [-1, 2, -1]]  # 9 names no page
    assert slots == [31, 16, -1, -1, -1, -1, 8, -1, -1, -1]


def test_plain_attention():
    """One key gives its v; a mask that leaves nothing gives zeros; NaN that is not seen stays out."""
    q, k = torch.randn(2, 2, 64).bfloat16(), torch.randn(3, 1, 64).bfloat16()
    v = torch.randn(3, 1, 64).bfloat16()
    v[2] = float("nan")
    seen = torch.tensor([[False, False, False], [False, True, False]])
    out, size, _ = serving.attention(q, k, v, seen, 0.1)
    assert bool((out[0] == 0).all())
    assert torch.allclose(out[1], v[1].double().expand(2, 64), rtol=1e-12)
    assert torch.allclose(size[1], v[1].double().abs().expand(2, 64), rtol=1e-12)
    want = torch.softmax(q[:, 0].double() @ k[:, 0].double().t() * 0.1, -1)[:, :2]
    two, _, _ = serving.attention(q, k[:2], v[:2], torch.ones(2, 2, dtype=torch.bool), 0.1)
    ref = torch.softmax(q[:, 0].double() @ k[:2, 0].double().t() * 0.1, -1) @ v[:2, 0].double()
    assert want.shape == (2, 2) and torch.allclose(two[:, 0], ref, rtol=1e-12)
