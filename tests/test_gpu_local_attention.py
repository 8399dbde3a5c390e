"""Local attention and its gradients against their definition in 64 bits (tests/local_reference.py has the bounds)."""
import pytest
import torch

import fast_memory_b200 as fm
from tests.local_reference import Case, assert_within

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32

CASES = {
    "one token": dict(nq=(1,)),
    "one query, many keys": dict(nq=(1,), nk=(1000,), d=128),
    "tile edges": dict(nq=(127, 128, 129, 1), d=128, hq=4, h=2),
    "two tiles and a bit": dict(nq=(257,), nk=(385,), d=128, dtype=HF),
    "not causal": dict(nq=(140, 60), nk=(200, 300), causal=False),
    "not causal, window": dict(nq=(300,), nk=(333,), causal=False, window=50, d=128),
    "window": dict(nq=(500,), window=37),
    "window of one": dict(nq=(130,), window=1, d=128),
    "window, many tiles": dict(nq=(1100,), window=300, d=128, hq=3, h=3),
    "more queries than keys": dict(nq=(200, 90), nk=(70, 0)),            # the first queries see nothing
    "more queries than keys, not causal": dict(nq=(200, 3), nk=(70, 0), causal=False, window=90),
    "empty documents": dict(nq=(0, 50, 0, 3, 0), nk=(0, 60, 5, 3, 0)),
    "tail": dict(nq=(33, 90), tail=45, d=128),
    "prefix": dict(nq=(150, 200, 20), prefix=(40, 0, 999), window=16, d=128),
    "prefix beyond the window": dict(nq=(400,), nk=(700,), prefix=(130,), window=100, d=128, softcap=20.0),
    "capped": dict(nq=(260,), softcap=5.0, d=128, scale=0.3),
    "distance": dict(nq=(300,), slopes=True, hq=4, h=1, d=128),
    "distance, capped, not causal": dict(nq=(90, 150), slopes=True, softcap=15.0, causal=False, hq=6, h=2),
    "group of seven": dict(nq=(50, 141), hq=7, h=1, d=128),
    "group of three, two heads": dict(nq=(70, 1, 200), nk=(170, 30, 200), hq=6, h=2, dtype=HF),
    "token major": dict(nq=(200, 111), token_major=True, hq=4, h=2, d=128),
    "fp32": dict(nq=(70, 200), dtype=F, d=64, hq=2, h=1, slopes=True),
    "fp32, d 128": dict(nq=(131,), nk=(300,), dtype=F, d=128, window=100, softcap=10.0, prefix=(7,)),
    "fp32 token major": dict(nq=(65, 1), dtype=F, token_major=True, hq=4, h=2),
    "d 16": dict(nq=(100,), d=16),
    "d 32": dict(nq=(100, 30), d=32, dtype=HF),
    "d 256": dict(nq=(90,), nk=(140,), d=256),
    "many documents": dict(nq=tuple((i * 7) % 11 for i in range(70)), nk=tuple((i * 5) % 13 for i in range(70)), hq=2, h=2, d=128),
    "large logits": dict(nq=(300,), d=128, scale=1.0),
}


def _run(c, **kw):
    return fm.local_attention(c.q, c.k, c.v, c.scale, **(kw or c.kwargs()))


@pytest.mark.parametrize("name", CASES)
def test_forward(name):
    c = Case(**CASES[name])
    o, lse = _run(c)
    assert o.dtype == c.dtype and lse.dtype == torch.float32 and o.shape == c.q.shape and lse.shape == c.q.shape[:2]
    ro, rl, to, tl = c.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    blind = torch.isinf(rl)
    assert (o[blind] == 0).all()
    if len(c.nq) == 1 and c.q.shape[1] == c.nq[0]:
        o2, lse2 = _run(c, **c.kwargs(plain=True))
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("with_lse", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_backward(name, with_lse):
    c = Case(**CASES[name], seed=3)
    o, lse = _run(c)
    d_lse = c.d_lse if with_lse else None
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, d_lse=d_lse, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse, d_lse), ("dq", "dk", "dv")):
        assert got.dtype == c.dtype
        assert_within(got, want, bound, what)
    again = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, d_lse=d_lse, **c.kwargs())
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (F, 64)])
def test_random_calls(dtype, d):
    import random
    rng = random.Random(17)
    for n in range(12):
        h, g = rng.choice([(1, 1), (2, 2), (1, 5), (3, 1)])
        docs = rng.randint(1, 5)
        nq = [rng.choice([0, 1, 17, 63, 64, 130, 300]) for _ in range(docs)]
        c = Case(dtype=dtype, d=d, hq=h * g, h=h, nq=nq, nk=[x + rng.choice([0, 0, 5, 128, 333]) for x in nq], causal=rng.random() < 0.7,
                 window=rng.choice([0, 0, 3, 64, 129, 200]), softcap=rng.choice([0.0, 12.0]), slopes=rng.random() < 0.4,
                 prefix=[rng.randint(0, 150) for _ in range(docs)] if rng.random() < 0.4 else None, token_major=rng.random() < 0.3,
                 tail=rng.choice([0, 9]), seed=n)
        o, lse = _run(c)
        ro, rl, to, tl = c.forward()
        assert_within(lse, rl, tl, f"lse of call {n}")
        assert_within(o, ro, to, f"o of call {n}")
        grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
        for got, (want, bound), what in zip(grads, c.backward(o, lse), ("dq", "dk", "dv")):
            assert_within(got, want, bound, f"{what} of call {n}")


@pytest.mark.parametrize("softcap", [0.0, 9.0])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("dtype,nq", [(BF, (150,)), (HF, (3, 2)), (F, (70,))])
def test_scales_that_are_not_positive(dtype, nq, scale, softcap):
    """The largest score is then not the largest product, and a scale of 0 makes all keys equal."""
    c = Case(dtype=dtype, d=64, hq=4, h=2, nq=nq, nk=tuple(n + 200 for n in nq), window=180, softcap=softcap, scale=scale, seed=21)
    o, lse = _run(c)
    ro, rl, to, tl = c.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse), ("dq", "dk", "dv")):
        assert_within(got, want, bound, what)


@pytest.mark.parametrize("softcap,scale", [(0.01, 0.3), (2000.0, 0.05), (3.0, 1.5), (60.0, 3.0)])
def test_caps_of_every_size(softcap, scale):
    """Scores far below, about and far above the cap: each formula of tanh, forward and backward."""
    c = Case(dtype=BF, d=128, hq=2, h=1, nq=(200, 90), nk=(330, 90), softcap=softcap, scale=scale, seed=22)
    o, lse = _run(c)
    ro, rl, to, tl = c.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse), ("dq", "dk", "dv")):
        assert_within(got, want, bound, what)


@pytest.mark.parametrize("dtype,nq", [(HF, 2), (BF, 300), (F, 100)])
def test_a_wide_cap_costs_no_precision(dtype, nq):
    """cap tanh(s / cap) is off by 2^-21 |s| at most (the polynomial's 2e-7 and three roundings), not by a fraction of the cap: the
    bound on lse is the general one less what that grants the cap (2 2^-20 cap)."""
    cap = 20000.0
    c = Case(dtype=dtype, d=64, hq=2, h=1, nq=(nq,), nk=(nq + 50,), softcap=cap, seed=23)
    _, lse = _run(c)
    _, rl, _, tl = c.forward()
    assert_within(lse, rl, tl - 2 * 2.0 ** -20 * cap, "lse")


def _assert_rows(got, want, bound, rows, name):
    assert_within(got[:, rows], want[:, rows], bound[:, rows], name)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float16).min])
def test_hidden_values_take_no_part(dtype, d, bad):
    """Keys, values, queries and output gradients that a row does not see may hold anything."""
    c = Case(dtype=dtype, d=d, hq=2, h=1, nq=(100, 60, 200), window=70, tail=20, seed=8)
    clean = [t.clone() for t in (c.q, c.k, c.v, c.d_out)]
    o0, lse0 = _run(c)
    ro, rl, to, tl = c.forward()
    g0 = c.backward(o0, lse0)
    # document 1, the tail, and the last position of document 2 (which only its own query sees)
    for t in (c.q, c.k, c.v, c.d_out):
        t[:, 100:160] = bad
        t[:, 360:] = bad
    c.k[:, 359] = bad
    c.v[:, 359] = bad
    o, lse = _run(c)
    rows = torch.ones(380, dtype=torch.bool, device="cuda")
    rows[100:160] = rows[359:] = False
    _assert_rows(o, ro, to, rows, "o")
    _assert_rows(lse, rl, tl, rows, "lse")
    assert (o[:, 360:] == 0).all() and torch.isinf(lse[:, 360:]).all()
    if bad != bad:
        assert torch.isnan(o[:, 359]).all() and torch.isnan(o[:, 101:160]).all()
    o1, lse1 = o0.clone(), lse0.clone()                    # what the caller has: the clean rows, and what became of the others
    o1[:, 100:160], lse1[:, 100:160] = o[:, 100:160], lse[:, 100:160]
    c.k[:, 359], c.v[:, 359] = clean[1][:, 359], clean[2][:, 359]
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o1, lse1, c.d_out, **c.kwargs())
    rows[359] = True
    for got, (want, bound), name in zip(grads, g0, ("dq", "dk", "dv")):
        _assert_rows(got, want, bound, rows, name)
        assert (got[:, 360:] == 0).all()


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64)])
def test_one_bad_value_reaches_the_rows_that_see_it(dtype, d):
    c = Case(dtype=dtype, d=d, nq=(300,), seed=2)
    o0, lse0 = _run(c)
    ro, rl, to, tl = c.forward()
    g0 = c.backward(o0, lse0)
    c.v[0, 150, 7] = float("nan")
    o, lse = _run(c)
    at = torch.arange(300, device="cuda")
    assert_within(lse, rl, tl, "lse")
    _assert_rows(o, ro, to, at < 150, "o")
    assert torch.isnan(o[:, 150:, 7]).all()
    assert torch.isfinite(o[:, :, :7]).all() and torch.isfinite(o[:, :, 8:]).all()
    c = Case(dtype=dtype, d=d, nq=(300,), seed=2)
    c.d_out[1, 40, 3] = float("nan")                       # keys up to 40 get it, dv in column 3 only
    dq, dk, dv = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o0, lse0, c.d_out, **c.kwargs())
    assert torch.isnan(dv[:, :41, 3]).all() and torch.isfinite(dv[:, :41, 4:]).all()
    _assert_rows(dk, *g0[1], at > 40, "dk")
    _assert_rows(dv, *g0[2], at > 40, "dv")
    assert torch.isnan(dk[:, :41]).all() and torch.isnan(dq[1, 40]).all() and torch.isfinite(dq[0]).all()


def test_gradient_against_differences():
    """The directional derivative of a loss over o and lse, by central differences of the fp32 operator: h = 2^-7 leaves an
    error of h^2 / 6 of the third derivative and 2^-24 |loss| / h of rounding, together well under 1e-2 of the derivative."""
    c = Case(dtype=F, d=32, hq=4, h=2, nq=(40, 60), nk=(50, 75), window=30, softcap=8.0, slopes=True, prefix=(5, 0), seed=4)
    kw = c.kwargs()
    g = torch.Generator().manual_seed(9)
    dirs = [torch.randn(t.shape, generator=g).cuda() / t.numel() ** 0.5 for t in (c.q, c.k, c.v)]

    def loss(q, k, v):
        o, lse = fm.local_attention(q, k, v, c.scale, **kw)
        return (o.double() * c.d_out.double()).sum() + (lse.double() * c.d_lse.double()).sum()

    leaves = [t.clone().requires_grad_() for t in (c.q, c.k, c.v)]
    loss(*leaves).backward()
    for i, x in enumerate(dirs):
        h = 2.0 ** -7
        moved = [[t + s * h * (x if j == i else 0) for j, t in enumerate((c.q, c.k, c.v))] for s in (1, -1)]
        diff = float(loss(*moved[0]) - loss(*moved[1])) / (2 * h)
        want = float((leaves[i].grad.double() * x.double()).sum())
        assert abs(diff - want) <= 1e-2 * abs(want) + 2.0 ** -24 * 1000 / h * 4, (i, diff, want)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F, 64)])
def test_autograd_is_the_explicit_backward(dtype, d):
    c = Case(dtype=dtype, d=d, hq=4, h=2, nq=(90, 80), seed=6)
    leaves = [t.detach().clone().requires_grad_() for t in (c.q, c.k, c.v)]
    o, lse = fm.local_attention(*leaves, c.scale, **c.kwargs())
    ((o * c.d_out).sum() + (lse * c.d_lse).sum()).backward()
    o2, lse2 = _run(c)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    want = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o2, lse2, c.d_out, d_lse=c.d_lse, **c.kwargs())
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    # a loss that reads one result only; an expanded output gradient
    leaves = [t.detach().clone().requires_grad_() for t in (c.q, c.k, c.v)]
    o, lse = fm.local_attention(*leaves, c.scale, **c.kwargs())
    o.sum().backward()
    want = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o2, lse2, torch.ones_like(o2), **c.kwargs())
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    leaves = [t.detach().clone().requires_grad_() for t in (c.q, c.k, c.v)]
    _, lse = fm.local_attention(*leaves, c.scale, **c.kwargs())
    lse.sum().backward()
    assert torch.equal(leaves[2].grad, torch.zeros_like(leaves[2]))


def test_registered_operators():
    c = Case(d=64, nq=(40, 30), hq=2, h=1)
    kw = c.kwargs()
    cu = kw["cu_seqlens_q"]
    args = (c.q.clone().requires_grad_(), c.k, c.v, c.scale, True, 0, 0.0, None, cu, cu, None)
    torch.library.opcheck(torch.ops.fast_memory_b200.local_attention.default, args,
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    o, lse = _run(c)
    torch.library.opcheck(torch.ops.fast_memory_b200.local_attention_backward.default,
                          (c.q, c.k, c.v, o, lse, c.d_out, None, c.scale, True, 0, 0.0, None, cu, cu, None),
                          test_utils=("test_schema", "test_faketensor"))
    compiled = torch.compile(lambda q, k, v: fm.local_attention(q, k, v, c.scale, **kw), backend="aot_eager")(c.q, c.k, c.v)
    assert torch.equal(compiled[0], o) and torch.equal(compiled[1], lse)


@pytest.mark.parametrize("dtype", [BF, F])
def test_strides_alignment_and_views(dtype):
    """Any layout gives what its contiguous copy gives."""
    c = Case(dtype=dtype, d=64, hq=4, h=2, nq=(150,), seed=5)
    o0, lse0 = _run(c)
    g0 = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o0, lse0, c.d_out, **c.kwargs())

    def offset(t):                                         # rows that start off the 16-byte grid
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return buf.copy_(t)

    def columns(t):                                        # the last dim is not contiguous
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def sliced(t):                                         # part of a wider projection, [tokens, heads, 2 d]
        wide = torch.full((t.shape[1], t.shape[0], 2 * t.shape[2]), float("nan"), dtype=t.dtype, device="cuda")
        wide[..., :t.shape[2]] = t.transpose(0, 1)
        return wide[..., :t.shape[2]].transpose(0, 1)

    for f in (offset, columns, sliced):
        q, k, v, g = (f(t) for t in (c.q, c.k, c.v, c.d_out))
        o, lse = fm.local_attention(q, k, v, c.scale, **c.kwargs())
        assert torch.equal(o, o0) and torch.equal(lse, lse0)
        for got, want in zip(fm.local_attention_backward(q, k, v, c.scale, o, lse, g, **c.kwargs()), g0):
            assert torch.equal(got, want)
    one = c.v[:1, :, :].expand(2, -1, -1)                  # shared by broadcasting
    o, _ = fm.local_attention(c.q, c.k, one, c.scale, **c.kwargs())
    o1, _ = fm.local_attention(c.q, c.k, one.contiguous(), c.scale, **c.kwargs())
    assert torch.equal(o, o1)


@pytest.mark.parametrize("dtype", [BF, F])
def test_backward_takes_any_layout_of_out(dtype):
    """``out`` and ``lse`` of a merge may be views: not on a 16-byte boundary, or token major."""
    c = Case(dtype=dtype, d=64, hq=4, h=2, nq=(90, 40), window=50, seed=24)
    o, lse = _run(c)
    want = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    odd = torch.empty(o.numel() + 1, dtype=dtype, device="cuda")[1:].view(o.shape).copy_(o)
    odd_lse = torch.empty(lse.numel() + 1, device="cuda")[1:].view(lse.shape).copy_(lse)
    for a, b in ((odd, odd_lse), (o.transpose(0, 1).contiguous().transpose(0, 1), lse.t().contiguous().t())):
        got = fm.local_attention_backward(c.q, c.k, c.v, c.scale, a, b, c.d_out, **c.kwargs())
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gradient_of_a_broadcast_input():
    c = Case(d=64, hq=2, h=2, nq=(100,), seed=5)
    v = c.v[:1].clone().requires_grad_()
    o, lse = fm.local_attention(c.q, c.k, v.expand(2, -1, -1), c.scale)
    (o * c.d_out).sum().backward()
    _, _, dv = fm.local_attention_backward(c.q, c.k, v.detach().expand(2, -1, -1), c.scale, o.detach(), lse.detach(), c.d_out)
    assert torch.equal(v.grad, dv.sum(0, keepdim=True))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F, 64)])
def test_captured_and_replayed(dtype, d):
    """Two graphs, replayed on two streams at once with new inputs and new documents, and an eager call beside them."""
    cases = [Case(dtype=dtype, d=d, hq=4, h=2, nq=(300, 100), window=90, seed=i) for i in range(2)]
    graphs, outs, kws = [], [], []
    for c in cases:
        kw = c.kwargs()
        o, lse = fm.local_attention(c.q, c.k, c.v, c.scale, **kw)                    # first call outside the capture
        fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **kw)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, lse = fm.local_attention(c.q, c.k, c.v, c.scale, **kw)
            grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **kw)
        graphs.append(g)
        outs.append((o, lse, *grads))
        kws.append(kw)
    fresh = [Case(dtype=dtype, d=d, hq=4, h=2, nq=(170, 230), window=90, seed=10 + i) for i in range(2)]
    for c, f, kw in zip(cases, fresh, kws):
        for name in ("q", "k", "v", "d_out"):
            getattr(c, name).copy_(getattr(f, name))
        kw["cu_seqlens_q"].copy_(f.kwargs()["cu_seqlens_q"])
        kw["cu_seqlens_k"].copy_(f.kwargs()["cu_seqlens_k"])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = fm.local_attention(fresh[0].q, fresh[0].k, fresh[0].v, fresh[0].scale, **fresh[0].kwargs())
    torch.cuda.synchronize()
    for f, got in zip(fresh, outs):
        o, lse = _run(f)
        want = (o, lse, *fm.local_attention_backward(f.q, f.k, f.v, f.scale, o, lse, f.d_out, **f.kwargs()))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(eager[0], outs[0][0])


def test_merged_with_a_memory():
    """Local attention over new keys and a memory of old ones, merged, is attention over both; the gradients of the merged
    result come from the two backward passes with the merged (out, lse)."""
    H, G, N, S, d, C = 2, 2, 512, 160, 64, 4
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()
    k_old, v_old, k, v, q, d_out = rnd(H, N, d), rnd(H, N, d), rnd(H, S, d), rnd(H, S, d), rnd(H * G, S, d), rnd(H * G, S, d)
    sm = d ** -0.5
    mem = fm.Memory.build(k_old, v_old, A=rnd(H, C, d), bucket_size=N)                 # every bucket holds every key
    o_l, lse_l = fm.local_attention(q, k, v, sm, window=50)
    o_m, lse_m = mem.query(q, sm)
    out, lse = fm.merge(o_l, lse_l, o_m, lse_m)
    dq_l, dk, dv = fm.local_attention_backward(q, k, v, sm, out.bfloat16(), lse, d_out, window=50)
    dq_m, dk_old, dv_old = mem.query_backward(q, sm, out.bfloat16(), lse, d_out)
    # dense in 64 bits
    x = [t.double().requires_grad_() for t in (q, k, v, k_old, v_old)]
    keys, vals = torch.cat([x[3], x[1]], 1).repeat_interleave(G, 0), torch.cat([x[4], x[2]], 1).repeat_interleave(G, 0)
    i, j = torch.arange(S, device="cuda")[:, None], torch.arange(S, device="cuda")[None, :]
    mask = torch.cat([torch.ones(S, N, dtype=torch.bool, device="cuda"), (j <= i) & (j > i - 50)], 1)
    s = (x[0] @ keys.transpose(1, 2) * sm).masked_fill(~mask, float("-inf"))
    ref = torch.softmax(s, -1) @ vals
    (ref * d_out.double()).sum().backward()
    # bf16 results of size <= 1 over weights that sum to one: two roundings of each part, 2^-8 each, of |o| <= max|v|
    u = 2.0 ** -8
    ref = ref.detach()
    assert (out.double() - ref).abs().max() <= 3 * u * float(vals.detach().abs().max()) / 4
    assert (lse.double() - torch.logsumexp(s, -1)).abs().max() <= 1e-3
    for got, want in ((dq_l.double() + dq_m.double(), x[0].grad), (dk.double(), x[1].grad), (dv.double(), x[2].grad),
                      (dk_old.double(), x[3].grad), (dv_old.double(), x[4].grad)):
        # every term is rounded to 2^-8 of itself; the terms of a row sum to at most this multiple of the largest gradient
        assert (got - want).abs().max() <= 8 * u * float(want.abs().max())


def test_refusals():
    c = Case(d=64, nq=(40,), hq=2, h=1)
    q, k, v, s = c.q, c.k, c.v, c.scale
    o, lse = fm.local_attention(q, k, v, s)
    cases = [
        (ValueError, lambda: fm.local_attention(q[0], k, v, s)),
        (ValueError, lambda: fm.local_attention(q, k, v[:, :-1], s)),
        (TypeError, lambda: fm.local_attention(q, k.half(), v.half(), s)),
        (TypeError, lambda: fm.local_attention(q.double(), k.double(), v.double(), s)),
        (ValueError, lambda: fm.local_attention(torch.cat([q, q[:1]]), torch.cat([k, k]), torch.cat([v, v]), s)),
        (fm.FastMemError, lambda: fm.local_attention(q[..., :48].contiguous(), k[..., :48].contiguous(), v[..., :48].contiguous(), s)),
        (ValueError, lambda: fm.local_attention(q, k, v, s, window=-1)),
        (ValueError, lambda: fm.local_attention(q, k, v, s, window=2.5)),
        (ValueError, lambda: fm.local_attention(q, k, v, s, softcap=-1.0)),
        (ValueError, lambda: fm.local_attention(q, k, v, s, softcap=float("nan"))),
        (TypeError, lambda: fm.local_attention(q, k, v, s, slopes=torch.ones(1, device="cuda"))),
        (ValueError, lambda: fm.local_attention(q, k, v, s, slopes=torch.ones(2, device="cuda", requires_grad=True))),
        (ValueError, lambda: fm.local_attention(q, k, v, s, slopes=torch.ones(2))),
        (ValueError, lambda: fm.local_attention(q, k, v, s, cu_seqlens_k=[0, 40])),
        (ValueError, lambda: fm.local_attention(q, k, v, s, cu_seqlens_q=[0, 41])),
        (ValueError, lambda: fm.local_attention(q, k, v, s, cu_seqlens_q=[0, 20, 10])),
        (ValueError, lambda: fm.local_attention(q, k, v, s, cu_seqlens_q=[0, 20, 40], cu_seqlens_k=[0, 40])),
        (ValueError, lambda: fm.local_attention(q, k[:, :30], v[:, :30], s, cu_seqlens_q=[0, 40])),
        (TypeError, lambda: fm.local_attention(q, k, v, s, cu_seqlens_q=torch.tensor([0.0, 40.0], device="cuda"))),
        (ValueError, lambda: fm.local_attention(q, k, v, s, cu_seqlens_q=torch.tensor([0, 40]))),
        (ValueError, lambda: fm.local_attention(q, k, v, s, prefix=[1, 2])),
        (fm.FastMemError, lambda: fm.local_attention(q.cpu(), k, v, s)),
        (TypeError, lambda: fm.local_attention_backward(q, k, v, s, o.float(), lse, c.d_out)),
        (TypeError, lambda: fm.local_attention_backward(q, k, v, s, o, lse.bfloat16(), c.d_out)),
        (ValueError, lambda: fm.local_attention_backward(q, k, v, s, o, lse[:1], c.d_out)),
        (ValueError, lambda: fm.local_attention_backward(q, k, v, s, o, lse, c.d_out[:, :20])),
    ]
    for n, (error, call) in enumerate(cases):
        with pytest.raises(error):
            call()
            print("call", n, "was not refused")
    assert fm.local_attention(q[:, :0], k, v, s)[0].shape == (2, 0, 64)
    o, lse = fm.local_attention(q, k[:, :0], v[:, :0], s)
    assert (o == 0).all() and torch.isinf(lse).all()
    dq, dk, dv = fm.local_attention_backward(q, k[:, :0], v[:, :0], s, o, lse, c.d_out)
    assert (dq == 0).all() and dk.shape == (1, 0, 64)


def test_wrong_prefix_sums_stay_inside_the_arrays():
    """Numbers on the device cannot be checked by the host: they are forced into the arrays."""
    c = Case(d=64, nq=(200,), hq=2, h=1)
    for cu in ([0, 150, 90, 400], [0, -5, 2 ** 30, 200], [7, 50, 60, 70], [0, 200, 200, 200]):
        t = torch.tensor(cu, dtype=torch.int32, device="cuda")
        o, lse = fm.local_attention(c.q, c.k, c.v, c.scale, cu_seqlens_q=t, cu_seqlens_k=t, prefix=torch.tensor([-4, 1000, 3], device="cuda"))
        fm.local_attention_backward(c.q, c.k, c.v, c.scale, torch.zeros_like(o), torch.zeros_like(lse), c.d_out, cu_seqlens_q=t, cu_seqlens_k=t)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nq,nk,hq,d", [(256, 100, 1, 64), (256, 100, 1, 128), (300, 70, 1, 128), (200, 40, 1, 64), (128, 50, 2, 128), (64, 20, 4, 64)])
def test_rows_without_a_key_beside_rows_with_one(nq, nk, hq, d, dtype):
    """A block of two query tiles, the first of them whole and blind: its rows are zero, whatever the queries hold."""
    c = Case(dtype=dtype, d=d, hq=hq, h=1, nq=(nq,) * 6, nk=(nk,) * 6, seed=30)
    ro, rl, to, tl = c.forward()
    blind = torch.isinf(rl)
    assert int(blind.sum()) == 6 * hq * (nq - nk)
    for _ in range(20):
        o, lse = _run(c)
        assert (o[blind] == 0).all()
        assert_within(lse, rl, tl, "lse")
        assert_within(o, ro, to, "o")


@pytest.mark.parametrize("dtype", [BF, F])
def test_strides_of_dims_of_size_one(dtype):
    """One KV head, or one new token, cut from a buffer whose rows have an odd width."""
    c = Case(dtype=dtype, d=64, hq=1, h=1, nq=(3,), seed=33)
    wide = lambda t: torch.zeros(2, t.shape[1] * 64 + 1, dtype=dtype, device="cuda")[:, :-1].unflatten(1, t.shape[1:])[:1].copy_(t)
    q, k, v, g = (wide(t) for t in (c.q, c.k, c.v, c.d_out))
    assert q.is_contiguous() and q.stride(0) % 8
    o, lse = _run(c)
    o1, lse1 = fm.local_attention(q, k, v, c.scale, **c.kwargs())
    assert torch.equal(o, o1) and torch.equal(lse, lse1)
    want = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    assert all(torch.equal(a, b) for a, b in zip(want, fm.local_attention_backward(q, k, v, c.scale, o, lse, g, **c.kwargs())))
    cache = fm.PagedCache(1, 64, n_pages=2, n_seqs=1, max_len=16, page_size=16, dtype=dtype)
    cache.append([0], k, v, [0, 3])
    one = torch.zeros(3, 1, 131, dtype=dtype, device="cuda")[:, :, :64][:1].copy_(c.q[:, 2:])
    assert one.is_contiguous()
    cache.append([0], one, one)
    assert torch.equal(cache.gather([0], [0, 4])[0], torch.cat([c.k, c.q[:, 2:]], 1))
    a, b = cache.attend(one, c.scale), cache.attend(one.clone(memory_format=torch.contiguous_format), c.scale)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_traced_and_transformed_calls():
    """A traced graph holds the operators and computes them again; a forward-mode derivative is refused; vmap loops."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    c, f = Case(d=64, nq=(40, 30), hq=2, h=1, seed=34), Case(d=64, nq=(40, 30), hq=2, h=1, seed=35)
    kw = c.kwargs()
    cu = kw["cu_seqlens_q"]

    def step(q, k, v, g, cu):
        o, lse = fm.local_attention(q, k, v, c.scale, cu_seqlens_q=cu)
        return (o, lse, *fm.local_attention_backward(q, k, v, c.scale, o, lse, g, cu_seqlens_q=cu))

    want = step(f.q, f.k, f.v, f.d_out, cu)
    for how in ({}, {"pre_dispatch": True}, {"tracing_mode": "fake"}):
        graph = make_fx(step, **how)(c.q, c.k, c.v, c.d_out, cu)
        assert all(torch.equal(a, b) for a, b in zip(graph(f.q, f.k, f.v, f.d_out, cu), want)), how
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(c.q, c.q)
        with pytest.raises(fm.FastMemError, match="forward-mode"):
            fm.local_attention(dual, c.k, c.v, c.scale)
        with pytest.raises(fm.FastMemError, match="forward-mode"):
            fm.local_attention_backward(c.q, c.k, c.v, c.scale, want[0], want[1], dual)
    o, lse = torch.func.vmap(lambda q: fm.local_attention(q, c.k, c.v, c.scale, **kw))(torch.stack([c.q, f.q]))
    for i, q in enumerate((c.q, f.q)):
        o1, lse1 = fm.local_attention(q, c.k, c.v, c.scale, **kw)
        assert torch.equal(o[i], o1) and torch.equal(lse[i], lse1)


@pytest.mark.parametrize("skip", [0, 1])
@pytest.mark.parametrize("name,how", [
    ("forward and gradients", dict(nq=(300, 70), nk=(300, 400), hq=2, h=1, d=128)),
    ("cut over CTAs", dict(nq=(200,), nk=(900,), hq=2, h=1, d=64, dtype=HF, softcap=9.0)),
    ("few queries", dict(nq=(1, 2, 1), nk=(500, 90, 300), hq=4, h=1, d=128)),
])
def test_waits_that_give_up(name, how, skip):
    """With the test hook every CTA leaves out a tile; the waits for it run out after 20 ms, the CTA unwinds and computes its rows one
    at a time.  The results are the same to rounding, and so is the next call."""
    import time
    from fast_memory_b200 import _lib as L
    c = Case(**how, seed=37)
    kw = c.kwargs()
    ro, rl, to, tl = c.forward()
    want_o, want_lse = _run(c)
    grads = c.backward(want_o, want_lse)
    lib = L.lib()
    torch.cuda.synchronize()
    assert lib.fm_test_set_tc_hooks(20, skip) == 0
    try:
        start = time.perf_counter()
        o, lse = fm.local_attention(c.q, c.k, c.v, c.scale, **kw)
        torch.cuda.synchronize()
        middle = time.perf_counter()
        got = fm.local_attention_backward(c.q, c.k, c.v, c.scale, want_o, want_lse, c.d_out, **kw)
        torch.cuda.synchronize()
        end = time.perf_counter()
    finally:
        assert lib.fm_test_set_tc_hooks(0, -1) == 0
    assert 0.02 <= middle - start and (skip or 0.04 <= end - middle)
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    for g, (want, bound), what in zip(got, grads, ("dq", "dk", "dv")):
        assert_within(g, want, bound, what)
    o, lse = _run(c)
    assert torch.equal(o, want_o) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("how", [dict(nq=(300,)), dict(nq=(300,), hq=4, h=2, dtype=HF, slopes=True), dict(nq=(3,), nk=(300,), hq=2)])
@pytest.mark.parametrize("softcap", [2.0, 30.0])
def test_hidden_scores_choose_no_bits(how, softcap):
    """With a cap there are two formulas of tanh.  Keys behind a position, and queries before one, leave every bit of what does not
    see them (is not seen by them) as it was, whether their scores are small or large."""
    c = Case(**{"d": 128, "hq": 2, "h": 1, "softcap": softcap, "seed": 38, **how})
    S, N = c.q.shape[1], c.k.shape[1]
    t, j = (150, 150) if S == N else (1, N - S + 1)                # query t is the first to see key j
    o, lse = _run(c)
    backward = lambda: fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    dq, dk, dv = backward()
    for factor in (40.0, 0.0):
        was = c.k.clone()
        c.k[:, j:] *= factor
        o1, lse1 = _run(c)
        dq1 = backward()[0]
        assert torch.equal(o1[:, :t], o[:, :t]) and torch.equal(lse1[:, :t], lse[:, :t]) and torch.equal(dq1[:, :t], dq[:, :t])
        c.k.copy_(was)
        was = c.q.clone()
        c.q[:, :t] *= factor
        _, dk1, dv1 = backward()
        assert torch.equal(dk1[:, j:], dk[:, j:]) and torch.equal(dv1[:, j:], dv[:, j:])
        o1, lse1 = _run(c)
        assert torch.equal(o1[:, t:], o[:, t:]) and torch.equal(lse1[:, t:], lse[:, t:])
        c.q.copy_(was)


def test_a_result_that_no_loss_reads_costs_nothing(monkeypatch):
    """A loss over o alone hands the backward pass no LSE gradient (not a tensor of zeros)."""
    from fast_memory_b200 import local
    c = Case(d=64, nq=(90,), seed=39)
    leaves = [t.detach().clone().requires_grad_() for t in (c.q, c.k, c.v)]
    calls = []
    inner = local._local_bwd
    monkeypatch.setattr(local, "_local_bwd", lambda *a: calls.append((a[5] is None, a[6] is None)) or inner(*a))
    o, lse = fm.local_attention(*leaves, c.scale)
    (o * c.d_out).sum().backward(retain_graph=True)
    lse.sum().backward(retain_graph=True)
    (o.sum() + lse.sum()).backward()
    assert calls == [(False, True), (False, False), (False, False)]


@pytest.mark.parametrize("softcap", [0.0, 6.0])
@pytest.mark.parametrize("nq,nk", [((2048,), (2048,)), ((40, 200), (1500, 900))])
@pytest.mark.parametrize("size", [2.0 ** -18, 2.0 ** -12, 1.0, 2.0 ** 10])
def test_fp16_gradients_of_every_size(size, nq, nk, softcap):
    """Output gradients as losses of any scale give them.  With B = max(8 |dO|, |delta|) dS is held times more than 2^5 / B, so that a
    subnormal one is off by up to 2^-25 / 2^5 B = 2^-30 B; P is held times 2^12: 2^-37.  The results' own last place: 2^-25."""
    c = Case(dtype=HF, d=64, hq=2, h=1, nq=nq, nk=nk, causal=False, softcap=softcap, scale=1.0, seed=40)
    c.q *= 0.125
    c.d_out *= size
    o, lse = _run(c)
    B = max(8 * float(c.d_out.abs().max()), float((c.d_out.double() * o.double()).sum(-1).abs().max()))
    c.tiny = lambda n: n * 2.0 ** -30 * B * c.scale
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse), ("dq", "dk", "dv")):
        assert_within(got, want, bound + 2.0 ** -25, what)


def test_fp16_gradients_of_a_document_stand_alone():
    """How large a neighbour's output gradients are changes no bit; nor do those of rows that see no key."""
    c = Case(dtype=HF, d=128, hq=4, h=2, nq=(200, 300, 50), nk=(200, 300, 20), seed=41)
    o, lse = _run(c)
    backward = lambda: fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    want = backward()
    c.d_out[:, 200:500] *= 2.0 ** 9
    c.d_out[:, 500:530] = 60000.0                          # of the third document: blind
    got = backward()
    for a, b in zip(got, want):
        assert torch.equal(a[:, :200], b[:, :200]) and torch.equal(a[:, 500:], b[:, 500:])


@pytest.mark.parametrize("nq,n,heads,floor", [(1, 4096, 300, 2.0 ** -40), (200, 8192, 80, 2.0 ** -28)])
@pytest.mark.parametrize("below", [18.3, 23.4, 26.5])
def test_fp16_weights_far_below_the_largest(nq, n, heads, floor, below):
    """One key of weight 1 and no value, the others of weight 2^-below that make up the result.  A weight is off by its rounding or by
    2^-25 of what the kernel holds 1 as: 2^15 where rows are few, 2^3 elsewhere; the result's own last place is 2^-25.  As many
    heads as keep the kernels from cutting a row's keys into parts, which have references of their own."""
    c = Case(dtype=HF, d=64, hq=heads, h=heads, nq=(nq,), nk=(n,), causal=False, scale=1.0, seed=42)
    c.q.zero_(), c.k.zero_()
    c.q[..., 0], c.k[:, 0, 0] = 4.0, below * 0.6931471805599453 / 4
    c.v[:, 0], c.v[:, 1:] = 0.0, c.v[:, 1:].abs() + 0.5
    c.tiny = lambda n: n * floor
    o, lse = _run(c)
    ro, rl, to, tl = c.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to + 2.0 ** -25, "o")


@pytest.mark.parametrize("name,how", [
    ("group of 12", dict(hq=24, h=2, nq=(50, 3), nk=(130, 90), d=128)),
    ("group of 16, few rows", dict(hq=16, h=1, nq=(1, 1, 1), nk=(200, 70, 900), d=64, dtype=HF, window=150)),
    ("group of 17, few rows", dict(hq=34, h=2, nq=(1, 1, 2), nk=(200, 70, 500), d=128, softcap=12.0)),
    ("group of 40", dict(hq=40, h=1, nq=(33, 70), d=64, dtype=HF, slopes=True)),
    ("group of 100", dict(hq=100, h=1, nq=(30,), nk=(300,), d=128, prefix=(20,), window=90)),
    ("group of 128", dict(hq=128, h=1, nq=(9, 21), d=128, causal=False)),
    ("group of 130", dict(hq=130, h=1, nq=(20, 5), nk=(90, 5), d=64)),
    ("group of 40, fp32", dict(hq=40, h=1, nq=(33,), d=64, dtype=F)),
])
def test_many_query_heads_a_key_head(name, how):
    """Up to 16 the kernel of few rows takes them, up to 128 a query tile, beyond that the CUDA cores."""
    c = Case(**how, seed=43)
    o, lse = _run(c)
    ro, rl, to, tl = c.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, d_lse=c.d_lse, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse, c.d_lse), ("dq", "dk", "dv")):
        assert_within(got, want, bound, what)


@pytest.mark.parametrize("how", [
    dict(nq=tuple(1 + (i * 37) % 23 for i in range(700)), hq=2, h=1, d=64, prefix=tuple(i % 5 for i in range(700)), softcap=9.0, tail=11),
    dict(nq=tuple((i * 29) % 7 if i % 90 else 400 for i in range(600)), nk=tuple((i * 31) % 9 if i % 90 else 500 for i in range(600)), hq=2, h=2, d=128,
         dtype=HF, window=100),
    dict(nq=tuple(1 + i % 3 for i in range(500)), nk=tuple(1 + i % 3 + i % 70 for i in range(500)), hq=4, h=1, d=128),
])
def test_hundreds_of_documents(how):
    c = Case(**how, seed=44)
    o, lse = _run(c)
    ro, rl, to, tl = c.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse), ("dq", "dk", "dv")):
        assert_within(got, want, bound, what)


@pytest.mark.parametrize("how", [
    dict(nq=(4500,), hq=2, h=1, d=128, window=2000, prefix=(300,)),
    dict(nq=(5000,), hq=1, h=1, d=64, dtype=HF, softcap=20.0),
    dict(nq=(700,), nk=(9000,), hq=4, h=1, d=128, slopes=True),
    dict(nq=(3000,), hq=1, h=1, d=32, causal=False),
    dict(nq=(1500,), nk=(2500,), hq=1, h=1, d=256, window=700),
])
def test_long_rows(how):
    c = Case(**how, seed=45)
    o, lse = _run(c)
    ro, rl, to, tl = c.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse), ("dq", "dk", "dv")):
        assert_within(got, want, bound, what)


@pytest.mark.parametrize("dtype,nq", [(HF, 2), (BF, 300), (F, 100)])
@pytest.mark.parametrize("cap", [1e30, 1e37, 3e38])
def test_a_cap_out_of_reach_changes_nothing(dtype, nq, cap):
    """(s / cap)^2 / 3 of a score is nothing in 32 bits; scale / cap, which does not fit a normal number, must not stand in its way."""
    c = Case(dtype=dtype, d=64, hq=2, h=1, nq=(nq,), nk=(nq + 50,), scale=1e-4, seed=47)
    c.q *= 300.0
    c.k *= 100.0
    o, lse = _run(c)
    kw = dict(c.kwargs(), softcap=cap)
    o1, lse1 = fm.local_attention(c.q, c.k, c.v, c.scale, **kw)
    assert torch.equal(o, o1) and torch.equal(lse, lse1)
    want = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    got = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_diverged_step_ends_soon():
    """Queries that are all NaN make every row NaN, and each ends with its first key (all keys a row one at a time: 35 and 110 ms)."""
    c = Case(d=128, hq=8, h=8, nq=(4096,), window=2048, seed=48)
    o, lse = _run(c)
    fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    c.q.fill_(float("nan"))
    kw = c.kwargs()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    a.record()
    o, lse = fm.local_attention(c.q, c.k, c.v, c.scale, **kw)
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **kw)
    b.record()
    torch.cuda.synchronize()
    assert all(torch.isnan(t).all() for t in (o, lse, *grads))
    assert a.elapsed_time(b) < 20.0


@pytest.mark.parametrize("nq,nk", [((1,), (268,)), ((3, 40), (200, 90))])
@pytest.mark.parametrize("size", [1.0, 64.0])
def test_fp16_gradients_of_keys_that_weigh_little(size, nq, nk):
    """Output gradients of usual size leave dS as it is: what is subnormal is off by 2^-25 and no more, however large others are."""
    c = Case(dtype=HF, d=128, hq=4, h=2, nq=nq, nk=nk, scale=1.0, seed=49)
    c.d_out *= size
    o, lse = _run(c)
    grads = fm.local_attention_backward(c.q, c.k, c.v, c.scale, o, lse, c.d_out, **c.kwargs())
    for got, (want, bound), what in zip(grads, c.backward(o, lse), ("dq", "dk", "dv")):
        assert_within(got, want, bound + 2.0 ** -25, what)
