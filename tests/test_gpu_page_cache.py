"""The page operations of a cache against a model that keeps every sequence as a list of rows and deals out pages one at a time,
and attention over the cache against its definition in 64 bits."""
import random

import pytest
import torch

import fast_memory_b200 as fm
from fast_memory_b200 import _lib as L
from tests.local_reference import Case, assert_within

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


class Model:
    def __init__(self, cache):
        self.c = cache
        self.rows = [[] for _ in range(cache.n_seqs)]          # token contents (k, v) of every sequence
        self.pages = [[] for _ in range(cache.n_seqs)]
        self.refs = [0] * cache.n_pages

    def take(self):
        at = self.refs.index(0)
        self.refs[at] = 1
        return at

    def append(self, seqs, k, v, cu):
        for i, s in enumerate(seqs):
            self.rows[s] += [(k[:, t], v[:, t]) for t in range(cu[i], cu[i + 1])]
            while len(self.pages[s]) * self.c.page_size < len(self.rows[s]):
                self.pages[s].append(self.take())

    def fork(self, parents, children):
        for a, b in zip(parents, children):
            full = len(self.rows[a]) // self.c.page_size
            self.pages[b] = self.pages[a][:full]
            for x in self.pages[b]:
                self.refs[x] += 1
            if len(self.rows[a]) % self.c.page_size:
                self.pages[b].append(self.take())
            self.rows[b] = list(self.rows[a])

    def free(self, seqs):
        for s in seqs:
            for x in self.pages[s]:
                self.refs[x] -= 1
            self.pages[s], self.rows[s] = [], []

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        moved = dict(zip([x for x in range(n, len(self.refs)) if self.refs[x]], [x for x in range(n) if not self.refs[x]]))
        for a, b in moved.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.pages = [[moved.get(x, x) for x in p] for p in self.pages]

    def same(self):
        c = self.c
        assert c.refcounts.tolist() == self.refs
        assert c.lengths.tolist() == [len(r) for r in self.rows]
        width = c.page_table.shape[1]
        assert c.page_table.tolist() == [p + [-1] * (width - len(p)) for p in self.pages]
        some = [s for s in range(c.n_seqs) if self.rows[s]]
        cu = [0]
        for s in some:
            cu.append(cu[-1] + len(self.rows[s]))
        if some:
            k, v = c.gather(some, cu)
            assert torch.equal(k, torch.stack([r[0] for s in some for r in self.rows[s]], 1))
            assert torch.equal(v, torch.stack([r[1] for s in some for r in self.rows[s]], 1))


def _new(cache, n, gen):
    return [torch.randn(cache.n_heads, n, cache.d, generator=gen).to(cache.k_pages.dtype).cuda() for _ in range(2)]


@pytest.mark.parametrize("dtype,d,page,H", [(BF, 128, 64, 2), (HF, 64, 16, 3), (F, 32, 32, 1), (BF, 16, 256, 2)])
def test_random_operations(dtype, d, page, H):
    rng, gen = random.Random(5), torch.Generator().manual_seed(5)
    c = fm.PagedCache(H, d, n_pages=300, n_seqs=12, max_len=12 * page, page_size=page, dtype=dtype)
    m = Model(c)
    for _ in range(40):
        what = rng.choice(["append", "append", "append", "fork", "free", "compact"])
        if what == "append":
            seqs = rng.sample(range(12), rng.randint(1, 8))
            new = [min(rng.choice([0, 1, 1, page - 1, page, 2 * page + 3]), 12 * page - len(m.rows[s])) for s in seqs]
            cu = [sum(new[:i]) for i in range(len(new) + 1)]
            k, v = _new(c, cu[-1], gen)
            c.append(seqs, k, v, cu)
            m.append(seqs, k, v, cu)
        elif what == "fork":
            empty = [s for s in range(12) if not m.rows[s]]
            children = empty[:rng.randint(0, len(empty))]
            parents = [rng.randrange(12) for _ in children]    # among them empty ones, and one with several children
            c.fork(parents, children)
            m.fork(parents, children)
        elif what == "free":
            seqs = rng.sample(range(12), rng.randint(0, 4))
            c.free(seqs)
            m.free(seqs)
        else:
            c.compact()
            m.compact()
        m.same()
    c.check()


def test_appending_one_token_a_sequence_and_strides():
    gen = torch.Generator().manual_seed(1)
    c = fm.PagedCache(2, 64, n_pages=40, n_seqs=5, max_len=100, page_size=16)
    m = Model(c)
    for step in range(40):
        wide = torch.randn(5, 2, 3 * 64, generator=gen).to(BF).cuda()          # [tokens, heads, q | k | v]
        k, v = wide[..., 64:128].transpose(0, 1), wide[..., 128:].transpose(0, 1)
        seqs = [4, 2, 0, 1, 3]
        c.append(torch.tensor(seqs, device="cuda"), k, v)
        m.append(seqs, k.contiguous(), v.contiguous(), list(range(6)))
    m.same()
    # tokens behind the last sequence's are left out; an empty call does nothing
    k, v = _new(c, 9, gen)
    c.append([1, 3], k, v, [0, 4, 7])
    m.append([1, 3], k, v, [0, 4, 7])
    c.append([], k[:, :0], v[:, :0])
    m.same()
    c.check()


def test_refused_calls_change_nothing():
    gen = torch.Generator().manual_seed(2)
    c = fm.PagedCache(1, 64, n_pages=8, n_seqs=4, max_len=96, page_size=16)
    m = Model(c)
    k, v = _new(c, 70, gen)
    c.append([0, 1], k, v, [0, 40, 70])                       # 3 + 2 pages
    m.append([0, 1], k, v, [0, 40, 70])
    before = [t.clone() for t in (c.k_pages, c.v_pages, c.page_table, c.lengths, c.refcounts)]
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    calls = [
        ("too few", lambda: c.append([2], k, v, [0, 49])),                       # 4 pages, 3 are free
        ("too few", lambda: c.append([2, 3], k, v, [0, 33, 34])),
        ("outgrow", lambda: c.append([0], k, v, [0, 57])),
        ("named twice", lambda: c.append([2, 2], k, v, [0, 1, 2])),
        ("out of range", lambda: c.append([4], k, v, [0, 1])),
        ("out of range", lambda: c.append([-1], k, v, [0, 1])),
        ("do not rise", lambda: c.append([2, 3], k, v, dev([0, 5, 3]))),
        ("do not rise", lambda: c.append([2, 3], k, v, dev([0, 5, 71]))),
        ("do not rise", lambda: c.append([2, 3], k, v, dev([1, 5, 6]))),
        ("holds tokens", lambda: c.fork([0], [1])),
        ("named twice", lambda: c.fork([0, 1], [2, 2])),
        ("out of range", lambda: c.fork([9], [2])),
        ("out of range", lambda: c.fork([0], [9])),
        ("named twice", lambda: c.free([0, 1, 0])),
        ("out of range", lambda: c.free([0, 7])),
    ]
    for text, call in calls:
        call()
        with pytest.raises(fm.FastMemError, match=text):
            c.check()
        c.check()                                               # reported once
        assert all(torch.equal(a, b) for a, b in zip(before, (c.k_pages, c.v_pages, c.page_table, c.lengths, c.refcounts)))
    m.same()
    errors = [
        (ValueError, lambda: c.append([0, 1], k, v, [0, 1])),
        (ValueError, lambda: c.append([0], k[0], v[0], [0, 1])),
        (TypeError, lambda: c.append([0], k.half(), v.half(), [0, 1])),
        (ValueError, lambda: c.append([0], k, v, [0, 71])),
        (ValueError, lambda: c.append([0], k, v)),
        (ValueError, lambda: c.fork([0, 1], [2])),
        (ValueError, lambda: c.free([0, 1, 2, 3, 0])),
        (ValueError, lambda: c.copy_pages([0], [1, 2])),
        (ValueError, lambda: c.gather([0], [0, 3, 4])),
        (ValueError, lambda: c.gather([0], dev([0, 3]))),
        (TypeError, lambda: c.free(torch.tensor([0.5], device="cuda"))),
        (fm.FastMemError, lambda: c.append([0], k.cpu(), v.cpu(), [0, 1])),
        (ValueError, lambda: fm.PagedCache(1, 64, n_pages=0, n_seqs=1, max_len=10)),
        (ValueError, lambda: fm.PagedCache.over(c.k_pages, c.v_pages, c.page_table, c.lengths[:2], c.refcounts)),
        (TypeError, lambda: fm.PagedCache.over(c.k_pages, c.v_pages, c.page_table.long(), c.lengths, c.refcounts)),
        (fm.FastMemError, lambda: fm.PagedCache(1, 64, n_pages=4, n_seqs=1, max_len=48, page_size=24).compact()),
    ]
    for n, (error, call) in enumerate(errors):
        with pytest.raises(error):
            call()
            print("call", n, "was not refused")
    c.check()


def test_copy_pages_and_gather_parts():
    gen = torch.Generator().manual_seed(3)
    c = fm.PagedCache(2, 64, n_pages=64, n_seqs=2, max_len=400, page_size=32)
    k, v = _new(c, 300, gen)
    c.append([1], k, v, [0, 300])
    src = [0, 3, 5, 64, -1]
    c.copy_pages(src, [20, 21, 22, 23, 24])                    # pairs with a page that does not exist are passed over
    for a, b in ((0, 20), (3, 21), (5, 22)):
        assert torch.equal(c.k_pages[a], c.k_pages[b]) and torch.equal(c.v_pages[a], c.v_pages[b])
    assert (c.k_pages[23:25] == 0).all()
    kk, vv = c.gather([1, 0, 1], torch.tensor([0, 50, 60, 90], device="cuda"), starts=[7, 0, 290], n_tokens=95)
    assert torch.equal(kk[:, :50], k[:, 7:57]) and torch.equal(vv[:, :50], v[:, 7:57])
    assert (kk[:, 50:60] == 0).all() and torch.equal(kk[:, 60:70], k[:, 290:]) and (vv[:, 70:] == 0).all()


def _filled(case, page, seqs_total, order_seed=0, poison=False):
    """A cache whose sequences hold the documents of ``case`` in a shuffled order of sequences and pages."""
    rng = random.Random(order_seed)
    n_pages = sum(-(-n // page) for n in case.nk) + 5
    width = max(1, max(-(-n // page) for n in case.nk)) + 1
    H, d = case.h, case.d
    kp = torch.full((n_pages, H, page, d), float("nan") if poison else 0.0, dtype=case.dtype, device="cuda")
    vp = kp.clone()
    table = torch.full((seqs_total, width), -1, dtype=torch.int32)
    lengths, refs = torch.zeros(seqs_total, dtype=torch.int32), torch.zeros(n_pages, dtype=torch.int32)
    seqs, free = rng.sample(range(seqs_total), len(case.nk)), rng.sample(range(n_pages), n_pages)
    for t, s in enumerate(seqs):
        lengths[s] = case.nk[t]
        for x in range(-(-case.nk[t] // page)):
            at = free.pop()
            table[s, x], refs[at] = at, 1
            a, b = case.ck[t] + x * page, min(case.ck[t] + (x + 1) * page, case.ck[t + 1])
            kp[at, :, :b - a], vp[at, :, :b - a] = case.k[:, a:b], case.v[:, a:b]
    return fm.PagedCache.over(kp, vp, table.cuda(), lengths.cuda(), refs.cuda()), seqs


PAGED = {
    "decode": dict(nq=(1,) * 9, nk=(1, 16, 17, 63, 64, 65, 300, 128, 1000), hq=8, h=2, d=128, page=16),
    "decode, page 256": dict(nq=(1,) * 4, nk=(5, 256, 257, 700), hq=4, h=4, d=64, page=256, dtype=HF),
    "decode, one long sequence": dict(nq=(1,), nk=(9000,), hq=8, h=2, d=128, page=64),
    "decode, window and prefix": dict(nq=(1, 1, 1), nk=(700, 90, 3000), hq=4, h=1, d=128, page=32, window=100, prefix=(5, 200, 33)),
    "decode, group of seven, capped": dict(nq=(1,) * 3, nk=(40, 333, 2000), hq=7, h=1, d=128, page=64, softcap=9.0),
    "chunks": dict(nq=(40, 1, 0, 130, 257), nk=(40, 500, 20, 390, 1000), hq=4, h=2, d=128, page=64),
    "chunks, page 16": dict(nq=(129, 64), nk=(700, 64), hq=4, h=1, d=64, page=16, slopes=True, dtype=HF),
    "chunks, window": dict(nq=(200, 33), nk=(900, 1500), hq=2, h=2, d=128, page=128, window=150, softcap=20.0),
    "not causal": dict(nq=(30, 5), nk=(90, 300), hq=4, h=2, d=128, page=32, causal=False),
    "lengths shorter than the queries": dict(nq=(20, 9), nk=(12, 0), hq=2, h=1, d=64, page=16),
    "fp32": dict(nq=(1, 30), nk=(80, 300), hq=2, h=1, d=64, page=16, dtype=F),
    "d 32": dict(nq=(1, 30), nk=(80, 300), hq=2, h=1, d=32, page=16),
    "tail": dict(nq=(5, 1), nk=(5, 44), hq=4, h=2, d=128, page=16, tail=7),
}


@pytest.mark.parametrize("poison", [False, True])
@pytest.mark.parametrize("name", PAGED)
def test_attention_over_pages(name, poison):
    """``poison``: the rows of the pool that hold no token are NaN."""
    how = dict(PAGED[name])
    page = how.pop("page")
    case = Case(**how, seed=11)
    cache, seqs = _filled(case, page, len(case.nk) + 3, poison=poison)
    kw = case.kwargs()
    kw.pop("cu_seqlens_k")
    o, lse = cache.attend(case.q, case.scale, seqs=seqs, **kw)
    ro, rl, to, tl = case.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
    if all(n == 1 for n in case.nq) and case.q.shape[1] == len(case.nq):
        kw.pop("cu_seqlens_q")
        o2, lse2 = cache.attend(case.q, case.scale, seqs=torch.tensor(seqs, device="cuda"), **kw)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_paged_refusals():
    c = fm.PagedCache(2, 64, n_pages=8, n_seqs=3, max_len=64, page_size=16)
    q = torch.zeros(4, 3, 64, dtype=BF, device="cuda")
    o, lse = c.attend(q, 1.0)
    assert (o == 0).all() and torch.isinf(lse).all()           # empty sequences
    errors = [
        (ValueError, lambda: c.attend(q[:, :2], 1.0)),
        (ValueError, lambda: c.attend(q, 1.0, seqs=[0, 1])),
        (ValueError, lambda: c.attend(q, 1.0, cu_seqlens_q=[0, 1])),
        (ValueError, lambda: c.attend(q, 1.0, cu_seqlens_q=[0, 1, 2, 5])),
        (ValueError, lambda: c.attend(q[:3], 1.0)),
        (ValueError, lambda: c.attend(q[..., :32], 1.0)),
        (TypeError, lambda: c.attend(q.half(), 1.0)),
        (ValueError, lambda: c.attend(q, 1.0, window=-2)),
        (ValueError, lambda: c.attend(q, 1.0, prefix=[1])),
        (fm.FastMemError, lambda: c.attend(q.cpu(), 1.0)),
        (TypeError, lambda: fm.paged_attention(q, c.k_pages, c.v_pages, c.page_table.long(), c.lengths, 1.0)),
        (ValueError, lambda: fm.paged_attention(q, c.k_pages.transpose(0, 1).contiguous().transpose(0, 1), c.v_pages, c.page_table, c.lengths, 1.0)),
    ]
    for n, (error, call) in enumerate(errors):
        with pytest.raises(error):
            call()
            print("call", n, "was not refused")
    # tables and lengths that point outside stay inside the pool
    c.page_table.fill_(10 ** 6)
    c.lengths.fill_(10 ** 6)
    c.attend(q, 1.0, seqs=[7, -3, 1])
    torch.cuda.synchronize()


def test_a_serving_step_captured_and_replayed():
    """append + attend + merge with a memory as one graph, replayed while the sequences grow over page borders."""
    gen = torch.Generator().manual_seed(4)
    H, G, d, B = 2, 2, 64, 3
    c = fm.PagedCache(H, d, n_pages=40, n_seqs=B, max_len=160, page_size=16)
    plain = fm.PagedCache(H, d, n_pages=40, n_seqs=B, max_len=160, page_size=16)
    k0, v0 = _new(c, 30, gen)
    for x in (c, plain):
        x.append([0, 1, 2], k0, v0, [0, 15, 15, 30])
    mk, mv = _new(c, 256, gen)
    mem = fm.Memory.build(mk, mv, A=torch.randn(H, 4, d, generator=gen).to(BF).cuda(), bucket_size=64)
    q, k, v = torch.empty(H * G, B, d, dtype=BF, device="cuda"), *(torch.empty(H, B, d, dtype=BF, device="cuda") for _ in range(2))
    seqs = torch.arange(B, dtype=torch.int32, device="cuda")
    sm = d ** -0.5

    def step(x):
        x.append(seqs, k, v)
        o, lse = x.attend(q, sm, window=20)
        om, lm = mem.query(q, sm)
        return fm.merge(o, lse, om, lm)

    for t in (q, k, v):
        t.copy_(torch.randn(t.shape, generator=gen))
    side = torch.cuda.Stream()
    state = [t.clone() for t in (c.page_table, c.lengths, c.refcounts)]
    with torch.cuda.stream(side):
        step(c)
        torch.cuda.synchronize()
        for t, s in zip((c.page_table, c.lengths, c.refcounts), state):
            t.copy_(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, lse = step(c)
    torch.cuda.synchronize()
    for _ in range(40):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen))
        graph.replay()
        want = step(plain)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert torch.equal(c.page_table, plain.page_table) and torch.equal(c.refcounts, plain.refcounts)
    c.check()


def test_from_the_cache_into_a_memory():
    """What leaves the window is gathered from the cache and becomes a memory; window and memory together are attention over
    everything."""
    gen = torch.Generator().manual_seed(6)
    H, G, d, N, W = 2, 2, 64, 600, 100
    c = fm.PagedCache(H, d, n_pages=24, n_seqs=2, max_len=700, page_size=32)
    k, v = _new(c, N, gen)
    c.append([1], k, v, [0, N])
    q = torch.randn(H * G, 1, d, generator=gen).to(BF).cuda()
    sm = d ** -0.5
    old_k, old_v = c.gather([1], [0, N - W])
    mem = fm.Memory.build(old_k, old_v, A=torch.randn(H, 2, d, generator=gen).to(BF).cuda(), bucket_size=N - W)
    o, lse = fm.merge(*c.attend(q, sm, seqs=[1], window=W), *mem.query(q, sm))
    s = (q.double() @ k.double().repeat_interleave(G, 0).transpose(1, 2)) * sm
    ref = torch.softmax(s, -1) @ v.double().repeat_interleave(G, 0)
    assert (o.double() - ref).abs().max() <= 3 * 2.0 ** -8 * float(v.abs().max()) / 4
    assert (lse.double() - torch.logsumexp(s, -1)).abs().max() <= 1e-3


@pytest.mark.parametrize("nq,nk,hq,d", [(256, 100, 1, 128), (128, 50, 2, 64)])
def test_rows_without_a_key_beside_rows_with_one_over_pages(nq, nk, hq, d):
    """Lengths shorter than the queries, the first query tile of a block whole and blind."""
    case = Case(hq=hq, h=1, d=d, nq=(nq,) * 3, nk=(nk,) * 3, seed=31)
    cache, seqs = _filled(case, 16, 5, poison=True)
    kw = case.kwargs()
    kw.pop("cu_seqlens_k")
    ro, rl, to, tl = case.forward()
    blind = torch.isinf(rl)
    assert blind.any()
    for _ in range(20):
        o, lse = cache.attend(case.q, case.scale, seqs=seqs, **kw)
        assert (o[blind] == 0).all()
        assert_within(lse, rl, tl, "lse")
        assert_within(o, ro, to, "o")


def test_traced_attention_over_pages():
    """A traced graph holds the operator; a backward pass through its result says that there is none; page operations are not traced."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    case = Case(hq=4, h=2, d=64, nq=(5, 40), nk=(30, 90), seed=36)
    cache, seqs = _filled(case, 16, 3)
    seqs = torch.tensor(seqs, dtype=torch.int32, device="cuda")
    kw = case.kwargs()
    kw.pop("cu_seqlens_k")
    f = lambda q: cache.attend(q, case.scale, seqs=seqs, **kw)
    q2 = case.q.flip(1).contiguous()
    want = f(q2)
    for how in ({}, {"pre_dispatch": True}):
        graph = make_fx(f, **how)(case.q)
        assert all(torch.equal(a, b) for a, b in zip(graph(q2), want))
    o, lse = torch.compile(f, backend="aot_eager")(q2)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    leaf = q2.clone().requires_grad_()
    o, lse = f(leaf)
    assert torch.equal(o.detach(), want[0]) and torch.equal(lse.detach(), want[1])
    with pytest.raises(RuntimeError, match="no autograd"):
        o.sum().backward()
    with torch.no_grad():
        assert not f(leaf)[0].requires_grad
    with forward_ad.dual_level(), pytest.raises(fm.FastMemError, match="forward-mode"):
        f(forward_ad.make_dual(q2, q2))
    k = torch.zeros(2, 1, 64, dtype=case.dtype, device="cuda")
    before = cache.lengths.clone()
    for call in (lambda t: cache.append(seqs[:1], t, t) or t, lambda t: cache.free(seqs) or t, lambda t: cache.fork(seqs, seqs) or t,
                 lambda t: cache.compact() or t, lambda t: cache.copy_pages(seqs, seqs) or t,
                 lambda t: cache.gather(seqs[:1], torch.tensor([0, 1], device="cuda"), n_tokens=1)[0]):
        with pytest.raises(fm.FastMemError, match="traced"):
            make_fx(call)(k)
    assert torch.equal(cache.lengths, before)
    torch.compile(lambda t: cache.append(seqs[:1], t, t), backend="aot_eager")(k)
    before[seqs[0]] += 1
    assert torch.equal(cache.lengths, before)
    cache.check()


def test_two_host_threads_share_a_cache():
    """Both enqueue on the default stream; rows that a kernel of their own copies, pages dealt out in whatever order."""
    import threading
    gen = torch.Generator().manual_seed(12)
    H, d, n, rounds = 8, 128, 40, 25
    c = fm.PagedCache(H, d, n_pages=2 * (n * rounds // 16 + 2), n_seqs=2, max_len=n * rounds, page_size=16)
    new = [_new(c, n * rounds, gen) for _ in range(2)]

    def run(s):
        k, v = new[s]
        for i in range(rounds):
            c.append([s], k[:, i * n:(i + 1) * n], v[:, i * n:(i + 1) * n], [0, n])

    threads = [threading.Thread(target=run, args=(s,)) for s in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    c.check()
    for s in range(2):
        k, v = c.gather([s], [0, n * rounds])
        assert torch.equal(k, new[s][0]) and torch.equal(v, new[s][1])


def test_sequence_numbers_of_64_bits():
    gen = torch.Generator().manual_seed(13)
    c = fm.PagedCache(1, 64, n_pages=4, n_seqs=2, max_len=32, page_size=16)
    k, v = _new(c, 5, gen)
    c.append(torch.tensor([1], device="cuda"), k, v, torch.tensor([0, 5], device="cuda"))
    c.check()
    c.free(torch.tensor([2 ** 32 + 1], device="cuda"))
    with pytest.raises(fm.FastMemError, match="out of range"):
        c.check()
    assert c.lengths.tolist() == [0, 5]


@pytest.mark.parametrize("how", [
    dict(hq=4, h=1, nq=(1,) * 31 + (400,), nk=tuple(40 + 9 * i for i in range(31)) + (900,)),            # many rows a sequence on average
    dict(hq=2, h=2, nq=(1,) * 60 + (500,), nk=tuple(30 + 7 * i for i in range(60)) + (800,), window=120),  # few
])
def test_single_tokens_and_a_chunk_in_one_call(how):
    case = Case(d=128, **how, seed=46)
    cache, seqs = _filled(case, 32, len(case.nk), poison=True)
    kw = case.kwargs()
    kw.pop("cu_seqlens_k")
    o, lse = cache.attend(case.q, case.scale, seqs=seqs, **kw)
    ro, rl, to, tl = case.forward()
    assert_within(lse, rl, tl, "lse")
    assert_within(o, ro, to, "o")
