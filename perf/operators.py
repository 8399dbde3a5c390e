"""The operators around a memory's near context, as cases: attention over local keys with its gradients, attention of new
tokens over a paged cache, and the page operations of that cache.

``run`` computes a case in its plain form (elementary torch operations in 32 bits) or, where ``own`` is true, through
``fast_memory_b200``.  Lengths of documents and sequences come from the case alone (``mix``), values from the seed."""
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- cases ---------------------------------------------------------------------------------------------------------
def _attend(name, kind, dtype, hq, h, d, docs, s, past=0, causal=True, window=0, softcap=0.0, slopes=False, prefix=0,
            token_major=False, d_lse=False, mix=1):
    return {"name": name, "kind": kind, "dtype": dtype, "hq": hq, "h": h, "d": d, "docs": docs, "s": s, "past": past,
            "causal": causal, "window": window, "softcap": softcap, "slopes": slopes, "prefix": prefix,
            "token_major": token_major, "d_lse": d_lse, "mix": mix}


def _paged(name, dtype, hq, h, d, seqs, new, context, page, window=0, softcap=0.0, slopes=False, prefix=0, mix=1):
    return {"name": name, "kind": "paged", "dtype": dtype, "hq": hq, "h": h, "d": d, "seqs": seqs, "new": new, "context": context,
            "page": page, "window": window, "softcap": softcap, "slopes": slopes, "prefix": prefix, "mix": mix}


def _pages(name, kind, dtype, h, d, seqs, context, new, page, mix=1):
    return {"name": name, "kind": kind, "dtype": dtype, "h": h, "d": d, "seqs": seqs, "context": context, "new": new, "page": page,
            "mix": mix}


def listed():
    return [
        # a short prompt of one sequence on one KV head's group: nothing but latency
        _attend("attend short", "attend", "bf16", 4, 1, 128, 1, 33),
        # the single-head fp32 workload: the last 512 positions of 4096, full precision
        _attend("attend fp32", "attend", "fp32", 1, 1, 64, 1, 512, past=3584),
        # prefill of the 32-head workload: 8192 queries a head over a local window of 4096 keys
        _attend("attend window", "attend", "bf16", 32, 32, 128, 1, 8192, window=4096),
        # training on one odd-sized sequence, grouped heads, distance bias, fp16 with head dim 64, activations [tokens, heads, d]
        _attend("train small", "train", "fp16", 8, 2, 64, 1, 777, slopes=True, token_major=True),
        # training on 16 packed documents of unequal length: capped scores, a prefix every token sees, a loss that reads the LSE
        _attend("train documents", "train", "bf16", 8, 8, 128, 16, 16384, softcap=30.0, prefix=96, d_lse=True, mix=5),
        # training on one long sequence with a local window, 32 query heads over 8 KV heads
        _attend("train window", "train", "bf16", 32, 8, 128, 1, 8192, window=4096),
        # decode: one new token for each of 64 sequences of unequal length, 32 query heads over 8 KV heads
        _paged("paged decode", "bf16", 32, 8, 128, 64, 1, 16384, 64, mix=2),
        # decode of a single sequence with a long context: few rows, one long axis
        _paged("paged decode one", "fp16", 32, 8, 128, 1, 1, 131072, 128),
        # prompts that arrive in chunks: up to 1024 new tokens of four sequences over what is cached, small pages, capped scores
        _paged("paged chunk", "bf16", 32, 8, 128, 4, 1024, 16384, 16, softcap=50.0, mix=3),
        # parallel sampling: every sequence forked, one token appended to each fork, the forks freed again
        _pages("pages fork", "fork", "bf16", 8, 128, 64, 2048, 1, 64, mix=4),
        # the smallest step of a server: one token for each of four sequences, then dropped
        _pages("pages fork small", "fork", "fp16", 2, 64, 4, 200, 1, 16),
        # memory pressure: half of the sequences evicted, the pool compacted, new prompts admitted; then the other half
        _pages("pages compact", "compact", "bf16", 8, 128, 64, 4096, 4096, 64, mix=6),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "train", "train", "paged", "paged", "paged", "fork", "compact"])
    mix = rng.randrange(1 << 20)
    h, g = rng.choice([(1, 1), (1, 4), (2, 3), (2, 4), (4, 2), (8, 1), (8, 4), (4, 7), (16, 1), (32, 1)])
    if kind in ("attend", "train"):
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        d = rng.choice([64, 128, 128])
        # the score matrix stays within the largest listed case's: 32 heads x 8192 x 8192; fp32 within a sixteenth
        # of it, and half of it where every key is visible
        causal = rng.random() < 0.85
        most = 32 * 8192 * 8192 // (16 if dtype == "fp32" else 1) // (1 if causal else 2)
        s = _log(rng, 1, 8192)
        past = rng.choice([0, 0, _log(rng, 1, 4096)])
        docs = min(s, rng.choice([1, 1, _log(rng, 2, 16)]))
        while h * g * s * (s + past * docs) > most:
            s, past, docs = max(1, s // 2), past // 2, max(1, docs // 2)
        return {k: v for k, v in _attend("", kind, dtype, h * g, h, d, docs, s, past, causal,
                                         rng.choice([0, 0, _log(rng, 16, 4096)]), rng.choice([0.0, 0.0, 20.0 + 30.0 * rng.random()]),
                                         rng.random() < 0.3, rng.choice([0, 0, _log(rng, 4, 256)]), rng.random() < 0.3,
                                         rng.random() < 0.3, mix).items() if k != "name"}
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([16, 32, 64, 128])
    d = rng.choice([64, 128, 128])
    if kind == "paged":
        seqs, context = _log(rng, 1, 64), _log(rng, 128, 32768)
        new = rng.choice([1, 1, _log(rng, 2, 1024)])
        while seqs * context * h * d > 64 * 16384 * 8 * 128 or seqs * h * g * new * (context + new) > 4 * 32 * 1024 * 17408:
            seqs, context, new = max(1, seqs // 2), max(128, context // 2), max(1, new // 2)
        return {k: v for k, v in _paged("", dtype, h * g, h, d, seqs, new, context, page, rng.choice([0, 0, _log(rng, 64, 4096)]),
                                        rng.choice([0.0, 0.0, 20.0 + 30.0 * rng.random()]), rng.random() < 0.3,
                                        rng.choice([0, 0, _log(rng, 4, 256)]), mix).items() if k != "name"}
    h = min(h, 8)
    seqs, context = _log(rng, 2, 64), _log(rng, 40, 4096)
    new = rng.choice([1, _log(rng, 2, 64)]) if kind == "fork" else _log(rng, 16, 4096)
    return {k: v for k, v in _pages("", kind, dtype, h, d, seqs, context, new, page, mix).items() if k != "name"}


# ---- lengths: from the case alone ----------------------------------------------------------------------------------
def _doc_lengths(case):
    """Query and key counts of every document: the queries are cut at random places, each has 0 .. past earlier keys."""
    rng = random.Random(case["mix"])
    n, s = case["docs"], case["s"]
    cuts = sorted(rng.sample(range(1, s), n - 1)) if n > 1 else []
    nq = np.diff([0] + cuts + [s])
    past = [case["past"] if n == 1 else rng.randint(0, case["past"]) for _ in range(n)]
    return nq, nq + np.asarray(past)


def _prefixes(case, count):
    rng = random.Random(case["mix"] + 1)
    return [rng.randint(0, case["prefix"]) for _ in range(count)]


def _seq_lengths(case):
    """New tokens and lengths after them of every cached sequence; the longest has the case's context."""
    rng = random.Random(case["mix"])
    n = case["seqs"]
    new = [case["new"] if case["new"] == 1 or i == 0 else rng.randint(1, case["new"]) for i in range(n)]
    old = [case["context"] if i == 0 else rng.randint(case["context"] // 16, case["context"]) for i in range(n)]
    return np.asarray(new), np.asarray(old) + np.asarray(new)


def _pairs(case, nq, nk, prefix):
    """Visible (query, key) pairs of one head, and keys that some query sees, over all documents."""
    pairs = seen = 0
    w = case["window"] or 1 << 40
    for n_q, n_k, pre in zip(nq, nk, prefix):
        pos = np.arange(n_q, dtype=np.int64) + (n_k - n_q)
        lo = np.maximum(pos - w + 1, 0)
        hi = np.minimum(pos if case.get("causal", True) else pos + w - 1, n_k - 1)
        pre = min(pre, n_k)
        pairs += int((np.maximum(hi + 1 - np.maximum(lo, pre), 0) + pre).sum())
        seen += int(pre + max(0, hi.max() + 1 - max(lo.min(), pre)))
    return pairs, seen


# ---- inputs --------------------------------------------------------------------------------------------------------
def _int32(values):
    return torch.tensor([int(x) for x in values], dtype=torch.int32, device="cuda")


def _slopes(hq):
    """Geometric slopes, one a query head."""
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / hq) for i in range(hq)], dtype=torch.float32, device="cuda")


def _prepare_attend(case, gen, dtype):
    hq, h, d = case["hq"], case["h"], case["d"]
    nq, nk = _doc_lengths(case)
    s, n = int(nq.sum()), int(nk.sum())

    def rows(heads, count):
        if case["token_major"]:  # activations as a projection leaves them, [tokens, heads, d]
            return torch.randn(count, heads, d, generator=gen, device="cuda").to(dtype).transpose(0, 1)
        return torch.randn(heads, count, d, generator=gen, device="cuda").to(dtype)

    st = {"q": rows(hq, s), "k": rows(h, n), "v": rows(h, n), "scale": d ** -0.5, "cu_q": None, "cu_k": None}
    st["cu_q"], st["cu_k"] = _int32(np.concatenate([[0], nq.cumsum()])), _int32(np.concatenate([[0], nk.cumsum()]))
    st["prefix"] = _int32(_prefixes(case, case["docs"])) if case["prefix"] else None
    st["slopes"] = _slopes(hq) if case["slopes"] else None
    if case["kind"] == "train":
        st["d_out"] = rows(hq, s)
        st["d_lse"] = torch.randn(hq, s, generator=gen, device="cuda") if case["d_lse"] else None
    return st


def _page_state(case, lengths, n_pages, gen, dtype, rows=None):
    """A pool whose pages are dealt out to the sequences in a shuffled order, as a server's are after a while.  ``rows``: rows
    of the page table (more than there are sequences where forks will need them)."""
    h, d, page = case["h"], case["d"], case["page"]
    rng = random.Random(case["mix"] + 2)
    counts = [-(-int(x) // page) for x in lengths]
    free = list(range(n_pages if case["kind"] == "paged" else sum(counts)))
    rng.shuffle(free)
    longest = max(-(-(int(x) + case["new"]) // page) for x in lengths)
    table = np.full((rows or len(lengths), longest), -1, dtype=np.int32)
    refs = np.zeros(n_pages, dtype=np.int32)
    for i, c in enumerate(counts):
        table[i, :c] = [free.pop() for _ in range(c)]
        refs[table[i, :c]] = 1
    full = np.zeros(rows or len(lengths), dtype=np.int32)
    full[:len(lengths)] = lengths
    return {"k_pages": torch.randn(n_pages, h, page, d, generator=gen, device="cuda", dtype=dtype),
            "v_pages": torch.randn(n_pages, h, page, d, generator=gen, device="cuda", dtype=dtype),
            "table": torch.from_numpy(table).cuda(), "lengths": torch.from_numpy(full).cuda(),
            "refs": torch.from_numpy(refs).cuda(), "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_paged(case, gen, dtype):
    new, lengths = _seq_lengths(case)
    n_pages = sum(-(-int(x) // case["page"]) for x in lengths) + 3
    st = _page_state(case, lengths, n_pages, gen, dtype)
    st["q"] = torch.randn(case["hq"], int(new.sum()), case["d"], generator=gen, device="cuda").to(dtype)
    st["cu_q"] = _int32(np.concatenate([[0], new.cumsum()]))
    st["scale"] = case["d"] ** -0.5
    st["prefix"] = _int32(_prefixes(case, case["seqs"])) if case["prefix"] else None
    st["slopes"] = _slopes(case["hq"]) if case["slopes"] else None
    return st


def _new_rows(case, count, gen, dtype):
    return [torch.randn(case["h"], count, case["d"], generator=gen, device="cuda").to(dtype) for _ in range(2)]


def _cycle_lengths(case):
    rng = random.Random(case["mix"])
    n = case["seqs"]
    lengths = [case["context"] if i == 0 else rng.randint(max(1, case["context"] // 4), case["context"]) for i in range(n)]
    new = [case["new"] if i < 2 or case["new"] == 1 else rng.randint(1, case["new"]) for i in range(n)]
    return lengths, new


def _prepare_fork(case, gen, dtype):
    lengths, new = _cycle_lengths(case)
    n, page = case["seqs"], case["page"]
    n_pages = sum(-(-x // page) for x in lengths) + sum(-(-(x % page + y) // page) for x, y in zip(lengths, new)) + 5
    st = _page_state(case, lengths, n_pages, gen, dtype, rows=2 * n)
    st["parents"], st["children"] = _int32(range(n)), _int32(range(n, 2 * n))
    st["cu_new"] = _int32(np.concatenate([[0], np.cumsum(new)]))
    st["k_new"], st["v_new"] = _new_rows(case, sum(new), gen, dtype)
    return st


def _prepare_compact(case, gen, dtype):
    _, new = _cycle_lengths(case)
    n, page = case["seqs"], case["page"]
    n_pages = sum(-(-x // page) for x in new) + 7
    st = _page_state(case, new, n_pages, gen, dtype)
    for name, part in (("even", range(0, n, 2)), ("odd", range(1, n, 2))):
        st[name] = _int32(part)
        st["cu_" + name] = _int32(np.concatenate([[0], np.cumsum([new[i] for i in part])]))
        st["k_" + name], st["v_" + name] = _new_rows(case, sum(new[i] for i in part), gen, dtype)
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]
    make = {"attend": _prepare_attend, "train": _prepare_attend, "paged": _prepare_paged, "fork": _prepare_fork,
            "compact": _prepare_compact}[case["kind"]]
    st = make(case, gen, dtype)
    st["case"] = dict(case)
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _mask(case, p, j, prefix):
    """Key position j is visible from query position p of its document."""
    w = case["window"]
    near = j <= p if case.get("causal", True) else j < p + w if w else torch.ones_like(j <= p)
    if w:
        near = near & (j > p - w)
    return near if prefix is None else near | (j < prefix)


def _scores(case, q, k, scale, slopes, p, j):
    """Scaled scores, capped, less the distance bias: q [..., G, S, d], k [..., 1, N, d], slopes [H, G, 1, 1].  Returns them and
    the derivative of the cap."""
    s = (q @ k.transpose(-1, -2)) * scale
    slope = None
    if case["softcap"]:
        t = torch.tanh(s / case["softcap"])
        s, slope = t * case["softcap"], 1.0 - t * t
    if slopes is not None:
        s = s - slopes * (p - j).abs().float()
    return s, slope


def _softmax(s, visible):
    s = torch.where(visible, s, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total), (m + torch.log(total)).squeeze(-1)


def _where(cu, count):
    """Document and place inside it of each of ``count`` packed rows."""
    i = torch.arange(count, device="cuda", dtype=torch.int32)
    doc = torch.bucketize(i, cu[1:], right=True)
    return doc, i - cu[doc]


def _plain_attend(st):
    case, dtype = st["case"], st["q"].dtype
    h, d = case["h"], case["d"]
    g, s_len, n_len = case["hq"] // h, st["q"].shape[1], st["k"].shape[1]
    q, k, v = st["q"].float().reshape(h, g, s_len, d), st["k"].float()[:, None], st["v"].float()[:, None]
    doc_q, p = _where(st["cu_q"], s_len)
    doc_k, j = _where(st["cu_k"], n_len)
    shift = (st["cu_k"][1:] - st["cu_k"][:-1]) - (st["cu_q"][1:] - st["cu_q"][:-1])
    p, j = (p + shift[doc_q])[:, None], j[None, :]
    prefix = None if st["prefix"] is None else st["prefix"][doc_q][:, None]
    visible = _mask(case, p, j, prefix) & (doc_q[:, None] == doc_k[None, :])
    slopes = None if st["slopes"] is None else st["slopes"].reshape(h, g, 1, 1)
    s, cap = _scores(case, q, k, st["scale"], slopes, p, j)
    w, lse = _softmax(s, visible)
    del s
    o = w @ v
    out = [o.reshape(case["hq"], s_len, d).to(dtype), lse.reshape(case["hq"], s_len)]
    if case["kind"] == "attend":
        return out
    d_o = st["d_out"].float().reshape(h, g, s_len, d)
    dv = (w.transpose(-1, -2) @ d_o).sum(1)
    dot = (d_o * o).sum(-1, keepdim=True)
    if st["d_lse"] is not None:
        dot = dot - st["d_lse"].reshape(h, g, s_len, 1)
    ds = w * (d_o @ v.transpose(-1, -2) - dot)
    del w
    if cap is not None:
        ds = ds * cap
    ds = ds * st["scale"]
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).sum(1)
    return out + [dq.reshape(case["hq"], s_len, d).to(dtype), dk.to(dtype), dv.to(dtype)]


def _plain_paged(st):
    case, dtype = st["case"], st["q"].dtype
    h, d, n, most = case["h"], case["d"], case["seqs"], case["new"]
    g = case["hq"] // h
    doc, place = _where(st["cu_q"], st["q"].shape[1])
    q = torch.zeros(n, h, g, most, d, device="cuda")
    q[doc, :, :, place] = st["q"].float().reshape(h, g, -1, d).permute(2, 0, 1, 3)
    pages = st["table"].clamp(min=0)
    k = st["k_pages"][pages].float().permute(0, 2, 1, 3, 4).reshape(n, h, 1, -1, d)
    v = st["v_pages"][pages].float().permute(0, 2, 1, 3, 4).reshape(n, h, 1, -1, d)
    new = st["cu_q"][1:] - st["cu_q"][:-1]
    length = st["lengths"][:, None, None, None, None]
    p = torch.arange(most, device="cuda")[:, None] + (st["lengths"] - new)[:, None, None, None, None]
    j = torch.arange(k.shape[-2], device="cuda")[None, :]
    prefix = None if st["prefix"] is None else st["prefix"][:, None, None, None, None]
    visible = _mask(case, p, j, prefix) & (j < length)
    slopes = None if st["slopes"] is None else st["slopes"].reshape(h, g, 1, 1)
    s, _ = _scores(case, q, k, st["scale"], slopes, p, j)
    w, lse = _softmax(s, visible)
    del s
    o = (w @ v)[doc, :, :, place].permute(1, 2, 0, 3).reshape(case["hq"], -1, d)
    return [o.to(dtype), lse[doc, :, :, place].permute(1, 2, 0).reshape(case["hq"], -1)]


def _plain_free_pages(st, count):
    """The ``count`` lowest free pages."""
    return torch.sort((st["refs"] != 0).to(torch.uint8), stable=True).indices[:count].int()


def _plain_fork(st, parents, children):
    page = st["k_pages"].shape[2]
    length = st["lengths"][parents]
    full, rest = (length // page)[:, None], length % page
    rows, col = st["table"][parents], torch.arange(st["table"].shape[1], device="cuda")[None, :]
    some = (rest > 0).nonzero()[:, 0]
    fresh = _plain_free_pages(st, some.numel())
    st["refs"].index_add_(0, rows[col < full], torch.ones_like(rows[col < full]))
    st["refs"][fresh] = 1
    old = rows[some, full[some, 0]]
    child = torch.where(col < full, rows, -1)
    child[some, full[some, 0]] = fresh
    st["table"][children], st["lengths"][children] = child, length
    who, where = (torch.arange(page, device="cuda")[None, :] < rest[some][:, None]).nonzero(as_tuple=True)
    for pages in (st["k_pages"], st["v_pages"]):
        pages[fresh[who], :, where] = pages[old[who], :, where]


def _plain_append(st, seqs, k_new, v_new, cu):
    page = st["k_pages"].shape[2]
    new, start = cu[1:] - cu[:-1], st["lengths"][seqs]
    have, want = -(-start // page), -(-(start + new) // page)
    col = torch.arange(st["table"].shape[1], device="cuda")[None, :]
    who, where = ((col >= have[:, None]) & (col < want[:, None])).nonzero(as_tuple=True)
    fresh = _plain_free_pages(st, who.numel())
    st["table"][seqs[who], where] = fresh
    st["refs"][fresh] = 1
    st["lengths"][seqs] = start + new
    doc, place = _where(cu, k_new.shape[1])
    place = place + start[doc]
    to = st["table"][seqs[doc], place // page]
    st["k_pages"][to, :, place % page] = k_new.transpose(0, 1)
    st["v_pages"][to, :, place % page] = v_new.transpose(0, 1)


def _plain_free(st, seqs):
    rows = st["table"][seqs]
    used = rows[rows >= 0]
    st["refs"].index_add_(0, used, torch.full_like(used, -1))
    st["table"][seqs] = -1
    st["lengths"][seqs] = 0


def _plain_compact(st):
    live = st["refs"] > 0
    at = torch.arange(live.numel(), device="cuda", dtype=torch.int32)
    count = live.sum()
    src, dst = at[live & (at >= count)], at[~live & (at < count)]
    st["k_pages"][dst], st["v_pages"][dst] = st["k_pages"][src], st["v_pages"][src]
    st["refs"][dst] = st["refs"][src]
    st["refs"][src] = 0
    to = at.clone()
    to[src] = dst
    st["table"].copy_(torch.where(st["table"] >= 0, to[st["table"].clamp(min=0)], -1))


def _buffers(st):
    return [st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["refs"], st["status"]]


def _plain(st):
    kind = st["case"]["kind"]
    if kind in ("attend", "train"):
        return _plain_attend(st)
    if kind == "paged":
        return _plain_paged(st)
    if kind == "fork":
        _plain_fork(st, st["parents"], st["children"])
        _plain_append(st, st["children"], st["k_new"], st["v_new"], st["cu_new"])
        _plain_free(st, st["children"])
    else:
        _plain_free(st, st["odd"])
        _plain_compact(st)
        _plain_append(st, st["odd"], st["k_odd"], st["v_odd"], st["cu_odd"])
        _plain_free(st, st["even"])
        _plain_compact(st)
        _plain_append(st, st["even"], st["k_even"], st["v_even"], st["cu_even"])
    return _buffers(st)


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _own(st):
    import fast_memory_b200 as fm
    case = st["case"]
    kind = case["kind"]
    if kind in ("attend", "train"):
        how = dict(causal=case["causal"], window=case["window"], softcap=case["softcap"], slopes=st["slopes"], cu_seqlens_q=st["cu_q"],
                   cu_seqlens_k=st["cu_k"], prefix=st["prefix"])
        o, lse = fm.local_attention(st["q"], st["k"], st["v"], st["scale"], **how)
        if kind == "attend":
            return [o, lse]
        return [o, lse, *fm.local_attention_backward(st["q"], st["k"], st["v"], st["scale"], o, lse, st["d_out"], d_lse=st["d_lse"], **how)]
    cache = fm.PagedCache.over(st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["refs"], st["status"])
    if kind == "paged":
        return list(cache.attend(st["q"], st["scale"], cu_seqlens_q=st["cu_q"], window=case["window"], softcap=case["softcap"],
                                 slopes=st["slopes"], prefix=st["prefix"]))
    if kind == "fork":
        cache.fork(st["parents"], st["children"])
        cache.append(st["children"], st["k_new"], st["v_new"], cu_new=st["cu_new"])
        cache.free(st["children"])
    else:
        cache.free(st["odd"])
        cache.compact()
        cache.append(st["odd"], st["k_odd"], st["v_odd"], cu_new=st["cu_odd"])
        cache.free(st["even"])
        cache.compact()
        cache.append(st["even"], st["k_even"], st["v_even"], cu_new=st["cu_even"])
    return _buffers(st)


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    e = _SIZE[case["dtype"]]
    d, h, kind = case["d"], case["h"], case["kind"]
    if kind in ("attend", "train"):
        nq, nk = _doc_lengths(case)
        pairs, _ = _pairs(case, nq, nk, _prefixes(case, len(nq)))
        s, n, hq = int(nq.sum()), int(nk.sum()), case["hq"]
        rows, keys = hq * s * (d * e), h * n * (d * e)
        if kind == "attend":
            return {"bytes": 2 * rows + 2 * keys + 4 * hq * s, "flops": 4 * d * pairs * hq}
        # forward and backward as one pass: q, k, v and d_out in, o, lse and the three gradients out; two products forward,
        # five backward
        return {"bytes": 4 * rows + 4 * keys + (8 if case["d_lse"] else 4) * hq * s, "flops": 14 * d * pairs * hq}
    if kind == "paged":
        new, lengths = _seq_lengths(case)
        pairs, seen = _pairs(case, new, lengths, _prefixes(case, len(new)))
        rows = case["hq"] * int(new.sum())
        return {"bytes": 2 * rows * d * e + 4 * rows + 2 * h * seen * d * e, "flops": 4 * d * pairs * case["hq"]}
    lengths, new = _cycle_lengths(case)
    page, row = case["page"], 2 * h * d * e
    if kind == "fork":
        partial = sum(x % page for x in lengths)
        entries = sum(-(-(x + y) // page) for x, y in zip(lengths, new))
        return {"bytes": 2 * row * (partial + sum(new)) + 24 * entries, "flops": 0}
    pages = [-(-x // page) for x in new]
    low = min(sum(pages[0::2]), sum(pages[1::2]))
    return {"bytes": 2 * row * sum(new) + 2 * (2 * row * page * low) + 16 * sum(pages), "flops": 0}


# ---- from the definition, in 64 bits -------------------------------------------------------------------------------
def _exact_rows(case, q, k, v, scale, slope, prefix):
    """One head of one document: o and lse of q [n, d] over k, v [m, d], the queries being the last positions."""
    n, m = q.shape[0], k.shape[0]
    logits = torch.einsum("id,jd->ij", q, k) * scale
    if case["softcap"]:
        logits = case["softcap"] * torch.tanh(logits / case["softcap"])
    dist = torch.arange(m - n, m, device=q.device, dtype=torch.float64)[:, None] - torch.arange(m, device=q.device, dtype=torch.float64)
    if slope is not None:
        logits = logits - slope * dist.abs()
    w = case["window"] if case["window"] else float("inf")
    hidden = (dist >= w) | ((dist < 0) if case.get("causal", True) else (dist <= -w))
    if prefix:
        hidden[:, :prefix] = False
    lse = torch.logsumexp(logits.masked_fill(hidden, float("-inf")), -1)
    blind = hidden.all(-1)
    weights = torch.exp(logits - torch.where(blind, 0.0, lse)[:, None]).masked_fill(hidden, 0.0)
    return torch.einsum("ij,jd->id", weights, v), lse


def _exact_attend(case, st):
    g = case["hq"] // case["h"]
    train = case["kind"] == "train"
    q, k, v = (st[x].double().contiguous() for x in "qkv")
    o, lse = torch.zeros_like(q), torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    cq, ck = st["cu_q"].tolist(), st["cu_k"].tolist()
    for t in range(case["docs"]):
        a, b, x, y = cq[t], cq[t + 1], ck[t], ck[t + 1]
        prefix = 0 if st["prefix"] is None else int(st["prefix"][t])
        for i in range(case["hq"]):
            qi, ki, vi = (z.clone().requires_grad_(train) for z in (q[i, a:b], k[i // g, x:y], v[i // g, x:y]))
            slope = None if st["slopes"] is None else st["slopes"][i].double()
            oi, li = _exact_rows(case, qi, ki, vi, st["scale"], slope, prefix)
            o[i, a:b], lse[i, a:b] = oi.detach(), li.detach()
            if train:
                loss = (oi * st["d_out"][i, a:b].double()).sum()
                if st["d_lse"] is not None:
                    seen = torch.isfinite(li)
                    loss = loss + (li[seen] * st["d_lse"][i, a:b][seen].double()).sum()
                gq, gk, gv = torch.autograd.grad(loss, (qi, ki, vi))
                dq[i, a:b] = torch.nan_to_num(gq)
                dk[i // g, x:y] += torch.nan_to_num(gk)
                dv[i // g, x:y] += torch.nan_to_num(gv)
    return [o, lse, dq, dk, dv] if train else [o, lse]


def _exact_paged(case, st):
    g = case["hq"] // case["h"]
    q = st["q"].double()
    o, lse = torch.zeros_like(q), torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    cq, lengths, table = st["cu_q"].tolist(), st["lengths"].tolist(), st["table"].tolist()
    for t in range(case["seqs"]):
        a, b, n = cq[t], cq[t + 1], lengths[t]
        prefix = 0 if st["prefix"] is None else int(st["prefix"][t])
        used = [x for x in table[t] if x >= 0]
        for i in range(case["h"]):
            k, v = (torch.cat([st[z][x, i] for x in used])[:n].double() for z in ("k_pages", "v_pages"))
            for m in range(i * g, (i + 1) * g):
                slope = None if st["slopes"] is None else st["slopes"][m].double()
                o[m, a:b], lse[m, a:b] = _exact_rows(case, q[m, a:b], k, v, st["scale"], slope, prefix)
    return [o, lse]


class _Pool:
    """The page operations one page at a time, on host lists; the pages' rows follow by plain copies."""

    def __init__(self, st):
        self.k, self.v = st["k_pages"].double(), st["v_pages"].double()
        self.rows = [[x for x in r if x >= 0] for r in st["table"].tolist()]
        self.width = st["table"].shape[1]
        self.lengths, self.refs = st["lengths"].tolist(), st["refs"].tolist()
        self.page = self.k.shape[2]

    def take(self):
        at = self.refs.index(0)
        self.refs[at] = 1
        return at

    def fork(self, parent, child):
        n, rest = divmod(self.lengths[parent], self.page)
        self.rows[child] = self.rows[parent][:n]
        for x in self.rows[child]:
            self.refs[x] += 1
        if rest:
            new, old = self.take(), self.rows[parent][n]
            for z in (self.k, self.v):
                z[new, :, :rest] = z[old, :, :rest]
            self.rows[child].append(new)
        self.lengths[child] = self.lengths[parent]

    def append(self, seq, k, v):
        done, count = 0, k.shape[1]
        while len(self.rows[seq]) * self.page < self.lengths[seq] + count:
            self.rows[seq].append(self.take())
        while done < count:
            at, off = divmod(self.lengths[seq], self.page)
            n = min(self.page - off, count - done)
            for z, new in ((self.k, k), (self.v, v)):
                z[self.rows[seq][at], :, off:off + n] = new[:, done:done + n].double()
            done, self.lengths[seq] = done + n, self.lengths[seq] + n

    def free(self, seq):
        for x in self.rows[seq]:
            self.refs[x] -= 1
        self.rows[seq], self.lengths[seq] = [], 0

    def compact(self):
        count = sum(r > 0 for r in self.refs)
        holes = [x for x in range(count) if self.refs[x] == 0]
        moved = dict(zip([x for x in range(count, len(self.refs)) if self.refs[x] > 0], holes))
        for old, new in moved.items():
            self.refs[new], self.refs[old] = self.refs[old], 0
            for z in (self.k, self.v):
                z[new] = z[old]
        self.rows = [[moved.get(x, x) for x in r] for r in self.rows]

    def answer(self):
        table = torch.tensor([r + [-1] * (self.width - len(r)) for r in self.rows], dtype=torch.int32)
        return [self.k, self.v, table, torch.tensor(self.lengths, dtype=torch.int32), torch.tensor(self.refs, dtype=torch.int32), None]


def _exact_pages(case, st):
    pool = _Pool(st)

    def append(seqs, name):
        cu = st["cu_" + name].tolist()
        for i, x in enumerate(seqs):
            pool.append(x, st["k_" + name][:, cu[i]:cu[i + 1]], st["v_" + name][:, cu[i]:cu[i + 1]])

    if case["kind"] == "fork":
        children = st["children"].tolist()
        for x, y in zip(st["parents"].tolist(), children):
            pool.fork(x, y)
        append(children, "new")
        for x in children:
            pool.free(x)
    else:
        for name in ("odd", "even"):
            seqs = st[name].tolist()
            for x in seqs:
                pool.free(x)
            pool.compact()
            append(seqs, name)
    return pool.answer()


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("attend", "train"):
        return _exact_attend(case, st)
    return _exact_paged(case, st) if kind == "paged" else _exact_pages(case, st)
