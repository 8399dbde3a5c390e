"""Local attention from its definition in 64 bits, with bounds on what a 32-bit / 16-bit computation of it may be off by.

Bounds.  u = eps / 2 of the element type (one rounding), e = 2^-23 (one fp32 operation of a tensor core, which may truncate).
A score is a sum of d products: off by at most  delta = d e scale max(|q|.|k|) + 2^-20 (1 + largest |score|)  (the second part:
scaling, cap, distance, exponent).  A softmax weight is then off by a factor 1 +- 2 delta, and by u where it is rounded to the
element type as the operand of the second product; n summands add n e of the sum of their magnitudes; results are rounded
once (u).  In fp16 a rounded weight below 2^-14 is off by up to 2^-25 absolutely.  Each function below adds these up."""
import torch

E = 2.0 ** -23


def visible(nq, nk, causal, window, prefix, device):
    p = (torch.arange(nq, device=device) + (nk - nq))[:, None]
    j = torch.arange(nk, device=device)[None, :]
    near = (j <= p) if causal else torch.ones(nq, nk, dtype=torch.bool, device=device)
    if window:
        near = near & ((p - j).abs() < window)
    return near | (j < prefix), (p - j).abs().double()


class Case:
    """One call: tensors on the device, options, and the documents as host lists."""

    def __init__(self, dtype=torch.bfloat16, hq=2, h=1, d=64, nq=(100,), nk=None, causal=True, window=0, softcap=0.0, slopes=False, prefix=None,
                 token_major=False, seed=0, scale=None, tail=0):
        g = torch.Generator().manual_seed(seed)
        self.nq, self.nk = list(nq), list(nk if nk is not None else nq)
        self.hq, self.h, self.d, self.dtype = hq, h, d, dtype
        S, N = sum(self.nq) + tail, sum(self.nk) + tail

        def rows(heads, n):
            if token_major:
                return torch.randn(n, heads, d, generator=g).to(dtype).cuda().transpose(0, 1)
            return torch.randn(heads, n, d, generator=g).to(dtype).cuda()

        self.q, self.k, self.v, self.d_out = rows(hq, S), rows(h, N), rows(h, N), rows(hq, S)
        self.d_lse = torch.randn(hq, S, generator=g).cuda()
        self.scale = d ** -0.5 if scale is None else scale
        cu = lambda ns: [sum(ns[:i]) for i in range(len(ns) + 1)]
        self.cq, self.ck = cu(self.nq), cu(self.nk)
        self.prefix = list(prefix) if prefix is not None else None
        self.opts = dict(causal=causal, window=window, softcap=softcap)
        self.slopes = torch.tensor([2.0 ** (-4.0 * (i + 1) / hq) for i in range(hq)]).cuda() if slopes else None

    def kwargs(self, plain=False):
        """``plain``: without prefix sums, where there is one document and no tail."""
        kw = dict(self.opts, slopes=self.slopes)
        if not plain:
            kw["cu_seqlens_q"] = torch.tensor(self.cq, dtype=torch.int32, device="cuda")
            kw["cu_seqlens_k"] = torch.tensor(self.ck, dtype=torch.int32, device="cuda")
        if self.prefix is not None:
            kw["prefix"] = torch.tensor(self.prefix, dtype=torch.int32, device="cuda")
        return kw

    def blocks(self):
        """(document's mask, distances, query slice, key slice) per document"""
        for t in range(len(self.nq)):
            pre = self.prefix[t] if self.prefix is not None else 0
            m, dist = visible(self.nq[t], self.nk[t], self.opts["causal"], self.opts["window"], pre, self.q.device)
            yield m, dist, slice(self.cq[t], self.cq[t + 1]), slice(self.ck[t], self.ck[t + 1])

    def _scores(self, i, q, k, mask, dist):
        s = (q @ k.T) * self.scale
        mag = (q.abs() @ k.abs().T) * abs(self.scale)
        dcap = torch.ones_like(s)
        cap = self.opts["softcap"]
        if cap:
            t = torch.tanh(s / cap)
            s, dcap = cap * t, 1 - t * t
        if self.slopes is not None:
            s = s - self.slopes[i].double() * dist
        seen = s[mask]
        big = float(seen.abs().max()) if seen.numel() else 0.0
        delta = self.d * E * (float(mag[mask].max()) if seen.numel() else 0.0) + 2.0 ** -20 * (1 + big + cap)
        return s, dcap, delta

    @property
    def u(self):
        return torch.finfo(self.dtype).eps / 2

    def tiny(self, n):
        return n * 2.0 ** -25 if self.dtype == torch.float16 else 0.0

    def forward(self):
        """(o, lse, bound on o, bound on lse) in 64 bits"""
        o = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        lse = torch.full(self.q.shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
        to, tl = torch.zeros_like(o), torch.zeros_like(lse)
        for mask, dist, a, b in self.blocks():
            for i in range(self.hq):
                q, k, v = self.q[i, a].double(), self.k[i // (self.hq // self.h), b].double(), self.v[i // (self.hq // self.h), b].double()
                s, _, delta = self._scores(i, q, k, mask, dist)
                s = s.masked_fill(~mask, float("-inf"))
                l = torch.logsumexp(s, -1) if s.shape[1] else lse[i, a]
                w = torch.exp(s - torch.where(torch.isinf(l), 0.0, l)[:, None]).masked_fill(~mask, 0.0)
                o[i, a], lse[i, a] = w @ v, l
                n = s.shape[1]
                vmax = float(v.abs().max()) if n else 0.0
                to[i, a] = (2 * self.u + 4 * delta + n * E) * (w @ v.abs()) + self.tiny(n) * vmax + 1e-30
                tl[i, a] = 2 * delta + n * E + 2.0 ** -20 * (1 + torch.nan_to_num(l, neginf=0.0).abs())
        return o, lse, to, tl

    def backward(self, out, lse, d_lse=None):
        """Gradients by the formulas for the given (out, lse), and their bounds."""
        z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
        dq, dk, dv, tq, tk, tv = z(self.q), z(self.k), z(self.v), z(self.q), z(self.k), z(self.v)
        for mask, dist, a, b in self.blocks():
            for i in range(self.hq):
                m = i // (self.hq // self.h)
                q, k, v, g, o = (x.double() for x in (self.q[i, a], self.k[m, b], self.v[m, b], self.d_out[i, a], out[i, a]))
                s, dcap, delta = self._scores(i, q, k, mask, dist)
                l = lse[i, a].double()
                p = torch.exp(s - torch.where(torch.isinf(l), 0.0, l)[:, None]).masked_fill(~mask | torch.isinf(l)[:, None], 0.0)
                D = (g * o).sum(-1) - (0 if d_lse is None else d_lse[i, a].double())
                ds = p * (g @ v.T - D[:, None]) * dcap * self.scale
                mag = p * abs(self.scale) * (g.abs() @ v.abs().T + ((g * o).abs().sum(-1) + (0 if d_lse is None else d_lse[i, a].double().abs()))[:, None])
                delta = delta + 2.0 ** -20 * (1 + float(torch.nan_to_num(l, neginf=0.0).abs().max()) if l.numel() else 0.0)
                es = self.u * ds.abs() + mag * (2 * delta + 2 * self.d * E)
                ep = p * (self.u + 2 * delta)
                nq, nk = s.shape
                gr = self.hq // self.h
                dq[i, a] = ds @ k
                tq[i, a] = (es + ds.abs() * nk * E) @ k.abs() + self.tiny(nk) * float(k.abs().max() if nk else 0) + 1e-30
                dk[m, b] += ds.T @ q
                tk[m, b] += (es + ds.abs() * nq * gr * E).T @ q.abs() + self.tiny(nq) * float(q.abs().max() if nq else 0) + 1e-30
                dv[m, b] += p.T @ g
                tv[m, b] += (ep + p * nq * gr * E).T @ g.abs() + self.tiny(nq) * float(g.abs().max() if nq else 0) + 1e-30
        return [(x, t + self.u * x.abs()) for x, t in ((dq, tq), (dk, tk), (dv, tv))]


def assert_within(got, want, bound, name):
    got = got.double()
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf), f"{name}: infinite elsewhere"
    assert not torch.isnan(got).any(), f"{name}: NaN"
    err = torch.where(inf, 0.0, (torch.where(inf, 0.0, got) - torch.where(inf, 0.0, want)).abs())
    over = err - bound
    if over.numel():
        at = int(over.argmax())
        assert over.max() <= 0, f"{name}: off by {float(err.flatten()[at]):.3g} where {float(bound.flatten()[at]):.3g} is allowed (element {at})"
