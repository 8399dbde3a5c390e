// What the kernels of local attention share: the documents, which keys a query sees, where a key row lies (in a packed
// array or in the pages of a cache), and the one-row-at-a-time forms that every call can fall back on.
//
//   p = n_k - n_q + i                      position of query i of a document with n_q queries and n_k keys
//   s = scale q.k;  c = cap tanh(s / cap)  (cap > 0);  b = c - slope_head |p - j|
//   key j < n_k is visible iff  j < prefix  or  p - w < j <= p  (causal)  /  |p - j| < w  (not causal); w = 0: no bound
//   lse = log sum_j e^b,   o = sum_j e^(b - lse) v_j;   nothing visible: lse = -inf, o = 0
// The visible keys of a query are therefore at most two runs, [0, prefix) and a run around p, and the queries that see
// a key are one run: loops walk runs and never touch a hidden key or query.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "mma_utils.cuh"

namespace fm {

struct LocalParams {
    const void *q, *k, *v;
    int64_t q_sh, q_st, k_sh, k_st, v_sh, v_st;      // strides in elements: head, row
    int Hq, H, G, d;
    int S, N;                                        // packed query / key rows
    int n_docs;
    const int32_t *cu_q, *cu_k, *prefix;             // may be null: one document; a query each (paged); no prefix
    const float *slopes;
    float scale, cap;
    int window, causal;                              // window 0: unbounded
    const int32_t *table, *lengths, *seqs;           // paged: table != null
    int table_ld, page_shift, n_pages, n_seqs;
    void *o;
    float *lse;                                      // [Hq, S]
    // how long a pipeline wait may take before the CTA gives up and, a hook for the test of that path only, the tile of every CTA whose
    // load is left out (-1: none)
    uint64_t wait_ns;
    int skip_tile;
};

struct BwdParams {
    const void *dout;
    int64_t do_sh, do_st;
    const float *lse, *delta;                        // delta = rowsum(dO * O) - d_lse
    const float *range;                              // fp16 on the tensor cores: [Hq, S], how large a row's dP - delta gets; else null
    float *tops;                                     // and [Hq, S] for the largest of 32 rows of a query tile, at the first of them
    void *dq, *dk, *dv;                              // [Hq, S, d], [H, N, d] twice
};

struct Doc {
    int q0, nq, k0, nk, prefix, seq;
};

// Document t, with every number forced into its array: a wrong prefix array gives wrong results, never a wrong address.
// t = n_docs is what lies behind the last document: its queries see no key (KEYS false), its keys no query (KEYS true).
template <bool KEYS = false> __device__ __forceinline__ Doc local_doc(const LocalParams &p, int t)
{
    Doc D;
    const bool tail = t >= p.n_docs;
    if (p.cu_q) {
        D.q0 = t ? min(max(p.cu_q[t], 0), p.S) : 0;
        D.nq = (tail ? p.S : min(max(p.cu_q[t + 1], D.q0), p.S)) - D.q0;
    } else if (p.table) {
        D.q0 = min(t, p.S);
        D.nq = tail ? p.S - D.q0 : min(1, p.S - D.q0);
    } else {
        D.q0 = tail ? p.S : 0;
        D.nq = tail ? 0 : p.S;
    }
    D.seq = D.k0 = 0;
    if (p.table) {
        D.seq = tail ? 0 : min(max(p.seqs ? p.seqs[t] : t, 0), p.n_seqs - 1);
        D.nk = min(max(p.lengths[D.seq], 0), p.table_ld << p.page_shift);
    } else if (p.cu_k) {
        D.k0 = t ? min(max(p.cu_k[t], 0), p.N) : 0;
        D.nk = (tail ? p.N : min(max(p.cu_k[t + 1], D.k0), p.N)) - D.k0;
    } else {
        D.k0 = tail ? p.N : 0;
        D.nk = tail ? 0 : p.N;
    }
    if (tail) (KEYS ? D.nq : D.nk) = 0;
    D.prefix = p.prefix && !tail ? min(max(p.prefix[t], 0), D.nk) : 0;
    return D;
}

// Document that packed row r belongs to: the last t with cu[t] <= r.
__device__ __forceinline__ int local_find(const int32_t *__restrict__ cu, int n_docs, int r)
{
    int lo = 0, hi = n_docs + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= r) lo = mid; else hi = mid;
    }
    return lo;
}

// The run of keys around position pos: [lo, hi).  The prefix comes on top of it.
__device__ __forceinline__ int2 local_run(const LocalParams &p, int pos, int nk)
{
    const int lo = p.window ? max(pos - p.window + 1, 0) : 0;
    const int hi = p.causal ? pos + 1 : (p.window ? int(min(int64_t(pos) + p.window, int64_t(nk))) : nk);
    return make_int2(lo, min(hi, nk));
}

// The run of queries [lo, hi) of a document that see key j.
__device__ __forceinline__ int2 local_query_run(const LocalParams &p, const Doc &D, int j)
{
    if (j < D.prefix) return make_int2(0, D.nq);
    const int shift = D.nk - D.nq;
    const int64_t lo = p.causal ? j : (p.window ? int64_t(j) - p.window + 1 : int64_t(shift));
    const int64_t hi = p.window ? int64_t(j) + p.window : int64_t(shift) + D.nq;
    return make_int2(int(max(lo - shift, int64_t(0))), int(min(hi - shift, int64_t(D.nq))));
}

// Row of key j of document D and KV head h, in elements from the start of k (or v).
__device__ __forceinline__ int64_t local_key_row(const LocalParams &p, const Doc &D, int h, int j, int64_t sh, int64_t st)
{
    if (p.table) {
        const int page = min(max(p.table[int64_t(D.seq) * p.table_ld + (j >> p.page_shift)], 0), p.n_pages - 1);
        return (((int64_t(page) * p.H + h) << p.page_shift) + (j & ((1 << p.page_shift) - 1))) * p.d;
    }
    return int64_t(h) * sh + int64_t(D.k0 + j) * st;
}

// Elements of a row that a lane of a warp holds: lane, lane + 32, ...
template <typename T, int D> struct RowRegs {
    static constexpr int N = (D + 31) / 32;
    float x[N];
    __device__ __forceinline__ void load(const T *row)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (threadIdx.x & 31) + 32 * i;
            x[i] = c < D ? Elem<T>::to_f32(row[c]) : 0.f;
        }
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.f;
    }
    __device__ __forceinline__ void store(T *row, float f) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = (threadIdx.x & 31) + 32 * i;
            if (c < D) row[c] = Elem<T>::from_f32(x[i] * f);
        }
    }
    __device__ __forceinline__ float dot(const RowRegs &o) const
    {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(x[i], o.x[i], s);
#pragma unroll
        for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        return s;
    }
    __device__ __forceinline__ void axpy(float a, const RowRegs &o)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = fmaf(a, o.x[i], x[i]);
    }
};

// Score of a pair from its product, and the derivative of the cap.
__device__ __forceinline__ float local_score(const LocalParams &p, float qk, float slope, int dist, float &dcap)
{
    float s = qk * p.scale;
    dcap = 1.f;
    if (p.cap > 0.f) {
        const float t = tanhf(s / p.cap);
        s = t * p.cap;
        dcap = 1.f - t * t;
    }
    return s - slope * fabsf(float(dist));
}

// ---- one row by a warp: right for every type, size, stride and value ---------------------------------------------------
// Rows whose tensor-core result is not finite come here too: 0 * NaN of a hidden key is not theirs.  A row that turns out to be NaN as a
// whole ends there: after a diverged step every row comes here.
template <typename T, int DIM> __device__ __forceinline__ void local_row_forward(const LocalParams &p, const Doc &D, int head, int i)
{
    const int h = head / p.G, pos = D.nk - D.nq + i;
    const float slope = p.slopes ? p.slopes[head] : 0.f;
    RowRegs<T, DIM> q, k, acc;
    q.load(static_cast<const T *>(p.q) + int64_t(head) * p.q_sh + int64_t(D.q0 + i) * p.q_st);
    acc.zero();
    float m = -INFINITY, l = 0.f;
    const int2 run = local_run(p, pos, D.nk);
    for (int part = 0; part < 2; ++part) {
        const int lo = part ? max(run.x, D.prefix) : 0, hi = part ? run.y : D.prefix;
        for (int j = lo; j < hi; ++j) {
            float dcap;
            k.load(static_cast<const T *>(p.k) + local_key_row(p, D, h, j, p.k_sh, p.k_st));
            const float b = local_score(p, q.dot(k), slope, pos - j, dcap);
            k.load(static_cast<const T *>(p.v) + local_key_row(p, D, h, j, p.v_sh, p.v_st));
            if (b > m) {                                       // (a NaN score falls through and makes l and acc NaN)
                const float f = m == -INFINITY ? 0.f : expf(m - b);
                l *= f;
#pragma unroll
                for (int c = 0; c < RowRegs<T, DIM>::N; ++c) acc.x[c] *= f;
                m = b;
            }
            const float e = b == -INFINITY ? 0.f : expf(b - m);
            l += e;
            acc.axpy(e, k);
            if (l != l) part = 2, j = hi;                      // the row is NaN, whatever comes
        }
    }
    const int64_t row = int64_t(head) * p.S + D.q0 + i;
    acc.store(static_cast<T *>(p.o) + row * DIM, l == 0.f ? 0.f : 1.f / l);
    if ((threadIdx.x & 31) == 0) p.lse[row] = l == 0.f ? -INFINITY : m + logf(l);
}

// P and dS of one pair.
template <typename T, int DIM>
__device__ __forceinline__ float2 local_pair(const LocalParams &p, const RowRegs<T, DIM> &q, const RowRegs<T, DIM> &k, const RowRegs<T, DIM> &dout,
                                             const RowRegs<T, DIM> &v, float slope, int dist, float lse, float delta)
{
    float dcap;
    const float b = local_score(p, q.dot(k), slope, dist, dcap);
    const float w = expf(b - lse);
    return make_float2(w, w * (dout.dot(v) - delta) * dcap * p.scale);
}

template <typename T, int DIM> __device__ __forceinline__ void local_row_dq(const LocalParams &p, const BwdParams &g, const Doc &D, int head, int i)
{
    const int h = head / p.G, pos = D.nk - D.nq + i;
    const int64_t row = int64_t(head) * p.S + D.q0 + i;
    const float slope = p.slopes ? p.slopes[head] : 0.f, lse = g.lse[row], delta = g.delta[row];
    RowRegs<T, DIM> q, k, v, dout, acc;
    acc.zero();
    if (lse != -INFINITY) {
        q.load(static_cast<const T *>(p.q) + int64_t(head) * p.q_sh + int64_t(D.q0 + i) * p.q_st);
        dout.load(static_cast<const T *>(g.dout) + int64_t(head) * g.do_sh + int64_t(D.q0 + i) * g.do_st);
        const int2 run = local_run(p, pos, D.nk);
        for (int part = 0; part < 2; ++part) {
            const int lo = part ? max(run.x, D.prefix) : 0, hi = part ? run.y : D.prefix;
            for (int j = lo; j < hi; ++j) {
                k.load(static_cast<const T *>(p.k) + local_key_row(p, D, h, j, p.k_sh, p.k_st));
                v.load(static_cast<const T *>(p.v) + local_key_row(p, D, h, j, p.v_sh, p.v_st));
                const float ds = local_pair(p, q, k, dout, v, slope, pos - j, lse, delta).y;
                acc.axpy(ds, k);
                if (ds != ds) part = 2, j = hi;
            }
        }
    }
    acc.store(static_cast<T *>(g.dq) + row * DIM, 1.f);
}

template <typename T, int DIM> __device__ __forceinline__ void local_row_dkv(const LocalParams &p, const BwdParams &g, const Doc &D, int h, int j)
{
    RowRegs<T, DIM> q, k, v, dout, dk, dv;
    k.load(static_cast<const T *>(p.k) + local_key_row(p, D, h, j, p.k_sh, p.k_st));
    v.load(static_cast<const T *>(p.v) + local_key_row(p, D, h, j, p.v_sh, p.v_st));
    dk.zero();
    dv.zero();
    const int2 run = local_query_run(p, D, j);
    for (int head = h * p.G; head < (h + 1) * p.G; ++head) {
        const float slope = p.slopes ? p.slopes[head] : 0.f;
        for (int i = run.x; i < run.y; ++i) {
            const int64_t row = int64_t(head) * p.S + D.q0 + i;
            const float lse = g.lse[row];
            if (lse == -INFINITY) continue;
            q.load(static_cast<const T *>(p.q) + int64_t(head) * p.q_sh + int64_t(D.q0 + i) * p.q_st);
            dout.load(static_cast<const T *>(g.dout) + int64_t(head) * g.do_sh + int64_t(D.q0 + i) * g.do_st);
            const float2 pd = local_pair(p, q, k, dout, v, slope, D.nk - D.nq + i - j, lse, g.delta[row]);
            dv.axpy(pd.x, dout);
            dk.axpy(pd.y, q);
            if (pd.x != pd.x) head = (h + 1) * p.G, i = run.y;  // (then pd.y is NaN too)
        }
    }
    const int64_t row = int64_t(h) * p.N + D.k0 + j;
    dk.store(static_cast<T *>(g.dk) + row * DIM, 1.f);
    dv.store(static_cast<T *>(g.dv) + row * DIM, 1.f);
}

// The same as calls: what a kernel of few microseconds next to never does must not fill its instruction cache.
template <typename T, int DIM> __device__ __noinline__ void local_row_forward_call(const LocalParams &p, const Doc &D, int head, int i)
{
    local_row_forward<T, DIM>(p, D, head, i);
}
template <typename T, int DIM> __device__ __noinline__ void local_row_dkv_call(const LocalParams &p, const BwdParams &g, const Doc &D, int h, int j)
{
    local_row_dkv<T, DIM>(p, g, D, h, j);
}

// f(T{}) for an element type, f(T{}, std::integral_constant<int, D>{}) for an element type and a head dim
template <typename F> int with_type(int dtype, F &&f)
{
    if (dtype == FM_F32) return f(float{});
    if (dtype == FM_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}
template <typename F> int with_type_and_dim(int dtype, int d, F &&f)
{
    return with_type(dtype, [&](auto t) -> int {
        switch (d) {
        case 16: return f(t, std::integral_constant<int, 16>{});
        case 32: return f(t, std::integral_constant<int, 32>{});
        case 64: return f(t, std::integral_constant<int, 64>{});
        case 128: return f(t, std::integral_constant<int, 128>{});
        default: return f(t, std::integral_constant<int, 256>{});
        }
    });
}

// ---- backward a row a warp, head dim 256 ------------------------------------------------------------------------------------------
int local_rows_bwd(const LocalParams &p, const BwdParams &g, int dtype, cudaStream_t st);

}  // namespace fm
