// Local attention on the CUDA cores, fp32 arithmetic throughout: fp32 inputs, and the head dims the tensor-core kernels are not
// built for.  64 x 64 tiles in shared memory, 256 threads, 4 x 4 products a thread (4 x d/16 in the second products).  Bound by latency:
// two CTAs fit an SM (registers), 14 warps of them are there on average, and a tile's four barriers separate its loads from its
// products; the FMA pipe is at 34 % of its issue rate, with shared memory (8 16-byte loads for 64 FMAs) the next most waited for.
//
//   forward   block = 64 tokens of one head; a key tile: S = Q K^T, running maximum over 16 threads by shuffles, P through shared
//             memory, O += P V.  K and V take turns in one buffer, so that two or three CTAs of an SM cover each other's loads.
//             Sums over a tile are formed apart and then added: the rounding error of a long row grows with the square
//             root of (64 + tiles), not of all its keys.  Few blocks: key tiles are cut over blockIdx.y and joined by
//             local_combine, as in the tensor-core forward.
//   dQ        block = 64 tokens of one head over the key tiles;  dK, dV: block = 64 keys of one KV head over the query tiles of
//             every head of its group.  No atomics.
// Rows that are not the document's are zero in the tiles; results that are not finite are computed again a pair at a time.
// One head, fp32, d = 64, the last 512 of 4096 positions: 37 us a call, 28 of them here and 6 in the join (a warp a row and no tiles: 1880 us).
#include "local_attn.cuh"
#include "local_tc.cuh"

#include <type_traits>

namespace fm {

namespace {

constexpr int kB = 64;                              // rows of a tile
constexpr int kT = 256;
constexpr int kLdP = kB + 4;

template <int D> struct Lay {
    static constexpr int kLd = D + 4;               // floats a row: rows land four banks apart
    static constexpr int kTileF = kB * kLd;
    static constexpr int W = D >= 64 ? 4 : D / 16;  // consecutive columns of a thread in the second products
    static constexpr int M = D / (16 * W);          // and how many such pieces it has
};

template <typename T> __device__ __forceinline__ float4 load4(const T *p)
{
    if constexpr (std::is_same<T, float>::value) return *reinterpret_cast<const float4 *>(p);
    else {
        const uint2 raw = *reinterpret_cast<const uint2 *>(p);
        const T *e = reinterpret_cast<const T *>(&raw);
        return make_float4(Elem<T>::to_f32(e[0]), Elem<T>::to_f32(e[1]), Elem<T>::to_f32(e[2]), Elem<T>::to_f32(e[3]));
    }
}

// row(r): pointer of row r of the tile or null (zeros)
template <typename T, int D, typename F> __device__ __forceinline__ void load_tile(float *dst, F &&row)
{
#pragma unroll
    for (int x = threadIdx.x; x < kB * D / 4; x += kT) {
        const int r = x / (D / 4), c = x % (D / 4) * 4;
        const T *src = row(r);
        *reinterpret_cast<float4 *>(dst + r * Lay<D>::kLd + c) = src ? load4(src + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
}

// acc[i][j] = A[ty * 4 + i] . B[tx + 16 j]
template <int D> __device__ __forceinline__ void dot_tile(const float *A, const float *B, float (&acc)[4][4])
{
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll 4
    for (int k = 0; k < D; k += 4) {
        float4 a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4 *>(A + (ty * 4 + i) * Lay<D>::kLd + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4 *>(B + (tx + 16 * j) * Lay<D>::kLd + k);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[i][j] = fmaf(a[i].x, b[j].x, acc[i][j]);
                acc[i][j] = fmaf(a[i].y, b[j].y, acc[i][j]);
                acc[i][j] = fmaf(a[i].z, b[j].z, acc[i][j]);
                acc[i][j] = fmaf(a[i].w, b[j].w, acc[i][j]);
            }
    }
}

template <int W> __device__ __forceinline__ void load_w(float (&v)[W], const float *p)
{
    if constexpr (W == 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = p[i];
    }
}

// out[i][m][w] += sum_k P[ty * 4 + i][k] V[k][m * 16 W + tx W + w]; TRANS: P[k][ty * 4 + i]
template <int D, bool TRANS> __device__ __forceinline__ void accumulate_tile(const float *P, const float *V, float (&out)[4][Lay<D>::M][Lay<D>::W])
{
    constexpr int W = Lay<D>::W, M = Lay<D>::M;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll 2
    for (int k = 0; k < kB; k += 4) {
        float p[4][4];                              // [i][k]
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = *reinterpret_cast<const float4 *>(TRANS ? P + (k + i) * kLdP + ty * 4 : P + (ty * 4 + i) * kLdP + k);
            if (TRANS) { p[0][i] = f.x; p[1][i] = f.y; p[2][i] = f.z; p[3][i] = f.w; }
            else { p[i][0] = f.x; p[i][1] = f.y; p[i][2] = f.z; p[i][3] = f.w; }
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int m = 0; m < M; ++m) {
                float v[W];
                load_w<W>(v, V + (k + kk) * Lay<D>::kLd + m * 16 * W + tx * W);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int w = 0; w < W; ++w) out[i][m][w] = fmaf(p[i][kk], v[w], out[i][m][w]);
            }
    }
}

template <int D, typename F> __device__ __forceinline__ void each_column(F &&f)
{
    const int tx = threadIdx.x & 15;
#pragma unroll
    for (int m = 0; m < Lay<D>::M; ++m)
#pragma unroll
        for (int w = 0; w < Lay<D>::W; ++w) f(m, w, m * 16 * Lay<D>::W + tx * Lay<D>::W + w);
}

template <typename T, int D> struct Rows {
    const LocalParams &p;
    const Doc &doc;
    int h;
    __device__ __forceinline__ const T *key(const void *base, int64_t sh, int64_t st, int j) const
    {
        return j < doc.nk ? static_cast<const T *>(base) + local_key_row(p, doc, h, j, sh, st) : nullptr;
    }
};

// ltc::find_block for the whole CTA
template <bool KEYS> __device__ __forceinline__ int cta_block(const LocalParams &p, int b, Doc &doc)
{
    __shared__ Doc found;
    __shared__ int index;
    if (threadIdx.x < 32) {
        Doc d;
        const int i = ltc::find_block<KEYS>(p, kB, b, d);
        if (threadIdx.x == 0) { found = d; index = i; }
    }
    __syncthreads();
    doc = found;
    return index;
}

template <typename T, int D> constexpr int fwd_smem() { return (2 * Lay<D>::kTileF + kB * kLdP) * 4; }

template <typename T, int D>
__global__ void __launch_bounds__(kT) local_simt_fwd_kernel(const __grid_constant__ LocalParams p, float *part_o, float *part_lse)
{
    extern __shared__ __align__(16) float sm[];
    float *Q = sm, *KV = Q + Lay<D>::kTileF, *P = KV + Lay<D>::kTileF;
    __shared__ int bad[kB];
    constexpr int W = Lay<D>::W, M = Lay<D>::M;
    const int nb = gridDim.x / p.Hq, head = blockIdx.x / nb, h = head / p.G;
    Doc doc;
    const int index = cta_block<false>(p, nb - 1 - int(blockIdx.x % nb), doc);
    if (index < 0) return;
    const Rows<T, D> rows{p, doc, h};
    const int t0 = index * kB, t1 = min(t0 + kB, doc.nq), shift = doc.nk - doc.nq;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const float slope = p.slopes ? p.slopes[head] : 0.f;
    const T *qb = static_cast<const T *>(p.q) + int64_t(head) * p.q_sh;
    load_tile<T, D>(Q, [&](int r) { return t0 + r < t1 ? qb + int64_t(doc.q0 + t0 + r) * p.q_st : nullptr; });
    if (tid < kB) bad[tid] = 0;

    const int lo = local_run(p, shift + t0, doc.nk).x, hi = local_run(p, shift + t1 - 1, doc.nk).y;
    const int n_pre = (doc.prefix + kB - 1) / kB, first = max(lo / kB, n_pre);
    const int tiles = n_pre + (hi > lo ? max((hi + kB - 1) / kB - first, 0) : 0);
    const int n0 = int(int64_t(tiles) * blockIdx.y / gridDim.y), n1 = int(int64_t(tiles) * (blockIdx.y + 1) / gridDim.y);

    int2 run[4];
    float m[4], l[4], acc[4][M][W];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        run[i] = local_run(p, shift + t0 + ty * 4 + i, doc.nk);
        m[i] = -INFINITY;
        l[i] = 0.f;
        each_column<D>([&](int a, int b, int) { acc[i][a][b] = 0.f; });
    }
    for (int n = n0; n < n1; ++n) {
        const int j0 = (n < n_pre ? n : first + n - n_pre) * kB;
        __syncthreads();                             // the tile before has been read
        load_tile<T, D>(KV, [&](int r) { return rows.key(p.k, p.k_sh, p.k_st, j0 + r); });
        __syncthreads();
        float s[4][4], part[4][M][W];
        dot_tile<D>(Q, KV, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = j0 + tx + 16 * j;
                float dcap;
                s[i][j] = local_score(p, s[i][j], slope, shift + t0 + ty * 4 + i - key, dcap);
                if (!((key >= run[i].x && key < run[i].y) || key < doc.prefix)) s[i][j] = -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float mn = fmaxf(m[i], top), ref = mn == -INFINITY ? 0.f : mn, f = expf(m[i] - ref);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = expf(s[i][j] - ref);
                sum += s[i][j];
                P[(ty * 4 + i) * kLdP + tx + 16 * j] = s[i][j];
            }
            m[i] = mn;
            l[i] = fmaf(l[i], f, sum);               // this thread's columns; the 16 threads are added up at the end
            each_column<D>([&](int a, int b, int) { acc[i][a][b] *= f; part[i][a][b] = 0.f; });
        }
        __syncthreads();                             // K has been read, P is complete
        load_tile<T, D>(KV, [&](int r) { return rows.key(p.v, p.v_sh, p.v_st, j0 + r); });
        __syncthreads();
        accumulate_tile<D, false>(P, KV, part);
#pragma unroll
        for (int i = 0; i < 4; ++i) each_column<D>([&](int a, int b, int) { acc[i][a][b] += part[i][a][b]; });
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int o = 8; o; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
        const int token = t0 + ty * 4 + i;
        if (token >= t1) continue;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        const int64_t row = int64_t(head) * p.S + doc.q0 + token;
        float worst = l[i] * 0.f;
        if (gridDim.y == 1) {
            T *dst = static_cast<T *>(p.o) + row * D;
            each_column<D>([&](int a, int b, int c) {
                const float x = acc[i][a][b] * inv;
                worst = fmaf(x, 0.f, worst);
                dst[c] = Elem<T>::from_f32(x);
            });
        } else {
            float *dst = part_o + (int64_t(blockIdx.y) * p.Hq * p.S + row) * D;
            each_column<D>([&](int a, int b, int c) {
                const float x = acc[i][a][b] * inv;
                worst = fmaf(x, 0.f, worst);
                dst[c] = x;
            });
        }
        if (worst != 0.f) bad[ty * 4 + i] = 1;
        if (tx == 0 && gridDim.y == 1) p.lse[row] = l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
        if (tx == 0 && gridDim.y > 1) part_lse[int64_t(blockIdx.y) * p.Hq * p.S + row] = l[i] == 0.f ? -INFINITY : m[i] + logf(l[i]);
    }
    __syncthreads();
    if (gridDim.y == 1) {
        for (int r = tid >> 5; r < t1 - t0; r += kT / 32)
            if (bad[r]) local_row_forward<T, D>(p, doc, head, t0 + r);
    } else if (tid < t1 - t0 && bad[tid]) {
        part_lse[(int64_t(blockIdx.y) * p.Hq + head) * p.S + doc.q0 + t0 + tid] = __int_as_float(0x7fc00000);
    }
}

template <typename T, int D> constexpr int dq_smem() { return (4 * Lay<D>::kTileF + kB * kLdP) * 4; }

template <typename T, int D>
__global__ void __launch_bounds__(kT) local_simt_dq_kernel(const __grid_constant__ LocalParams p, const __grid_constant__ BwdParams g)
{
    extern __shared__ __align__(16) float sm[];
    float *Q = sm, *DO = Q + Lay<D>::kTileF, *K = DO + Lay<D>::kTileF, *V = K + Lay<D>::kTileF, *dS = V + Lay<D>::kTileF;
    __shared__ int bad[kB];
    constexpr int W = Lay<D>::W, M = Lay<D>::M;
    const int nb = gridDim.x / p.Hq, head = blockIdx.x / nb, h = head / p.G;
    Doc doc;
    const int index = cta_block<false>(p, nb - 1 - int(blockIdx.x % nb), doc);
    if (index < 0) return;
    const Rows<T, D> rows{p, doc, h};
    const int t0 = index * kB, t1 = min(t0 + kB, doc.nq), shift = doc.nk - doc.nq;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const float slope = p.slopes ? p.slopes[head] : 0.f;
    const T *qb = static_cast<const T *>(p.q) + int64_t(head) * p.q_sh, *db = static_cast<const T *>(g.dout) + int64_t(head) * g.do_sh;
    load_tile<T, D>(Q, [&](int r) { return t0 + r < t1 ? qb + int64_t(doc.q0 + t0 + r) * p.q_st : nullptr; });
    load_tile<T, D>(DO, [&](int r) { return t0 + r < t1 ? db + int64_t(doc.q0 + t0 + r) * g.do_st : nullptr; });
    if (tid < kB) bad[tid] = 0;
    const int lo = local_run(p, shift + t0, doc.nk).x, hi = local_run(p, shift + t1 - 1, doc.nk).y;
    const int n_pre = (doc.prefix + kB - 1) / kB, first = max(lo / kB, n_pre);
    const int tiles = n_pre + (hi > lo ? max((hi + kB - 1) / kB - first, 0) : 0);
    int2 run[4];
    float lse[4], delta[4], acc[4][M][W];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int token = t0 + ty * 4 + i;
        run[i] = make_int2(0, 0);
        lse[i] = INFINITY;
        delta[i] = 0.f;
        if (token < t1) {
            run[i] = local_run(p, shift + token, doc.nk);
            const float x = g.lse[int64_t(head) * p.S + doc.q0 + token];
            lse[i] = x == -INFINITY ? INFINITY : x;
            delta[i] = g.delta[int64_t(head) * p.S + doc.q0 + token];
        }
        each_column<D>([&](int a, int b, int) { acc[i][a][b] = 0.f; });
    }
    for (int n = 0; n < tiles; ++n) {
        const int j0 = (n < n_pre ? n : first + n - n_pre) * kB;
        __syncthreads();
        load_tile<T, D>(K, [&](int r) { return rows.key(p.k, p.k_sh, p.k_st, j0 + r); });
        load_tile<T, D>(V, [&](int r) { return rows.key(p.v, p.v_sh, p.v_st, j0 + r); });
        __syncthreads();
        float s[4][4], dp[4][4], part[4][M][W];
        dot_tile<D>(Q, K, s);
        dot_tile<D>(DO, V, dp);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = j0 + tx + 16 * j;
                float dcap;
                const float b = local_score(p, s[i][j], slope, shift + t0 + ty * 4 + i - key, dcap);
                const bool vis = (key >= run[i].x && key < run[i].y) || (key < doc.prefix && t0 + ty * 4 + i < t1);
                dS[(ty * 4 + i) * kLdP + tx + 16 * j] = vis ? expf(b - lse[i]) * (dp[i][j] - delta[i]) * dcap * p.scale : 0.f;
            }
            each_column<D>([&](int a, int b, int) { part[i][a][b] = 0.f; });
        }
        __syncthreads();
        accumulate_tile<D, false>(dS, K, part);
#pragma unroll
        for (int i = 0; i < 4; ++i) each_column<D>([&](int a, int b, int) { acc[i][a][b] += part[i][a][b]; });
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int token = t0 + ty * 4 + i;
        if (token >= t1) continue;
        T *dst = static_cast<T *>(g.dq) + (int64_t(head) * p.S + doc.q0 + token) * D;
        float worst = 0.f;
        each_column<D>([&](int a, int b, int c) {
            worst = fmaf(acc[i][a][b], 0.f, worst);
            dst[c] = Elem<T>::from_f32(acc[i][a][b]);
        });
        if (worst != 0.f) bad[ty * 4 + i] = 1;
    }
    __syncthreads();
    for (int r = tid >> 5; r < t1 - t0; r += kT / 32)
        if (bad[r]) local_row_dq<T, D>(p, g, doc, head, t0 + r);
}

template <typename T, int D> constexpr int dkv_smem() { return (4 * Lay<D>::kTileF + 2 * kB * kLdP) * 4; }

template <typename T, int D>
__global__ void __launch_bounds__(kT) local_simt_dkv_kernel(const __grid_constant__ LocalParams p, const __grid_constant__ BwdParams g)
{
    extern __shared__ __align__(16) float sm[];
    float *Q = sm, *DO = Q + Lay<D>::kTileF, *K = DO + Lay<D>::kTileF, *V = K + Lay<D>::kTileF, *P = V + Lay<D>::kTileF, *dS = P + kB * kLdP;
    __shared__ int bad[kB];
    constexpr int W = Lay<D>::W, M = Lay<D>::M;
    const int nb = gridDim.x / p.H, h = blockIdx.x / nb;
    Doc doc;
    const int index = cta_block<true>(p, blockIdx.x % nb, doc);
    if (index < 0) return;
    const Rows<T, D> rows{p, doc, h};
    const int j0 = index * kB, j1 = min(j0 + kB, doc.nk), shift = doc.nk - doc.nq;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    load_tile<T, D>(K, [&](int r) { return rows.key(p.k, p.k_sh, p.k_st, j0 + r); });
    load_tile<T, D>(V, [&](int r) { return rows.key(p.v, p.v_sh, p.v_st, j0 + r); });
    if (tid < kB) bad[tid] = 0;
    int2 span = make_int2(local_query_run(p, doc, j0).x, local_query_run(p, doc, j1 - 1).y);
    if (j0 < doc.prefix) span = make_int2(0, doc.nq);
    int2 run[4];                                     // of this thread's key columns
    float dk[4][M][W], dv[4][M][W];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int key = j0 + tx + 16 * j;
        run[j] = key < j1 ? local_query_run(p, doc, key) : make_int2(0, 0);
        each_column<D>([&](int a, int b, int) { dk[j][a][b] = dv[j][a][b] = 0.f; });
    }
    for (int head = h * p.G; head < (h + 1) * p.G; ++head) {
        const float slope = p.slopes ? p.slopes[head] : 0.f;
        const T *qb = static_cast<const T *>(p.q) + int64_t(head) * p.q_sh, *db = static_cast<const T *>(g.dout) + int64_t(head) * g.do_sh;
        for (int t0 = span.x / kB * kB; t0 < span.y; t0 += kB) {
            __syncthreads();
            load_tile<T, D>(Q, [&](int r) { return t0 + r < doc.nq ? qb + int64_t(doc.q0 + t0 + r) * p.q_st : nullptr; });
            load_tile<T, D>(DO, [&](int r) { return t0 + r < doc.nq ? db + int64_t(doc.q0 + t0 + r) * g.do_st : nullptr; });
            __syncthreads();
            float s[4][4], dp[4][4], part[4][M][W];
            dot_tile<D>(Q, K, s);
            dot_tile<D>(DO, V, dp);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int token = t0 + ty * 4 + i;
                float lse = INFINITY, delta = 0.f;
                if (token < doc.nq) {
                    const float x = g.lse[int64_t(head) * p.S + doc.q0 + token];
                    lse = x == -INFINITY ? INFINITY : x;
                    delta = g.delta[int64_t(head) * p.S + doc.q0 + token];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float dcap;
                    const float b = local_score(p, s[i][j], slope, shift + token - (j0 + tx + 16 * j), dcap);
                    const bool vis = token >= run[j].x && token < run[j].y;
                    const float w = vis ? expf(b - lse) : 0.f;
                    P[(ty * 4 + i) * kLdP + tx + 16 * j] = w;
                    dS[(ty * 4 + i) * kLdP + tx + 16 * j] = vis ? w * (dp[i][j] - delta) * dcap * p.scale : 0.f;
                }
                each_column<D>([&](int a, int b, int) { part[i][a][b] = 0.f; });
            }
            __syncthreads();
            accumulate_tile<D, true>(P, DO, part);
#pragma unroll
            for (int i = 0; i < 4; ++i) each_column<D>([&](int a, int b, int) { dv[i][a][b] += part[i][a][b]; part[i][a][b] = 0.f; });
            accumulate_tile<D, true>(dS, Q, part);
#pragma unroll
            for (int i = 0; i < 4; ++i) each_column<D>([&](int a, int b, int) { dk[i][a][b] += part[i][a][b]; });
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int key = j0 + ty * 4 + i;
        if (key >= j1) continue;
        const int64_t row = (int64_t(h) * p.N + doc.k0 + key) * D;
        float worst = 0.f;
        each_column<D>([&](int a, int b, int c) {
            worst = fmaf(dk[i][a][b], 0.f, fmaf(dv[i][a][b], 0.f, worst));
            static_cast<T *>(g.dk)[row + c] = Elem<T>::from_f32(dk[i][a][b]);
            static_cast<T *>(g.dv)[row + c] = Elem<T>::from_f32(dv[i][a][b]);
        });
        if (worst != 0.f) bad[ty * 4 + i] = 1;
    }
    __syncthreads();
    for (int r = tid >> 5; r < j1 - j0; r += kT / 32)
        if (bad[r]) local_row_dkv<T, D>(p, g, doc, h, j0 + r);
}

int64_t blocks_of(int64_t rows, int64_t docs) { return std::min<int64_t>(rows, (rows + docs * (kB - 1)) / kB); }

struct Shape {
    int64_t blocks;
    int parts;
};
// As in the tensor-core forward: key tiles are cut where the blocks fill less than half of the chip.
Shape shape_of(const LocalParams &p)
{
    Shape s{blocks_of(p.S, p.n_docs + (p.cu_q ? 1 : 0)) * p.Hq, 1};
    int64_t keys = p.table ? int64_t(p.table_ld) << p.page_shift : p.N;
    if (p.window && !p.prefix) keys = std::min<int64_t>(keys, int64_t(p.window) * (p.causal ? 1 : 2) + kB);
    const int64_t slots = 2 * sm_count();
    if (s.blocks > 0 && s.blocks * 2 <= slots) s.parts = int(std::max<int64_t>(1, std::min<int64_t>(slots / s.blocks, ceil_div(keys, kB) / 2)));
    return s;
}

template <typename T, int D> int fwd(const LocalParams &p, void *ws, cudaStream_t st)
{
    const Shape s = shape_of(p);
    float *part_lse = static_cast<float *>(ws), *part_o = part_lse + (size_t(s.parts) * p.Hq * p.S + 31) / 32 * 32;
    FM_CUDA_OK(func_attr_cached((const void *)local_simt_fwd_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, fwd_smem<T, D>()));
    local_simt_fwd_kernel<T, D><<<dim3(unsigned(s.blocks), unsigned(s.parts)), kT, fwd_smem<T, D>(), st>>>(p, part_o, part_lse);
    FM_LAUNCHED("local_simt_fwd_kernel");
    return s.parts > 1 ? local_combine(p, Elem<T>::id, part_o, part_lse, s.parts, st) : FM_OK;
}

template <typename T, int D> int bwd(const LocalParams &p, const BwdParams &g, cudaStream_t st)
{
    if (p.S > 0) {
        FM_CUDA_OK(func_attr_cached((const void *)local_simt_dq_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, dq_smem<T, D>()));
        local_simt_dq_kernel<T, D><<<unsigned(blocks_of(p.S, p.n_docs + (p.cu_q ? 1 : 0)) * p.Hq), kT, dq_smem<T, D>(), st>>>(p, g);
        FM_LAUNCHED("local_simt_dq_kernel");
    }
    if (p.N > 0) {
        FM_CUDA_OK(func_attr_cached((const void *)local_simt_dkv_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, dkv_smem<T, D>()));
        local_simt_dkv_kernel<T, D><<<unsigned(blocks_of(p.N, p.n_docs + (p.cu_k ? 1 : 0)) * p.H), kT, dkv_smem<T, D>(), st>>>(p, g);
        FM_LAUNCHED("local_simt_dkv_kernel");
    }
    return FM_OK;
}

}  // namespace

size_t local_simt_fwd_workspace(const LocalParams &p)
{
    const Shape s = shape_of(p);
    return s.parts > 1 ? (size_t(s.parts) * p.Hq * p.S * (p.d + 1) + 64) * sizeof(float) : 0;
}

int local_simt_fwd(const LocalParams &p, int dtype, void *ws, cudaStream_t st)
{
    return with_type_and_dim(dtype, p.d, [&](auto t, auto dim) { return fwd<decltype(t), decltype(dim)::value>(p, ws, st); });
}

int local_simt_bwd(const LocalParams &p, const BwdParams &g, int dtype, cudaStream_t st)
{
    return with_type_and_dim(dtype, p.d, [&](auto t, auto dim) -> int {
        using T = decltype(t);
        constexpr int D = decltype(dim)::value;
        if constexpr (D <= 128) return bwd<T, D>(p, g, st);
        else return local_rows_bwd(p, g, Elem<T>::id, st);       // four tiles of 256 columns do not fit an SM
    });
}

}  // namespace fm
