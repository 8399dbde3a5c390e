// What the tcgen05 kernels of local attention share: tile shapes, the list of key tiles of a block of queries, the loads of a
// key tile from a packed array or from pages, bounded waits, and the rank of a block among the documents.
#pragma once

#include "local_attn.cuh"
#include "tc_utils.cuh"

namespace fm {
namespace ltc {

constexpr int kTile = 128;                          // rows of a query tile = keys of a key tile = UMMA M = TMEM lanes
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// fp16 reaches from 2^-24 to 2^16 only: what is rounded to it is held times a power of two where it would leave that.
template <typename T> constexpr bool kNarrow = std::is_same<T, __half>::value;

// byte offset of column block c (64 elements) of a tile: [128 rows][128 bytes], 128-byte swizzle
constexpr uint32_t kBlock = kTile * 128;

__device__ __forceinline__ uint32_t bar_addr(const uint64_t *b) { return tc::smem_addr(b); }

// K-major operand of a tile: K step ks (16 elements)
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, int ks) { return tc::smem_desc_sw128(tile + uint32_t(ks >> 2) * kBlock + uint32_t(ks & 3) * 32u); }
// MN-major operand of a tile (the contraction runs over its ROWS): K step ks = rows 16 ks ..
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int ks) { return tc::smem_desc_mn_sw128(tile + uint32_t(ks) * 2048u, kBlock); }

// and what a K step adds to the descriptor of step 0
__host__ __device__ constexpr uint32_t step_k(int ks) { return (uint32_t(ks >> 2) * kBlock + uint32_t(ks & 3) * 32u) >> 4; }
__host__ __device__ constexpr uint32_t step_mn(int ks) { return uint32_t(ks) * 2048u >> 4; }

// ---- two fp32 numbers an instruction ------------------------------------------------------------------------------------
// A pair takes the FMA pipe as long as two single operations, but one issue slot.  (Moving part of the exponentials from the
// special-function unit, 16 a cycle and SM, to a polynomial on the FMA pipe was measured and made every kernel here slower: a
// pair costs 27 cycles of a scheduler's pipe that way, 16 on the special-function unit.)
typedef uint64_t f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b)
{
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ f32x2 pair(uint32_t a, uint32_t b) { return pair(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 split(f32x2 x)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ f32x2 exp2_pair(f32x2 x)
{
    const float2 v = split(x);
    return pair(fast_exp2(v.x), fast_exp2(v.y));
}

// tanh(k s) for |k s| <= 0.4: s (k + k^3 s^2 p(k^2 s^2)), p the polynomial of degree 2 of least relative error, 2e-7 in fp32.  k is
// multiplied into the coefficients: five operations a pair.
struct ShortTanh {
    f32x2 k, c0, c1, c2;
    __device__ __forceinline__ ShortTanh(float x)
    {
        const float x2 = x * x, x3 = x * x2, x5 = x3 * x2, x7 = x5 * x2;
        k = pair(x, x);
        c0 = pair(-0.333318823f * x3, -0.333318823f * x3);
        c1 = pair(0.13277629f * x5, 0.13277629f * x5);
        c2 = pair(-0.0477942206f * x7, -0.0477942206f * x7);
    }
    __device__ __forceinline__ f32x2 operator()(f32x2 s) const
    {
        const f32x2 u = mul2(s, s);
        return mul2(s, fma2(fma2(fma2(c2, u, c1), u, c0), u, k));
    }
};
// tanh x = 1 - 2 / (1 + e^2x): e^2x = inf gives 1, 0 gives -1.
__device__ __forceinline__ float tanh_far(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(x * (2.f * kLog2e))));
    return fmaf(-2.f, r, 1.f);
}
// Near 0 that difference is off by 1e-7 whatever x is, which the cap multiplies: there the polynomial.
__device__ __forceinline__ float tanh_any(float x)
{
    const float u = x * x, low = x * fmaf(fmaf(fmaf(-0.0477942206f, u, 0.13277629f), u, -0.333318823f), u, 1.f);
    return fabsf(x) <= 0.4f ? low : tanh_far(x);
}

// t = tanh(s k).  Which formula a score takes follows from that score alone: up to |s k| = 0.4 the short one, else tanh_any's.  A warp whose
// rows (valid: the lane holds one) all stay below does without the other; the bits are the same either way, so that nothing of another
// row and nothing hidden reaches a result.  Outside of [2^-18, 2^17] k's powers leave fp32's range: there the short one gets the
// product.  Scores are usually small against their cap.  More tiers, a shorter one up to 0.2 or a longer one up to 0.7,
// cost more in code than they save: chunked prompts 860 us, with this one alone 770.
__device__ __forceinline__ void cap_scores(f32x2 (&t)[16], const uint32_t (&s)[32], float k, bool valid)
{
    const bool folds = k >= 0x1p-18f && k <= 0x1p17f;
    float big[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 32; c += 2) big[c >> 1 & 1] = max3(big[c >> 1 & 1], fabsf(__uint_as_float(s[c])), fabsf(__uint_as_float(s[c + 1])));
    const float top = valid ? fmaxf(big[0], big[1]) * (folds ? k : INFINITY) : 0.f;
    const ShortTanh tanh_pair(folds ? k : 1.f);
    if (__all_sync(0xffffffffu, top <= 0.4f)) {
#pragma unroll
        for (int c = 0; c < 16; ++c) t[c] = tanh_pair(pair(s[2 * c], s[2 * c + 1]));
    } else {
        const float first = folds ? 1.f : k;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            asm volatile("" ::: "memory");                                     // a pair at a time: interleaved, this branch costs the usual one registers
            const float a = __uint_as_float(s[2 * c]), b = __uint_as_float(s[2 * c + 1]);
            const float2 low = split(tanh_pair(mul2(pair(a, b), pair(first, first))));
            t[c] = pair(fabsf(a * k) <= 0.4f ? low.x : tanh_far(a * k), fabsf(b * k) <= 0.4f ? low.y : tanh_far(b * k));
        }
    }
}

// 32 accumulator columns of a row, scaled and rounded, into a tile in shared memory (128-byte swizzle; dst: the tile, generic
// address) or straight to the row.  Returns false if one of them is not finite.  A thread's row written straight costs 32
// lines an instruction; through shared memory and a TMA store it costs four.
template <typename T> __device__ __forceinline__ bool put_row(const uint32_t (&o)[32], float f, unsigned char *tile, T *row_ptr, int row, int col)
{
    uint4 v[4];
    uint32_t *w = reinterpret_cast<uint32_t *>(v);
    float worst = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float a = __uint_as_float(o[2 * i]) * f, b = __uint_as_float(o[2 * i + 1]) * f;
        worst = fmaf(a, 0.f, fmaf(b, 0.f, worst));                             // NaN as soon as one is not finite
        w[i] = pack2<T>(a, b);
    }
    if (tile) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4 *>(tile + (col >> 6) * kBlock + row * 128 + ((((col & 63) >> 3) + i) ^ (row & 7)) * 16) = v[i];
    } else if (row_ptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<uint4 *>(row_ptr + col)[i] = v[i];
    }
    return worst == 0.f;
}

// A value that is the same in every lane, so that the compiler can see it.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Blocks of `per` rows, document by document (`KEYS`: of keys, else of queries): the document of block number `b` and which of its
// blocks that is (-1: there is no such block).  Called by one whole warp; every lane gets the answer.  Documents come, 32 at
// a time, in the order of what a block of theirs costs: blocks of keys by falling number of queries, blocks of queries by rising
// number of keys (they are handed out from the last one).  The grids have the KV head as their fastest index: then the long
// blocks of every head run first and the short ones fill the gaps at the end.  (One head after the other, 8192 tokens with a window of
// 4096 waited 13 % longer for the last key block, 8 % for the last query block.)
template <bool KEYS> __device__ __forceinline__ int find_block(const LocalParams &p, int per, int b, Doc &doc)
{
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int t0 = 0; t0 <= p.n_docs; t0 += 32) {
        const int t = t0 + lane;
        Doc D = {};
        if (t <= p.n_docs) D = local_doc<KEYS>(p, t);
        int n = ((KEYS ? D.nk : D.nq) + per - 1) / per, from = lane;             // from: the lane that has this place's document
        if (p.n_docs > 1) {
            const int cost = KEYS ? -D.nq : D.nk;
            int rank = 0;
#pragma unroll
            for (int l = 0; l < 32; ++l) {
                const int other = __shfl_sync(0xffffffffu, cost, l);
                rank += other < cost || (other == cost && l < lane);
            }
#pragma unroll
            for (int l = 0; l < 32; ++l)
                if (__shfl_sync(0xffffffffu, rank, l) == lane) from = l;
            n = __shfl_sync(0xffffffffu, n, from);
        }
        int s = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        const int total = __shfl_sync(0xffffffffu, s, 31);
        if (b < before + total) {
            const int at = __ffs(__ballot_sync(0xffffffffu, b < before + s)) - 1, l = __shfl_sync(0xffffffffu, from, at);
            doc.q0 = __shfl_sync(0xffffffffu, D.q0, l);
            doc.nq = __shfl_sync(0xffffffffu, D.nq, l);
            doc.k0 = __shfl_sync(0xffffffffu, D.k0, l);
            doc.nk = __shfl_sync(0xffffffffu, D.nk, l);
            doc.prefix = __shfl_sync(0xffffffffu, D.prefix, l);
            doc.seq = __shfl_sync(0xffffffffu, D.seq, l);
            return b - before - __shfl_sync(0xffffffffu, s - n, at);
        }
        before += total;
    }
    doc = Doc{};
    return -1;
}

}  // namespace ltc

// CUDA-core tiles: every type and head dim.
size_t local_simt_fwd_workspace(const LocalParams &p);
int local_simt_fwd(const LocalParams &p, int dtype, void *ws, cudaStream_t st);
int local_simt_bwd(const LocalParams &p, const BwdParams &g, int dtype, cudaStream_t st);
// Joins the parts [parts, Hq S, d], fp32 rows and their LSE, that a forward kernel left (local_attn.cu).
int local_combine(const LocalParams &p, int dtype, const float *part_o, const float *part_lse, int parts, cudaStream_t st);

// Whether a call goes to the tcgen05 kernels, their launches and tensor maps.
int local_query_map(CUtensorMap *map, const LocalParams &p, const void *q, int64_t sh, int64_t st, int dtype);
int local_key_map(CUtensorMap *map, const LocalParams &p, const void *k, int64_t sh, int64_t st, int dtype, int rows = ltc::kTile);
int local_tc_bwd(const LocalParams &p, const BwdParams &g, int dtype, float *parts, cudaStream_t st);
size_t local_tc_bwd_workspace(const LocalParams &p);        // of `parts`
int local_tc_fwd(const LocalParams &p, int dtype, void *ws, cudaStream_t st);
size_t local_tc_fwd_workspace(const LocalParams &p);
bool local_tc_fits(const LocalParams &p, int dtype);

// Few queries a document (mma.sync): the same for it.
bool local_decode_fits(const LocalParams &p, int dtype);
size_t local_decode_workspace(const LocalParams &p);
int local_decode_fwd(const LocalParams &p, int dtype, void *ws, cudaStream_t st);

}  // namespace fm
