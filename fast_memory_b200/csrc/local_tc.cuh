// What the tcgen05 kernels of local attention share: tile shapes, the list of key tiles of a block of queries, the loads of a
// key tile from a packed array or from pages, bounded waits, and the rank of a block among the documents.
#pragma once

#include "local_attn.cuh"
#include "tc_utils.cuh"

namespace fm {
namespace ltc {

constexpr int kTile = 128;                          // rows of a query tile = keys of a key tile = UMMA M = TMEM lanes
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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
// The softmax of a tile is issue-bound unless its arithmetic goes two scores at a time, and bound by the special-function unit
// (16 exponentials a cycle and SM: 1024 cycles a tile, as long as two of its products) unless some of its exponentials go
// to the FMA pipe.
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

__device__ __forceinline__ f32x2 exp2_sfu(f32x2 x)
{
    const float2 v = split(x);
    return pair(fast_exp2(v.x), fast_exp2(v.y));
}

// 2^x on the FMA pipe, x <= 120: x = n + f with n the nearest whole number (the sum with 1.5 2^23 holds it in its low bits),
// 2^f by the degree-5 polynomial of least relative error on [-1/2, 1/2] (7e-8; 2.4e-7 with fp32 rounding), n added to the
// exponent.  x is cut at -126: no exact zeros come out of this one.
__device__ __forceinline__ f32x2 exp2_fma(f32x2 x)
{
    const float2 v = split(x);
    const f32x2 y = pair(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
    const f32x2 t = add2(y, pair(12582912.f, 12582912.f));
    const f32x2 f = add2(y, mul2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f)));
    f32x2 q = fma2(f, pair(1.32917648e-3f, 1.32917648e-3f), pair(9.67562478e-3f, 9.67562478e-3f));
    q = fma2(q, f, pair(5.55065386e-2f, 5.55065386e-2f));
    q = fma2(q, f, pair(2.40221202e-1f, 2.40221202e-1f));
    q = fma2(q, f, pair(6.93147004e-1f, 6.93147004e-1f));
    q = fma2(q, f, pair(1.f, 1.f));
    const float2 a = split(q), b = split(t);
    return pair(__float_as_uint(a.x) + (__float_as_uint(b.x) << 23), __float_as_uint(a.y) + (__float_as_uint(b.y) << 23));
}

// Exponential of score pair i of a row; MIX: three of eight go to the FMA pipe.
template <bool MIX> __device__ __forceinline__ f32x2 exp2_pair(f32x2 x, int i)
{
    if (MIX && (i & 7) >= 5) return exp2_fma(x);
    return exp2_sfu(x);
}

// tanh of a pair, |x| <= 0.7: x + x^3 p(x^2), p of degree 4 with the least error on that range (5e-8 in fp32).
constexpr float kTanhRange = 0.7f;
__device__ __forceinline__ f32x2 tanh_small(f32x2 x)
{
    const f32x2 u = mul2(x, x);
    f32x2 q = fma2(u, pair(-5.13866311e-3f, -5.13866311e-3f), pair(2.00919714e-2f, 2.00919714e-2f));
    q = fma2(q, u, pair(-5.35588600e-2f, -5.35588600e-2f));
    q = fma2(q, u, pair(1.33291110e-1f, 1.33291110e-1f));
    q = fma2(q, u, pair(-3.33331913e-1f, -3.33331913e-1f));
    return fma2(mul2(x, u), q, x);
}
// tanh x = 1 - 2 / (1 + e^2x): e^2x = inf gives 1, 0 gives -1
__device__ __forceinline__ float tanh_any(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(x * (2.f * kLog2e))));
    return fmaf(-2.f, r, 1.f);
}

// A value that is the same in every lane, so that the compiler can see it.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Blocks of `per` rows, document by document (`KEYS`: of keys, else of queries): which document and which block of it is
// block number `b`?  Called by one whole warp; .x = document (n_docs: the tail), .y = block; .x = -1: there is no such block.
template <bool KEYS> __device__ __forceinline__ int2 find_block(const LocalParams &p, int per, int b)
{
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int t0 = 0; t0 <= p.n_docs; t0 += 32) {
        const int t = t0 + lane;
        int n = 0;
        if (t <= p.n_docs) {
            const Doc D = local_doc<KEYS>(p, t);
            n = ((KEYS ? D.nk : D.nq) + per - 1) / per;
        }
        int s = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        const int total = __shfl_sync(0xffffffffu, s, 31);
        if (b < before + total) {
            const unsigned m = __ballot_sync(0xffffffffu, b < before + s);
            const int l = __ffs(m) - 1;
            const int first = before + __shfl_sync(0xffffffffu, s - n, l);
            return make_int2(t0 + l, b - first);
        }
        before += total;
    }
    return make_int2(-1, 0);
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
int local_key_map(CUtensorMap *map, const LocalParams &p, const void *k, int64_t sh, int64_t st, int dtype);
int local_tc_bwd(const LocalParams &p, const BwdParams &g, int dtype, cudaStream_t st);
int local_tc_fwd(const LocalParams &p, int dtype, void *ws, cudaStream_t st);
size_t local_tc_fwd_workspace(const LocalParams &p);
bool local_tc_fits(const LocalParams &p, int dtype);

}  // namespace fm
