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
