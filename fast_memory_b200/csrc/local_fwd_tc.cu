// Local attention forward on the 5th-generation tensor cores, 16-bit types, head dim 64 or 128.
//
// A CTA owns two query tiles of 128 rows - row = (token, head of the group), so that a tile reads its KV head's keys once for
// the whole group - and streams the key tiles that either of them sees:
//     S [128 x 128] = Q K^T        A = Q, B = K, both K-major in shared memory (TMA, 128-byte swizzle); fp32 in TMEM
//     P = 2^(s - m)                thread = row: 128 scores in registers, running maximum m and sum l, no shuffles;
//                                  P goes back to TMEM over S as packed 16-bit: the A operand of the second product
//     O [128 x d] += P V           B = V, the same tile layout read MN-major; fp32 in TMEM (S0 S1 O0 O1 = 512 columns)
// The two tiles take turns: while one's 128 threads do a softmax, the tensor core works for the other.  m is only moved when a
// row's maximum has grown by more than 2^8 (the sums are fp32 and P is a floating-point number: a late reference costs no
// accuracy), so O is rescaled in TMEM a few times a row instead of once a tile.
// l sums the unrounded p; P is rounded to the element type because the second product takes 16-bit operands.
//
//   warps 0-3, 4-7   softmax and epilogue of tile 0, 1 (a warp reaches its own quarter of the TMEM lanes)
//   warp 8           one thread issues all products
//   warp 9           TMA: query tiles, then K and V tiles through one ring; a paged tile is one box a page, its addresses looked
//                    up by the lanes side by side.  Rows behind the document's last key are zeroed in the V tile: they would
//                    meet P = 0, and 0 * NaN is NaN
// A hidden key INSIDE the document can still hold a NaN value.  It shows as a result that is not finite; such rows are computed
// again, one key at a time (local_row_forward).  The same happens to all rows of a CTA whose pipeline wait gave up.
//
// Few blocks (a chunk over a long cache): the key tiles of a block are cut over blockIdx.y; the parts leave normalised partial
// rows and their LSE in the workspace, and local_combine joins them.
#include "local_tc.cuh"

namespace fm {

namespace {

using namespace ltc;

constexpr int kThreads = 384;
constexpr int kMmaWarp = 8, kLoadWarp = 9;        // warps 10 and 11 complete the third warpgroup: registers are split by warpgroup
constexpr float kLazy = 8.f;                        // how far (log2) a row maximum may outgrow the reference before O is rescaled

template <int D> struct Cfg {
    static constexpr uint32_t kTileBytes = uint32_t(D / 64) * kBlock;
    static constexpr int kRing = D == 128 ? 5 : 8;  // K and V tiles in flight or in use
    static constexpr uint32_t kSmem = (2 + kRing) * kTileBytes + 1024;
};

struct Block {
    Doc D;
    int h, tokens;                                  // KV head; tokens of a query tile
    int t0[2], t1[2];                               // tokens of each tile in the document, [t0, t1)
    int lo[2], hi[2];                               // key tiles of each tile behind the prefix's, [lo, hi)
    int n_pre, lo0;                                 // key tiles of the prefix; first one behind them that any tile sees
    int n0, n1;                                     // this CTA's part of the list
    __device__ __forceinline__ int key_tile(int n) const { return n < n_pre ? n : lo0 + n - n_pre; }
    __device__ __forceinline__ bool active(int s, int n) const
    {
        const int kt = key_tile(n);
        return t0[s] < t1[s] && (n < n_pre || (kt >= lo[s] && kt < hi[s]));
    }
};

template <int D> struct Shared {
    uint64_t q_full[2], full[Cfg<D>::kRing], empty[Cfg<D>::kRing], tail;
    uint64_t s_full[2], p_full[2], o_done[2], drain;
    uint32_t tmem_slot;
    int abort;
    Block b;
};

__device__ __forceinline__ void make_block(const LocalParams &p, Block &b, int doc, int index, int h, int part, int parts)
{
    b.D = local_doc(p, doc);
    b.h = h;
    b.tokens = kTile / p.G;
    const int shift = b.D.nk - b.D.nq;
    b.n_pre = (b.D.prefix + kTile - 1) / kTile;
    int first = 1 << 30, last = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        b.t0[s] = min((2 * index + s) * b.tokens, b.D.nq);
        b.t1[s] = min(b.t0[s] + b.tokens, b.D.nq);
        b.lo[s] = b.hi[s] = 0;
        if (b.t0[s] < b.t1[s]) {
            const int lo = local_run(p, shift + b.t0[s], b.D.nk).x, hi = local_run(p, shift + b.t1[s] - 1, b.D.nk).y;
            b.lo[s] = max(lo / kTile, b.n_pre);
            b.hi[s] = hi > lo ? max((hi + kTile - 1) / kTile, b.lo[s]) : b.lo[s];
            if (b.hi[s] > b.lo[s]) { first = min(first, b.lo[s]); last = max(last, b.hi[s]); }
        }
    }
    b.lo0 = first;
    const int n = b.n_pre + max(last - first, 0);
    b.n0 = int(int64_t(n) * part / parts);
    b.n1 = int(int64_t(n) * (part + 1) / parts);
}

// Column c of the tile is a visible key if it lies in [a, b) or below pre.
__device__ __forceinline__ void mask_scores(uint32_t (&s)[4][32], int a, int b, int pre)
{
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            const int j = x * 32 + c;
            if (!((j >= a && j < b) || j < pre)) s[x][c] = 0xff800000u;
        }
}

// Scores in log2 units after scale, cap and distance; what is left to multiply is 1.
__device__ __forceinline__ void shape_scores(const LocalParams &p, uint32_t (&s)[4][32], float slope2, float fp)
{
    if (p.cap > 0.f) {
        // cap tanh(x) = cap - 2 cap / (1 + e^2x): e^2x = inf gives cap, 0 gives -cap
        const float k = 2.f * kLog2e * p.scale / p.cap, c2 = p.cap * kLog2e;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int c = 0; c < 32; ++c) {
                const float e = fast_exp2(__uint_as_float(s[x][c]) * k);
                float r;
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
                s[x][c] = __float_as_uint(fmaf(-2.f * c2, r, c2));
            }
    } else {
        const float k = p.scale * kLog2e;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int c = 0; c < 32; ++c) s[x][c] = __float_as_uint(__uint_as_float(s[x][c]) * k);
    }
    if (slope2 != 0.f) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int c = 0; c < 32; ++c)
                s[x][c] = __float_as_uint(fmaf(-slope2, fabsf(fp - float(x * 32 + c)), __uint_as_float(s[x][c])));
    }
}

template <typename T, int D> __device__ __forceinline__ void redo_rows(const LocalParams &p, const Block &b, unsigned rows, int token0, int row0)
{
    while (rows) {
        const int r = row0 + __ffs(rows) - 1;
        rows &= rows - 1;
        local_row_forward<T, D>(p, b.D, b.h * p.G + r % p.G, token0 + r / p.G);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
local_fwd_kernel(const __grid_constant__ LocalParams p, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, uint32_t idesc_s, uint32_t idesc_o, float *part_o, float *part_lse)
{
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(16) Shared<D> sh;
    using C = Cfg<D>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (tc::smem_addr(smem_dyn) + 1023u) & ~1023u;
    unsigned char *base_ptr = smem_dyn + (base - tc::smem_addr(smem_dyn));
    const uint32_t ring0 = base + 2 * C::kTileBytes;
    volatile int *abort_flag = &sh.abort;

    if (warp == 0) {
        // the last blocks of a document have the most keys (causal): they go first
        const int nb = gridDim.x / p.H, h = blockIdx.x / nb, parts = gridDim.y;
        const int2 at = find_block<false>(p, 2 * (kTile / p.G), nb - 1 - int(blockIdx.x % nb));
        if (lane == 0) {
            if (at.x >= 0) make_block(p, sh.b, at.x, at.y, h, blockIdx.y, parts);
            else { sh.b.t0[0] = sh.b.t1[0] = sh.b.t0[1] = sh.b.t1[1] = 0; sh.b.n0 = sh.b.n1 = 0; }
        }
    }
    if (warp == kMmaWarp) tc::tmem_alloc(tc::smem_addr(&sh.tmem_slot), 512);
    if (warp == kLoadWarp && lane == 0) {
        for (int s = 0; s < 2; ++s) {
            tc::mbar_init(bar_addr(&sh.q_full[s]), 1);
            tc::mbar_init(bar_addr(&sh.s_full[s]), 1);
            tc::mbar_init(bar_addr(&sh.p_full[s]), 4);
            tc::mbar_init(bar_addr(&sh.o_done[s]), 1);
        }
        for (int i = 0; i < C::kRing; ++i) {
            tc::mbar_init(bar_addr(&sh.full[i]), 1);
            tc::mbar_init(bar_addr(&sh.empty[i]), 1);
        }
        tc::mbar_init(bar_addr(&sh.tail), 1);
        tc::mbar_init(bar_addr(&sh.drain), 1);
        tc::mbar_fence_init();
        sh.abort = 0;
        tc::prefetch_tensormap(&tm_q);
        tc::prefetch_tensormap(&tm_k);
        tc::prefetch_tensormap(&tm_v);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Block &b = sh.b;
    const uint32_t tmem = sh.tmem_slot;
    const int n0 = b.n0, n1 = b.n1;

    // 384 threads x 168 registers at launch = 256 x 216 + 128 x 72
    if (warp >= 8) {
        tc::set_registers_down<72>();
        if (warp == kLoadWarp) {
            // ---- loads ----------------------------------------------------------------------------------------------------
            if (n1 > n0) {
                if (lane < 2 && b.t0[lane] < b.t1[lane]) {
                    const int s = lane;
                    const uint32_t bytes = uint32_t(D / 64) * 128u * p.G * b.tokens, bar = bar_addr(&sh.q_full[s]);
                    tc::mbar_arrive_expect_tx(bar, bytes);
                    for (int c = 0; c < D / 64; ++c)
                        tc::tma_load_4d(base + s * C::kTileBytes + c * kBlock, &tm_q, c * 64, 0, b.D.q0 + b.t0[s], b.h, bar);
                }
                const int page = p.table ? 1 << p.page_shift : kTile;
                const int boxes = page >= kTile ? 1 : kTile / page;
                const int box_rows = min(page, kTile);
                int issued = 0;
                bool ok = true;
                for (int n = n0; n < n1 && ok; ++n) {
                    const int j0 = b.key_tile(n) * kTile, rows = b.D.nk - j0;      // rows of the tile that are keys of the document
                    const int live = rows >= kTile ? boxes : (rows + box_rows - 1) / box_rows;
                    for (int kv = 0; kv < 2 && ok; ++kv, ++issued) {
                        const int slot = issued % C::kRing;
                        if (issued >= C::kRing) ok = tc::mbar_wait_or_abort(bar_addr(&sh.empty[slot]), ((issued / C::kRing) & 1) ^ 1, abort_flag);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        const uint32_t dst = ring0 + slot * C::kTileBytes;
                        const bool cut = kv == 1 && rows < kTile;                  // a V tile whose last rows must be zeroed
                        const uint32_t bar = bar_addr(cut ? &sh.tail : &sh.full[slot]);
                        if (lane == 0) tc::mbar_arrive_expect_tx(bar, uint32_t(live) * box_rows * (D * 2));
                        __syncwarp();
                        for (int i = lane; i < live * (D / 64); i += 32) {
                            const int x = i / (D / 64), c = i % (D / 64);
                            int y, z;
                            if (p.table) {
                                const int j = j0 + x * box_rows;
                                z = min(max(p.table[int64_t(b.D.seq) * p.table_ld + (j >> p.page_shift)], 0), p.n_pages - 1) * p.H + b.h;
                                y = j & (page - 1);
                            } else {
                                y = b.D.k0 + j0;
                                z = b.h;
                            }
                            tc::tma_load_3d(dst + c * kBlock + x * box_rows * 128, kv ? &tm_v : &tm_k, c * 64, y, z, bar);
                        }
                        if (cut) {                                                 // at most once a CTA: the document's last tile
                            ok = tc::mbar_wait_or_abort(bar, 0, abort_flag);
                            ok = __all_sync(0xffffffffu, ok);
                            if (!ok) break;
                            for (int i = rows * 8 + lane; i < kTile * 8; i += 32)
    #pragma unroll
                                for (int c = 0; c < D / 64; ++c)
                                    *reinterpret_cast<uint4 *>(base_ptr + (dst - base) + c * kBlock + i * 16) = make_uint4(0, 0, 0, 0);
                            tc::fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) tc::mbar_arrive(bar_addr(&sh.full[slot]));
                        }
                    }
                }
                if (!ok) {
                    // unwind: every copy in flight lands before the CTA's shared memory goes away
                    if (lane == 0) *abort_flag = 1;
                    for (int i = max(issued - C::kRing, 0); i < issued; ++i) tc::mbar_wait(bar_addr(&sh.full[i % C::kRing]), (i / C::kRing) & 1);
                    for (int s = 0; s < 2; ++s)
                        if (b.t0[s] < b.t1[s]) tc::mbar_wait(bar_addr(&sh.q_full[s]), 0);
                }
            }
        } else if (warp == kMmaWarp) {
            // ---- products -------------------------------------------------------------------------------------------------
            if (lane == 0 && n1 > n0) {
                bool ok = true;
                int done[2] = {0, 0};                                              // key tiles of each query tile so far
                auto ring_wait = [&](int i) { ok = ok && tc::mbar_wait_or_abort(bar_addr(&sh.full[i % C::kRing]), (i / C::kRing) & 1, abort_flag); };
                auto scores = [&](int s, int n) {                                  // S of query tile s and key tile n
                    const uint32_t q = base + s * C::kTileBytes, k = ring0 + ((2 * (n - n0)) % C::kRing) * C::kTileBytes;
    #pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) tc::umma_f16(tmem + s * 128, desc_k(q, ks), desc_k(k, ks), idesc_s, ks > 0);
                    tc::umma_commit(bar_addr(&sh.s_full[s]));
                };
                ring_wait(0);
                for (int s = 0; s < 2; ++s)
                    if (b.t0[s] < b.t1[s]) ok = ok && tc::mbar_wait_or_abort(bar_addr(&sh.q_full[s]), 0, abort_flag);
                if (ok) {
                    for (int s = 0; s < 2; ++s)
                        if (b.active(s, n0)) scores(s, n0);
                    tc::umma_commit(bar_addr(&sh.empty[0]));
                }
                for (int n = n0; n < n1 && ok; ++n) {
                    const int vi = 2 * (n - n0) + 1;
                    const uint32_t v = ring0 + (vi % C::kRing) * C::kTileBytes;
                    ring_wait(vi);
                    for (int s = 0; s < 2 && ok; ++s) {
                        if (b.active(s, n)) {
                            ok = tc::mbar_wait_or_abort(bar_addr(&sh.p_full[s]), done[s] & 1, abort_flag);
                            if (!ok) break;
                            tc::fence_after_sync();
    #pragma unroll
                            for (int ks = 0; ks < kTile / 16; ++ks)
                                tc::umma_f16_ts(tmem + 256 + s * 128, tmem + s * 128 + ks * 8, desc_mn(v, ks), idesc_o, done[s] > 0 || ks > 0);
                            tc::umma_commit(bar_addr(&sh.o_done[s]));
                            ++done[s];
                        }
                        if (s == 1) tc::umma_commit(bar_addr(&sh.empty[vi % C::kRing]));
                        if (n + 1 < n1) {
                            if (s == 0) ring_wait(vi + 1);
                            if (ok && b.active(s, n + 1)) scores(s, n + 1);
                            if (s == 1) tc::umma_commit(bar_addr(&sh.empty[(vi + 1) % C::kRing]));
                        }
                    }
                }
                if (!ok) *abort_flag = 1;
                tc::umma_commit(bar_addr(&sh.drain));
                tc::mbar_wait(bar_addr(&sh.drain), 0);
            }
        }
    } else {
        tc::set_registers_up<216>();
        // ---- softmax and epilogue ---------------------------------------------------------------------------------------
        const int s = warp >> 2, row = tid & 127;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + s * 128 + lanes, t_o = tmem + 256 + s * 128 + lanes;
        const int token = b.t0[s] + row / p.G, head = b.h * p.G + row % p.G;
        const bool valid = row < b.tokens * p.G && token < b.t1[s];
        const int pos = b.D.nk - b.D.nq + token;
        const int2 run = local_run(p, pos, b.D.nk);
        const int pos_lo = b.D.nk - b.D.nq + b.t0[s], pos_hi = b.D.nk - b.D.nq + b.t1[s] - 1;
        const int safe_lo = p.window ? pos_hi - p.window + 1 : 0;              // keys in [safe_lo, safe_hi) are seen by every row
        const int safe_hi = local_run(p, pos_lo, b.D.nk).y;
        const float slope2 = p.slopes && valid ? p.slopes[head] * kLog2e : 0.f;
        const bool shaped = p.cap > 0.f || p.slopes || !(p.scale > 0.f);
        const float mul = shaped ? 1.f : p.scale * kLog2e;
        float m = -INFINITY, l = 0.f;
        int done = 0;
        bool ok = true;
        for (int n = n0; n < n1; ++n) {
            if (!b.active(s, n)) continue;
            const int j0 = b.key_tile(n) * kTile;
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.s_full[s]), done & 1, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::fence_after_sync();
            uint32_t x[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc::tmem_ld_x32(t_s + c * 32, x[c]);
#pragma unroll
            for (int c = 0; c < 4; ++c) tc::tmem_ld_wait(x[c]);
            if (shaped) shape_scores(p, x, slope2, float(pos - j0));
            if (!(j0 + kTile <= b.D.prefix || (j0 >= safe_lo && j0 + kTile <= safe_hi))) mask_scores(x, run.x - j0, run.y - j0, b.D.prefix - j0);
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 32; ++c)
#pragma unroll
                for (int y = 0; y < 4; ++y) mx[y] = fmaxf(mx[y], __uint_as_float(x[y][c]));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * mul;
            if (done == 0) m = top;
            else {
                const bool grow = top > m + kLazy || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? fast_exp2(m - top) : 1.f;           // 0 where nothing was seen before
                    ok = tc::mbar_wait_or_abort(bar_addr(&sh.o_done[s]), (done - 1) & 1, abort_flag);
                    if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                    tc::fence_after_sync();
                    if (grow) { m = top; l *= f; }
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tc::tmem_ld_x16(t_o + c * 16, o);
                        tc::tmem_ld_wait16(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tc::tmem_st_x16(t_o + c * 16, o);
                    }
                }
            }
            const float sub = m == -INFINITY ? 0.f : m;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float a = fast_exp2(fmaf(__uint_as_float(x[c][2 * i]), mul, -sub)), d = fast_exp2(fmaf(__uint_as_float(x[c][2 * i + 1]), mul, -sub));
                    sum[(2 * i) & 3] += a;
                    sum[(2 * i + 1) & 3] += d;
                    pk[i] = pack2<T>(a, d);
                }
                tc::tmem_st_x16(t_s + c * 16, pk);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tc::tmem_st_wait();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar_addr(&sh.p_full[s]));
            ++done;
        }
        if (ok && done > 0) {
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.o_done[s]), (done - 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok) *abort_flag = 1;
        tc::fence_after_sync();
        const int64_t out_row = int64_t(head) * p.S + b.D.q0 + token;
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const float lse = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        bool fine = ok && l < INFINITY && l >= 0.f;
        if (ok && b.t0[s] < b.t1[s]) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (done) {
                    tc::tmem_ld_x32(t_o + c * 32, o);
                    tc::tmem_ld_wait(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                float worst = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float f = __uint_as_float(o[i]) * inv;
                    o[i] = __float_as_uint(f);
                    worst = fmaf(f, 0.f, worst);                               // NaN as soon as one is not finite
                }
                fine = fine && worst == 0.f;
                if (valid) {
                    if (gridDim.y == 1) {
                        uint4 *dst = reinterpret_cast<uint4 *>(static_cast<T *>(p.o) + out_row * D + c * 32);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            dst[i] = make_uint4(pack2<T>(__uint_as_float(o[8 * i]), __uint_as_float(o[8 * i + 1])),
                                                pack2<T>(__uint_as_float(o[8 * i + 2]), __uint_as_float(o[8 * i + 3])),
                                                pack2<T>(__uint_as_float(o[8 * i + 4]), __uint_as_float(o[8 * i + 5])),
                                                pack2<T>(__uint_as_float(o[8 * i + 6]), __uint_as_float(o[8 * i + 7])));
                    } else {
                        uint4 *dst = reinterpret_cast<uint4 *>(part_o + (int64_t(blockIdx.y) * p.Hq * p.S + out_row) * D + c * 32);
#pragma unroll
                        for (int i = 0; i < 8; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
        }
        if (gridDim.y == 1) {
            if (valid) p.lse[out_row] = lse;
            const unsigned again = __ballot_sync(0xffffffffu, valid && !fine);
            __syncwarp();
            if (again) redo_rows<T, D>(p, b, again, b.t0[s], row & ~31);
        } else if (valid) {
            part_lse[int64_t(blockIdx.y) * p.Hq * p.S + out_row] = fine ? lse : __int_as_float(0x7fc00000);
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
}

// Blocks of query tiles, at most, and the parts that their key tiles are cut into: only where the blocks fill less than half
// of the SMs, with at least four key tiles a part.
struct Shape {
    int64_t blocks;
    int parts;
};
Shape shape_of(const LocalParams &p)
{
    const int per = 2 * (ltc::kTile / p.G);
    const int docs = p.n_docs + (p.cu_q ? 1 : 0);
    Shape s;
    s.blocks = std::min<int64_t>(p.S, (int64_t(p.S) + int64_t(docs) * (per - 1)) / per) * p.H;
    int64_t keys = p.table ? int64_t(p.table_ld) << p.page_shift : p.N;
    if (p.window && !p.prefix) keys = std::min<int64_t>(keys, int64_t(p.window) * (p.causal ? 1 : 2) + per);
    const int64_t tiles = ceil_div(keys, ltc::kTile);
    s.parts = 1;
    if (s.blocks > 0 && s.blocks * 2 <= sm_count()) s.parts = int(std::max<int64_t>(1, std::min<int64_t>(sm_count() / s.blocks, tiles / 4)));
    return s;
}

template <typename T, int D> int launch(const LocalParams &p, int dtype, void *ws, cudaStream_t st)
{
    using C = Cfg<D>;
    const Shape sh = shape_of(p);
    CUtensorMap tm_q, tm_k, tm_v;
    if (int rc = local_query_map(&tm_q, p, p.q, p.q_sh, p.q_st, dtype)) return rc;
    if (int rc = local_key_map(&tm_k, p, p.k, p.k_sh, p.k_st, dtype)) return rc;
    if (int rc = local_key_map(&tm_v, p, p.v, p.v_sh, p.v_st, dtype)) return rc;
    float *part_lse = static_cast<float *>(ws), *part_o = part_lse + (size_t(sh.parts) * p.Hq * p.S + 31) / 32 * 32;
    const bool bf16 = dtype == FM_BF16;
    FM_CUDA_OK(func_attr_cached((const void *)local_fwd_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem));
    local_fwd_kernel<T, D><<<dim3(unsigned(sh.blocks), unsigned(sh.parts)), kThreads, C::kSmem, st>>>(
        p, tm_q, tm_k, tm_v, tc::instr_desc_f16(bf16, ltc::kTile, ltc::kTile), tc::instr_desc_f16(bf16, ltc::kTile, D, false, true), part_o, part_lse);
    FM_LAUNCHED("local_fwd_kernel");
    return sh.parts > 1 ? local_combine(p, dtype, part_o, part_lse, sh.parts, st) : FM_OK;
}

}  // namespace

// Queries as (d, head of the group, token, KV head): a box is one tile of rows (token, head).  A dim of size one may have any
// stride, so that 0 becomes something a tensor map takes.
int local_query_map(CUtensorMap *map, const LocalParams &p, const void *q, int64_t sh, int64_t st, int dtype)
{
    auto bytes = [](int64_t stride) { return uint64_t(stride > 0 ? stride * 2 : 16); };
    const uint64_t dims[4] = {uint64_t(p.d), uint64_t(p.G), uint64_t(p.S), uint64_t(p.H)};
    const uint64_t strides[3] = {bytes(sh), bytes(st), bytes(sh * p.G)};
    const uint32_t box[4] = {64, uint32_t(p.G), uint32_t(ltc::kTile / p.G), 1};
    return make_tensor_map(map, q, dtype, 4, dims, strides, box);
}

// Keys as (d, row, KV head), or pages as (d, row of the page, page x head): a box is one tile, or the part of it in one page.
int local_key_map(CUtensorMap *map, const LocalParams &p, const void *k, int64_t sh, int64_t st, int dtype)
{
    auto bytes = [](int64_t stride) { return uint64_t(stride > 0 ? stride * 2 : 16); };
    const int64_t page = int64_t(1) << p.page_shift;
    const uint64_t dims[3] = {uint64_t(p.d), uint64_t(p.table ? page : p.N), uint64_t(p.table ? int64_t(p.n_pages) * p.H : p.H)};
    const uint64_t strides[2] = {p.table ? uint64_t(p.d) * 2 : bytes(st), p.table ? uint64_t(page) * p.d * 2 : bytes(sh)};
    const uint32_t box[3] = {64, uint32_t(p.table ? std::min<int64_t>(page, ltc::kTile) : ltc::kTile), 1};
    return make_tensor_map(map, k, dtype, 3, dims, strides, box);
}

// 16-bit types, head dim 64 or 128, a group that fits a tile, and at least one key (a tensor map has no empty dims).
bool local_tc_fits(const LocalParams &p, int dtype)
{
    return (dtype == FM_BF16 || dtype == FM_F16) && (p.d == 64 || p.d == 128) && p.G <= ltc::kTile &&
           (p.table ? p.table_ld > 0 && int64_t(p.n_pages) * p.H < (int64_t(1) << 31) : p.N > 0);
}

size_t local_tc_fwd_workspace(const LocalParams &p)
{
    const Shape s = shape_of(p);
    return s.parts > 1 ? (size_t(s.parts) * p.Hq * p.S * (p.d + 1) + 64) * sizeof(float) : 0;
}

int local_tc_fwd(const LocalParams &p, int dtype, void *ws, cudaStream_t st)
{
    if (dtype == FM_BF16) return p.d == 128 ? launch<__nv_bfloat16, 128>(p, dtype, ws, st) : launch<__nv_bfloat16, 64>(p, dtype, ws, st);
    return p.d == 128 ? launch<__half, 128>(p, dtype, ws, st) : launch<__half, 64>(p, dtype, ws, st);
}

}  // namespace fm
