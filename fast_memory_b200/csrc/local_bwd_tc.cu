// Gradients of local attention on the 5th-generation tensor cores, 16-bit types, head dim 64 or 128.
//
//   P = e^(b - lse),  dP = dO V^T,  dS = P (dP - delta) (1 - tanh^2),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K
// Two kernels, seven products instead of the five that one kernel with global reductions of dQ would do: no atomics, the same
// bits every time, and no fp32 copy of dQ (twice its size, written and read back).
//
// local_dkv_kernel: a CTA owns 128 keys of one KV head and walks the query tiles (128 rows = tokens x heads of the group, so
// that the sum over the group is part of the contraction) that see them.  Everything is transposed - lane = key:
//     S^T = K Q^T    dP^T = V dO^T    (SS)      P^T, dS^T go back to TMEM over S^T, dP^T as 16-bit A operands
//     dV += P^T dO   dK += dS^T Q     (TS, B read MN-major from the very tiles that served K-major above)
// S^T | dP^T | dV | dK fill the 512 columns.  The order S(j+1) behind dV(j) and dP(j+1) behind dK(j) lets the exponentials of one
// tile run under the products of its neighbours although nothing is double-buffered in TMEM.  Two warpgroups share the 128
// lanes, 64 columns (queries) each; lse and delta of a column come from shared memory as broadcasts.
//
// local_dq_kernel: a CTA owns one query tile and walks its key tiles; lane = query row.  S is double-buffered: S(j+2), dP(j+1)
// and dQ(j) are under way while tile j+1 is worked on.  dS overwrites S.
//
// 32 over 8 heads, 8192 tokens, window 4096, d = 128: dK, dV 668 us (1230 TFLOP/s of its four products, 75 % of cuBLAS's measured
// rate), dQ 485 us (1270 TFLOP/s of its three).  A tile of dK, dV takes 3050 cycles, 2080 of them products and 800 the wait for the
// next S^T, which cannot start before dV has read this P^T: TMEM has no room for another.  Halves of 64 queries, so that
// the warpgroups run apart, took 767 us: a product with N = 64 costs 48 cycles, not 32 (shared-memory reads).
//
// P and dS are rounded to the element type because the products take 16-bit operands; sums are fp32 (TMEM) and rounded once.
// scale is applied to the sums.  fp16 has no room below 2^-14 and above 2^16: there P is held as 2^12 P, and dS times the power of two
// that brings the largest of 8 |dO| and |delta| - of a row for dQ, of the query tiles that a CTA walks for dK - into [2^6, 2^13); the
// sums are divided by them.  Weights keep all their bits down to 2^-26, dS down to 2^-20 of that largest or further, whatever size a
// loss gives its gradient; dP - delta may be 2^3 times that largest before a dS overflows (values of 20 and more).  dQ goes first and
// leaves the largest of each 32 rows for dK, dV.  (16 packed documents, 16384 tokens: 8 us more than without.)
// Rows of a tile that are not the document's are zero where a contraction runs over them; a hidden NaN inside the document shows as a
// result that is not finite, and such rows are computed again one pair at a time, as are all rows of a CTA whose pipeline wait
// gave up.
#include "local_tc.cuh"

#include <type_traits>

namespace fm {

namespace {

using namespace ltc;

constexpr int kThreads = 384;
constexpr int kMmaWarp = 8, kLoadWarp = 9, kStatWarp = 10;

template <int D> struct Bytes {
    static constexpr uint32_t kTileB = uint32_t(D / 64) * kBlock;
};

// Powers of two by which fp16 operands are held larger than they are.
constexpr float kLogP = 12.f, kPUp = 4096.f;
__device__ __forceinline__ float scale_up(float range)
{
    const int e = int(__float_as_uint(range) >> 23) - 127;                     // range lies in [2^e, 2^(e + 1))
    const int up = e < 6 ? min(6 - e, 100) : e > 12 ? max(12 - e, -100) : 0;
    return range < 0x1p-126f ? 1.f : __int_as_float((up + 127) << 23);
}

// ======================================================= dK, dV ============================================================
template <int D> struct DkvCfg {
    static constexpr uint32_t kTileB = Bytes<D>::kTileB;
    static constexpr int kStages = D == 128 ? 2 : 4;             // query tiles (Q and dO) in flight or in use
    static constexpr uint32_t kSmem = (2 + 2 * kStages) * kTileB + 1024;
};

template <int DIM> struct DkvShared {
    uint64_t kv_full, full[DkvCfg<DIM>::kStages], empty[DkvCfg<DIM>::kStages], tail;
    uint64_t stat_full[2], stat_empty[2];
    uint64_t s_full, p_full, dp_full, ds_full, drain;
    uint32_t tmem_slot;
    int abort;
    int h, j0, q_lo, n_q;                                        // head, first key, first query tile, query tiles
    Doc D;
    alignas(16) float lse2[2][kTile], delta[2][kTile];           // negated; delta too if there is no cap
    alignas(16) float slope2[kTile], place[kTile];               // negated slope; token of a column, from the tile's first
    alignas(16) int token[kTile];
    float up;                                                    // dS is held times this (fp16)
};

template <typename T, int DIM, bool CAP, bool SLOPES>
__global__ void __launch_bounds__(kThreads, 1)
local_dkv_kernel(const __grid_constant__ LocalParams p, const __grid_constant__ BwdParams g, const __grid_constant__ CUtensorMap tm_q,
                 const __grid_constant__ CUtensorMap tm_do, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv, uint32_t idesc_s, uint32_t idesc_o,
                 float *parts)
{
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(16) DkvShared<DIM> sh;
    using C = DkvCfg<DIM>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (tc::smem_addr(smem_dyn) + 1023u) & ~1023u;
    unsigned char *base_ptr = smem_dyn + (base - tc::smem_addr(smem_dyn));
    const uint32_t s_k = base, s_v = base + C::kTileB, s_q0 = base + 2 * C::kTileB;      // stage i: Q, then dO
    volatile int *abort_flag = &sh.abort;
    const int tokens = kTile / p.G, rows = tokens * p.G;

    if (warp == 0) {
        const int h = blockIdx.x % p.H;
        Doc doc;
        const int index = find_block<true>(p, kTile, blockIdx.x / p.H, doc);   // (the most queries first)
        if (lane == 0) {
            sh.h = h;
            sh.n_q = 0;
            sh.j0 = -1;
            if (index >= 0) {
                sh.D = doc;
                sh.j0 = index * kTile;
                const int last = min(sh.j0 + kTile, sh.D.nk) - 1;
                int2 run = make_int2(local_query_run(p, sh.D, sh.j0).x, local_query_run(p, sh.D, last).y);
                if (sh.j0 < sh.D.prefix) run = make_int2(0, sh.D.nq);
                const int lo = run.x / tokens, n = run.y > run.x ? (run.y + tokens - 1) / tokens - lo : 0;
                const int from = int(int64_t(n) * blockIdx.y / gridDim.y), to = int(int64_t(n) * (blockIdx.y + 1) / gridDim.y);
                sh.q_lo = lo + from;                             // this CTA's part of the query tiles
                sh.n_q = to - from;
            }
        }
    }
    if (warp == kMmaWarp) tc::tmem_alloc(tc::smem_addr(&sh.tmem_slot), 512);
    if (warp == kLoadWarp && lane == 0) {
        tc::mbar_init(bar_addr(&sh.kv_full), 1);
        for (int i = 0; i < C::kStages; ++i) {
            tc::mbar_init(bar_addr(&sh.full[i]), 1);
            tc::mbar_init(bar_addr(&sh.empty[i]), 1);
        }
        tc::mbar_init(bar_addr(&sh.tail), 1);
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(bar_addr(&sh.stat_full[i]), 1);
            tc::mbar_init(bar_addr(&sh.stat_empty[i]), 8);
        }
        tc::mbar_init(bar_addr(&sh.s_full), 1);
        tc::mbar_init(bar_addr(&sh.p_full), 8);
        tc::mbar_init(bar_addr(&sh.dp_full), 1);
        tc::mbar_init(bar_addr(&sh.ds_full), 8);
        tc::mbar_init(bar_addr(&sh.drain), 1);
        tc::mbar_fence_init();
        sh.abort = 0;
        tc::prefetch_tensormap(&tm_q);
        tc::prefetch_tensormap(&tm_do);
        tc::prefetch_tensormap(&tm_k);
        tc::prefetch_tensormap(&tm_v);
    }
    if (tid < kTile) {
        sh.token[tid] = tid / p.G;
        sh.place[tid] = float(tid / p.G);
        sh.slope2[tid] = 0.f;
    }
    // rows that no load writes: a group that does not divide the tile
    for (int i = rows * 8 + tid; i < kTile * 8; i += kThreads)
        for (int c = 0; c < 2 * C::kStages * (DIM / 64); ++c)
            *reinterpret_cast<uint4 *>(base_ptr + 2 * C::kTileB + c * kBlock + i * 16) = make_uint4(0, 0, 0, 0);
    tc::fence_proxy_async_smem();
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sh.tmem_slot;
    const int n_q = sh.n_q, q_lo = sh.q_lo, h = sh.h, j0 = sh.j0;
    const Doc &D = sh.D;

    if (warp >= 8) {
        tc::set_registers_down<72>();
        if (warp == kLoadWarp) {
            if (n_q > 0) {
                if (lane == 0) {
                    tc::mbar_arrive_expect_tx(bar_addr(&sh.kv_full), 2 * C::kTileB);
                    for (int c = 0; c < DIM / 64; ++c) {
                        tc::tma_load_3d(s_k + c * kBlock, &tm_k, c * 64, D.k0 + j0, h, bar_addr(&sh.kv_full));
                        tc::tma_load_3d(s_v + c * kBlock, &tm_v, c * 64, D.k0 + j0, h, bar_addr(&sh.kv_full));
                    }
                }
                bool ok = true, tail_open = false;
                int i = 0;
                for (; i < n_q; ++i) {
                    const int slot = i % C::kStages, t0 = (q_lo + i) * tokens;
                    if (i >= C::kStages) ok = tc::mbar_wait_or_abort(bar_addr(&sh.empty[slot]), ((i / C::kStages) & 1) ^ 1, abort_flag, p.wait_ns);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const bool cut = t0 + tokens > D.nq;                       // the document's last queries
                    const uint32_t bar = bar_addr(cut ? &sh.tail : &sh.full[slot]);
                    const uint32_t dst = s_q0 + slot * 2 * C::kTileB;
                    if (i == p.skip_tile) continue;                            // never, but in a test
                    if (lane == 0) {
                        tc::mbar_arrive_expect_tx(bar, 2u * (DIM / 64) * 128u * rows);
                        for (int c = 0; c < DIM / 64; ++c) {
                            tc::tma_load_4d(dst + c * kBlock, &tm_q, c * 64, 0, D.q0 + t0, h, bar);
                            tc::tma_load_4d(dst + C::kTileB + c * kBlock, &tm_do, c * 64, 0, D.q0 + t0, h, bar);
                        }
                    }
                    if (cut) {
                        ok = tc::mbar_wait_or_abort(bar, 0, abort_flag, p.wait_ns);
                        ok = __all_sync(0xffffffffu, ok);
                        tail_open = !ok;
                        if (!ok) break;
                        for (int x = (D.nq - t0) * p.G * 8 + lane; x < rows * 8; x += 32)
                            for (int c = 0; c < 2 * (DIM / 64); ++c)
                                *reinterpret_cast<uint4 *>(base_ptr + (dst - base) + c * kBlock + x * 16) = make_uint4(0, 0, 0, 0);
                        tc::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(bar_addr(&sh.full[slot]));
                    }
                }
                if (!ok && lane == 0) *abort_flag = 1;
                // whoever gave up: every copy in flight lands before the CTA's shared memory goes away
                tc::mbar_wait(bar_addr(&sh.kv_full), 0);
                for (int x = max(i - C::kStages, 0); x < i; ++x)
                    if (x != p.skip_tile) tc::mbar_wait(bar_addr(&sh.full[x % C::kStages]), (x / C::kStages) & 1);
                if (tail_open) tc::mbar_wait(bar_addr(&sh.tail), 0);
            }
        } else if (warp == kStatWarp) {
            bool ok = true;
            float lse[4], delta[4], up = 1.f;
            auto fetch = [&](int i) {                            // a tile's numbers, a tile ahead
                const int t0 = (q_lo + i) * tokens;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = lane + 32 * x, token = t0 + r / p.G;
                    lse[x] = -INFINITY;
                    delta[x] = 0.f;
                    if (i < n_q && r < rows && token < D.nq) {
                        const int64_t at = int64_t(h * p.G + r % p.G) * p.S + D.q0 + token;
                        lse[x] = g.lse[at];
                        delta[x] = g.delta[at];
                    }
                }
            };
            fetch(0);
            if constexpr (kNarrow<T>) {
                float top = 0.f;
                for (int x = lane; x < 4 * n_q; x += 32) {
                    const int r = (x & 3) * 32, token = (q_lo + (x >> 2)) * tokens + r / p.G;
                    if (r < rows && token < D.nq) top = fmaxf(top, g.tops[int64_t(h * p.G + r % p.G) * p.S + D.q0 + token]);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                up = scale_up(top);
                if (lane == 0) sh.up = up;                       // (there with the first tile's numbers)
                up /= kPUp;
            }
            if (n_q > 0 && p.slopes)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = lane + 32 * x;
                    if (r < rows) sh.slope2[r] = -p.slopes[h * p.G + r % p.G] * kLog2e;
                }
            for (int i = 0; i < n_q; ++i) {
                const int buf = i & 1;
                if (i >= 2) ok = tc::mbar_wait_or_abort(bar_addr(&sh.stat_empty[buf]), ((i >> 1) & 1) ^ 1, abort_flag, p.wait_ns);
                if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = lane + 32 * x;
                    // no such row, or one that sees nothing: P = 0
                    sh.lse2[buf][r] = lse[x] == -INFINITY ? -INFINITY : kNarrow<T> ? fmaf(-lse[x], kLog2e, kLogP) : -lse[x] * kLog2e;
                    sh.delta[buf][r] = (CAP ? delta[x] : -delta[x]) * up;
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(bar_addr(&sh.stat_full[buf]));
                fetch(i + 1);
            }
            if (!ok && lane == 0) *abort_flag = 1;
        } else if (warp == kMmaWarp && n_q > 0) {
            const uint32_t tm = uniform(int(tmem));
            const int n = uniform(n_q);
            const bool leader = tc::elect_one();
            bool ok = true;
            auto wait = [&](uint64_t *bar, int parity) { ok = ok && tc::mbar_wait_or_abort(bar_addr(bar), parity, abort_flag, p.wait_ns); };
            auto q_tile = [&](int i) { return s_q0 + (i % C::kStages) * 2 * C::kTileB; };
            auto wait_q = [&](int i) { wait(&sh.full[i % C::kStages], (i / C::kStages) & 1); };
            auto product = [&](uint32_t d, uint32_t a_tile, uint32_t b_tile, uint64_t *bar) {            // S^T or dP^T
                const uint64_t a = desc_k(a_tile, 0), b = desc_k(b_tile, 0);
#pragma unroll
                for (int ks = 0; ks < DIM / 16; ++ks) tc::umma_f16_if(leader && ok, d, a + step_k(ks), b + step_k(ks), idesc_s, ks > 0);
                tc::umma_commit_if(leader && ok, bar_addr(bar));               // (nothing is announced once a wait gave up)
            };
            auto gather = [&](uint32_t d, uint32_t a, uint32_t b_tile, bool more) {                       // dV or dK
                const uint64_t b = desc_mn(b_tile, 0);
#pragma unroll
                for (int ks = 0; ks < kTile / 16; ++ks)
                    tc::umma_f16_ts_if(leader && ok, d, a + (ks >> 2) * 64 + (ks & 3) * 8, b + step_mn(ks), idesc_o, more || ks > 0);
            };
            wait(&sh.kv_full, 0);
            wait_q(0);
            product(tm, s_k, q_tile(0), &sh.s_full);
            product(tm + 128, s_v, q_tile(0) + C::kTileB, &sh.dp_full);
            for (int i = 0; i < n; ++i) {
                if (i + 1 < n) wait_q(i + 1);                                  // there long before P is
                wait(&sh.p_full, i & 1);
                tc::fence_after_sync();
                gather(tm + 256, tm, q_tile(i) + C::kTileB, i > 0);
                if (i + 1 < n) product(tm, s_k, q_tile(i + 1), &sh.s_full);
                wait(&sh.ds_full, i & 1);
                tc::fence_after_sync();
                gather(tm + 384, tm + 128, q_tile(i), i > 0);
                tc::umma_commit_if(leader && ok, bar_addr(&sh.empty[i % C::kStages]));
                if (i + 1 < n) product(tm + 128, s_v, q_tile(i + 1) + C::kTileB, &sh.dp_full);
            }
            if (leader && !ok) *abort_flag = 1;
            tc::umma_commit_if(leader, bar_addr(&sh.drain));
            tc::mbar_wait(bar_addr(&sh.drain), 0);
        }
    } else {
        tc::set_registers_up<216>();
        const int half = warp >> 2, row = tid & 127, j = j0 + row;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + half * 64 + lanes, t_dp = tmem + 128 + half * 64 + lanes;
        const bool valid = j0 >= 0 && j < D.nk;
        int2 run = make_int2(0, 0), all = make_int2(0, 0);       // queries that see this key; that see every key of the tile
        if (n_q > 0) {
            const int last = min(j0 + kTile, D.nk) - 1;
            if (valid) run = local_query_run(p, D, j);
            all = make_int2(local_query_run(p, D, last).x, local_query_run(p, D, max(j0, min(D.prefix, last))).y);
        }
        const f32x2 scale2 = pair(p.scale * kLog2e, p.scale * kLog2e), c2 = pair(p.cap * kLog2e, p.cap * kLog2e);
        const f32x2 minus = pair(-1.f, -1.f);
        const float kc = p.cap > 0.f ? p.scale / p.cap : 0.f;
        bool ok = true;
        for (int i = 0; i < n_q; ++i) {
            const int buf = i & 1, t0 = (q_lo + i) * tokens;
            const f32x2 dist0 = pair(float(D.nk - D.nq + t0 - j), float(D.nk - D.nq + t0 - j));
            const bool masked = !(all.x <= t0 && min(t0 + tokens, D.nq) <= all.y);
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.stat_full[buf]), (i >> 1) & 1, abort_flag, p.wait_ns) &&
                 tc::mbar_wait_or_abort(bar_addr(&sh.s_full), i & 1, abort_flag, p.wait_ns);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::fence_after_sync();
            f32x2 pr[32];                                        // P; with a cap, P times its derivative, negated (tanh^2 - 1: one operation)
            unsigned seen[2] = {0xffffffffu, 0xffffffffu};
            if (masked) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    unsigned m = 0;
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        const int token = t0 + sh.token[half * 64 + x * 32 + c];
                        m |= (token >= run.x && token < run.y) ? 1u << c : 0u;
                    }
                    seen[x] = m;
                }
            }
            auto weights = [&](auto with_mask) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t s[32], pk[16];
                    tc::tmem_ld_x32(t_s + x * 32, s);
                    tc::tmem_ld_wait(s);
                    const int col0 = half * 64 + x * 32;
                    const ulonglong2 *lse2 = reinterpret_cast<const ulonglong2 *>(&sh.lse2[buf][col0]);
                    f32x2 t[16];
                    if constexpr (CAP) cap_scores(t, s, kc, valid);
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const f32x2 n = (c & 1) ? lse2[c >> 1].y : lse2[c >> 1].x;
                        f32x2 e = CAP ? fma2(t[c], c2, n) : fma2(pair(s[2 * c], s[2 * c + 1]), scale2, n);
                        if constexpr (SLOPES) {
                            const float2 d = split(add2(dist0, *reinterpret_cast<const f32x2 *>(&sh.place[col0 + 2 * c])));
                            e = fma2(*reinterpret_cast<const f32x2 *>(&sh.slope2[col0 + 2 * c]), pair(fabsf(d.x), fabsf(d.y)), e);
                        }
                        float2 w = split(exp2_pair(e));
                        if constexpr (decltype(with_mask)::value) {
                            w.x = (seen[x] >> (2 * c) & 1u) ? w.x : 0.f;
                            w.y = (seen[x] >> (2 * c + 1) & 1u) ? w.y : 0.f;
                        }
                        pk[c] = pack2<T>(w.x, w.y);
                        pr[x * 16 + c] = CAP ? mul2(pair(w.x, w.y), fma2(t[c], t[c], minus)) : pair(w.x, w.y);
                    }
                    tc::tmem_st_x16(t_s + x * 16, pk);
                }
            };
            if (masked) weights(std::true_type{});
            else weights(std::false_type{});
            tc::tmem_st_wait();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar_addr(&sh.p_full));
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.dp_full), i & 1, abort_flag, p.wait_ns);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::fence_after_sync();
            const float up = kNarrow<T> ? sh.up * ((CAP ? -1.f : 1.f) / kPUp) : 1.f;
            const f32x2 up2 = pair(up, up);                      // of dP (fp16)
            auto gradients = [&](auto with_mask) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t s[32], pk[16];
                    tc::tmem_ld_x32(t_dp + x * 32, s);
                    tc::tmem_ld_wait(s);
                    const ulonglong2 *delta = reinterpret_cast<const ulonglong2 *>(&sh.delta[buf][half * 64 + x * 32]);
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const f32x2 n = (c & 1) ? delta[c >> 1].y : delta[c >> 1].x;
                        const f32x2 dp = pair(s[2 * c], s[2 * c + 1]);
                        float2 w = split(mul2(pr[x * 16 + c], kNarrow<T> ? fma2(dp, up2, n) : CAP ? fma2(dp, minus, n) : add2(dp, n)));
                        if constexpr (decltype(with_mask)::value) {          // P = 0 is not enough: dP may be NaN there
                            w.x = (seen[x] >> (2 * c) & 1u) ? w.x : 0.f;
                            w.y = (seen[x] >> (2 * c + 1) & 1u) ? w.y : 0.f;
                        }
                        pk[c] = pack2<T>(w.x, w.y);
                    }
                    tc::tmem_st_x16(t_dp + x * 16, pk);
                }
            };
            if (masked) gradients(std::true_type{});
            else gradients(std::false_type{});
            tc::tmem_st_wait();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                tc::mbar_arrive(bar_addr(&sh.ds_full));
                tc::mbar_arrive(bar_addr(&sh.stat_empty[buf]));
            }
        }
        if (ok && n_q > 0) {
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.drain), 0, abort_flag, p.wait_ns);
            ok = __all_sync(0xffffffffu, ok) && !*abort_flag;
        }
        ok = tc::named_barrier_and(1, 256, ok);                                // all warps go on together
        if (!ok) *abort_flag = 1;
        tc::fence_after_sync();
        // first warpgroup: dV, second: dK; a whole tile goes out through the shared memory of K or V, which no product reads any more
        bool fine = ok;
        const float down = !kNarrow<T> || n_q == 0 ? 1.f : half ? 1.f / sh.up : 1.f / kPUp, f = (half ? p.scale : 1.f) * down;
        const bool whole = ok && j0 >= 0 && j0 + kTile <= D.nk && gridDim.y == 1;
        if (gridDim.y > 1) {
            // parts stay fp32, and local_dkv_join looks for what is not finite
            float *out = parts + ((int64_t(blockIdx.y) * 2 + half) * p.H * p.N + int64_t(h) * p.N + D.k0 + j) * DIM;
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) {
                uint32_t o[32];
                if (ok && n_q > 0) {
                    tc::tmem_ld_x32(tmem + 256 + half * 128 + lanes + c * 32, o);
                    tc::tmem_ld_wait(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = ok ? 0u : 0x7fc00000u;
                }
                if constexpr (kNarrow<T>) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
                }
                if (valid) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) reinterpret_cast<uint4 *>(out + c * 32)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
            fine = true;
        } else if (ok && j0 >= 0) {
            T *out = valid ? static_cast<T *>(half ? g.dk : g.dv) + (int64_t(h) * p.N + D.k0 + j) * DIM : nullptr;
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) {
                uint32_t o[32];
                if (n_q > 0) {
                    tc::tmem_ld_x32(tmem + 256 + half * 128 + lanes + c * 32, o);
                    tc::tmem_ld_wait(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                const bool good = put_row<T>(o, f, whole ? base_ptr + half * C::kTileB : nullptr, out, row, c * 32);
                fine = fine && good;
            }
        }
        if (whole) tc::fence_proxy_async_smem();
        const bool any = tc::named_barrier_or(1, 256, valid && !fine);         // (both warpgroups redo a row together)
        if (whole && row == 0) {
            for (int c = 0; c < DIM / 64; ++c) tc::tma_store_3d(half ? &tm_dk : &tm_dv, c * 64, D.k0 + j0, h, base + half * C::kTileB + c * kBlock);
            tc::tma_store_commit();
            if (any) tc::tma_store_wait_all();
            else tc::tma_store_wait_read();
        }
        unsigned again = 0;
        if (any) {
            tc::named_barrier(1, 256);
            again = __ballot_sync(0xffffffffu, valid && !fine);
        }
        while (again) {
            const int r = (row & ~31) + __ffs(again) - 1;
            again &= again - 1;
            local_row_dkv<T, DIM>(p, g, D, h, j0 + r);
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
}

// Sums the parts of dV and dK in their order: a warp a key row.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) local_dkv_join(const __grid_constant__ LocalParams p, const __grid_constant__ BwdParams g, const float *parts, int n)
{
    const int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) >> 5, rows = int64_t(p.H) * p.N;
    if (row >= rows) return;
    constexpr int E = DIM / 32;
    const int c = (threadIdx.x & 31) * E;
    float dv[E] = {}, dk[E] = {}, worst = 0.f;
#pragma unroll 4
    for (int i = 0; i < n; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dv[e] += parts[(int64_t(2 * i) * rows + row) * DIM + c + e];
            dk[e] += parts[(int64_t(2 * i + 1) * rows + row) * DIM + c + e];
        }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        dk[e] *= p.scale;
        worst = fmaf(dv[e], 0.f, fmaf(dk[e], 0.f, worst));
        static_cast<T *>(g.dv)[row * DIM + c + e] = Elem<T>::from_f32(dv[e]);
        static_cast<T *>(g.dk)[row * DIM + c + e] = Elem<T>::from_f32(dk[e]);
    }
    if (__any_sync(0xffffffffu, worst != 0.f)) {
        const int r = int(row % p.N);
        const Doc doc = local_doc<true>(p, p.cu_k ? local_find(p.cu_k, p.n_docs, r) : 0);
        local_row_dkv_call<T, DIM>(p, g, doc, int(row / p.N), r - doc.k0);
    }
}

// ========================================================= dQ ==============================================================
template <int D> struct DqCfg {
    static constexpr uint32_t kTileB = Bytes<D>::kTileB;
    static constexpr int kRing = D == 128 ? 5 : 8;               // K and V tiles in flight or in use
    static constexpr uint32_t kSmem = (2 + kRing) * kTileB + 1024;
};

template <int DIM> struct DqShared {
    uint64_t q_full, full[DqCfg<DIM>::kRing], empty[DqCfg<DIM>::kRing], tail;
    uint64_t s_full[2], dp_full, ds_full, drain;
    uint32_t tmem_slot;
    int abort;
    int h, t0, t1, n_pre, lo, n_k;                               // query tokens [t0, t1); key tiles: prefix, then lo ..; n_k in all
    Doc D;
};

template <typename T, int DIM, bool CAP, bool SLOPES>
__global__ void __launch_bounds__(kThreads, 1)
local_dq_kernel(const __grid_constant__ LocalParams p, const __grid_constant__ BwdParams g, const __grid_constant__ CUtensorMap tm_q,
                const __grid_constant__ CUtensorMap tm_do, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ CUtensorMap tm_dq, uint32_t idesc_s, uint32_t idesc_o)
{
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(16) DqShared<DIM> sh;
    using C = DqCfg<DIM>;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (tc::smem_addr(smem_dyn) + 1023u) & ~1023u;
    unsigned char *base_ptr = smem_dyn + (base - tc::smem_addr(smem_dyn));
    const uint32_t s_q = base, s_do = base + C::kTileB, ring0 = base + 2 * C::kTileB;
    volatile int *abort_flag = &sh.abort;
    const int tokens = kTile / p.G, rows = tokens * p.G;

    if (warp == 0) {
        const int nb = gridDim.x / p.H, h = blockIdx.x % p.H;
        Doc doc;
        const int index = find_block<false>(p, tokens, nb - 1 - int(blockIdx.x / p.H), doc);   // (the most keys first)
        if (lane == 0) {
            sh.h = h;
            sh.t0 = sh.t1 = sh.n_pre = sh.lo = sh.n_k = 0;
            if (index >= 0) {
                const Doc &D = sh.D = doc;
                sh.t0 = index * tokens;
                sh.t1 = min(sh.t0 + tokens, D.nq);
                const int lo = local_run(p, D.nk - D.nq + sh.t0, D.nk).x, hi = local_run(p, D.nk - D.nq + sh.t1 - 1, D.nk).y;
                sh.n_pre = (D.prefix + kTile - 1) / kTile;
                sh.lo = max(lo / kTile, sh.n_pre);
                sh.n_k = sh.n_pre + (hi > lo ? max((hi + kTile - 1) / kTile - sh.lo, 0) : 0);
            }
        }
    }
    if (warp == kMmaWarp) tc::tmem_alloc(tc::smem_addr(&sh.tmem_slot), 512);
    if (warp == kLoadWarp && lane == 0) {
        tc::mbar_init(bar_addr(&sh.q_full), 1);
        for (int i = 0; i < C::kRing; ++i) {
            tc::mbar_init(bar_addr(&sh.full[i]), 1);
            tc::mbar_init(bar_addr(&sh.empty[i]), 1);
        }
        tc::mbar_init(bar_addr(&sh.tail), 1);
        tc::mbar_init(bar_addr(&sh.s_full[0]), 1);
        tc::mbar_init(bar_addr(&sh.s_full[1]), 1);
        tc::mbar_init(bar_addr(&sh.dp_full), 1);
        tc::mbar_init(bar_addr(&sh.ds_full), 8);
        tc::mbar_init(bar_addr(&sh.drain), 1);
        tc::mbar_fence_init();
        sh.abort = 0;
        tc::prefetch_tensormap(&tm_q);
        tc::prefetch_tensormap(&tm_do);
        tc::prefetch_tensormap(&tm_k);
        tc::prefetch_tensormap(&tm_v);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sh.tmem_slot;                          // S0, S1, dP, dQ
    const int n_k = sh.n_k, n_pre = sh.n_pre, lo = sh.lo, h = sh.h, t0 = sh.t0, t1 = sh.t1;
    const Doc &D = sh.D;
    auto key_tile = [&](int n) { return n < n_pre ? n : lo + n - n_pre; };

    if (warp >= 8) {
        tc::set_registers_down<72>();
        if (warp == kLoadWarp) {
            if (lane == 0 && n_k > 0) {
                tc::mbar_arrive_expect_tx(bar_addr(&sh.q_full), 2u * (DIM / 64) * 128u * rows);
                for (int c = 0; c < DIM / 64; ++c) {
                    tc::tma_load_4d(s_q + c * kBlock, &tm_q, c * 64, 0, D.q0 + t0, h, bar_addr(&sh.q_full));
                    tc::tma_load_4d(s_do + c * kBlock, &tm_do, c * 64, 0, D.q0 + t0, h, bar_addr(&sh.q_full));
                }
            }
            bool ok = true, tail_open = false;
            int i = 0;
            for (; i < 2 * n_k; ++i) {
                const int slot = i % C::kRing, kt = key_tile(i >> 1), live = D.nk - kt * kTile;
                if (i >= C::kRing) ok = tc::mbar_wait_or_abort(bar_addr(&sh.empty[slot]), ((i / C::kRing) & 1) ^ 1, abort_flag, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const bool cut = !(i & 1) && live < kTile;                     // the K tile's rows behind the last key meet dS = 0
                const uint32_t bar = bar_addr(cut ? &sh.tail : &sh.full[slot]), dst = ring0 + slot * C::kTileB;
                if (i == p.skip_tile) continue;                                // never, but in a test
                if (lane == 0) {
                    tc::mbar_arrive_expect_tx(bar, C::kTileB);
                    for (int c = 0; c < DIM / 64; ++c) tc::tma_load_3d(dst + c * kBlock, (i & 1) ? &tm_v : &tm_k, c * 64, D.k0 + kt * kTile, h, bar);
                }
                if (cut) {
                    ok = tc::mbar_wait_or_abort(bar, 0, abort_flag, p.wait_ns);
                    ok = __all_sync(0xffffffffu, ok);
                    tail_open = !ok;
                    if (!ok) break;
                    for (int x = live * 8 + lane; x < kTile * 8; x += 32)
                        for (int c = 0; c < DIM / 64; ++c)
                            *reinterpret_cast<uint4 *>(base_ptr + (dst - base) + c * kBlock + x * 16) = make_uint4(0, 0, 0, 0);
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(bar_addr(&sh.full[slot]));
                }
            }
            if (!ok && lane == 0) *abort_flag = 1;
            if (n_k > 0) tc::mbar_wait(bar_addr(&sh.q_full), 0);
            for (int x = max(i - C::kRing, 0); x < i; ++x)
                if (x != p.skip_tile) tc::mbar_wait(bar_addr(&sh.full[x % C::kRing]), (x / C::kRing) & 1);
            if (tail_open) tc::mbar_wait(bar_addr(&sh.tail), 0);
        } else if (warp == kMmaWarp && n_k > 0) {
            const uint32_t tm = uniform(int(tmem));
            const int tiles = uniform(n_k);
            const bool leader = tc::elect_one();
            bool ok = true;
            auto wait = [&](uint64_t *bar, int parity) { ok = ok && tc::mbar_wait_or_abort(bar_addr(bar), parity, abort_flag, p.wait_ns); };
            auto tile = [&](int i) { return ring0 + (i % C::kRing) * C::kTileB; };                        // i = 2 n: K, 2 n + 1: V
            auto product = [&](uint32_t d, uint32_t a_tile, int i, uint64_t *bar) {                       // S or dP
                wait(&sh.full[i % C::kRing], (i / C::kRing) & 1);
                const uint64_t a = desc_k(a_tile, 0), b = desc_k(tile(i), 0);
#pragma unroll
                for (int ks = 0; ks < DIM / 16; ++ks) tc::umma_f16_if(leader && ok, d, a + step_k(ks), b + step_k(ks), idesc_s, ks > 0);
                tc::umma_commit_if(leader && ok, bar_addr(bar));               // (nothing is announced once a wait gave up)
                if (i & 1) tc::umma_commit_if(leader && ok, bar_addr(&sh.empty[i % C::kRing]));
            };
            wait(&sh.q_full, 0);
            product(tm, s_q, 0, &sh.s_full[0]);
            product(tm + 256, s_do, 1, &sh.dp_full);
            if (tiles > 1) product(tm + 128, s_q, 2, &sh.s_full[1]);
            for (int n = 0; n < tiles; ++n) {
                wait(&sh.ds_full, n & 1);
                tc::fence_after_sync();
                if (n + 1 < tiles) product(tm + 256, s_do, 2 * n + 3, &sh.dp_full);
                const uint64_t k = desc_mn(tile(2 * n), 0);
#pragma unroll
                for (int ks = 0; ks < kTile / 16; ++ks)
                    tc::umma_f16_ts_if(leader && ok, tm + 384, tm + (n & 1) * 128 + (ks >> 2) * 64 + (ks & 3) * 8, k + step_mn(ks), idesc_o, n > 0 || ks > 0);
                tc::umma_commit_if(leader && ok, bar_addr(&sh.empty[(2 * n) % C::kRing]));
                if (n + 2 < tiles) product(tm + (n & 1) * 128, s_q, 2 * n + 4, &sh.s_full[n & 1]);
            }
            if (leader && !ok) *abort_flag = 1;
            tc::umma_commit_if(leader, bar_addr(&sh.drain));
            tc::mbar_wait(bar_addr(&sh.drain), 0);
        }
    } else {
        tc::set_registers_up<216>();
        const int half = warp >> 2, row = tid & 127, token = t0 + row / p.G, head = h * p.G + row % p.G;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t t_dp = tmem + 256 + half * 64 + lanes;
        const bool valid = row < rows && token < t1;
        const int64_t out_row = int64_t(head) * p.S + D.q0 + token;
        const int shift = D.nk - D.nq, pos = shift + token;
        float lse2 = INFINITY, delta = 0.f, slope2 = 0.f;
        if (valid) {
            const float x = g.lse[out_row];
            lse2 = x == -INFINITY ? INFINITY : x * kLog2e;
            delta = g.delta[out_row];
            slope2 = p.slopes ? p.slopes[head] * kLog2e : 0.f;
        }
        const int2 run = valid ? local_run(p, pos, D.nk) : make_int2(0, 0);
        const int pre = valid ? D.prefix : 0;
        const int safe_lo = p.window ? shift + t1 - p.window : 0, safe_hi = n_k > 0 ? local_run(p, shift + t0, D.nk).y : 0;
        const f32x2 scale2 = pair(p.scale * kLog2e, p.scale * kLog2e), c2 = pair(p.cap * kLog2e, p.cap * kLog2e);
        const f32x2 minus = pair(-1.f, -1.f);
        float up = 1.f;
        if constexpr (kNarrow<T>) {
            float top = valid ? g.range[out_row] : 0.f;
            up = scale_up(top);
            delta *= up;
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (lane == 0 && half == 0 && valid) g.tops[out_row] = top;
        }
        const f32x2 up2 = CAP ? pair(-up, -up) : pair(up, up);                 // of dP (fp16)
        const f32x2 nlse = pair(-lse2, -lse2), sdelta = CAP ? pair(delta, delta) : pair(-delta, -delta), nslope = pair(-slope2, -slope2);
        const float kc = p.cap > 0.f ? p.scale / p.cap : 0.f;
        bool ok = true;
        for (int n = 0; n < n_k; ++n) {
            const int j0 = key_tile(n) * kTile, b = n & 1, col0 = j0 + half * 64;
            const bool masked = !(j0 + kTile <= D.prefix || (j0 >= safe_lo && j0 + kTile <= safe_hi));
            const uint32_t t_s = tmem + b * 128 + half * 64 + lanes;
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.s_full[b]), (n >> 1) & 1, abort_flag, p.wait_ns);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::fence_after_sync();
            f32x2 pr[32];                                        // P; with a cap, P times its derivative, negated (tanh^2 - 1: one operation)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t s[32];
                tc::tmem_ld_x32(t_s + x * 32, s);
                tc::tmem_ld_wait(s);
                f32x2 t[16];
                if constexpr (CAP) cap_scores(t, s, kc, valid);
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    f32x2 e = CAP ? fma2(t[c], c2, nlse) : fma2(pair(s[2 * c], s[2 * c + 1]), scale2, nlse);
                    if constexpr (SLOPES) {
                        const float d = float(pos - col0 - x * 32 - 2 * c);
                        e = fma2(nslope, pair(fabsf(d), fabsf(d - 1.f)), e);
                    }
                    e = exp2_pair(e);
                    pr[x * 16 + c] = CAP ? mul2(e, fma2(t[c], t[c], minus)) : e;
                }
            }
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.dp_full), n & 1, abort_flag, p.wait_ns);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tc::fence_after_sync();
            auto gradients = [&](auto with_mask) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t s[32], pk[16];
                    tc::tmem_ld_x32(t_dp + x * 32, s);
                    tc::tmem_ld_wait(s);
                    const int a = run.x - col0 - x * 32, e = run.y - col0 - x * 32, q = pre - col0 - x * 32;
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const f32x2 dp = pair(s[2 * c], s[2 * c + 1]);
                        float2 w = split(mul2(pr[x * 16 + c], kNarrow<T> ? fma2(dp, up2, sdelta) : CAP ? fma2(dp, minus, sdelta) : add2(dp, sdelta)));
                        if constexpr (decltype(with_mask)::value) {
                            const int i = 2 * c;
                            if (!((i >= a && i < e) || i < q)) w.x = 0.f;
                            if (!((i + 1 >= a && i + 1 < e) || i + 1 < q)) w.y = 0.f;
                        }
                        pk[c] = pack2<T>(w.x, w.y);
                    }
                    tc::tmem_st_x16(t_s + x * 16, pk);
                }
            };
            if (masked) gradients(std::true_type{});
            else gradients(std::false_type{});
            tc::tmem_st_wait();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar_addr(&sh.ds_full));
        }
        if (ok && n_k > 0) {
            ok = tc::mbar_wait_or_abort(bar_addr(&sh.drain), 0, abort_flag, p.wait_ns);
            ok = __all_sync(0xffffffffu, ok) && !*abort_flag;
        }
        ok = tc::named_barrier_and(1, 256, ok);                                // all warps go on together
        if (!ok) *abort_flag = 1;
        tc::fence_after_sync();
        bool fine = ok;
        const bool whole = ok && t1 - t0 == tokens;
        // each warpgroup writes its half of the columns
        if (ok && t0 < t1) {
            T *out = valid ? static_cast<T *>(g.dq) + out_row * DIM : nullptr;
#pragma unroll
            for (int c = 0; c < DIM / 64; ++c) {
                const int col = half * (DIM / 2) + c * 32;
                uint32_t o[32];
                if (n_k > 0) {
                    tc::tmem_ld_x32(tmem + 384 + lanes + col, o);
                    tc::tmem_ld_wait(o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
                const bool good = put_row<T>(o, kNarrow<T> ? p.scale / up : p.scale, whole ? base_ptr : nullptr, out, row, col);
                fine = fine && good;
            }
        }
        if (whole) tc::fence_proxy_async_smem();
        const bool any = tc::named_barrier_or(1, 256, valid && !fine);
        if (whole && tid == 0) {
            for (int c = 0; c < DIM / 64; ++c) tc::tma_store_4d(&tm_dq, c * 64, 0, D.q0 + t0, h, s_q + c * kBlock);
            tc::tma_store_commit();
            if (any) tc::tma_store_wait_all();
            else tc::tma_store_wait_read();
        }
        unsigned again = 0;
        if (any) {
            tc::named_barrier(1, 256);
            again = __ballot_sync(0xffffffffu, valid && !fine);
        }
        while (again) {
            const int r = (row & ~31) + __ffs(again) - 1;
            again &= again - 1;
            local_row_dq<T, DIM>(p, g, D, h * p.G + r % p.G, t0 + r / p.G);
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
}

// Key blocks, at most, and the parts that the query tiles of a block are cut into: only where the blocks fill less than half of the
// SMs, with at least two query tiles a part.
struct KeyShape {
    int64_t blocks;
    int parts;
};
KeyShape key_shape(const LocalParams &p)
{
    const int docs = p.n_docs + (p.cu_k ? 1 : 0), tokens = kTile / p.G;
    KeyShape s{std::min<int64_t>(p.N, (int64_t(p.N) + int64_t(docs) * (kTile - 1)) / kTile) * p.H, 1};
    int64_t rows = p.S;
    if (p.window && !p.prefix) rows = std::min<int64_t>(rows, int64_t(p.window) * (p.causal ? 1 : 2) + kTile);
    if (s.blocks > 0 && s.blocks * 2 <= sm_count())
        s.parts = int(std::max<int64_t>(1, std::min<int64_t>(sm_count() / s.blocks, ceil_div(rows, tokens) / 2)));
    return s;
}

template <typename T, int DIM> int launch(const LocalParams &p, const BwdParams &g, int dtype, float *parts, cudaStream_t st)
{
    const int tokens = kTile / p.G, docs = p.n_docs + (p.cu_q ? 1 : 0);
    CUtensorMap tm_q, tm_do, tm_k, tm_v, tm_dq, tm_dk, tm_dv;
    if (int rc = local_query_map(&tm_q, p, p.q, p.q_sh, p.q_st, dtype)) return rc;
    if (int rc = local_query_map(&tm_do, p, g.dout, g.do_sh, g.do_st, dtype)) return rc;
    if (int rc = local_key_map(&tm_k, p, p.k, p.k_sh, p.k_st, dtype)) return rc;
    if (int rc = local_key_map(&tm_v, p, p.v, p.v_sh, p.v_st, dtype)) return rc;
    if (int rc = local_query_map(&tm_dq, p, g.dq, int64_t(p.S) * DIM, DIM, dtype)) return rc;
    if (int rc = local_key_map(&tm_dk, p, g.dk, int64_t(p.N) * DIM, DIM, dtype)) return rc;
    if (int rc = local_key_map(&tm_dv, p, g.dv, int64_t(p.N) * DIM, DIM, dtype)) return rc;
    const bool bf16 = dtype == FM_BF16;
    const uint32_t idesc_s = tc::instr_desc_f16(bf16, kTile, kTile), idesc_o = tc::instr_desc_f16(bf16, kTile, DIM, false, true);
    const int64_t q_blocks = std::min<int64_t>(p.S, (int64_t(p.S) + int64_t(docs) * (tokens - 1)) / tokens) * p.H;
    const KeyShape ks = key_shape(p);
    auto launch_mode = [&](auto cap, auto slopes) -> int {
        auto *dkv = local_dkv_kernel<T, DIM, decltype(cap)::value, decltype(slopes)::value>;
        auto *dq = local_dq_kernel<T, DIM, decltype(cap)::value, decltype(slopes)::value>;
        FM_CUDA_OK(func_attr_cached((const void *)dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DkvCfg<DIM>::kSmem));
        FM_CUDA_OK(func_attr_cached((const void *)dq, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DqCfg<DIM>::kSmem));
        dq<<<unsigned(q_blocks), kThreads, DqCfg<DIM>::kSmem, st>>>(p, g, tm_q, tm_do, tm_k, tm_v, tm_dq, idesc_s, idesc_o);
        FM_LAUNCHED("local_dq_kernel");
        dkv<<<dim3(unsigned(ks.blocks), unsigned(ks.parts)), kThreads, DkvCfg<DIM>::kSmem, st>>>(p, g, tm_q, tm_do, tm_k, tm_v, tm_dk, tm_dv, idesc_s, idesc_o, parts);
        FM_LAUNCHED("local_dkv_kernel");
        if (ks.parts > 1) {
            local_dkv_join<T, DIM><<<unsigned(ceil_div(int64_t(p.H) * p.N * 32, 256)), 256, 0, st>>>(p, g, parts, ks.parts);
            FM_LAUNCHED("local_dkv_join");
        }
        return FM_OK;
    };
    if (p.cap > 0.f) return p.slopes ? launch_mode(std::true_type{}, std::true_type{}) : launch_mode(std::true_type{}, std::false_type{});
    return p.slopes ? launch_mode(std::false_type{}, std::true_type{}) : launch_mode(std::false_type{}, std::false_type{});
}

}  // namespace

size_t local_tc_bwd_workspace(const LocalParams &p)
{
    const KeyShape s = key_shape(p);
    return s.parts > 1 ? size_t(s.parts) * 2 * p.H * p.N * p.d * sizeof(float) : 0;
}

int local_tc_bwd(const LocalParams &p, const BwdParams &g, int dtype, float *parts, cudaStream_t st)
{
    if (dtype == FM_BF16) return p.d == 128 ? launch<__nv_bfloat16, 128>(p, g, dtype, parts, st) : launch<__nv_bfloat16, 64>(p, g, dtype, parts, st);
    return p.d == 128 ? launch<__half, 128>(p, g, dtype, parts, st) : launch<__half, 64>(p, g, dtype, parts, st);
}

}  // namespace fm
