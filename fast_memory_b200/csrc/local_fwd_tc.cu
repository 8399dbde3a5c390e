// Local attention forward on the 5th-generation tensor cores, 16-bit types, head dim 64 or 128.
//
// A CTA owns two query tiles of 128 rows - row = (token, head of the group), so that a tile reads its KV head's keys once for
// the whole group - and streams the key tiles that either of them sees, in steps of 64 keys:
//     S [128 x 64] = Q K^T         A = Q, B = K, both K-major in shared memory (TMA, 128-byte swizzle); fp32 in TMEM
//     P = 2^(s - m)                thread = row: 64 scores in registers, sum l, no shuffles; P goes back to TMEM over S as
//                                  packed 16-bit: the A operand of the second product
//     O [128 x d] += P V           B = V, the same tile layout read MN-major; fp32 in TMEM
// TMEM: two buffers of S for each tile and O of each, 512 columns.  S of step k + 1 is under way while step k is in the softmax,
// so that neither waits for the other: the special-function unit (16 exponentials a cycle: 1024 cycles for 128 keys of a tile)
// and the tensor core (1280 cycles; a product with N = 64 and both operands in shared memory takes 48 cycles, not 32) are
// both busy.  With steps of 128 keys TMEM holds one buffer of S, and a tile's softmax (2000 cycles) and products (1500 with their
// hand-over) take turns.
// The reference m is the maximum of the row's first step and is renewed only when a step's sum of p exceeds 2^12: the sums are
// fp32 and P is a floating-point number, so a reference that is too small costs no accuracy.  Most steps then
// need no maximum at all, and O is rescaled in TMEM next to never.  fp16, with bits down to 2^-24 and a top of 2^16, takes 1/8 of
// the maximum and 2^15: a weight is off by 2^-28 of the largest at most, over 2^17 keys half a step of the result.
// l sums the unrounded p; P is rounded to the element type because the second product takes 16-bit operands.
// 32 heads of 8192 tokens, window 4096, d = 128: 385 to 400 us, 1030 TFLOP/s and more (63 % of cuBLAS's measured bf16 rate).  A step of both tiles takes
// 1300 to 1600 cycles.  What is between that and the whole time: about 3000 cycles at the start and 4000 at the end of a block.
//
//   warps 0-3, 4-7   softmax and epilogue of tile 0, 1 (a warp reaches its own quarter of the TMEM lanes).  Two threads a row
//                    would keep the special-function unit 15 % busier, but the barrier and the bookkeeping that they need
//                    in every step cost more than that
//   warps 8, 9       issue the products of tile 0, 1
//   warp 10          TMA: query tiles, then K and V tiles through one ring; a paged tile is one box a page, its addresses looked
//                    up by the lanes side by side.  Rows behind the document's last key are zeroed in the V tile: they would
//                    meet P = 0, and 0 * NaN is NaN
// A hidden key INSIDE the document can still hold a NaN value.  It shows as a result that is not finite; such rows are computed
// again, one key at a time (local_row_forward).  The same happens to all rows of a CTA whose pipeline wait gave up.
//
// Few blocks (a chunk over a long cache): the key tiles of a block are cut over blockIdx.y; the parts leave normalised partial
// rows and their LSE in the workspace, and local_combine joins them.
#include "local_tc.cuh"

#include <type_traits>

namespace fm {

namespace {

using namespace ltc;

constexpr int kThreads = 384;
constexpr int kMmaWarp = 8, kLoadWarp = 10;         // warp 11 completes the third warpgroup: registers are split by warpgroup
constexpr int kStep = 64;                           // keys of a step: half a key tile
template <typename T> constexpr float kBelow = kNarrow<T> ? 3.f : 0.f;                    // what a reference lies below the maximum
template <typename T> constexpr float kMostSum = kNarrow<T> ? 32768.f : 4096.f;          // sum of a step's p from which it is renewed

template <int D> struct Cfg {
    static constexpr uint32_t kTileBytes = uint32_t(D / 64) * kBlock;
    static constexpr int kRing = D == 128 ? 5 : 8;  // K and V tiles in flight or in use
};

struct Block {
    Doc D;
    int h, tokens;                                  // KV head; tokens of a query tile
    int t0[2], t1[2];                               // tokens of each tile in the document, [t0, t1)
    int lo[2], hi[2];                               // steps (of 64 keys) of each tile behind the prefix's, [lo, hi)
    int pre_steps;                                  // steps of the prefix (seen by both)
    int n_pre, lo0;                                 // key tiles of the prefix; first one behind them that any tile sees
    int n0, n1;                                     // this CTA's part of the list of key tiles
    __device__ __forceinline__ int key_tile(int n) const { return n < n_pre ? n : lo0 + n - n_pre; }
};

// Which steps a query tile takes part in, as registers of one role.
struct Steps {
    int on, pre, lo, hi, n_pre, lo0;
    __device__ __forceinline__ Steps(const Block &b, int s)
        : on(uniform(b.t0[s] < b.t1[s])), pre(uniform(b.pre_steps)), lo(uniform(b.lo[s])), hi(uniform(b.hi[s])), n_pre(uniform(b.n_pre)), lo0(uniform(b.lo0)) {}
    // step u (0, 1) of tile n of the list, as its number among the document's steps
    __device__ __forceinline__ int step(int n, int u) const { return 2 * (n < n_pre ? n : lo0 + n - n_pre) + u; }
    __device__ __forceinline__ bool active(int n, int u) const
    {
        const int e = step(n, u);
        return on && (e < pre || (e >= lo && e < hi));
    }
};

template <int D> struct Shared {
    uint64_t q_full[2], full[Cfg<D>::kRing], empty[Cfg<D>::kRing], tail;
    uint64_t s_full[2][2], p_full[2][2], o_done[2][2], drain[2];
    uint32_t tmem_slot;
    int abort;
    Block b;
};
template <int D> constexpr uint32_t smem_bytes() { return (2 + Cfg<D>::kRing) * Cfg<D>::kTileBytes + uint32_t(sizeof(Shared<D>)); }

__device__ __forceinline__ void make_block(const LocalParams &p, Block &b, const Doc &doc, int index, int h, int part, int parts)
{
    b.D = doc;
    b.h = h;
    b.tokens = kTile / p.G;
    const int shift = b.D.nk - b.D.nq;
    b.n_pre = (b.D.prefix + kTile - 1) / kTile;
    b.pre_steps = (b.D.prefix + kStep - 1) / kStep;
    int first = 1 << 30, last = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        b.t0[s] = min((2 * index + s) * b.tokens, b.D.nq);
        b.t1[s] = min(b.t0[s] + b.tokens, b.D.nq);
        b.lo[s] = b.hi[s] = 0;
        if (b.t0[s] < b.t1[s]) {
            const int lo = local_run(p, shift + b.t0[s], b.D.nk).x, hi = local_run(p, shift + b.t1[s] - 1, b.D.nk).y;
            b.lo[s] = max(lo / kStep, b.pre_steps);
            b.hi[s] = hi > lo ? max((hi + kStep - 1) / kStep, b.lo[s]) : b.lo[s];
            if (b.hi[s] > b.lo[s]) { first = min(first, b.lo[s] / 2); last = max(last, (b.hi[s] + 1) / 2); }
        }
    }
    first = max(first, b.n_pre);                    // (a step that shares its tile with the prefix's last one is in that tile)
    b.lo0 = first;
    const int n = b.n_pre + max(last - first, 0);
    b.n0 = int(int64_t(n) * part / parts);
    b.n1 = int(int64_t(n) * (part + 1) / parts);
}

// Bits [0, x) of a word, for any x.
__device__ __forceinline__ uint32_t bits_below(int x) { return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u; }
// Column c is a visible key if it lies in [a, b) or below pre; the others become `hidden`.
__device__ __forceinline__ void mask_scores(uint32_t (&s)[32], int a, int b, int pre, uint32_t hidden)
{
    const uint32_t seen = (bits_below(b) & ~bits_below(a)) | bits_below(pre);
#pragma unroll
    for (int c = 0; c < 32; ++c) s[c] = (seen & (1u << c)) ? s[c] : hidden;
}

// Scores after scale, cap and distance (fp: the row's position less the first column's).  What is left to multiply them with to
// get log2 units (left_over): the cap if it comes last.
template <bool CAP, bool SLOPES>
__device__ __forceinline__ void shape_scores(const LocalParams &p, uint32_t (&s)[32], float slope2, float fp, bool valid)
{
    const float c2 = CAP ? p.cap * kLog2e : p.scale * kLog2e;
    f32x2 t[16];
    if constexpr (CAP) cap_scores(t, s, p.scale / p.cap, valid);
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        f32x2 e = CAP ? t[c] : pair(s[2 * c], s[2 * c + 1]);
        if constexpr (SLOPES) e = fma2(pair(-slope2, -slope2), pair(fabsf(fp - float(2 * c)), fabsf(fp - float(2 * c + 1))), mul2(e, pair(c2, c2)));
        const float2 v = split(e);
        s[2 * c] = __float_as_uint(v.x);
        s[2 * c + 1] = __float_as_uint(v.y);
    }
}
template <bool CAP, bool SLOPES> __device__ __forceinline__ float left_over(const LocalParams &p)
{
    return SLOPES ? 1.f : (CAP ? p.cap : p.scale) * kLog2e;
}

__device__ __forceinline__ float row_max(const uint32_t (&x)[32])
{
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 32; c += 2) mx[c >> 1 & 3] = max3(mx[c >> 1 & 3], __uint_as_float(x[c]), __uint_as_float(x[c + 1]));
    return max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
}

// P = 2^(s mul - sub) of 32 columns as packed 16-bit into TMEM; adds the unrounded p to sum.
template <typename T> __device__ __forceinline__ void exp_scores(const uint32_t (&x)[32], float mul, float sub, uint32_t t_p, f32x2 (&sum)[2])
{
    const f32x2 m2 = pair(mul, mul), n2 = pair(-sub, -sub);
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const f32x2 e = exp2_pair(fma2(pair(x[2 * i], x[2 * i + 1]), m2, n2));
        sum[i & 1] = add2(sum[i & 1], e);
        const float2 v = split(e);
        pk[i] = pack2<T>(v.x, v.y);
    }
    tc::tmem_st_x16(t_p, pk);
}
__device__ __forceinline__ float total(const f32x2 (&sum)[2])
{
    const float2 v = split(add2(sum[0], sum[1]));
    return v.x + v.y;
}

template <typename T, int D> __device__ __forceinline__ void redo_rows(const LocalParams &p, const Block &b, unsigned rows, int token0, int row0)
{
    while (rows) {
        const int r = row0 + __ffs(rows) - 1;
        rows &= rows - 1;
        local_row_forward<T, D>(p, b.D, b.h * p.G + r % p.G, token0 + r / p.G);
    }
}

template <typename T, int D, bool CAP, bool SLOPES>
__global__ void __launch_bounds__(kThreads, 1)
local_fwd_kernel(const __grid_constant__ LocalParams p, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o, uint32_t idesc_s, uint32_t idesc_o, float *part_o, float *part_lse)
{
    extern __shared__ __align__(1024) unsigned char smem_dyn[];
    using C = Cfg<D>;
    Shared<D> &sh = *reinterpret_cast<Shared<D> *>(smem_dyn + (2 + C::kRing) * C::kTileBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = tc::smem_addr(smem_dyn);
    const uint32_t ring0 = base + 2 * C::kTileBytes;
    volatile int *abort_flag = &sh.abort;

    const Block &b = sh.b;
    // The loading warp makes the barriers and the block and starts loading at once; everybody meets when it has filled the ring.
    auto meet = [&] {
        tc::fence_before_sync();
        tc::named_barrier(3, kThreads);
        tc::fence_after_sync();
    };
    if (warp == kLoadWarp) {
        if (lane == 0) {
            tc::prefetch_tensormap(&tm_q);
            tc::prefetch_tensormap(&tm_k);
            tc::prefetch_tensormap(&tm_v);
            for (int s = 0; s < 2; ++s) {
                tc::mbar_init(bar_addr(&sh.q_full[s]), 1);
                tc::mbar_init(bar_addr(&sh.drain[s]), 1);
                for (int u = 0; u < 2; ++u) {
                    tc::mbar_init(bar_addr(&sh.s_full[s][u]), 1);
                    tc::mbar_init(bar_addr(&sh.p_full[s][u]), 4);
                    tc::mbar_init(bar_addr(&sh.o_done[s][u]), 1);
                }
            }
            for (int i = 0; i < C::kRing; ++i) {
                tc::mbar_init(bar_addr(&sh.full[i]), 1);
                tc::mbar_init(bar_addr(&sh.empty[i]), 2);                          // both product warps let go of it
            }
            tc::mbar_init(bar_addr(&sh.tail), 1);
            tc::mbar_fence_init();
            sh.abort = 0;
        }
        // the last blocks of a document have the most keys (causal): they go first
        const int nb = gridDim.x / p.H;
        Doc doc;
        const int index = find_block<false>(p, 2 * (kTile / p.G), nb - 1 - int(blockIdx.x / p.H), doc);
        if (lane == 0) {
            if (index >= 0) make_block(p, sh.b, doc, index, blockIdx.x % p.H, blockIdx.y, gridDim.y);
            else sh.b = Block{};
        }
        __syncwarp();
    } else {
        if (warp == kMmaWarp) tc::tmem_alloc(tc::smem_addr(&sh.tmem_slot), 512);
        meet();
    }
    const int n0 = b.n0, n1 = b.n1;

    // 384 threads x 168 registers at launch = 256 x 216 + 128 x 72
    if (warp >= 8) {
        tc::set_registers_down<72>();
        if (warp == kLoadWarp) {
            // ---- loads ----------------------------------------------------------------------------------------------------
            int issued = 0;
            bool ok = true, met = false, tail_open = false;
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
                // lane x * (d / 64) + c loads column block c of the tile's box x; its page is looked up a tile ahead
                const int box = lane / (D / 64), col = lane % (D / 64);
                auto look_up = [&](int n) {
                    const int j = b.key_tile(n) * kTile + box * box_rows;
                    if (!p.table || n >= n1 || box >= boxes || j >= b.D.nk) return 0;
                    return min(max(p.table[int64_t(b.D.seq) * p.table_ld + (j >> p.page_shift)], 0), p.n_pages - 1);
                };
                int page_id = look_up(n0);
                for (int n = n0; n < n1 && ok; ++n) {
                    const int j0 = b.key_tile(n) * kTile, rows = b.D.nk - j0;      // rows of the tile that are keys of the document
                    const int live = rows >= kTile ? boxes : (rows + box_rows - 1) / box_rows;
                    const int next_id = look_up(n + 1);
                    const int y = p.table ? (j0 + box * box_rows) & (page - 1) : b.D.k0 + j0, z = p.table ? page_id * p.H + b.h : b.h;
                    for (int kv = 0; kv < 2; ++kv) {
                        const int slot = issued % C::kRing;
                        const bool cut = kv == 1 && rows < kTile;                  // a V tile whose last rows must be zeroed
                        const bool skip = issued == p.skip_tile;                   // never, but in a test
                        if (!met && (issued >= C::kRing || cut)) {
                            meet();
                            met = true;
                        }
                        if (issued >= C::kRing) ok = tc::mbar_wait_or_abort(bar_addr(&sh.empty[slot]), ((issued / C::kRing) & 1) ^ 1, abort_flag, p.wait_ns);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        const uint32_t dst = ring0 + slot * C::kTileBytes;
                        const uint32_t bar = bar_addr(cut ? &sh.tail : &sh.full[slot]);
                        if (lane == 0 && !skip) tc::mbar_arrive_expect_tx(bar, uint32_t(live) * box_rows * (D * 2));
                        __syncwarp();
                        if (box < live && !skip) tc::tma_load_3d(dst + col * kBlock + box * box_rows * 128, kv ? &tm_v : &tm_k, col * 64, y, z, bar);
                        if (cut && !skip) {                                        // at most once a CTA: the document's last tile
                            ok = tc::mbar_wait_or_abort(bar, 0, abort_flag, p.wait_ns);
                            ok = __all_sync(0xffffffffu, ok);
                            tail_open = !ok;
                            if (!ok) break;
                            for (int i = rows * 8 + lane; i < kTile * 8; i += 32)
#pragma unroll
                                for (int c = 0; c < D / 64; ++c)
                                    *reinterpret_cast<uint4 *>(smem_dyn + (dst - base) + c * kBlock + i * 16) = make_uint4(0, 0, 0, 0);
                            tc::fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) tc::mbar_arrive(bar_addr(&sh.full[slot]));
                        }
                        ++issued;
                    }
                    page_id = next_id;
                }
            }
            if (!met) meet();
            if (!ok && lane == 0) *abort_flag = 1;
            // whoever gave up: every copy in flight lands before the CTA's shared memory goes away
            for (int i = max(issued - C::kRing, 0); i < issued; ++i)
                if (i != p.skip_tile) tc::mbar_wait(bar_addr(&sh.full[i % C::kRing]), (i / C::kRing) & 1);
            if (tail_open) tc::mbar_wait(bar_addr(&sh.tail), 0);
            for (int s = 0; s < 2; ++s)
                if (n1 > n0 && b.t0[s] < b.t1[s]) tc::mbar_wait(bar_addr(&sh.q_full[s]), 0);
        } else if (warp < kLoadWarp && n1 > n0) {
            // ---- products of one query tile: S runs two steps ahead of P V -----------------------------------------------------
            const int s = warp - kMmaWarp, m0 = uniform(n0), m1 = uniform(n1);
            const uint32_t t_s = uniform(int(sh.tmem_slot)) + s * 128, t_o = t_s + 256;
            const Steps st(b, s);
            const bool leader = tc::elect_one();
            bool ok = true;                                                    // (what the leader's waits said; the others follow the same path)
            auto wait = [&](uint64_t *bar, int parity) { ok = ok && tc::mbar_wait_or_abort(bar_addr(bar), parity, abort_flag, p.wait_ns); };
            auto ring_wait = [&](int i) { wait(&sh.full[i % C::kRing], (i / C::kRing) & 1); };
            auto commit = [&](uint64_t *bar) { tc::umma_commit_if(leader && ok, bar_addr(bar)); };          // (nothing is announced once a wait gave up)
            const uint64_t q = desc_k(base + s * C::kTileBytes, 0);
            int sn = m0, su = 0, ns = 0, done = 0;                             // the step whose S comes next; steps issued, and multiplied with V
            // S up to two steps ahead, but no further than the tile behind `n`: the ring has to turn.  A key tile that is passed is let go of.
            auto scores = [&](int n) {
                while (ns - done < 2 && sn < m1 && sn <= n + 1) {
                    const int i = 2 * (sn - m0);
                    if (su == 0) ring_wait(i);
                    if (st.active(sn, su)) {
                        const uint64_t k = desc_k(ring0 + (i % C::kRing) * C::kTileBytes, 0) + uint32_t(su * (kStep * 128) >> 4);
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) tc::umma_f16_if(leader && ok, t_s + (ns & 1) * kStep, q + step_k(ks), k + step_k(ks), idesc_s, ks > 0);
                        commit(&sh.s_full[s][ns & 1]);
                        ++ns;
                    }
                    if (su == 1) commit(&sh.empty[i % C::kRing]);
                    sn += su;
                    su ^= 1;
                }
            };
            if (st.on) wait(&sh.q_full[s], 0);
            for (int n = m0; n < m1; ++n) {
                const int i = 2 * (n - m0) + 1;
                scores(n);
                ring_wait(i);
                const uint64_t v = desc_mn(ring0 + (i % C::kRing) * C::kTileBytes, 0);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (st.active(n, u)) {
                        const int buf = done & 1;
                        wait(&sh.p_full[s][buf], (done >> 1) & 1);
                        tc::fence_after_sync();
#pragma unroll
                        for (int ks = 0; ks < kStep / 16; ++ks)
                            tc::umma_f16_ts_if(leader && ok, t_o, t_s + buf * kStep + ks * 8, v + step_mn(u * (kStep / 16) + ks), idesc_o,
                                               done > 0 || ks > 0);
                        commit(&sh.o_done[s][buf]);
                        ++done;
                    }
                    if (u == 1) commit(&sh.empty[i % C::kRing]);
                    scores(n);
                }
            }
            if (leader && !ok) *abort_flag = 1;
            tc::umma_commit_if(leader, bar_addr(&sh.drain[s]));
            tc::mbar_wait(bar_addr(&sh.drain[s]), 0);
        }
    } else {
        tc::set_registers_up<216>();
        // ---- softmax and epilogue ---------------------------------------------------------------------------------------
        const int s = warp >> 2, row = tid & 127;
        const uint32_t t_s = sh.tmem_slot + s * 128 + (uint32_t((warp & 3) * 32) << 16), t_o = t_s + 256;
        const int token = b.t0[s] + row / p.G, head = b.h * p.G + row % p.G;
        const bool valid = row < b.tokens * p.G && token < b.t1[s];
        const int shift = b.D.nk - b.D.nq, pos = shift + token;
        const int safe_lo = p.window ? shift + b.t1[s] - p.window : 0;         // keys in [safe_lo, safe_hi) are seen by every row
        const int safe_hi = local_run(p, shift + b.t0[s], b.D.nk).y;
        constexpr bool shaped = CAP || SLOPES;
        const float mul = left_over<CAP, SLOPES>(p);                           // positive
        const float slope2 = p.slopes && valid ? p.slopes[head] * kLog2e : 0.f;
        const Steps st(b, s);
        float m = -INFINITY, l = 0.f;
        int done = 0;
        bool ok = true, fresh = true;                                          // fresh: a row of the warp has no reference yet
        for (int n = n0; n < n1 && ok; ++n)
#pragma unroll 1
            for (int u = 0; u < 2; ++u) {
                if (!st.active(n, u)) continue;
                const int j0 = st.step(n, u) * kStep, buf = done & 1;
                const uint32_t t_p = t_s + buf * kStep;                        // S of this step, then P
                ok = tc::mbar_wait_or_abort(bar_addr(&sh.s_full[s][buf]), (done >> 1) & 1, abort_flag);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc::fence_after_sync();
                uint32_t x[2][32];
                f32x2 sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                tc::tmem_ld_x32(t_p, x[0]);
                tc::tmem_ld_wait(x[0]);
                tc::tmem_ld_x32(t_p + 32, x[1]);
                const bool masked = !(j0 + kStep <= b.D.prefix || (j0 >= safe_lo && j0 + kStep <= safe_hi));
                if (!fresh && !masked) {
                    // the usual step: half of the scores arrive under the exponentials of the others
                    if constexpr (shaped) shape_scores<CAP, SLOPES>(p, x[0], slope2, float(pos - j0), valid);
                    exp_scores<T>(x[0], mul, m, t_p, sums);
                    tc::tmem_ld_wait(x[1]);
                    if constexpr (shaped) shape_scores<CAP, SLOPES>(p, x[1], slope2, float(pos - j0 - 32), valid);
                    exp_scores<T>(x[1], mul, m, t_p + 16, sums);
                } else {
                    tc::tmem_ld_wait(x[1]);
                    const int2 run = local_run(p, pos, b.D.nk);
                    auto mask = [&](uint32_t hidden) {
                        mask_scores(x[0], run.x - j0, run.y - j0, b.D.prefix - j0, hidden);
                        mask_scores(x[1], run.x - j0 - 32, run.y - j0 - 32, b.D.prefix - j0 - 32, hidden);
                    };
                    if constexpr (shaped) {
                        if (masked) mask(0u);                                  // (what is hidden must not cost the short formula)
                        shape_scores<CAP, SLOPES>(p, x[0], slope2, float(pos - j0), valid);
                        shape_scores<CAP, SLOPES>(p, x[1], slope2, float(pos - j0 - 32), valid);
                    }
                    if (masked) mask(0xff800000u);
                    if (fresh && m == -INFINITY) m = fmaxf(row_max(x[0]), row_max(x[1])) * mul - kBelow<T>;
                    fresh = __any_sync(0xffffffffu, m == -INFINITY);
                    const float sub = m == -INFINITY ? 0.f : m;
                    exp_scores<T>(x[0], mul, sub, t_p, sums);
                    exp_scores<T>(x[1], mul, sub, t_p + 16, sums);
                }
                float sum = total(sums);
                const bool grow = sum > kMostSum<T>;
                if (__any_sync(0xffffffffu, grow)) {                           // rows that have outgrown their reference get a new one
                    const float top = fmaxf(row_max(x[0]), row_max(x[1])) * mul - kBelow<T>, f = grow ? fast_exp2(m - top) : 1.f;
                    if (done > 0) {
                        // every product into O has finished: the next one waits for this step's P
                        ok = tc::mbar_wait_or_abort(bar_addr(&sh.o_done[s][buf ^ 1]), ((done - 1) >> 1) & 1, abort_flag);
                        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                        tc::fence_after_sync();
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
                    if (grow) { m = top; l *= f; }
                    const float sub = m == -INFINITY ? 0.f : m;
                    sums[0] = sums[1] = pair(0.f, 0.f);
                    exp_scores<T>(x[0], mul, sub, t_p, sums);
                    exp_scores<T>(x[1], mul, sub, t_p + 16, sums);
                    sum = total(sums);
                }
                l += sum;
                tc::tmem_st_wait();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(bar_addr(&sh.p_full[s][buf]));
                ++done;
            }
        if (ok && done > 0) ok = tc::mbar_wait_or_abort(bar_addr(&sh.o_done[s][(done - 1) & 1]), ((done - 1) >> 1) & 1, abort_flag);
        ok = tc::named_barrier_and(1 + s, 128, ok && !*abort_flag);            // the tile's warps go on together
        if (!ok) *abort_flag = 1;
        tc::fence_after_sync();
        const int64_t out_row = int64_t(head) * p.S + b.D.q0 + token;
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const float lse = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        bool fine = ok && l < INFINITY && l >= 0.f;
        // a whole tile goes out through the query tile's shared memory: with a step done, the products that read it have finished, so its
        // load has long landed.  A tile that sees no key waits for nothing, while its load (the block's other tile sees some)
        // may still be in flight: its zeros go straight out
        const bool whole = ok && gridDim.y == 1 && done > 0 && b.t1[s] - b.t0[s] == b.tokens;
        if (ok && b.t0[s] < b.t1[s]) {
            unsigned char *tile = smem_dyn + s * C::kTileBytes;
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
                if (gridDim.y == 1) {
                    T *dst = valid ? static_cast<T *>(p.o) + out_row * D : nullptr;
                    const bool good = put_row<T>(o, inv, whole ? tile : nullptr, dst, row, c * 32);
                    fine = fine && good;
                } else {
                    float worst = 0.f;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float f = __uint_as_float(o[i]) * inv;
                        o[i] = __float_as_uint(f);
                        worst = fmaf(f, 0.f, worst);
                    }
                    fine = fine && worst == 0.f;
                    if (valid) {
                        uint4 *dst = reinterpret_cast<uint4 *>(part_o + (int64_t(blockIdx.y) * p.Hq * p.S + out_row) * D + c * 32);
#pragma unroll
                        for (int i = 0; i < 8; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
        }
        if (gridDim.y == 1) {
            if (valid) p.lse[out_row] = lse;
            if (whole) tc::fence_proxy_async_smem();
            const bool any = tc::named_barrier_or(1 + s, 128, valid && !fine);
            if (whole && row == 0) {                                           // (the same thread waits for its stores)
                for (int c = 0; c < D / 64; ++c) tc::tma_store_4d(&tm_o, c * 64, 0, b.D.q0 + b.t0[s], b.h, base + s * C::kTileBytes + c * kBlock);
                tc::tma_store_commit();
                if (any) tc::tma_store_wait_all();
                else tc::tma_store_wait_read();
            }
            if (any) {
                tc::named_barrier(1 + s, 128);                                 // every row of the tile has been written
                const unsigned again = __ballot_sync(0xffffffffu, valid && !fine);
                if (again) redo_rows<T, D>(p, b, again, b.t0[s], row & ~31);
            }
        } else if (valid) {
            part_lse[int64_t(blockIdx.y) * p.Hq * p.S + out_row] = fine ? lse : __int_as_float(0x7fc00000);
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    if (warp == kMmaWarp) tc::tmem_dealloc(sh.tmem_slot, 512);
}

// Blocks of query tiles, at most, and the parts that their key tiles are cut into: only where the blocks fill less than half
// of the SMs, with at least two key tiles a part.
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
    if (s.blocks > 0 && s.blocks * 2 <= sm_count()) s.parts = int(std::max<int64_t>(1, std::min<int64_t>(sm_count() / s.blocks, tiles / 2)));
    return s;
}

template <typename T, int D> int launch(const LocalParams &p, int dtype, void *ws, cudaStream_t st)
{
    const Shape sh = shape_of(p);
    CUtensorMap tm_q, tm_k, tm_v, tm_o;
    if (int rc = local_query_map(&tm_q, p, p.q, p.q_sh, p.q_st, dtype)) return rc;
    if (int rc = local_key_map(&tm_k, p, p.k, p.k_sh, p.k_st, dtype)) return rc;
    if (int rc = local_key_map(&tm_v, p, p.v, p.v_sh, p.v_st, dtype)) return rc;
    if (int rc = local_query_map(&tm_o, p, p.o, int64_t(p.S) * D, D, dtype)) return rc;
    float *part_lse = static_cast<float *>(ws), *part_o = part_lse + (size_t(sh.parts) * p.Hq * p.S + 31) / 32 * 32;
    const bool bf16 = dtype == FM_BF16;
    auto launch_mode = [&](auto cap, auto slopes) -> int {
        auto *kernel = local_fwd_kernel<T, D, decltype(cap)::value, decltype(slopes)::value>;
        FM_CUDA_OK(func_attr_cached((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<D>()));
        kernel<<<dim3(unsigned(sh.blocks), unsigned(sh.parts)), kThreads, smem_bytes<D>(), st>>>(
            p, tm_q, tm_k, tm_v, tm_o, tc::instr_desc_f16(bf16, ltc::kTile, kStep), tc::instr_desc_f16(bf16, ltc::kTile, D, false, true), part_o, part_lse);
        FM_LAUNCHED("local_fwd_kernel");
        return FM_OK;
    };
    const bool slopes = p.slopes || (!(p.scale > 0.f) && !(p.cap > 0.f));      // the plain form needs scores that grow with the products
    const int rc = p.cap > 0.f ? (slopes ? launch_mode(std::true_type{}, std::true_type{}) : launch_mode(std::true_type{}, std::false_type{}))
                               : (slopes ? launch_mode(std::false_type{}, std::true_type{}) : launch_mode(std::false_type{}, std::false_type{}));
    if (rc) return rc;
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

// Keys as (d, row, KV head), or pages as (d, row of the page, page x head): a box is one tile of
// `rows` keys, or the part of it in one page.
int local_key_map(CUtensorMap *map, const LocalParams &p, const void *k, int64_t sh, int64_t st, int dtype, int rows)
{
    auto bytes = [](int64_t stride) { return uint64_t(stride > 0 ? stride * 2 : 16); };
    const int64_t page = int64_t(1) << p.page_shift;
    const uint64_t dims[3] = {uint64_t(p.d), uint64_t(p.table ? page : p.N), uint64_t(p.table ? int64_t(p.n_pages) * p.H : p.H)};
    const uint64_t strides[2] = {p.table ? uint64_t(p.d) * 2 : bytes(st), p.table ? uint64_t(page) * p.d * 2 : bytes(sh)};
    const uint32_t box[3] = {64, uint32_t(p.table ? std::min<int64_t>(page, rows) : rows), 1};
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
