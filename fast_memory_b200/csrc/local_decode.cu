// Local attention of few queries a document over many keys - single new tokens, short drafts -, 16-bit types, head dim 64 or 128.
//
// Bound by HBM: a block has at most 16 rows (token x head of the group), one m16n8k16 tile, and every key and value that a block sees
// is read once for all heads of its group; a document of more rows has several blocks, which read its keys each.  What matters is that every SM always has loads in flight and that all end together:
//   * the key tiles (64 keys) of all (document, KV head, row block) items form ONE list that is cut into equal stretches, one a CTA
//     and two CTAs an SM, wherever that falls; an item that is cut leaves normalised partial rows, which local_decode_join adds up
//     in a fixed order (no atomics)
//   * warp 4 walks the stretch with TMA into a ring of three tiles (32 KB of K and V each), across items; what a tile belongs to
//     travels in its slot
//   * warps 0-3 take 16 keys of a tile each: S = Q K^T, running maximum and sum of their own, O += P V in registers.  They meet
//     only at the end of an item, to add up their four partial rows through shared memory.
// mma.sync is enough here: a tile is 64 products a warp, ~500 cycles, against ~900 that an SM's share of HBM needs for two CTAs'
// tiles; on tcgen05 112 of the 128 rows of a product would be empty.
// P is rounded to the element type as the operand of the second product; sums are fp32.  In fp16 the reference of a row is 2^-15 of its
// running maximum, so that P fills the type's range: a weight is off by 2^-40 of the largest at most, or by its rounding.
// 64 sequences of up to 16384 tokens, 32 over 8 heads, d = 128: 366 us, 98 % of the measured copy rate; one of 131072: 91 us (90 %) and
// 6.5 us for the join.  The tcgen05 forward, its key tiles cut over CTAs, took 534 and 135 us.
#include "local_tc.cuh"

#include <type_traits>

namespace fm {

namespace {

using namespace ltc;

constexpr int kKeys = 64;                           // keys of a tile
constexpr int kRows = 16;
constexpr int kRing = 3;
constexpr int kThreads = 160;
constexpr int kMinTiles = 4;                        // a CTA's stretch is at least this long
template <typename T> constexpr float kBelow = kNarrow<T> ? 15.f : 0.f;

// What a tile of the list is: written by the loading warp into the tile's slot.
struct Piece {
    Doc D;
    int h, t0, t1;                                  // KV head; tokens [t0, t1) of the row block
    int j0;                                         // first key
    int first, last;                                // of the CTA's part of the item
    int starts, ends;                               // the item starts / ends inside the CTA's stretch
    int more;                                       // CTAs that hold the rest of it
};

// Left for local_decode_join by each CTA: the item that starts in it and goes on (or none).
struct Cut {
    Doc D;
    int h, t0, t1, more;                            // more = 0: none
};

template <int D> struct Shared {
    alignas(1024) unsigned char tile[kRing][2][D / 64][kKeys * 128];
    alignas(16) float rows[2][kRows][D];            // partial rows on their way to another warp (not padded: two CTAs fit an SM to the byte)
    float m[2][kRows], l[2][kRows];
    uint64_t full[kRing], empty[kRing];
    Piece piece[kRing];
    int abort;
};

// Tiles and row blocks of a document: the tiles that any of its queries sees.
struct DocTiles {
    int blocks, n_pre, lo, n;
    __device__ __forceinline__ DocTiles(const LocalParams &p, const Doc &D)
    {
        const int tokens = kRows / p.G;
        blocks = (D.nq + tokens - 1) / tokens;
        n_pre = (D.prefix + kKeys - 1) / kKeys;
        const int a = local_run(p, D.nk - D.nq, D.nk).x, b = local_run(p, D.nk - 1, D.nk).y;
        lo = max(a / kKeys, n_pre);
        n = n_pre + (b > a ? max((b + kKeys - 1) / kKeys - lo, 0) : 0);
        n = max(n, 1);                              // an item without keys has one (hidden) tile, which writes its rows
    }
    __device__ __forceinline__ int tile(int i) const { return i < n_pre ? i : lo + i - n_pre; }
};

// A place in the list of tiles: document, (row block x KV head) of it, tile of that.
struct Walk {
    Doc d;
    int t, item, i, n, blocks, n_pre, lo;
    __device__ __forceinline__ void enter(const LocalParams &p, int doc)
    {
        t = doc;
        d = local_doc(p, t);
        const DocTiles x(p, d);
        n = x.n; blocks = x.blocks; n_pre = x.n_pre; lo = x.lo;
    }
    // Place number `a` of the list, by a whole warp; n_all: documents and what lies behind them.
    __device__ __forceinline__ void find(const LocalParams &p, int n_all, long long a)
    {
        const int lane = threadIdx.x & 31;
        long long before = 0;
        int at = 0;
        for (int t0 = 0; t0 < n_all; t0 += 32) {
            const long long mine = t0 + lane < n_all ? tiles_of(p, t0 + lane) : 0;
            long long s = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += y;
            }
            const long long total = __shfl_sync(0xffffffffu, s, 31);
            if (a < before + total) {
                const int l = __ffs(__ballot_sync(0xffffffffu, a < before + s)) - 1;
                at = t0 + l;
                before += __shfl_sync(0xffffffffu, s - mine, l);
                break;
            }
            before += total;
        }
        enter(p, at);
        const long long rest = a - before;
        item = int(rest / n);
        i = int(rest % n);
    }
    __device__ __forceinline__ static long long tiles_of(const LocalParams &p, int doc)
    {
        const Doc d = local_doc(p, doc);
        if (d.nq == 0) return 0;
        const DocTiles x(p, d);
        return (long long)x.n * x.blocks * p.H;
    }
    // The next place; there has to be one.
    __device__ __forceinline__ void next(const LocalParams &p)
    {
        if (++i < n) return;
        i = 0;
        if (++item < blocks * p.H) return;
        item = 0;
        int doc = t;
        do enter(p, ++doc); while (d.nq == 0);
    }
    // What the place is to a CTA whose stretch has `count` places of which this is number `done`.
    __device__ __forceinline__ Piece piece(const LocalParams &p, int done, int count, long long per) const
    {
        const int tokens = kRows / p.G;
        Piece q;
        q.D = d;
        q.h = item % p.H;
        q.t0 = item / p.H * tokens;
        q.t1 = min(q.t0 + tokens, d.nq);
        q.j0 = (i < n_pre ? i : lo + i - n_pre) * kKeys;
        q.first = i == 0 || done == 0;
        q.last = i == n - 1 || done == count - 1;
        q.starts = i == 0;
        q.ends = i == n - 1;
        q.more = int((n - 1 - i + per - 1) / per);
        return q;
    }
};

template <typename T, int D, bool CAP, bool SLOPES>
__global__ void __launch_bounds__(kThreads, 2)
local_decode_kernel(const __grid_constant__ LocalParams p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    float *part_o, float *part_lse, Cut *cuts)
{
    extern __shared__ __align__(1024) unsigned char smem_dyn[];
    Shared<D> &sh = *reinterpret_cast<Shared<D> *>(smem_dyn);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
    volatile int *abort_flag = &sh.abort;
    if (tid == 128) {
        tc::prefetch_tensormap(&tm_k);
        tc::prefetch_tensormap(&tm_v);
        for (int i = 0; i < kRing; ++i) {
            tc::mbar_init(bar_addr(&sh.full[i]), 1);
            tc::mbar_init(bar_addr(&sh.empty[i]), 4);
        }
        tc::mbar_fence_init();
        sh.abort = 0;
        cuts[cta].more = 0;
    }
    const int n_all = p.n_docs + (p.cu_q ? 1 : 0);  // with what lies behind the last document
    // every warp finds the CTA's stretch [a, b) of the list
    long long tiles = 0;
    for (int t = lane; t < n_all; t += 32) tiles += Walk::tiles_of(p, t);
#pragma unroll
    for (int o = 16; o; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    const long long per = max((tiles + gridDim.x - 1) / gridDim.x, (long long)kMinTiles), a = min(per * cta, tiles), b = min(a + per, tiles);
    __syncthreads();
    const int count = int(b - a);
    if (count <= 0) return;

    if (warp == 4) {
        // ---- loads ------------------------------------------------------------------------------------------------------------
        const int page = p.table ? 1 << p.page_shift : kKeys, boxes = page >= kKeys ? 1 : kKeys / page, box_rows = min(page, kKeys);
        const int box = lane / (D / 64), col = lane % (D / 64);
        Walk at;
        at.find(p, n_all, a);
        bool ok = true;
        int done = 0;
        for (; done < count; ++done) {
            if (done) at.next(p);
            const Piece q = at.piece(p, done, count, per);
            const int slot = done % kRing, rows = q.D.nk - q.j0;
            const int live = rows >= kKeys ? boxes : max(0, (rows + box_rows - 1) / box_rows);
            int y = q.D.k0 + q.j0, z = q.h;
            if (p.table && box < live) {
                const int j = q.j0 + box * box_rows;
                z = min(max(p.table[int64_t(q.D.seq) * p.table_ld + (j >> p.page_shift)], 0), p.n_pages - 1) * p.H + q.h;
                y = j & (page - 1);
            }
            if (done >= kRing) ok = tc::mbar_wait_or_abort(bar_addr(&sh.empty[slot]), ((done / kRing) & 1) ^ 1, abort_flag, p.wait_ns);
            if (!__all_sync(0xffffffffu, ok)) break;
            if (done == p.skip_tile) continue;                                 // never, but in a test
            if (lane == 0) {
                sh.piece[slot] = q;
                tc::mbar_arrive_expect_tx(bar_addr(&sh.full[slot]), 2u * uint32_t(live) * box_rows * (D * 2));
            }
            __syncwarp();
            if (box < live) {
                tc::tma_load_3d(tc::smem_addr(&sh.tile[slot][0][col][box * box_rows * 128]), &tm_k, col * 64, y, z, bar_addr(&sh.full[slot]));
                tc::tma_load_3d(tc::smem_addr(&sh.tile[slot][1][col][box * box_rows * 128]), &tm_v, col * 64, y, z, bar_addr(&sh.full[slot]));
            }
        }
        if (!ok && lane == 0) *abort_flag = 1;
        // nothing may still be in flight when the CTA goes
        for (int s = max(done - kRing, 0); s < done; ++s)
            if (s != p.skip_tile) tc::mbar_wait(bar_addr(&sh.full[s % kRing]), (s / kRing) & 1);
        return;
    }

    // ---- 16 keys of every tile ------------------------------------------------------------------------------------------------
    const int quad = lane >> 2, pos2 = (lane & 3) * 2;                         // this thread: rows quad and quad + 8, columns pos2, pos2 + 1 of 8
    const float mul = CAP || SLOPES ? 1.f : p.scale * kLog2e;
    uint32_t q[D / 16][4];
    float o[D / 8][4], m[2], l[2], slope2[2];
    int2 run[2];
    int pos[2];
    bool valid[2] = {false, false}, started = false;
    for (int it = 0; it < count; ++it) {
        const int slot = it % kRing;
        bool ok = tc::mbar_wait_or_abort(bar_addr(&sh.full[slot]), (it / kRing) & 1, abort_flag, p.wait_ns);
        ok = tc::named_barrier_and(1, 128, ok);                                // (the warps leave together, or not at all)
        if (!ok) {
            // a wait gave up: the rest of the stretch goes row by row, parts of cut items by way of local_decode_join
            *abort_flag = 1;
            Walk at;
            at.find(p, n_all, a);
            bool from_start = false;
            for (int k = 0; k < count; ++k) {
                if (k) at.next(p);
                const Piece x = at.piece(p, k, count, per);
                if (x.first) from_start = x.starts;
                if (!x.last) continue;
                if (from_start && x.ends) {
                    for (int r = warp; r < (x.t1 - x.t0) * p.G; r += 4) local_row_forward<T, D>(p, x.D, x.h * p.G + r % p.G, x.t0 + r / p.G);
                } else if (warp == 0) {
                    if (lane < kRows) part_lse[(int64_t(cta) * 2 + (from_start ? 1 : 0)) * kRows + lane] = __int_as_float(0x7fc00000);
                    if (from_start && lane == 0) cuts[cta] = Cut{x.D, x.h, x.t0, x.t1, x.more};
                }
            }
            return;
        }
        const Piece &pc = sh.piece[slot];
        const int first = pc.first, last = pc.last, j0 = pc.j0;
        if (first) {
            started = pc.starts;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = quad + 8 * i, token = pc.t0 + r / p.G, head = pc.h * p.G + r % p.G;
                valid[i] = r < kRows / p.G * p.G && token < pc.t1;
                pos[i] = pc.D.nk - pc.D.nq + token;
                run[i] = valid[i] ? local_run(p, pos[i], pc.D.nk) : make_int2(0, 0);
                slope2[i] = SLOPES && p.slopes && valid[i] ? p.slopes[head] * kLog2e : 0.f;
                m[i] = -INFINITY;
                l[i] = 0.f;
                const T *src = static_cast<const T *>(p.q) + int64_t(head) * p.q_sh + int64_t(pc.D.q0 + token) * p.q_st;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    q[k][i] = valid[i] ? *reinterpret_cast<const uint32_t *>(src + k * 16 + pos2) : 0u;
                    q[k][i + 2] = valid[i] ? *reinterpret_cast<const uint32_t *>(src + k * 16 + 8 + pos2) : 0u;
                }
            }
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[c][i] = 0.f;
        }
        // S: two blocks of eight keys
        const uint32_t kt = tc::smem_addr(sh.tile[slot][0]), vt = tc::smem_addr(sh.tile[slot][1]);
        float s[2][4] = {};
        {
            const int r = warp * 16 + (lane & 7) + ((lane & 16) >> 1), odd = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                uint32_t f[4];                                                 // keys 0-7: k, k + 8; keys 8-15: k, k + 8
                const int c = 2 * k + odd;
                ldmatrix_x4(f, kt + (c >> 3) * (kKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                mma16816<T>(s[0], q[k], f[0], f[1]);
                mma16816<T>(s[1], q[k], f[2], f[3]);
            }
        }
        const int key0 = j0 + warp * 16 + pos2;
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = e >> 1, j = key0 + n * 8 + (e & 1);
                float x = s[n][e];
                if (CAP) x = p.cap * kLog2e * tanh_any(x * (p.scale / p.cap));
                else if (SLOPES) x *= p.scale * kLog2e;
                if (SLOPES) x -= slope2[i] * fabsf(float(pos[i] - j));
                if (!((j >= run[i].x && j < run[i].y) || (j < pc.D.prefix && valid[i]))) x = -INFINITY;
                s[n][e] = x;
                top[i] = fmaxf(top[i], x);
            }
        float f[2], sub[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
            const float mn = fmaxf(m[i], top[i] * mul - kBelow<T>);
            sub[i] = mn == -INFINITY ? 0.f : mn;
            f[i] = fast_exp2(m[i] - sub[i]);
            m[i] = mn;
            l[i] *= f[i];
        }
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
            for (int c = 0; c < D / 8; ++c) {
                o[c][0] *= f[0];
                o[c][1] *= f[0];
                o[c][2] *= f[1];
                o[c][3] *= f[1];
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = fast_exp2(fmaf(s[n][e], mul, -sub[e >> 1]));
                l[e >> 1] += s[n][e];
            }
        const uint32_t pa[4] = {pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]), pack2<T>(s[1][0], s[1][1]), pack2<T>(s[1][2], s[1][3])};
        // rows behind the last key would meet P = 0, and 0 * NaN is NaN
        if (j0 + warp * 16 + 16 > pc.D.nk) {
            const int live = max(pc.D.nk - j0 - warp * 16, 0);
            for (int x = lane; x < (16 - live) * 8 * (D / 64); x += 32) {
                const int c = x % (8 * (D / 64)), r = warp * 16 + live + x / (8 * (D / 64));
                *reinterpret_cast<uint4 *>(&sh.tile[slot][1][c >> 3][r * 128 + (c & 7) * 16]) = make_uint4(0, 0, 0, 0);
            }
            tc::fence_proxy_async_smem();                                      // (the slot's next load comes behind these stores)
            __syncwarp();
        }
        {
            const int r = warp * 16 + (lane & 15), odd = lane >> 4;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
                uint32_t b[4];
                const int ch = 2 * c + odd;
                ldmatrix_x4_trans(b, vt + (ch >> 3) * (kKeys * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                mma16816<T>(o[2 * c], pa, b[0], b[1]);
                mma16816<T>(o[2 * c + 1], pa, b[2], b[3]);
            }
        }
        if (!last) {
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar_addr(&sh.empty[slot]));
            continue;
        }
        // ---- the end of (this CTA's part of) an item: four partial rows become one -------------------------------------------------
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
#pragma unroll
        for (int half = 2; half; half >>= 1) {                                 // warps 2, 3 -> 0, 1; warp 1 -> 0
            if (warp >= half && warp < 2 * half) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = quad + 8 * i;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c)
                        *reinterpret_cast<float2 *>(&sh.rows[warp - half][r][c * 8 + pos2]) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
                    if ((lane & 3) == 0) {
                        sh.m[warp - half][r] = m[i];
                        sh.l[warp - half][r] = l[i];
                    }
                }
            }
            tc::named_barrier(1, 128);
            if (warp < half) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = quad + 8 * i;
                    const float m2 = sh.m[warp][r], mn = fmaxf(m[i], m2), ref = mn == -INFINITY ? 0.f : mn;
                    const float f1 = fast_exp2(m[i] - ref), f2 = fast_exp2(m2 - ref);
                    m[i] = mn;
                    l[i] = l[i] * f1 + sh.l[warp][r] * f2;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        const float2 v = *reinterpret_cast<const float2 *>(&sh.rows[warp][r][c * 8 + pos2]);
                        o[c][2 * i] = o[c][2 * i] * f1 + v.x * f2;
                        o[c][2 * i + 1] = o[c][2 * i + 1] * f1 + v.y * f2;
                    }
                }
            }
            tc::named_barrier(1, 128);
        }
        if (warp == 0) {
            const bool whole = started && pc.ends;
            const int64_t part = (int64_t(cta) * 2 + (started ? 1 : 0)) * kRows;
            unsigned again = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = quad + 8 * i, token = pc.t0 + r / p.G, head = pc.h * p.G + r % p.G;
                const float inv = l[i] > 0.f ? 1.f / l[i] : (l[i] == 0.f ? 0.f : l[i]);
                const float lse = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
                float worst = l[i] * 0.f;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    o[c][2 * i] *= inv;
                    o[c][2 * i + 1] *= inv;
                    worst = fmaf(o[c][2 * i], 0.f, fmaf(o[c][2 * i + 1], 0.f, worst));
                }
                worst += __shfl_xor_sync(0xffffffffu, worst, 1);
                worst += __shfl_xor_sync(0xffffffffu, worst, 2);
                const int64_t row = int64_t(head) * p.S + pc.D.q0 + token;
                if (whole && valid[i]) {
                    T *dst = static_cast<T *>(p.o) + row * D;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint32_t *>(dst + c * 8 + pos2) = pack2<T>(o[c][2 * i], o[c][2 * i + 1]);
                    if ((lane & 3) == 0) p.lse[row] = lse;
                } else if (!whole) {
                    float *dst = part_o + (part + r) * D;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) *reinterpret_cast<float2 *>(dst + c * 8 + pos2) = make_float2(o[c][2 * i], o[c][2 * i + 1]);
                    if ((lane & 3) == 0) part_lse[part + r] = worst == 0.f ? lse : __int_as_float(0x7fc00000);
                }
                const unsigned bad = __ballot_sync(0xffffffffu, whole && valid[i] && worst != 0.f && (lane & 3) == 0);
                for (int k = 0; k < 8; ++k) again |= (bad >> (4 * k) & 1u) << (8 * i + k);
            }
            if (started && !pc.ends && lane == 0) cuts[cta] = Cut{pc.D, pc.h, pc.t0, pc.t1, pc.more};
            __syncwarp();
            while (again) {
                const int r = __ffs(again) - 1;
                again &= again - 1;
                local_row_forward<T, D>(p, pc.D, pc.h * p.G + r % p.G, pc.t0 + r / p.G);
            }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(bar_addr(&sh.empty[slot]));
    }
}

// CTA c joins the item that started in CTA c of the other kernel and went on in the `more` CTAs behind it.  The warps are dealt out
// to its rows; those of one row take every n-th part and are added up in their order.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kRows) local_decode_join(const __grid_constant__ LocalParams p, const float *part_o, const float *part_lse, const Cut *cuts)
{
    __shared__ float sums[kRows][D];
    __shared__ float totals[kRows];
    const Cut cut = cuts[blockIdx.x];
    if (cut.more == 0) return;
    const int rows = (cut.t1 - cut.t0) * p.G, n = kRows / rows;                // warps a row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = warp % rows, mine = warp / rows;
    const int token = cut.t0 + r / p.G, head = cut.h * p.G + r % p.G;
    auto slot = [&](int i) { return (int64_t(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kRows + r; };
    float m = -INFINITY;
    bool bad = false;
    for (int i = lane; i <= cut.more; i += 32) {
        const float x = part_lse[slot(i)];
        bad = bad || x != x;
        m = fmaxf(m, x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    bad = __any_sync(0xffffffffu, bad);
    constexpr int N = D / 32;
    float acc[N] = {}, total = 0.f;
    if (mine < n && m > -INFINITY && !bad) {
#pragma unroll 8
        for (int i = mine; i <= cut.more; i += n) {                            // (parts that saw nothing are zero)
            const float w = expf(part_lse[slot(i)] - m);
            const float *src = part_o + slot(i) * D + lane * N;
            total += w;
#pragma unroll
            for (int c = 0; c < N; ++c) acc[c] = fmaf(w, src[c], acc[c]);
        }
    }
#pragma unroll
    for (int c = 0; c < N; ++c) sums[warp][lane * N + c] = acc[c];
    if (lane == 0) totals[warp] = total;
    __syncthreads();
    if (mine > 0) return;
    if (bad) {
        local_row_forward_call<T, D>(p, cut.D, head, token);
        return;
    }
    for (int i = 1; i < n; ++i) {
        total += totals[r + i * rows];
#pragma unroll
        for (int c = 0; c < N; ++c) acc[c] += sums[r + i * rows][lane * N + c];
    }
    const float inv = total > 0.f ? 1.f / total : 0.f;
    const int64_t row = int64_t(head) * p.S + cut.D.q0 + token;
    T *dst = static_cast<T *>(p.o) + row * D + lane * N;
#pragma unroll
    for (int c = 0; c < N; ++c) dst[c] = Elem<T>::from_f32(acc[c] * inv);
    if (lane == 0) p.lse[row] = total > 0.f ? m + logf(total) : -INFINITY;
}

struct Space {
    int ctas;
    size_t lse, o, bytes;                           // offsets: the cuts come first
};
Space space_of(const LocalParams &p)
{
    Space s;
    s.ctas = 2 * sm_count();
    s.lse = align_up(size_t(s.ctas) * sizeof(Cut), 256);
    s.o = s.lse + align_up(size_t(s.ctas) * 2 * kRows * sizeof(float), 256);
    s.bytes = s.o + size_t(s.ctas) * 2 * kRows * p.d * sizeof(float);
    return s;
}

template <typename T, int D> int launch(const LocalParams &p, int dtype, void *ws, cudaStream_t st)
{
    const Space s = space_of(p);
    CUtensorMap tm_k, tm_v;
    if (int rc = local_key_map(&tm_k, p, p.k, p.k_sh, p.k_st, dtype, kKeys)) return rc;
    if (int rc = local_key_map(&tm_v, p, p.v, p.v_sh, p.v_st, dtype, kKeys)) return rc;
    char *base = static_cast<char *>(ws);
    Cut *cuts = reinterpret_cast<Cut *>(base);
    float *part_lse = reinterpret_cast<float *>(base + s.lse), *part_o = reinterpret_cast<float *>(base + s.o);
    auto launch_mode = [&](auto cap, auto slopes) -> int {
        auto *kernel = local_decode_kernel<T, D, decltype(cap)::value, decltype(slopes)::value>;
        FM_CUDA_OK(func_attr_cached((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared<D>)));
        kernel<<<unsigned(s.ctas), kThreads, sizeof(Shared<D>), st>>>(p, tm_k, tm_v, part_o, part_lse, cuts);
        FM_LAUNCHED("local_decode_kernel");
        return FM_OK;
    };
    const bool slopes = p.slopes || !(p.scale > 0.f);
    const int rc = p.cap > 0.f ? (slopes ? launch_mode(std::true_type{}, std::true_type{}) : launch_mode(std::true_type{}, std::false_type{}))
                               : (slopes ? launch_mode(std::false_type{}, std::true_type{}) : launch_mode(std::false_type{}, std::false_type{}));
    if (rc) return rc;
    local_decode_join<T, D><<<unsigned(s.ctas), 32 * kRows, 0, st>>>(p, part_o, part_lse, cuts);
    FM_LAUNCHED("local_decode_join");
    return FM_OK;
}

}  // namespace

// Up to 16 rows a document on average, which is all that the host knows: a row block of the other kernel would be seven eighths empty.  64
// documents of one token over 8192 keys, 32 over 8 heads: 374 us, the other 429; of 4 tokens 374 and 433; of 8 tokens (two blocks) 668
// and 434.  The mean misses unequal documents: 300 single tokens over 2048 keys beside a prompt of 3500 over 8192, 8 heads,
// take 1393 us here and would take 690 there; 63 single tokens beside a chunk of 1024 go there, 549 us (here 1425).
bool local_decode_fits(const LocalParams &p, int dtype)
{
    return local_tc_fits(p, dtype) && p.G <= kRows && int64_t(p.S) * p.G <= int64_t(kRows) * p.n_docs;
}

size_t local_decode_workspace(const LocalParams &p) { return space_of(p).bytes; }

int local_decode_fwd(const LocalParams &p, int dtype, void *ws, cudaStream_t st)
{
    if (dtype == FM_BF16) return p.d == 128 ? launch<__nv_bfloat16, 128>(p, dtype, ws, st) : launch<__nv_bfloat16, 64>(p, dtype, ws, st);
    return p.d == 128 ? launch<__half, 128>(p, dtype, ws, st) : launch<__half, 64>(p, dtype, ws, st);
}

}  // namespace fm
