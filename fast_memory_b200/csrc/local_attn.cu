// Local attention: entry points, the kernels around the tiled ones (delta, joining of key parts), and the backward pass a row
// a warp for head dim 256 (local_attn.cuh has the mathematics).
//
// The row kernels hold a query (or a key) in registers and walk the runs of visible rows, one dot product and one shuffle
// reduction a pair: no tiles, no masks, fp32 throughout.
#include "local_tc.cuh"

namespace fm {

namespace {

constexpr int kRowThreads = 256;

// One warp a row: the parts' rows weighted by e^(lse_part - max).  A part that was not finite sends the row through
// local_row_forward, whose registers (64) must not decide how many rows an SM works on: 777 tokens of 8 heads 4.5 us, with 64 registers 5.7.
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads, 6) local_combine_kernel(const __grid_constant__ LocalParams p, const float *part_o, const float *part_lse, int parts)
{
    const int64_t row = (int64_t(blockIdx.x) * kRowThreads + threadIdx.x) >> 5, rows = int64_t(p.Hq) * p.S;
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    bool bad = false;
    for (int i = lane; i < parts; i += 32) {
        const float x = part_lse[i * rows + row];
        bad = bad || x != x;
        m = fmaxf(m, x);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (__any_sync(0xffffffffu, bad)) {
        const int r = int(row % p.S);
        const Doc doc = local_doc(p, p.cu_q ? local_find(p.cu_q, p.n_docs, r) : p.table ? r : 0);
        local_row_forward_call<T, D>(p, doc, int(row / p.S), r - doc.q0);
        return;
    }
    constexpr int N = (D + 31) / 32;                                           // N consecutive columns a lane
    if (lane * N >= D) return;
    float acc[N] = {}, total = 0.f;
    if (m > -INFINITY)
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {                                       // (parts that saw nothing are zero)
            const float w = expf(part_lse[i * rows + row] - m);
            total += w;
            const float *src = part_o + (i * rows + row) * D + lane * N;
#pragma unroll
            for (int c = 0; c < N; ++c) acc[c] = fmaf(w, src[c], acc[c]);
        }
    const float inv = total > 0.f ? 1.f / total : 0.f;
    T *dst = static_cast<T *>(p.o) + row * D + lane * N;
#pragma unroll
    for (int c = 0; c < N; ++c) dst[c] = Elem<T>::from_f32(acc[c] * inv);
    if (lane == 0) p.lse[row] = total > 0.f ? m + logf(total) : -INFINITY;
}

// delta[row] = dO . O - d_lse.  range (fp16 on the tensor cores): the larger of 8 max |dO| and |delta| of a row that sees a key, else 0.
// 16 bytes a lane, as many lanes a row as that takes; bound by HBM, so that a lane has the loads of
// several rows in flight (32 heads of 8192 rows, d = 128, bf16: 22.8 us, 90 % of the measured copy rate; a row at a time 26.5).
constexpr int kDeltaRows = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) local_delta_kernel(LocalParams p, BwdParams g, const T *o, const float *d_lse, float *delta, float *range)
{
    constexpr int E = 16 / sizeof(T), L = D / E < 32 ? D / E : 32, M = D / (E * L);      // elements a load, lanes a row, loads a lane and row
    const int64_t rows = int64_t(p.Hq) * p.S, w0 = (int64_t(blockIdx.x) * kRowThreads + threadIdx.x) / L * kDeltaRows;
    const int lane = threadIdx.x % L;
    uint4 u[kDeltaRows][M], v[kDeltaRows][M];
#pragma unroll
    for (int r = 0; r < kDeltaRows; ++r) {
        const unsigned w = unsigned(min(w0 + r, rows - 1));                    // (fewer than 2^31 rows)
        const T *a = o + int64_t(w) * D, *b = static_cast<const T *>(g.dout) + int64_t(w / p.S) * g.do_sh + int64_t(w % p.S) * g.do_st;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            u[r][m] = *reinterpret_cast<const uint4 *>(a + (m * L + lane) * E);
            v[r][m] = *reinterpret_cast<const uint4 *>(b + (m * L + lane) * E);
        }
    }
#pragma unroll
    for (int r = 0; r < kDeltaRows; ++r) {
        float x = 0.f;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const T *s = reinterpret_cast<const T *>(&u[r][m]), *t = reinterpret_cast<const T *>(&v[r][m]);
#pragma unroll
            for (int i = 0; i < E; ++i) x = fmaf(Elem<T>::to_f32(s[i]), Elem<T>::to_f32(t[i]), x);
        }
#pragma unroll
        for (int i = L / 2; i; i >>= 1) x += __shfl_xor_sync(0xffffffffu, x, i);
        if (lane == 0 && w0 + r < rows) {
            if (d_lse) x -= d_lse[w0 + r];
            delta[w0 + r] = x;
        }
        if constexpr (std::is_same<T, __half>::value) {
            if (range) {
                float top = 0.f;
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    const T *t = reinterpret_cast<const T *>(&v[r][m]);
#pragma unroll
                    for (int i = 0; i < E; ++i) top = fmaxf(top, fabsf(Elem<T>::to_f32(t[i])));
                }
#pragma unroll
                for (int i = L / 2; i; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
                if (lane == 0 && w0 + r < rows) {
                    top = fmaxf(8.f * top, fabsf(x));
                    range[w0 + r] = g.lse[w0 + r] > -INFINITY && top < INFINITY ? top : 0.f;
                }
            }
        }
    }
}

template <typename T, int D> __global__ void __launch_bounds__(kRowThreads) local_rows_dq_kernel(LocalParams p, BwdParams g)
{
    const int64_t w = (int64_t(blockIdx.x) * kRowThreads + threadIdx.x) >> 5;
    if (w >= int64_t(p.Hq) * p.S) return;
    const int head = int(w / p.S), r = int(w % p.S);
    const Doc doc = local_doc(p, p.cu_q ? local_find(p.cu_q, p.n_docs, r) : 0);
    local_row_dq<T, D>(p, g, doc, head, r - doc.q0);
}

template <typename T, int D> __global__ void __launch_bounds__(kRowThreads) local_rows_dkv_kernel(LocalParams p, BwdParams g)
{
    const int64_t w = (int64_t(blockIdx.x) * kRowThreads + threadIdx.x) >> 5;
    if (w >= int64_t(p.H) * p.N) return;
    const int h = int(w / p.N), r = int(w % p.N);
    const Doc doc = local_doc<true>(p, p.cu_k ? local_find(p.cu_k, p.n_docs, r) : 0);
    local_row_dkv<T, D>(p, g, doc, h, r - doc.k0);
}

inline unsigned row_grid(int64_t rows) { return unsigned(ceil_div(rows * 32, kRowThreads)); }

}  // namespace

int local_combine(const LocalParams &p, int dtype, const float *part_o, const float *part_lse, int parts, cudaStream_t st)
{
    return with_type_and_dim(dtype, p.d, [&](auto t, auto dim) -> int {
        local_combine_kernel<decltype(t), decltype(dim)::value><<<row_grid(int64_t(p.Hq) * p.S), kRowThreads, 0, st>>>(p, part_o, part_lse, parts);
        FM_LAUNCHED("local_combine_kernel");
        return FM_OK;
    });
}

int local_rows_bwd(const LocalParams &p, const BwdParams &g, int dtype, cudaStream_t st)
{
    constexpr int D = 256;
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        if (p.S > 0) {
            local_rows_dq_kernel<T, D><<<row_grid(int64_t(p.Hq) * p.S), kRowThreads, 0, st>>>(p, g);
            FM_LAUNCHED("local_rows_dq_kernel");
        }
        if (p.N > 0) {
            local_rows_dkv_kernel<T, D><<<row_grid(int64_t(p.H) * p.N), kRowThreads, 0, st>>>(p, g);
            FM_LAUNCHED("local_rows_dkv_kernel");
        }
        return FM_OK;
    });
}

static int local_params(const fm_local_attn_args *a, LocalParams &p)
{
    FM_REQUIRE(a, "local attention: null arguments");
    FM_REQUIRE(a->dtype == FM_F32 || a->dtype == FM_BF16 || a->dtype == FM_F16, "local attention: unknown element type %d", a->dtype);
    FM_REQUIRE(a->n_q_rows >= 0 && a->n_q_rows < (int64_t(1) << 30) && a->n_k_rows >= 0 && a->n_k_rows < (int64_t(1) << 30),
               "local attention: bad row counts %lld, %lld", (long long)a->n_q_rows, (long long)a->n_k_rows);
    FM_REQUIRE(a->n_kv_heads > 0 && a->n_q_heads > 0 && a->n_q_heads % a->n_kv_heads == 0,
               "local attention: %d query heads do not share %d KV heads evenly", a->n_q_heads, a->n_kv_heads);
    FM_REQUIRE(a->n_docs > 0 && a->window >= 0, "local attention: bad document count %d or window %d", a->n_docs, a->window);
    FM_REQUIRE(a->softcap >= 0.f && a->softcap < INFINITY, "local attention: the cap must be finite and not negative");
    FM_REQUIRE(int64_t(a->n_q_heads) * a->n_q_rows < (int64_t(1) << 31) && int64_t(a->n_kv_heads) * a->n_k_rows < (int64_t(1) << 31),
               "local attention: more than 2^31 rows over all heads");
    if (a->d != 16 && a->d != 32 && a->d != 64 && a->d != 128 && a->d != 256) {
        set_error("local attention: head dim %d (16, 32, 64, 128 and 256 are built)", a->d);
        return FM_ERR_UNSUPPORTED;
    }
    const int e = elem_bytes(a->dtype);
    uintptr_t grid = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v);
    grid |= uintptr_t((a->q_stride_head | a->q_stride_row | a->k_stride_head | a->k_stride_row | a->v_stride_head | a->v_stride_row) * e);
    FM_REQUIRE(grid % 16 == 0, "local attention: rows must start on 16-byte boundaries");
    p = LocalParams{};
    p.q = a->q; p.k = a->k; p.v = a->v;
    p.q_sh = a->q_stride_head; p.q_st = a->q_stride_row;
    p.k_sh = a->k_stride_head; p.k_st = a->k_stride_row;
    p.v_sh = a->v_stride_head; p.v_st = a->v_stride_row;
    p.Hq = a->n_q_heads; p.H = a->n_kv_heads; p.G = p.Hq / p.H; p.d = a->d;
    p.S = int(a->n_q_rows); p.N = int(a->n_k_rows);
    p.n_docs = a->n_docs;
    p.cu_q = a->cu_q; p.cu_k = a->cu_k; p.prefix = a->prefix;
    p.slopes = a->slopes; p.scale = a->sm_scale; p.cap = a->softcap;
    // A cap out of reach: what it changes of a score is less than half a bit for products up to 2^88, while scale / cap has few bits left
    // (below 2^-126) or none.
    if (fabsf(p.scale) <= p.cap * 0x1p-100f) p.cap = 0.f;
    p.window = a->window; p.causal = a->causal != 0;
    tc_test_hooks(p.wait_ns, p.skip_tile);
    if (a->page_table) {
        FM_REQUIRE(a->lengths && a->n_seqs > 0 && a->n_pages > 0 && a->n_pages < (int64_t(1) << 31), "paged attention: lengths, n_seqs and n_pages are needed");
        int shift = 0;
        while ((1 << shift) < a->page_size) ++shift;
        if (a->page_size < 16 || a->page_size > 256 || (1 << shift) != a->page_size) {
            set_error("paged attention: page size %d (a power of two from 16 to 256)", a->page_size);
            return FM_ERR_UNSUPPORTED;
        }
        FM_REQUIRE(a->page_table_width >= 0 && a->page_table_width < (int64_t(1) << 30 >> shift), "paged attention: page table too wide");
        FM_REQUIRE(a->cu_q || a->n_q_rows == a->n_docs, "paged attention: one query a sequence without cu_q");
        p.table = a->page_table; p.lengths = a->lengths; p.seqs = a->seqs;
        p.table_ld = int(a->page_table_width); p.page_shift = shift; p.n_pages = int(a->n_pages); p.n_seqs = a->n_seqs;
    } else {
        FM_REQUIRE(a->n_docs == 1 || (a->cu_q && a->cu_k), "local attention: several documents need cu_q and cu_k");
    }
    return FM_OK;
}

// Workspace of the backward pass: delta, the ranges, then the parts of dV and dK.
static size_t delta_bytes(const LocalParams &p) { return align_up(size_t(p.Hq) * size_t(p.S) * sizeof(float), 256); }
static size_t range_bytes(const LocalParams &p, int dtype)
{
    return dtype == FM_F16 && p.S > 0 && local_tc_fits(p, dtype) ? 2 * delta_bytes(p) : 0;
}
static size_t parts_bytes(const LocalParams &p, int dtype) { return p.S > 0 && local_tc_fits(p, dtype) ? local_tc_bwd_workspace(p) : 0; }

static size_t forward_workspace(const LocalParams &p, int dtype)
{
    if (local_decode_fits(p, dtype)) return local_decode_workspace(p);
    return local_tc_fits(p, dtype) ? local_tc_fwd_workspace(p) : local_simt_fwd_workspace(p);
}

}  // namespace fm

extern "C" {

size_t fm_local_attn_workspace_bytes(const fm_local_attn_args *a)
{
    fm::LocalParams p;
    if (fm::local_params(a, p) || p.S == 0) return 0;
    return fm::forward_workspace(p, a->dtype);
}

int fm_local_attn_fwd(const fm_local_attn_args *a, void *o, float *lse, void *workspace, size_t workspace_bytes, fm_stream_t stream)
{
    using namespace fm;
    LocalParams p;
    if (int rc = local_params(a, p)) return rc;
    if (p.S == 0) return FM_OK;
    FM_REQUIRE(p.q && o && lse && (p.table || p.N == 0 || (p.k && p.v)), "fm_local_attn_fwd: null pointer");
    const size_t need = forward_workspace(p, a->dtype);
    if (need && (workspace_bytes < need || !workspace)) {
        set_error("fm_local_attn_fwd: workspace of %zu bytes, %zu are needed", workspace_bytes, need);
        return FM_ERR_WORKSPACE;
    }
    FM_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && reinterpret_cast<uintptr_t>(o) % 16 == 0, "fm_local_attn_fwd: misaligned buffer");
    p.o = o;
    p.lse = lse;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (local_decode_fits(p, a->dtype)) return local_decode_fwd(p, a->dtype, workspace, st);
    if (local_tc_fits(p, a->dtype)) return local_tc_fwd(p, a->dtype, workspace, st);
    return local_simt_fwd(p, a->dtype, workspace, st);
}

size_t fm_local_attn_bwd_workspace_bytes(const fm_local_attn_args *a)
{
    fm::LocalParams p;
    return fm::local_params(a, p) ? 0 : fm::delta_bytes(p) + fm::range_bytes(p, a->dtype) + fm::parts_bytes(p, a->dtype);
}

int fm_local_attn_bwd(const fm_local_attn_args *a, const void *o, const float *lse, const void *d_o, int64_t do_stride_head,
                      int64_t do_stride_row, const float *d_lse, void *dq, void *dk, void *dv, void *workspace, size_t workspace_bytes,
                      fm_stream_t stream)
{
    using namespace fm;
    LocalParams p;
    if (int rc = local_params(a, p)) return rc;
    if (p.table) {
        set_error("fm_local_attn_bwd: a paged cache has no backward pass");
        return FM_ERR_UNSUPPORTED;
    }
    if (p.S == 0 && p.N == 0) return FM_OK;
    FM_REQUIRE(p.S == 0 || (p.q && o && lse && d_o && dq), "fm_local_attn_bwd: null pointer");
    FM_REQUIRE(p.N == 0 || (p.k && p.v && dk && dv), "fm_local_attn_bwd: null pointer");
    const size_t ranges = range_bytes(p, a->dtype), need = delta_bytes(p) + ranges + parts_bytes(p, a->dtype);
    if (need && (workspace_bytes < need || !workspace)) {
        set_error("fm_local_attn_bwd: workspace of %zu bytes, %zu are needed", workspace_bytes, need);
        return FM_ERR_WORKSPACE;
    }
    FM_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "fm_local_attn_bwd: misaligned buffer");
    FM_REQUIRE((reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) % 16 == 0, "fm_local_attn_bwd: misaligned buffer");
    FM_REQUIRE((reinterpret_cast<uintptr_t>(d_o) | reinterpret_cast<uintptr_t>(o) | uintptr_t((do_stride_head | do_stride_row) * elem_bytes(a->dtype))) % 16 == 0,
               "fm_local_attn_bwd: rows must start on 16-byte boundaries");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    float *delta = static_cast<float *>(workspace);
    float *range = ranges ? reinterpret_cast<float *>(static_cast<char *>(workspace) + delta_bytes(p)) : nullptr;
    BwdParams g{d_o, do_stride_head, do_stride_row, lse, delta, range, range ? range + delta_bytes(p) / sizeof(float) : nullptr, dq, dk, dv};
    if (p.S > 0) {
        const int rc = with_type_and_dim(a->dtype, p.d, [&](auto t, auto dim) -> int {
            using T = decltype(t);
            constexpr int lanes = decltype(dim)::value * sizeof(T) / 16;
            local_delta_kernel<T, decltype(dim)::value><<<unsigned(ceil_div(ceil_div(int64_t(p.Hq) * p.S, kDeltaRows) * std::min(lanes, 32), kRowThreads)), kRowThreads, 0, st>>>(p, g, static_cast<const T *>(o), d_lse, delta, range);
            FM_LAUNCHED("local_delta_kernel");
            return FM_OK;
        });
        if (rc) return rc;
    }
    if (p.S > 0 && local_tc_fits(p, a->dtype)) return local_tc_bwd(p, g, a->dtype, reinterpret_cast<float *>(static_cast<char *>(workspace) + delta_bytes(p) + ranges), st);
    return local_simt_bwd(p, g, a->dtype, st);
}

}  // extern "C"
