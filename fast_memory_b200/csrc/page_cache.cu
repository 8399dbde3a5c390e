// Pages of a cache: append, fork, free, compact, gather, copy.  Everything the operations decide - which pages a sequence
// gets, whether there are enough - is decided on the device, so that a captured graph can be replayed with other lengths.
//
// State: refcounts [n_pages] (0 = free), page_table [n_seqs, width] (-1 behind a sequence's last page), lengths [n_seqs].
// The r-th page that a call asks for is the r-th LOWEST free page: no free list has to be kept in step, and the same calls
// give the same tables.  A last page that is not full belongs to one sequence only (a fork copies its rows), so an append
// never writes into a shared page.
//
// An operation is a PLAN by one CTA (checks every index, counts what each sequence needs, ranks the free pages, writes the
// tables) and, where rows move, a copy kernel over the whole chip that reads the plan.  A plan that fails a check sets its
// bit in the status word and changes nothing, and its copy kernel finds `go` = 0.  The plan is bound by latency: two sweeps
// over the refcounts, 32 warps side by side, one ballot for 32 pages.  The copies are bound by HBM: 16 bytes a thread.
// 64 sequences of 4096 tokens, 8 heads, d = 128: evicting half, compacting and admitting new ones, twice over, 440-448 us (83 % of the
// measured copy rate with the plans between); one token for each of 64 forks, 37-39 us for three calls, most of it the host's;
// gathering 64 sequences 339 us (97 %).
#include "common.cuh"

namespace fm {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kCopyThreads = 256;
// 16-byte pieces (of K; V has as many) that the plan's CTA copies itself: 64 KB take it about 1.5 us, a launch of its own costs the
// host 2.5 us and the device as much.
constexpr int64_t kFewPieces = 2048;

struct Cache {
    char *k, *v;
    int32_t *table, *lengths, *refs, *status;
    int n_pages, n_seqs, width, shift, heads;
    int row16;                                    // 16-byte pieces of a row
};

// Head of the workspace, written by the plan and read by the copy kernel.
struct PlanHead {
    int go, count, pad[2];
};

__device__ __forceinline__ int pages_of(int len, int shift) { return (len + (1 << shift) - 1) >> shift; }

// Inclusive sum over the CTA's threads; `total` gets the sum.
__device__ __forceinline__ int block_scan(int x, int *warp_sums, int &total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    __syncthreads();                              // the sums of an earlier call have been read
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    return s + (warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0);
}

// Pages whose refcount is zero (or is not, LIVE) in ascending order: f(rank, page) for every page for which want(page) holds.
// Each warp ranks one stretch of the pool; `limit`: ranks from there on are not needed.  Returns how many there are.
template <typename W, typename F> __device__ __forceinline__ int rank_pages(int n_pages, int *warp_sums, W &&want, int limit, F &&f)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = ((n_pages + kPlanWarps - 1) / kPlanWarps + 31) & ~31;
    const int lo = min(warp * per, n_pages), hi = min(lo + per, n_pages);
    int mine = 0;
#pragma unroll 4
    for (int b = lo; b < hi; b += 32) mine += __popc(__ballot_sync(0xffffffffu, b + lane < hi && want(b + lane)));
    int total;
    const int incl = block_scan(lane == 0 ? mine : 0, warp_sums, total);       // lane 0's value: through this warp
    int base = __shfl_sync(0xffffffffu, incl, 0) - mine;
#pragma unroll 4
    for (int b = lo; b < hi && base < limit; b += 32) {
        const bool w = b + lane < hi && want(b + lane);
        const unsigned m = __ballot_sync(0xffffffffu, w);
        const int r = base + __popc(m & ((1u << lane) - 1u));
        if (w && r < limit) f(r, b + lane);
        base += __popc(m);
    }
    return total;
}

__device__ __forceinline__ void fail(int *err, int bit) { atomicOr(err, bit); }

// Marks sequence s as named by this call; false (and an error) if it is out of range or named twice.
__device__ __forceinline__ bool claim(const Cache &c, int s, int *mark, int *err)
{
    if (s < 0 || s >= c.n_seqs || atomicAdd(&mark[s], 1)) {
        fail(err, FM_CACHE_BAD_SEQ);
        return false;
    }
    return true;
}

// The length of a sequence as far as its table can hold it (a wrong length stays inside the table).
__device__ __forceinline__ int length_of(const Cache &c, int s) { return min(max(c.lengths[s], 0), c.width << c.shift); }

// Takes `need` (over all threads: `total`) pages per item.  off[i] (exclusive sums, off[n] = total) must be written.  Leaves
// the pages in alloc[0 .. total).  Called by every thread; returns false, with an error set, if the pool has too few.
__device__ __forceinline__ bool allocate(const Cache &c, int total, int32_t *alloc, int *warp_sums, int *err)
{
    if (total == 0) return true;
    const int free_pages = rank_pages(c.n_pages, warp_sums, [&](int p) { return c.refs[p] == 0; }, total,
                                      [&](int r, int p) { alloc[r] = p; });
    if (free_pages < total && threadIdx.x == 0) fail(err, FM_CACHE_NO_PAGES);
    __syncthreads();
    return *err == 0;
}

// Exclusive sums of need(i) over n items into off[0 .. n]; returns the sum.
template <typename F> __device__ __forceinline__ int scan_needs(int n, int32_t *off, int *warp_sums, F &&need)
{
    int base = 0;
    for (int b = 0; b < n; b += kPlanThreads) {
        const int i = b + threadIdx.x;
        const int x = i < n ? need(i) : 0;
        int total;
        const int incl = block_scan(x, warp_sums, total);
        if (i < n) off[i] = base + incl - x;
        base += total;
    }
    if (threadIdx.x == 0) off[n] = base;
    __syncthreads();
    return base;
}

// largest i with off[i] <= r, among n items
__device__ __forceinline__ int find_item(const int32_t *off, int n, int r)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (off[mid] <= r) lo = mid; else hi = mid;
    }
    return lo;
}

// workspace: PlanHead, mark [n_seqs], off [n + 1], start [n], src [n], alloc [n_pages] (append, fork)
struct PlanWs {
    PlanHead *head;
    int32_t *mark, *off, *start, *src, *alloc;
};
__host__ __device__ inline PlanWs plan_ws(void *ws, int n_seqs, int n)
{
    PlanWs w;
    w.head = static_cast<PlanHead *>(ws);
    w.mark = reinterpret_cast<int32_t *>(w.head + 1);
    w.off = w.mark + n_seqs;
    w.start = w.off + n + 1;
    w.src = w.start + n;
    w.alloc = w.src + n;
    return w;
}

__device__ __forceinline__ void clear_marks(const Cache &c, const PlanWs &w, int *err)
{
    for (int i = threadIdx.x; i < c.n_seqs; i += kPlanThreads) w.mark[i] = 0;
    if (threadIdx.x == 0) *err = 0;
    __syncthreads();
}

__device__ __forceinline__ void finish(const Cache &c, PlanHead *head, int count, const int *err)
{
    if (threadIdx.x == 0) {
        head->go = *err == 0;
        head->count = *err == 0 ? count : 0;
        if (*err) atomicOr(c.status, *err);
    }
}

// What is appended: rows of k and v, strides in bytes.
struct NewRows {
    const int32_t *seqs, *cu;
    const char *k, *v;
    int64_t k_sh, k_st, v_sh, v_st;
    int n, tokens;
};

// 32 tokens from t0 on and head h: their places are looked up once, then 16-byte pieces go side by side.  By a whole CTA.
__device__ __forceinline__ void append_rows(const Cache &c, const PlanWs &w, const NewRows &a, int t0, int h, int64_t *to)
{
    if (threadIdx.x < 32) {
        const int t = t0 + threadIdx.x;
        int64_t row = -1;
        if (t < (a.cu ? min(a.tokens, a.cu[a.n]) : a.tokens)) {
            const int i = a.cu ? find_item(a.cu, a.n, t) : t;
            const int at = w.start[i] + t - (a.cu ? a.cu[i] : i);
            const int page = c.table[int64_t(a.seqs[i]) * c.width + (at >> c.shift)];
            if (page >= 0 && page < c.n_pages) row = ((int64_t(page) * c.heads + h) << c.shift) + (at & ((1 << c.shift) - 1));
        }
        to[threadIdx.x] = row;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 32 * c.row16; x += blockDim.x) {
        const int t = x / c.row16, o = x % c.row16;
        const int64_t row = to[t];
        if (row < 0) continue;
        const uint4 k = *reinterpret_cast<const uint4 *>(a.k + h * a.k_sh + (t0 + t) * a.k_st + o * 16);
        const uint4 v = *reinterpret_cast<const uint4 *>(a.v + h * a.v_sh + (t0 + t) * a.v_st + o * 16);
        *reinterpret_cast<uint4 *>(c.k + (row * c.row16 + o) * 16) = k;
        *reinterpret_cast<uint4 *>(c.v + (row * c.row16 + o) * 16) = v;
    }
}

__global__ void __launch_bounds__(kCopyThreads) cache_append_rows(Cache c, NewRows a, void *ws)
{
    __shared__ int64_t to[32];
    const PlanWs w = plan_ws(ws, c.n_seqs, a.n);
    if (w.head->go) append_rows(c, w, a, blockIdx.x * 32, blockIdx.y, to);
}

// copy: the rows as well, where they are so few that another launch would take longer
__global__ void __launch_bounds__(kPlanThreads) cache_append_plan(Cache c, NewRows a, void *ws, bool copy)
{
    __shared__ int warp_sums[32], err;
    __shared__ int64_t to[32];
    const int32_t *seqs = a.seqs, *cu = a.cu;
    const int n = a.n, tokens = a.tokens;
    const PlanWs w = plan_ws(ws, c.n_seqs, n);
    clear_marks(c, w, &err);
    const int total = scan_needs(n, w.off, warp_sums, [&](int i) {
        const int s = seqs[i], a = cu ? cu[i] : i, b = cu ? cu[i + 1] : i + 1;
        if (a < 0 || b < a || b > tokens || (i == 0 && a != 0)) { fail(&err, FM_CACHE_BAD_SEQ); return 0; }
        if (!claim(c, s, w.mark, &err)) return 0;
        const int len = length_of(c, s);
        if (b - a > (c.width << c.shift) - len) { fail(&err, FM_CACHE_TOO_LONG); return 0; }
        w.start[i] = len;
        return pages_of(len + b - a, c.shift) - pages_of(len, c.shift);
    });
    if (!err && allocate(c, total, w.alloc, warp_sums, &err)) {
        for (int r = threadIdx.x; r < total; r += kPlanThreads) {
            const int i = find_item(w.off, n, r), page = w.alloc[r];
            c.table[int64_t(seqs[i]) * c.width + pages_of(w.start[i], c.shift) + (r - w.off[i])] = page;
            c.refs[page] = 1;
        }
        for (int i = threadIdx.x; i < n; i += kPlanThreads) c.lengths[seqs[i]] = w.start[i] + (cu ? cu[i + 1] - cu[i] : 1);
        if (copy) {
            __syncthreads();
            for (int t = 0; t < tokens; t += 32)
                for (int h = 0; h < c.heads; ++h) {
                    append_rows(c, w, a, t, h, to);
                    __syncthreads();
                }
        }
    }
    finish(c, w.head, n, &err);
}

// The rows of item i's partial page, head h, K or V: one contiguous run.  By the threads `first`, `first` + `step` ...
__device__ __forceinline__ void fork_rows(const Cache &c, const PlanWs &w, int i, int h, bool v, int first, int step)
{
    const int rows = w.start[i] & ((1 << c.shift) - 1);
    if (rows == 0) return;
    const int src = w.src[i], dst = w.alloc[w.off[i]];
    if (src < 0 || src >= c.n_pages) return;
    uint4 *pool = reinterpret_cast<uint4 *>(v ? c.v : c.k);
    const uint4 *from = pool + ((int64_t(src) * c.heads + h) << c.shift) * c.row16;
    uint4 *to = pool + ((int64_t(dst) * c.heads + h) << c.shift) * c.row16;
#pragma unroll 4
    for (int x = first; x < rows * c.row16; x += step) to[x] = from[x];
}

__global__ void __launch_bounds__(kCopyThreads) cache_fork_rows(Cache c, int n, void *ws)
{
    const PlanWs w = plan_ws(ws, c.n_seqs, n);
    if (w.head->go) fork_rows(c, w, blockIdx.x, blockIdx.y, blockIdx.z, threadIdx.x, kCopyThreads);
}

// copy: the rows as well, a warp a run, where they are so few that another launch would take longer
__global__ void __launch_bounds__(kPlanThreads) cache_fork_plan(Cache c, const int32_t *parents, const int32_t *children, int n, void *ws, bool copy)
{
    __shared__ int warp_sums[32], err;
    const PlanWs w = plan_ws(ws, c.n_seqs, n);
    clear_marks(c, w, &err);
    const int total = scan_needs(n, w.off, warp_sums, [&](int i) {
        const int from = parents[i], to = children[i];
        w.start[i] = 0;
        if (from < 0 || from >= c.n_seqs) { fail(&err, FM_CACHE_BAD_SEQ); return 0; }
        if (!claim(c, to, w.mark, &err)) return 0;
        if (c.lengths[to] != 0) { fail(&err, FM_CACHE_NOT_EMPTY); return 0; }
        const int len = length_of(c, from);
        w.start[i] = len;
        return (len & ((1 << c.shift) - 1)) ? 1 : 0;
    });
    if (!err && allocate(c, total, w.alloc, warp_sums, &err)) {
        // a warp an item: shared pages gain an owner, the partial page gets a copy
        for (int i = threadIdx.x >> 5; i < n; i += kPlanWarps) {
            const int len = w.start[i], full = len >> c.shift, used = pages_of(len, c.shift);
            const int32_t *from = c.table + int64_t(parents[i]) * c.width;
            int32_t *to = c.table + int64_t(children[i]) * c.width;
            for (int col = threadIdx.x & 31; col < used; col += 32) {
                int page = from[col];
                if (col < full) {
                    if (page >= 0 && page < c.n_pages) atomicAdd(&c.refs[page], 1);
                } else {
                    w.src[i] = page;
                    page = w.alloc[w.off[i]];
                    c.refs[page] = 1;
                }
                to[col] = page;
            }
            if ((threadIdx.x & 31) == 0) c.lengths[children[i]] = len;
        }
        if (copy) {
            __syncthreads();
            for (int x = threadIdx.x >> 5; x < 2 * n * c.heads; x += kPlanWarps) fork_rows(c, w, x / (2 * c.heads), x / 2 % c.heads, x & 1, threadIdx.x & 31, 32);
        }
    }
    finish(c, w.head, n, &err);
}

__global__ void __launch_bounds__(kPlanThreads) cache_free_plan(Cache c, const int32_t *seqs, int n, void *ws)
{
    __shared__ int err;
    const PlanWs w = plan_ws(ws, c.n_seqs, n);
    clear_marks(c, w, &err);
    for (int i = threadIdx.x; i < n; i += kPlanThreads) claim(c, seqs[i], w.mark, &err);
    __syncthreads();
    if (!err) {
        for (int i = threadIdx.x >> 5; i < n; i += kPlanWarps) {
            int32_t *row = c.table + int64_t(seqs[i]) * c.width;
            const int used = pages_of(length_of(c, seqs[i]), c.shift);
#pragma unroll 4
            for (int col = threadIdx.x & 31; col < used; col += 32) {
                const int page = row[col];
                if (page >= 0 && page < c.n_pages) atomicSub(&c.refs[page], 1);
                row[col] = -1;
            }
            __syncwarp();
            if ((threadIdx.x & 31) == 0) c.lengths[seqs[i]] = 0;
        }
    }
    finish(c, w.head, n, &err);
}

// workspace: PlanHead (go = live pages, count = moves), src [n_pages], dst [n_pages], to [n_pages] (where a moved page went)
__global__ void __launch_bounds__(kPlanThreads) cache_compact_plan(Cache c, void *ws)
{
    __shared__ int warp_sums[32];
    PlanHead *head = static_cast<PlanHead *>(ws);
    int32_t *src = reinterpret_cast<int32_t *>(head + 1), *dst = src + c.n_pages, *to = dst + c.n_pages;
    auto live = [&](int p) { return c.refs[p] > 0; };
    const int n_live = rank_pages(c.n_pages, warp_sums, live, 0, [](int, int) {});
    const int moves = rank_pages(c.n_pages, warp_sums, [&](int p) { return p >= n_live && live(p); }, c.n_pages, [&](int r, int p) { src[r] = p; });
    rank_pages(n_live, warp_sums, [&](int p) { return !live(p); }, moves, [&](int r, int p) { dst[r] = p; });
    for (int p = n_live + threadIdx.x; p < c.n_pages; p += kPlanThreads) to[p] = p;
    __syncthreads();
    for (int r = threadIdx.x; r < moves; r += kPlanThreads) {
        const int a = src[r], b = dst[r];
        c.refs[b] = c.refs[a];
        c.refs[a] = 0;
        to[a] = b;
    }
    if (threadIdx.x == 0) {
        head->go = n_live;
        head->count = moves;
    }
}

// Whole pages src[r] -> dst[r], K and V, dealt out in pieces of 16 bytes x 4 x threads; pieces of all moves form one list.
__device__ __forceinline__ void copy_pages_part(const Cache &c, const int32_t *src, const int32_t *dst, int64_t count)
{
    const int64_t page16 = (int64_t(c.heads) << c.shift) * c.row16;
    const int per = kCopyThreads * 4;
    const int64_t pieces = (page16 + per - 1) / per;
    for (int64_t x = blockIdx.x; x < 2 * count * pieces; x += gridDim.x) {
        const int64_t move = x / (2 * pieces), rest = x % (2 * pieces);
        const int a = src[move], b = dst[move];
        if (a < 0 || a >= c.n_pages || b < 0 || b >= c.n_pages) continue;
        uint4 *pool = reinterpret_cast<uint4 *>(rest >= pieces ? c.v : c.k);
        const int64_t o = (rest >= pieces ? rest - pieces : rest) * per + threadIdx.x;
        uint4 buf[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (o + i * kCopyThreads < page16) buf[i] = pool[a * page16 + o + i * kCopyThreads];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (o + i * kCopyThreads < page16) pool[b * page16 + o + i * kCopyThreads] = buf[i];
    }
}

__global__ void __launch_bounds__(kCopyThreads) cache_compact_move(Cache c, const void *ws)
{
    const PlanHead *head = static_cast<const PlanHead *>(ws);
    const int moves = head->count, n_live = head->go;
    if (moves == 0) return;
    const int32_t *src = reinterpret_cast<const int32_t *>(head + 1), *dst = src + c.n_pages, *to = dst + c.n_pages;
    const int64_t entries = int64_t(c.n_seqs) * c.width;
    for (int64_t x = int64_t(blockIdx.x) * kCopyThreads + threadIdx.x; x < entries; x += int64_t(gridDim.x) * kCopyThreads) {
        const int page = c.table[x];
        if (page >= n_live && page < c.n_pages) c.table[x] = to[page];
    }
    copy_pages_part(c, src, dst, moves);
}

__global__ void __launch_bounds__(kCopyThreads) cache_copy_pages(Cache c, const int32_t *src, const int32_t *dst, int64_t n)
{
    copy_pages_part(c, src, dst, n);
}

// Rows [start, start + n) of sequences as packed arrays [heads, tokens, d]; rows the sequence does not have are zero.
__global__ void __launch_bounds__(kCopyThreads) cache_gather_rows(Cache c, const int32_t *seqs, const int32_t *cu, const int32_t *starts, int n, int tokens,
                                                                  char *k_out, char *v_out)
{
    __shared__ int64_t from[32];
    const int t0 = blockIdx.x * 32, h = blockIdx.y;
    if (threadIdx.x < 32) {
        const int t = t0 + threadIdx.x;
        int64_t row = -1;
        if (t < tokens) {
            const int i = find_item(cu, n, t), s = seqs[i];
            if (t >= cu[i] && t < cu[i + 1] && s >= 0 && s < c.n_seqs) {
                const int at = (starts ? starts[i] : 0) + t - cu[i];
                if (at >= 0 && at < length_of(c, s)) {
                    const int page = c.table[int64_t(s) * c.width + (at >> c.shift)];
                    if (page >= 0 && page < c.n_pages) row = ((int64_t(page) * c.heads + h) << c.shift) + (at & ((1 << c.shift) - 1));
                }
            }
        }
        from[threadIdx.x] = row;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 32 * c.row16; x += kCopyThreads) {
        const int t = x / c.row16, o = x % c.row16;
        if (t0 + t >= tokens) break;
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (from[t] >= 0) {
            a = *reinterpret_cast<const uint4 *>(c.k + (from[t] * c.row16 + o) * 16);
            b = *reinterpret_cast<const uint4 *>(c.v + (from[t] * c.row16 + o) * 16);
        }
        const int64_t out = ((int64_t(h) * tokens + t0 + t) * c.row16 + o) * 16;
        *reinterpret_cast<uint4 *>(k_out + out) = a;
        *reinterpret_cast<uint4 *>(v_out + out) = b;
    }
}

int cache_of(const fm_page_cache *a, Cache &c)
{
    FM_REQUIRE(a && a->k_pages && a->v_pages && a->page_table && a->lengths && a->refcounts && a->status, "page cache: null pointer");
    FM_REQUIRE(a->dtype == FM_F32 || a->dtype == FM_BF16 || a->dtype == FM_F16, "page cache: unknown element type %d", a->dtype);
    FM_REQUIRE(a->n_pages > 0 && a->n_pages < (int64_t(1) << 31) && a->n_seqs > 0 && a->width >= 0 && a->n_heads > 0 && a->n_heads < 65536,
               "page cache: bad sizes");
    int shift = 0;
    while ((1 << shift) < a->page_size && shift < 30) ++shift;
    if (a->page_size < 16 || a->page_size > 256 || (1 << shift) != a->page_size) {
        set_error("page cache: page size %d (a power of two from 16 to 256)", a->page_size);
        return FM_ERR_UNSUPPORTED;
    }
    FM_REQUIRE(a->width < (int64_t(1) << 30 >> shift), "page cache: page table too wide");
    const int64_t bytes = int64_t(a->d) * elem_bytes(a->dtype);
    if (a->d <= 0 || a->d > 1024 || bytes % 16) {
        set_error("page cache: rows of %lld bytes (a multiple of 16 is needed)", (long long)bytes);
        return FM_ERR_UNSUPPORTED;
    }
    FM_REQUIRE((reinterpret_cast<uintptr_t>(a->k_pages) | reinterpret_cast<uintptr_t>(a->v_pages)) % 16 == 0, "page cache: pools must be 16-byte aligned");
    c = Cache{static_cast<char *>(a->k_pages), static_cast<char *>(a->v_pages), a->page_table, a->lengths, a->refcounts, a->status,
              int(a->n_pages), a->n_seqs, int(a->width), shift, a->n_heads, int(bytes / 16)};
    return FM_OK;
}

int check_ws(const fm_page_cache *a, int64_t n, void *ws, size_t bytes, const char *what)
{
    const size_t need = fm_page_cache_workspace_bytes(a, n);
    if (!ws || bytes < need) {
        set_error("%s: workspace of %zu bytes, %zu are needed", what, bytes, need);
        return FM_ERR_WORKSPACE;
    }
    return FM_OK;
}

}  // namespace

}  // namespace fm

extern "C" {

size_t fm_page_cache_workspace_bytes(const fm_page_cache *a, int64_t n)
{
    if (!a || n < 0 || a->n_pages < 0 || a->n_seqs < 0) return 0;
    const size_t plan = size_t(a->n_seqs) + 3 * size_t(n) + 1 + size_t(a->n_pages), compact = 3 * size_t(a->n_pages);
    return sizeof(fm::PlanHead) + 4 * std::max(plan, compact) + 16;
}

int fm_cache_append(const fm_page_cache *a, const int32_t *seqs, int64_t n, const int32_t *cu_new, const void *k_new, const void *v_new,
                    int64_t n_tokens, int64_t k_stride_head, int64_t k_stride_row, int64_t v_stride_head, int64_t v_stride_row,
                    void *workspace, size_t workspace_bytes, fm_stream_t stream)
{
    using namespace fm;
    Cache c;
    if (int rc = cache_of(a, c)) return rc;
    FM_REQUIRE(n >= 0 && n <= a->n_seqs && n_tokens >= 0 && n_tokens < (int64_t(1) << 30), "fm_cache_append: bad sizes (%lld sequences, %lld tokens)",
               (long long)n, (long long)n_tokens);
    if (n == 0) return FM_OK;
    FM_REQUIRE(seqs && (n_tokens == 0 || (k_new && v_new)), "fm_cache_append: null pointer");
    FM_REQUIRE(cu_new || n == n_tokens, "fm_cache_append: without cu_new every sequence gets one token");
    const int e = elem_bytes(a->dtype);
    FM_REQUIRE((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) % 16 == 0 &&
               ((k_stride_head | k_stride_row | v_stride_head | v_stride_row) * e) % 16 == 0, "fm_cache_append: rows must start on 16-byte boundaries");
    if (int rc = check_ws(a, n, workspace, workspace_bytes, "fm_cache_append")) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const NewRows rows{seqs, cu_new, static_cast<const char *>(k_new), static_cast<const char *>(v_new), k_stride_head * e, k_stride_row * e,
                       v_stride_head * e, v_stride_row * e, int(n), int(n_tokens)};
    const bool copy = n_tokens * c.heads * c.row16 <= kFewPieces;
    cache_append_plan<<<1, kPlanThreads, 0, st>>>(c, rows, workspace, copy);
    FM_LAUNCHED("cache_append_plan");
    if (n_tokens > 0 && !copy) {
        cache_append_rows<<<dim3(unsigned(ceil_div(n_tokens, 32)), unsigned(c.heads)), kCopyThreads, 0, st>>>(c, rows, workspace);
        FM_LAUNCHED("cache_append_rows");
    }
    return FM_OK;
}

int fm_cache_fork(const fm_page_cache *a, const int32_t *parents, const int32_t *children, int64_t n, void *workspace, size_t workspace_bytes,
                  fm_stream_t stream)
{
    using namespace fm;
    Cache c;
    if (int rc = cache_of(a, c)) return rc;
    FM_REQUIRE(n >= 0 && n <= a->n_seqs, "fm_cache_fork: %lld forks of %d sequences", (long long)n, a->n_seqs);
    if (n == 0) return FM_OK;
    FM_REQUIRE(parents && children, "fm_cache_fork: null pointer");
    if (int rc = check_ws(a, n, workspace, workspace_bytes, "fm_cache_fork")) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool copy = ((n * c.heads) << c.shift) * c.row16 <= kFewPieces;
    cache_fork_plan<<<1, kPlanThreads, 0, st>>>(c, parents, children, int(n), workspace, copy);
    FM_LAUNCHED("cache_fork_plan");
    if (!copy) {
        cache_fork_rows<<<dim3(unsigned(n), unsigned(c.heads), 2), kCopyThreads, 0, st>>>(c, int(n), workspace);
        FM_LAUNCHED("cache_fork_rows");
    }
    return FM_OK;
}

int fm_cache_free(const fm_page_cache *a, const int32_t *seqs, int64_t n, void *workspace, size_t workspace_bytes, fm_stream_t stream)
{
    using namespace fm;
    Cache c;
    if (int rc = cache_of(a, c)) return rc;
    FM_REQUIRE(n >= 0 && n <= a->n_seqs, "fm_cache_free: %lld of %d sequences", (long long)n, a->n_seqs);
    if (n == 0) return FM_OK;
    FM_REQUIRE(seqs, "fm_cache_free: null pointer");
    if (int rc = check_ws(a, n, workspace, workspace_bytes, "fm_cache_free")) return rc;
    cache_free_plan<<<1, kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(c, seqs, int(n), workspace);
    FM_LAUNCHED("cache_free_plan");
    return FM_OK;
}

int fm_cache_compact(const fm_page_cache *a, void *workspace, size_t workspace_bytes, fm_stream_t stream)
{
    using namespace fm;
    Cache c;
    if (int rc = cache_of(a, c)) return rc;
    if (int rc = check_ws(a, 0, workspace, workspace_bytes, "fm_cache_compact")) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cache_compact_plan<<<1, kPlanThreads, 0, st>>>(c, workspace);
    FM_LAUNCHED("cache_compact_plan");
    cache_compact_move<<<unsigned(sm_count() * 8), kCopyThreads, 0, st>>>(c, workspace);
    FM_LAUNCHED("cache_compact_move");
    return FM_OK;
}

int fm_cache_copy_pages(const fm_page_cache *a, const int32_t *src, const int32_t *dst, int64_t n, fm_stream_t stream)
{
    using namespace fm;
    Cache c;
    if (int rc = cache_of(a, c)) return rc;
    FM_REQUIRE(n >= 0, "fm_cache_copy_pages: %lld pages", (long long)n);
    if (n == 0) return FM_OK;
    FM_REQUIRE(src && dst, "fm_cache_copy_pages: null pointer");
    const int64_t page16 = (int64_t(c.heads) << c.shift) * c.row16;
    const int64_t pieces = 2 * n * ceil_div(page16, kCopyThreads * 4);
    cache_copy_pages<<<unsigned(std::min<int64_t>(pieces, sm_count() * 8)), kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(c, src, dst, n);
    FM_LAUNCHED("cache_copy_pages");
    return FM_OK;
}

int fm_cache_gather(const fm_page_cache *a, const int32_t *seqs, const int32_t *cu, const int32_t *starts, int64_t n, int64_t n_tokens, void *k_out,
                    void *v_out, fm_stream_t stream)
{
    using namespace fm;
    Cache c;
    if (int rc = cache_of(a, c)) return rc;
    FM_REQUIRE(n >= 0 && n < (int64_t(1) << 30) && n_tokens >= 0 && n_tokens < (int64_t(1) << 30), "fm_cache_gather: bad sizes");
    if (n_tokens == 0) return FM_OK;
    FM_REQUIRE(n > 0 && seqs && cu && k_out && v_out, "fm_cache_gather: null pointer");
    cache_gather_rows<<<dim3(unsigned(ceil_div(n_tokens, 32)), unsigned(c.heads)), kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        c, seqs, cu, starts, int(n), int(n_tokens), static_cast<char *>(k_out), static_cast<char *>(v_out));
    FM_LAUNCHED("cache_gather_rows");
    return FM_OK;
}

}  // extern "C"
