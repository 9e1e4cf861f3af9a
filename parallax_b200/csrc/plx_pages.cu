// The pages of a paged KV cache: copying them, forking rows (parallel sampling, beams), moving the live ones together,
// and listing the free ones.  A page is live while an active entry of some row's page table names it; nothing else is
// kept, so no count can drift from the tables.  All of it runs on the device without a word from the host, so a call can
// be captured; what a table holds beyond a row's active entries is not looked at, and page or row numbers out of range
// are passed over.
//
// Forking and compacting are two launches each.  The PLAN is one CTA: a bitmap of the live pages in shared memory (up to 524288
// pages; beyond that in global memory), filled from the active entries, counted once, from which ranks
// of live and free pages follow by popcount.  The APPLICATION is spread over the chip: table entries, and pages cut into
// pieces of 16 KB that CTAs take in turn, four 16-byte loads a thread in flight.  Copying is an application alone, freeing a plan that
// writes its lists.
#include <mutex>

#include "plx_common.cuh"
#include "plx_launch.h"
#include "plx_tma_host.h"

namespace plx {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256, kCopyUnroll = 4;              // 16 KB of a page per CTA and step
constexpr int kPieceChunks = kCopyThreads * kCopyUnroll;
constexpr int kMost = 1 << 30;                                  // pages, table entries, items of a list: strides of a CTA stay inside 32 bits
constexpr int kMaxBitmapWords = 32 * 1024;                      // bitmap and ranks, 128 KB of shared memory: 524288 pages

struct PoolArgs {
    void *k, *v;
    int n_pages, page_size, chunks_per_key;                     // 16-byte chunks of all heads of a key
    int chunks_per_row;                                         // of one head of a key
    int64_t k_sp, k_st, k_sh, v_sp, v_st, v_sh;                 // strides in 16-byte chunks
};

struct TableArgs {
    const int32_t *table, *lens;
    int32_t *new_table, *new_lens;
    int batch, pages_per_seq, shift, mask, n_pages;
    __device__ __forceinline__ int len(int b) const {
        const int64_t most = static_cast<int64_t>(pages_per_seq) << shift;
        return static_cast<int>(min(static_cast<int64_t>(max(lens[b], 0)), most));
    }
    __device__ __forceinline__ bool in_pool(int p) const { return static_cast<uint32_t>(p) < static_cast<uint32_t>(n_pages); }
};

// The live pages as bits, and after rank(): how many live pages lie before each word.
struct Bitmap {
    uint32_t *bits;
    int32_t *before;
    int words;
    __device__ __forceinline__ bool live(int p) const { return bits[p >> 5] >> (p & 31) & 1u; }
    __device__ __forceinline__ int live_before(int p) const { return before[p >> 5] + __popc(bits[p >> 5] & ((1u << (p & 31)) - 1u)); }
};

__device__ __forceinline__ int warp_scan(int x, int lane) {       // inclusive
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
    }
    return x;
}
// exclusive scan over the CTA; the total in `total`
__device__ __forceinline__ int cta_scan(int x, int *s_warp, int &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int incl = warp_scan(x, lane);
    __syncthreads();                       // s_warp may still be read from the scan before
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const int w = s_warp[lane];
        s_warp[lane] = warp_scan(w, lane);
    }
    __syncthreads();
    total = s_warp[31];
    return incl - x + (warp > 0 ? s_warp[warp - 1] : 0);
}

__device__ __forceinline__ void clear(const Bitmap &m) {
    for (int i = threadIdx.x; i < m.words; i += kPlanThreads) m.bits[i] = 0u;
    __syncthreads();
}
// The active entries of the table -> bits; len(b): the keys of row b.
template <typename Len>
__device__ __forceinline__ void mark(const Bitmap &m, const TableArgs &t, Len len) {
    // a warp takes 128 entries of a row at a time, of four rows at once: bound by the round trips for lengths and entries
    constexpr int kAhead = 4, kRows = 4;
    const int lane = threadIdx.x & 31, segments = (t.pages_per_seq + 32 * kAhead - 1) / (32 * kAhead), units = t.batch * segments;
    for (int unit0 = threadIdx.x >> 5; unit0 < units; unit0 += kRows * kPlanThreads / 32) {
        int p[kRows][kAhead], active[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int unit = unit0 + i * kPlanThreads / 32;
            active[i] = unit < units ? static_cast<int>(min((static_cast<int64_t>(max(len(unit / segments), 0)) + t.mask) >> t.shift,
                                                            static_cast<int64_t>(t.pages_per_seq))) : 0;
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int unit = unit0 + i * kPlanThreads / 32, b = unit / segments, j0 = (unit - b * segments) * 32 * kAhead + lane;
            const int32_t *row = t.table + static_cast<int64_t>(b) * t.pages_per_seq;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) p[i][u] = j0 + 32 * u < active[i] ? row[j0 + 32 * u] : -1;
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (t.in_pool(p[i][u])) atomicOr(m.bits + (p[i][u] >> 5), 1u << (p[i][u] & 31));
    }
    __syncthreads();
}
// -> the number of live pages
__device__ __forceinline__ int rank(const Bitmap &m, int *s_warp) {
    const int per = (m.words + kPlanThreads - 1) / kPlanThreads, w0 = threadIdx.x * per, w1 = min(w0 + per, m.words);
    int n = 0, total;
    for (int w = w0; w < w1; ++w) n += __popc(m.bits[w]);
    int at = cta_scan(n, s_warp, total);
    for (int w = w0; w < w1; ++w) {
        m.before[w] = at;
        at += __popc(m.bits[w]);
    }
    __syncthreads();
    return total;
}

// One copy: `keys` keys from the start of page src to page dst.
struct Move {
    int src, dst, keys;
};

// Piece `piece` of a move of `keys` keys: chunks piece * kPieceChunks .. of them.  FLAT: the keys of a page follow one another
// without gaps, so that a chunk lies where its number says.
template <bool FLAT>
__device__ __forceinline__ void copy_piece(const PoolArgs &pool, const Move &mv, int piece, bool second) {
    const int64_t sp = second ? pool.v_sp : pool.k_sp, st = second ? pool.v_st : pool.k_st, sh = second ? pool.v_sh : pool.k_sh;
    uint4 *base = static_cast<uint4 *>(second ? pool.v : pool.k);
    const uint4 *src = base + mv.src * sp;
    uint4 *dst = base + mv.dst * sp;
    const int n = mv.keys * pool.chunks_per_key, c0 = piece * kPieceChunks + threadIdx.x;
    uint4 x[kCopyUnroll];
    auto at = [&](int c) -> int64_t {
        if (FLAT) return c;
        const int key = c / pool.chunks_per_key, rest = c - key * pool.chunks_per_key, h = rest / pool.chunks_per_row;
        return key * st + h * sh + (rest - h * pool.chunks_per_row);
    };
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (c0 + u * kCopyThreads < n) x[u] = src[at(c0 + u * kCopyThreads)];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (c0 + u * kCopyThreads < n) dst[at(c0 + u * kCopyThreads)] = x[u];
}

__host__ __device__ inline int pieces_of(int keys, int chunks_per_key) { return (keys * chunks_per_key + kPieceChunks - 1) / kPieceChunks; }

// Pages src[i] -> dst[i]; grid (pieces of a page, 2: k and v, n).
template <bool FLAT>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const PoolArgs pool, const int32_t *src, const int32_t *dst) {
    grid_wait();
    const Move mv{src[blockIdx.z], dst[blockIdx.z], pool.page_size};
    if (static_cast<uint32_t>(mv.src) >= static_cast<uint32_t>(pool.n_pages) || static_cast<uint32_t>(mv.dst) >= static_cast<uint32_t>(pool.n_pages) ||
        mv.src == mv.dst)
        return;
    copy_piece<FLAT>(pool, mv, blockIdx.x, blockIdx.y != 0);
}

// What a plan leaves for the application, in the workspace.
struct Plan {
    int32_t *n_moves;      // and how many pages to move there are
    Move *moves;
    int32_t *map;          // compaction: where a page goes that lies behind the live ones
    int32_t *last;         // fork: the last mention of each row among the children, or -1
    int32_t *fresh;        // fork: the page that entry i of the lists gets; -1: none needed, -2: none left
    uint32_t *bits;        // bitmap and ranks of pools too large for shared memory (else null)
    int32_t *before;
};

extern __shared__ __align__(16) uint32_t pages_smem[];
__device__ __forceinline__ Bitmap bitmap_of(const Plan &plan, int n_pages) {
    const int words = (n_pages + 31) / 32;
    return plan.bits ? Bitmap{plan.bits, plan.before, words} : Bitmap{pages_smem, reinterpret_cast<int32_t *>(pages_smem) + words, words};
}

// ------------------------------------------------------------------------- //
// compaction
// ------------------------------------------------------------------------- //
// With n live pages, the i-th live page from n on goes to the i-th free page below n: as many of the one as of the
// other, and no page is both a source and a target.
constexpr int kHoles = 8192;              // targets that are passed on through shared memory; more, through the list of moves
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const TableArgs t, const Plan plan, int32_t *n_live) {
    __shared__ int s_warp[32];
    __shared__ int s_holes[kHoles];
    grid_wait();
    const Bitmap m = bitmap_of(plan, t.n_pages);
    clear(m);
    mark(m, t, [&](int b) { return t.len(b); });
    const int n = rank(m, s_warp);
    const int front = n < t.n_pages ? m.live_before(n) : n;       // live pages that stay
    const bool small = n - front <= kHoles;
    for (int p = threadIdx.x; p < n; p += kPlanThreads)
        if (!m.live(p)) {
            const int i = p - m.live_before(p);
            if (small) s_holes[i] = p;
            else plan.moves[i].dst = p;
        }
    __syncthreads();
    for (int p = n + threadIdx.x; p < t.n_pages; p += kPlanThreads)
        if (m.live(p)) {
            const int i = m.live_before(p) - front, to = small ? s_holes[i] : plan.moves[i].dst;
            plan.moves[i].src = p;
            plan.moves[i].dst = to;
            plan.map[p] = to;
        }
    if (threadIdx.x == 0) {
        *plan.n_moves = n - front;
        *n_live = n;
    }
}

template <bool FLAT>
__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(const PoolArgs pool, const TableArgs t, const Plan plan, const int32_t *n_live) {
    grid_wait();
    const int n = __ldcg(n_live), n_moves = __ldcg(plan.n_moves), pieces = pieces_of(pool.page_size, pool.chunks_per_key);
    const int64_t units = 2ll * n_moves * pieces;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int i = static_cast<int>(u / (2 * pieces)), rest = static_cast<int>(u - static_cast<int64_t>(i) * 2 * pieces);
        const Move mv{__ldcg(&plan.moves[i].src), __ldcg(&plan.moves[i].dst), pool.page_size};
        copy_piece<FLAT>(pool, mv, rest >> 1, rest & 1);
    }
    const int entries = t.batch * t.pages_per_seq;
    for (int64_t i64 = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x; i64 < entries; i64 += static_cast<int64_t>(gridDim.x) * kCopyThreads) {
        const int i = static_cast<int>(i64), b = i / t.pages_per_seq, j = i - b * t.pages_per_seq;
        int p = t.table[i];
        if ((static_cast<int64_t>(j) << t.shift) < t.len(b) && t.in_pool(p) && p >= n) p = __ldcg(plan.map + p);
        t.new_table[i] = p;
    }
}

// ------------------------------------------------------------------------- //
// forking rows
// ------------------------------------------------------------------------- //
// Row children[i] becomes row parents[i]: it shares the parent's whole pages and gets a page of its own for a last one
// that is not full, the next free one in the order of the lists.  Free are the pages that no row held BEFORE the call, those
// of the rows that are overwritten among them: they may be what is copied from.
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const TableArgs t, const Plan plan, const int32_t *parents, const int32_t *children, int n,
                                                                 int32_t *missing) {
    __shared__ int s_warp[32];
    grid_wait();
    const Bitmap m = bitmap_of(plan, t.n_pages);
    for (int b = threadIdx.x; b < t.batch; b += kPlanThreads) plan.last[b] = -1;
    clear(m);
    auto ok = [&](int i) {
        return static_cast<uint32_t>(parents[i]) < static_cast<uint32_t>(t.batch) && static_cast<uint32_t>(children[i]) < static_cast<uint32_t>(t.batch);
    };
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (ok(i)) atomicMax(plan.last + children[i], i);
    mark(m, t, [&](int b) { return t.len(b); });
    const int n_free = t.n_pages - rank(m, s_warp);
    int needed = 0;
    for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
        const int i = i0 + threadIdx.x;
        // (a row that is its own child keeps its page)
        const bool needs = i < n && ok(i) && __ldcg(plan.last + children[i]) == i && parents[i] != children[i] && (t.len(parents[i]) & t.mask) != 0;
        int total;
        const int at = needed + cta_scan(needs ? 1 : 0, s_warp, total);
        if (i < n) plan.fresh[i] = !needs ? -1 : at < n_free ? at : -2;      // the rank of its page among the free ones, for now
        if (needs && at < n_free) {
            const int parent = parents[i], len = t.len(parent);
            plan.moves[at].src = t.table[static_cast<int64_t>(parent) * t.pages_per_seq + (len >> t.shift)];
            plan.moves[at].keys = len & t.mask;
        }
        needed += total;
    }
    const int given = min(needed, n_free);
    __syncthreads();
    for (int w = threadIdx.x; w < m.words; w += kPlanThreads) {
        int at = 32 * w - m.before[w];                   // free pages before this word
        if (at >= given) continue;
        uint32_t free = ~m.bits[w];
        if (32 * (w + 1) > t.n_pages) free &= (1u << (t.n_pages & 31)) - 1u;
        for (; free && at < given; free &= free - 1u, ++at) plan.moves[at].dst = 32 * w + __ffs(free) - 1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (plan.fresh[i] >= 0) plan.fresh[i] = plan.moves[plan.fresh[i]].dst;
    if (threadIdx.x == 0) {
        *plan.n_moves = given;
        *missing = needed - given;
    }
}

template <bool FLAT>
__global__ void __launch_bounds__(kCopyThreads) fork_apply_kernel(const PoolArgs pool, const TableArgs t, const Plan plan, const int32_t *parents) {
    grid_wait();
    const int n_moves = __ldcg(plan.n_moves), pieces = pieces_of(pool.page_size, pool.chunks_per_key);
    const int64_t units = 2ll * n_moves * pieces;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int i = static_cast<int>(u / (2 * pieces)), rest = static_cast<int>(u - static_cast<int64_t>(i) * 2 * pieces);
        const Move mv{__ldcg(&plan.moves[i].src), __ldcg(&plan.moves[i].dst), __ldcg(&plan.moves[i].keys)};
        if (t.in_pool(mv.src)) copy_piece<FLAT>(pool, mv, rest >> 1, rest & 1);
    }
    const int entries = t.batch * t.pages_per_seq;
    for (int64_t i64 = static_cast<int64_t>(blockIdx.x) * kCopyThreads + threadIdx.x; i64 < entries; i64 += static_cast<int64_t>(gridDim.x) * kCopyThreads) {
        const int i = static_cast<int>(i64), b = i / t.pages_per_seq, j = i - b * t.pages_per_seq;
        const int by = __ldcg(plan.last + b), from = by < 0 ? b : parents[by], fresh = by < 0 ? -1 : __ldcg(plan.fresh + by);
        int p = t.table[static_cast<int64_t>(from) * t.pages_per_seq + j];
        if (fresh != -1 || j == 0) {
            const int len = by < 0 ? t.lens[b] : t.len(from);
            if (fresh != -1 && j == len >> t.shift) p = max(fresh, -1);
            // without a page for its last keys a row ends with the whole pages
            if (j == 0) t.new_lens[b] = fresh == -2 ? len & ~t.mask : len;
        }
        t.new_table[i] = p;
    }
}

// ------------------------------------------------------------------------- //
// freeing rows
// ------------------------------------------------------------------------- //
__global__ void __launch_bounds__(kPlanThreads) free_kernel(const TableArgs t, const Plan plan, const int32_t *rows, int n_rows, int32_t *free_list,
                                                            int32_t *n_free) {
    __shared__ int s_warp[32];
    grid_wait();
    const Bitmap m = bitmap_of(plan, t.n_pages);
    for (int b = threadIdx.x; b < t.batch; b += kPlanThreads) t.new_lens[b] = t.lens[b];
    clear(m);
    for (int i = threadIdx.x; i < n_rows; i += kPlanThreads)
        if (static_cast<uint32_t>(rows[i]) < static_cast<uint32_t>(t.batch)) t.new_lens[rows[i]] = 0;
    __syncthreads();
    mark(m, t, [&](int b) { return t.new_lens[b]; });
    const int n = t.n_pages - rank(m, s_warp);
    for (int p = threadIdx.x; p < t.n_pages; p += kPlanThreads)
        if (!m.live(p)) free_list[p - m.live_before(p)] = p;
    for (int i = n + threadIdx.x; i < t.n_pages; i += kPlanThreads) free_list[i] = -1;
    if (threadIdx.x == 0) *n_free = n;
}

// ------------------------------------------------------------------------- //
// host side
// ------------------------------------------------------------------------- //
template <typename... Params, typename... Args>
int launch(void (*kern)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t st = cudaLaunchKernelEx(&cfg, kern, args...);
    count_launch();
    return st == cudaSuccess && cudaGetLastError() == cudaSuccess ? PLX_OK : PLX_ERR_LAUNCH;
}

// shared memory of a plan: bitmap and ranks, or nothing where they live in the workspace
size_t plan_smem(int n_pages) {
    const int words = (n_pages + 31) / 32;
    return 2 * words <= kMaxBitmapWords ? 8u * words : 0;
}

template <auto kKernel>
bool opt_in() {
    static std::mutex mu;
    static bool done[tma::kMaxDevices] = {};
    return tma::opt_in_smem(kKernel, 4 * kMaxBitmapWords, done, mu);
}

size_t aligned(size_t bytes) { return (bytes + 15u) & ~static_cast<size_t>(15u); }

// The parts of a workspace; returns its size.  n_forks: 0 for compacting, kFree for freeing, which needs the bitmap alone.
constexpr int kFree = -1;
size_t lay_out(unsigned char *ws, int n_pages, int batch, int n_forks, Plan *plan) {
    size_t at = 0;
    auto part = [&](size_t bytes) {
        unsigned char *p = ws ? ws + at : nullptr;
        at += aligned(bytes);
        return p;
    };
    const size_t moves = n_forks > 0 ? n_forks : n_forks == kFree ? 0 : n_pages, words = (static_cast<size_t>(n_pages) + 31) / 32;
    const bool global = plan_smem(n_pages) == 0;
    Plan p{};
    p.n_moves = reinterpret_cast<int32_t *>(part(moves ? 4 : 0));
    p.moves = reinterpret_cast<Move *>(part(sizeof(Move) * moves));
    p.map = reinterpret_cast<int32_t *>(part(n_forks == 0 ? 4 * moves : 0));
    p.last = reinterpret_cast<int32_t *>(part(n_forks > 0 ? 4 * static_cast<size_t>(batch) : 0));
    p.fresh = reinterpret_cast<int32_t *>(part(n_forks > 0 ? 4 * moves : 0));
    p.bits = global ? reinterpret_cast<uint32_t *>(part(4 * words)) : nullptr;
    p.before = global ? reinterpret_cast<int32_t *>(part(4 * words)) : nullptr;
    if (plan) *plan = p;
    return at;
}

int log2_of(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

// PLX_OK and `a` filled, or the status to return; `flat`: see copy_piece
int make_pool(const plx_page_pool *p, PoolArgs &a, bool &flat) {
    if (!p || !p->k || !p->v || p->n_pages <= 0 || p->page_size <= 0 || p->heads_kv <= 0 || p->head_dim <= 0) return PLX_ERR_BAD_ARG;
    if ((p->page_size & (p->page_size - 1)) != 0 || p->head_dim % 8 != 0) return PLX_ERR_BAD_ARG;
    if (((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15u) != 0) return PLX_ERR_BAD_ARG;
    const int64_t strides[] = {p->k_stride_p, p->k_stride_t, p->k_stride_h, p->v_stride_p, p->v_stride_t, p->v_stride_h};
    for (int64_t s : strides)
        if (s < 0 || (s & 7) != 0) return PLX_ERR_BAD_ARG;
    if (p->n_pages > 1 && (p->k_stride_p == 0 || p->v_stride_p == 0)) return PLX_ERR_BAD_ARG;      // pages on top of each other
    const int64_t row = p->head_dim, key = row * p->heads_kv;
    if (key / 8 * p->page_size > INT32_MAX / 2 || p->n_pages > kMost) return PLX_ERR_UNSUPPORTED;
    a = PoolArgs{};
    a.k = p->k; a.v = p->v;
    a.n_pages = p->n_pages; a.page_size = p->page_size;
    a.chunks_per_key = static_cast<int>(key / 8); a.chunks_per_row = static_cast<int>(row / 8);
    a.k_sp = p->k_stride_p / 8; a.k_st = p->k_stride_t / 8; a.k_sh = p->k_stride_h / 8;
    a.v_sp = p->v_stride_p / 8; a.v_st = p->v_stride_t / 8; a.v_sh = p->v_stride_h / 8;
    auto dense = [&](int64_t st, int64_t sh) { return (p->page_size == 1 || st == key) && (p->heads_kv == 1 || sh == row); };
    flat = dense(p->k_stride_t, p->k_stride_h) && dense(p->v_stride_t, p->v_stride_h);
    return PLX_OK;
}

int make_table(const int32_t *table, const int32_t *lens, int batch, int pages_per_seq, int n_pages, int page_size, TableArgs &t) {
    if (!table || !lens || batch <= 0 || pages_per_seq <= 0 || n_pages <= 0 || page_size <= 0 || (page_size & (page_size - 1)) != 0) return PLX_ERR_BAD_ARG;
    if (static_cast<int64_t>(batch) * pages_per_seq > kMost || n_pages > kMost) return PLX_ERR_UNSUPPORTED;
    t = TableArgs{};
    t.table = table; t.lens = lens;
    t.batch = batch; t.pages_per_seq = pages_per_seq; t.n_pages = n_pages;
    t.shift = log2_of(page_size); t.mask = page_size - 1;
    return PLX_OK;
}

// CTAs of an application: what the pages and the entries at most ask for, up to 32 an SM, four times what is resident.
// (16384 pages of 16 keys, 8 heads of 128, 536 MB read and written: 8 an SM 107.6 us, 16 100.2, 32 97.1 with 4 loads a thread in flight; 98.0 to
// 101.7 with 8 or 2, 117 with 1 or 16.)
int apply_grid(const PoolArgs &pool, const TableArgs &t, int64_t moves) {
    const int sms = tma::sm_count();
    const int64_t units = 2 * moves * pieces_of(pool.page_size, pool.chunks_per_key);
    const int64_t entries = (static_cast<int64_t>(t.batch) * t.pages_per_seq + kCopyThreads - 1) / kCopyThreads;
    const int64_t want = units > entries ? units : entries, most = 32ll * sms;
    return static_cast<int>(want < most ? want : most);
}

}  // namespace

int launch_pages_copy(const plx_page_pool *p, const int32_t *src, const int32_t *dst, int n, cudaStream_t stream) {
    PoolArgs pool;
    bool flat;
    int st = make_pool(p, pool, flat);
    if (st != PLX_OK) return st;
    if (n < 0 || (n > 0 && (!src || !dst))) return PLX_ERR_BAD_ARG;
    if (n > kMost) return PLX_ERR_UNSUPPORTED;
    if ((st = check_device()) != PLX_OK) return st;
    const int pieces = pieces_of(pool.page_size, pool.chunks_per_key);
    for (int at = 0; at < n && st == PLX_OK; at += 65535) {          // the grid's third axis
        const dim3 grid(pieces, 2, n - at < 65535 ? n - at : 65535);
        st = flat ? launch(copy_kernel<true>, grid, kCopyThreads, 0, stream, pool, src + at, dst + at)
                  : launch(copy_kernel<false>, grid, kCopyThreads, 0, stream, pool, src + at, dst + at);
    }
    return st;
}

int pages_workspace_bytes(int n_pages, int batch, int n_forks, size_t *bytes) {
    if (n_pages <= 0 || batch <= 0 || n_forks < 0 || !bytes) return PLX_ERR_BAD_ARG;
    if (n_pages > kMost || batch > kMost || n_forks > kMost) return PLX_ERR_UNSUPPORTED;
    *bytes = lay_out(nullptr, n_pages, batch, n_forks, nullptr);
    return PLX_OK;
}
int pages_free_workspace_bytes(int n_pages, size_t *bytes) {
    if (n_pages <= 0 || !bytes) return PLX_ERR_BAD_ARG;
    if (n_pages > kMost) return PLX_ERR_UNSUPPORTED;
    *bytes = lay_out(nullptr, n_pages, 1, kFree, nullptr);
    return PLX_OK;
}

int launch_pages_compact(const plx_page_pool *p, const int32_t *table, const int32_t *lens, int batch, int pages_per_seq, int32_t *new_table, int32_t *n_live,
                         void *ws, size_t ws_bytes, cudaStream_t stream) {
    PoolArgs pool;
    TableArgs t;
    bool flat;
    int st = make_pool(p, pool, flat);
    if (st == PLX_OK) st = make_table(table, lens, batch, pages_per_seq, p->n_pages, p->page_size, t);
    if (st != PLX_OK) return st;
    if (!new_table || !n_live) return PLX_ERR_BAD_ARG;
    Plan plan;
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) != 0 || lay_out(static_cast<unsigned char *>(ws), p->n_pages, batch, 0, &plan) > ws_bytes) return PLX_ERR_WORKSPACE;
    t.new_table = new_table;
    if ((st = check_device()) != PLX_OK) return st;
    if (!opt_in<compact_plan_kernel>()) return PLX_ERR_LAUNCH;
    st = launch(compact_plan_kernel, dim3(1), kPlanThreads, plan_smem(p->n_pages), stream, t, plan, n_live);
    if (st != PLX_OK) return st;
    const int grid = apply_grid(pool, t, p->n_pages / 2);            // a move has a live page and a free one
    return flat ? launch(compact_apply_kernel<true>, dim3(grid), kCopyThreads, 0, stream, pool, t, plan, static_cast<const int32_t *>(n_live))
                : launch(compact_apply_kernel<false>, dim3(grid), kCopyThreads, 0, stream, pool, t, plan, static_cast<const int32_t *>(n_live));
}

int launch_pages_fork(const plx_page_pool *p, const int32_t *table, const int32_t *lens, int batch, int pages_per_seq, const int32_t *parents,
                      const int32_t *children, int n, int32_t *new_table, int32_t *new_lens, int32_t *missing, void *ws, size_t ws_bytes,
                      cudaStream_t stream) {
    PoolArgs pool;
    TableArgs t;
    bool flat;
    int st = make_pool(p, pool, flat);
    if (st == PLX_OK) st = make_table(table, lens, batch, pages_per_seq, p->n_pages, p->page_size, t);
    if (st != PLX_OK) return st;
    if (n <= 0 || !parents || !children || !new_table || !new_lens || !missing) return PLX_ERR_BAD_ARG;
    if (n > kMost) return PLX_ERR_UNSUPPORTED;
    Plan plan;
    if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) != 0 || lay_out(static_cast<unsigned char *>(ws), p->n_pages, batch, n, &plan) > ws_bytes) return PLX_ERR_WORKSPACE;
    t.new_table = new_table;
    t.new_lens = new_lens;
    if ((st = check_device()) != PLX_OK) return st;
    if (!opt_in<fork_plan_kernel>()) return PLX_ERR_LAUNCH;
    st = launch(fork_plan_kernel, dim3(1), kPlanThreads, plan_smem(p->n_pages), stream, t, plan, parents, children, n, missing);
    if (st != PLX_OK) return st;
    const int grid = apply_grid(pool, t, n);
    return flat ? launch(fork_apply_kernel<true>, dim3(grid), kCopyThreads, 0, stream, pool, t, plan, parents)
                : launch(fork_apply_kernel<false>, dim3(grid), kCopyThreads, 0, stream, pool, t, plan, parents);
}

int launch_pages_free(const int32_t *table, const int32_t *lens, int batch, int pages_per_seq, const int32_t *rows, int n_rows, int n_pages, int page_size,
                      int32_t *new_lens, int32_t *free_list, int32_t *n_free, void *ws, size_t ws_bytes, cudaStream_t stream) {
    TableArgs t;
    int st = make_table(table, lens, batch, pages_per_seq, n_pages, page_size, t);
    if (st != PLX_OK) return st;
    if (n_rows < 0 || (n_rows > 0 && !rows) || !new_lens || !free_list || !n_free) return PLX_ERR_BAD_ARG;
    if (n_rows > kMost) return PLX_ERR_UNSUPPORTED;
    Plan plan;
    const size_t need = lay_out(static_cast<unsigned char *>(ws), n_pages, batch, kFree, &plan);
    if (need > 0 && (!ws || (reinterpret_cast<uintptr_t>(ws) & 15u) != 0 || need > ws_bytes)) return PLX_ERR_WORKSPACE;
    t.new_lens = new_lens;
    if ((st = check_device()) != PLX_OK) return st;
    if (!opt_in<free_kernel>()) return PLX_ERR_LAUNCH;
    return launch(free_kernel, dim3(1), kPlanThreads, plan_smem(n_pages), stream, t, plan, rows, n_rows, free_list, n_free);
}

}  // namespace plx
