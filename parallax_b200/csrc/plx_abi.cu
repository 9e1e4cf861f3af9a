// extern "C" surface of libplx_sm100.so (declared in include/plx_abi.h):
// argument validation, kernel selection, launch accounting.
#include <algorithm>
#include <array>
#include <atomic>
#include <cmath>

#include "plx_common.cuh"
#include "plx_decode.h"
#include "plx_launch.h"

namespace plx {

static std::atomic<uint64_t> g_launches{0};
void count_launch() { g_launches.fetch_add(1, std::memory_order_relaxed); }

// The kernels are built for sm_100a only; anything else must fail loudly, not fall back.
int check_device() {
    static std::atomic<int> cached[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return PLX_ERR_DEVICE;
    if (dev >= 0 && dev < 64) {
        int c = cached[dev].load(std::memory_order_relaxed);
        if (c != 0) return c > 0 ? PLX_OK : PLX_ERR_DEVICE;
    }
    int major = 0;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess) return PLX_ERR_DEVICE;
    const bool ok = major == 10;
    if (dev >= 0 && dev < 64) cached[dev].store(ok ? 1 : -1, std::memory_order_relaxed);
    return ok ? PLX_OK : PLX_ERR_DEVICE;
}

static int check_train(const plx_train_problem *p) {
    if (!p) return PLX_ERR_BAD_ARG;
    if (p->batch <= 0 || p->heads_q <= 0 || p->heads_kv <= 0 || p->len_q <= 0 || p->len_k <= 0) return PLX_ERR_BAD_ARG;
    if (p->heads_q % p->heads_kv != 0) return PLX_ERR_BAD_ARG;
    if (p->window_left < -1) return PLX_ERR_BAD_ARG;
    if (p->dtype != PLX_BF16 && p->dtype != PLX_FP16) return PLX_ERR_UNSUPPORTED;
    if (p->head_dim != 64 && p->head_dim != 128) return PLX_ERR_UNSUPPORTED;
    if (p->cu_seqlens) {
        if (p->batch != 1 || p->n_seqs <= 0 || p->len_q != p->len_k) return PLX_ERR_BAD_ARG;
    }
    // 16-byte vector accesses: every stride must be a multiple of 8 elements
    const int64_t strides[] = {p->q_stride_b, p->q_stride_h, p->q_stride_t, p->kv_stride_b, p->kv_stride_h, p->kv_stride_t};
    for (int64_t s : strides)
        if (s < 0 || (s & 7) != 0) return PLX_ERR_BAD_ARG;
    if (static_cast<int64_t>(p->batch) * p->heads_q > 65535) return PLX_ERR_UNSUPPORTED;
    return PLX_OK;
}

static bool misaligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

// n bytes from x and m bytes from y have one in common (null: none)
static bool overlap(const void *x, size_t n, const void *y, size_t m) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
    return x && y && a < b + m && b < a + n;
}

static TrainArgs make_train_args(const plx_train_problem *p) {
    TrainArgs a{};
    a.cu = p->cu_seqlens;
    a.n_seqs = p->cu_seqlens ? p->n_seqs : 0;
    a.batch = p->batch;
    a.heads_q = p->heads_q;
    a.heads_kv = p->heads_kv;
    a.n_rep = p->heads_q / p->heads_kv;
    a.len_q = p->len_q;
    a.len_k = p->len_k;
    a.window = p->window_left;
    a.scale = p->qk_scale;
    a.c2 = p->qk_scale * kLog2e;
    a.q_sb = p->q_stride_b; a.q_sh = p->q_stride_h; a.q_st = p->q_stride_t;
    a.kv_sb = p->kv_stride_b; a.kv_sh = p->kv_stride_h; a.kv_st = p->kv_stride_t;
    a.st_sb = p->st_stride_b; a.st_sh = p->st_stride_h; a.st_st = p->st_stride_t;
    return a;
}

static size_t train_stat_rows(const plx_train_problem *p) {
    // one 64-row tile of slack: the dk/dv kernel fetches the statistics of whole 64-row tiles and the
    // last tile may reach past the last token
    return static_cast<size_t>(p->batch) * p->heads_q * p->len_q + 64;
}

static size_t train_ws_bytes(const plx_train_problem *p) {
    // per (batch, q head, token): an 8-float record plus a compact 4-float record (see bwd_stats_kernel)
    return train_stat_rows(p) * 12 * sizeof(float);
}

// Sinks of a problem into its arguments; none where no window hides a key.
static void set_sinks(TrainArgs &a, int32_t sink_tokens) {
    if (sink_tokens <= 0 || a.window < 0 || a.window >= a.len_k) return;
    a.sink = sink_tokens < a.len_k ? sink_tokens : a.len_k;
    a.sink_chunk = train_sink_chunk(a.sink, a.window, a.len_q);
    const int64_t longest = a.len_q;          // of a pack: one sequence may hold all tokens
    if (longest > a.sink_chunk) a.sink_slots = static_cast<int>(a.cu ? 2 * longest / a.sink_chunk + 1 : (longest + a.sink_chunk - 1) / a.sink_chunk);
}
// bytes of the chunks' parts, behind the statistics
static size_t train_sink_bytes(const TrainArgs &a, int head_dim) {
    const size_t tiles = (static_cast<size_t>(a.sink) + 127) / 128;
    return a.sink ? static_cast<size_t>(a.sink_slots) * tiles * a.batch * a.heads_kv * 2 * 128 * head_dim * sizeof(float) : 0;
}

static int check_decode(const plx_decode_problem *p) {
    if (!p) return PLX_ERR_BAD_ARG;
    if (p->batch <= 0 || p->heads_q <= 0 || p->heads_kv <= 0 || p->cache_len <= 0 || p->n_splits <= 0 ||
        p->n_splits > PLX_DECODE_MAX_SPLITS)
        return PLX_ERR_BAD_ARG;
    if (p->heads_q % p->heads_kv != 0 || p->window_left < -1 || p->kv_offset < 0 || p->total_len < 0) return PLX_ERR_BAD_ARG;
    if (p->dtype != PLX_BF16 && p->dtype != PLX_FP16) return PLX_ERR_UNSUPPORTED;
    if (p->head_dim != 64 && p->head_dim != 128) return PLX_ERR_UNSUPPORTED;
    const int64_t strides[] = {p->kv_stride_b, p->kv_stride_t, p->kv_stride_h};
    for (int64_t s : strides)
        if (s < 0 || (s & 7) != 0) return PLX_ERR_BAD_ARG;
    if (p->heads_q > 65535 || p->batch > 65535) return PLX_ERR_UNSUPPORTED;
    if (p->page_table) {
        if (p->page_size < 1 || (p->page_size & (p->page_size - 1)) != 0 || p->pages_per_seq < 1) return PLX_ERR_BAD_ARG;
        if (static_cast<int64_t>(p->pages_per_seq) * p->page_size < p->cache_len) return PLX_ERR_BAD_ARG;
        if (p->kv_offset != 0) return PLX_ERR_UNSUPPORTED;   // a paged cache is not key-sharded
    }
    return PLX_OK;
}

static size_t decode_ws_bytes(const plx_decode_problem *p) {
    const size_t bh = static_cast<size_t>(p->batch) * p->heads_q;
    const size_t groups = PLX_DECODE_GROUPS(p->n_splits);
    return bh * (p->n_splits + groups) * PLX_DECODE_PART_FLOATS(p->head_dim) * sizeof(float) + bh * (1 + groups) * sizeof(int);
}

// the checks of a decode call that do not concern the workspace: problem, pointers, alignment, device
static int check_decode_args(const plx_decode_problem *p, const void *q, const void *r, const void *k, const void *v,
                             const void *out, const void *part) {
    int st = check_decode(p);
    if (st != PLX_OK) return st;
    if (!q || !r || !k || !v || (!out && !part)) return PLX_ERR_BAD_ARG;
    if (misaligned16(q) || misaligned16(r) || misaligned16(k) || misaligned16(v) || (out && misaligned16(out)))
        return PLX_ERR_BAD_ARG;
    return check_device();
}

// fills the kernel-side exchange block from the C struct; PLX_OK or the status to return
static int make_exchange_args(const plx_exchange *x, ExchangeArgs &e) {
    if (x->world < 1 || x->world > PLX_EXCHANGE_MAX_RANKS || x->rank < 0 || x->rank >= x->world || x->n_records <= 0)
        return PLX_ERR_BAD_ARG;
    if (x->head_dim != 64 && x->head_dim != 128) return PLX_ERR_UNSUPPORTED;
    for (int r = 0; r < x->world; ++r) {
        if (!x->inbox[r] || misaligned16(x->inbox[r])) return PLX_ERR_BAD_ARG;
        e.inbox[r] = static_cast<float *>(x->inbox[r]);
    }
    e.world = x->world; e.rank = x->rank; e.n_records = x->n_records;
    e.status = x->status;
    e.wait_ms = x->wait_ms ? x->wait_ms : PLX_EXCHANGE_DEFAULT_WAIT_MS;
    return PLX_OK;
}

// where a step leaves copies of its inputs (null: nowhere)
struct StepCopies {
    void *q, *r;
    int32_t *lens;
    const int32_t *lens_src;   // host
};

// which keys a sweep takes and where its partial state goes, where that is not the ordinary way
struct Sweep {
    int sink = 0;              // keys in front that stay visible behind the window
    int first_key = 0;         // keys before it are not looked at
    int min_len = 1;           // shorter lengths count as it
    int part_stride = 1;       // records between those of two (batch, head)
    int under = 0;             // runs under the launch before it, which has waited for what came before both
    const plx_prefix *prefix = nullptr;   // keys in tensors of their own that every row begins with
};

static int run_decode(const plx_decode_problem *p, const void *q, const void *r, const void *k, const void *v, void *out,
                      float *part, const int32_t *seqused_k, const int32_t *cache_start, void *workspace,
                      size_t workspace_bytes, cudaStream_t stream, const plx_exchange *xch = nullptr,
                      const StepCopies *step = nullptr, const Sweep &sweep = Sweep()) {
    if (sweep.sink < 0) return PLX_ERR_BAD_ARG;
    int st = check_decode_args(p, q, r, k, v, out, part);
    if (st != PLX_OK) return st;
    if (sweep.sink > 0 && (p->kv_offset != 0 || xch)) return PLX_ERR_UNSUPPORTED;   // sinks of a cache that is not key-sharded
    if (p->n_splits > 1 && (!workspace || workspace_bytes < decode_ws_bytes(p) || misaligned16(workspace)))
        return PLX_ERR_WORKSPACE;
    DecodeArgs a{};
    a.q = q; a.r = r; a.k = k; a.v = v;
    a.out = part ? nullptr : out;
    a.part_out = part;
    a.part_stride = sweep.part_stride;
    a.sink = p->window_left >= 0 && p->window_left < p->cache_len ? (sweep.sink < p->cache_len ? sweep.sink : p->cache_len) : 0;
    a.first_key = sweep.first_key;
    a.min_len = sweep.min_len;
    a.under = sweep.under;
    if (sweep.prefix) {
        a.k_prefix = sweep.prefix->k; a.v_prefix = sweep.prefix->v;
        a.prefix_len = sweep.prefix->len;
        a.prefix_st = sweep.prefix->stride_t; a.prefix_sh = sweep.prefix->stride_h;
    }
    a.seqused = seqused_k;
    a.cache_start = cache_start;
    const size_t bh = static_cast<size_t>(p->batch) * p->heads_q;
    // workspace: split records | group records | per-(batch, head) counters | group counters
    const size_t rec = PLX_DECODE_PART_FLOATS(p->head_dim), groups = PLX_DECODE_GROUPS(p->n_splits);
    a.n_groups = static_cast<int>(groups);
    a.ws_parts = static_cast<float *>(workspace);
    if (workspace) {
        a.ws_gparts = a.ws_parts + bh * p->n_splits * rec;
        a.ws_counters = reinterpret_cast<int *>(a.ws_gparts + bh * groups * rec);
        a.ws_gcounters = a.ws_counters + bh;
    }
    a.batch = p->batch; a.heads_q = p->heads_q; a.heads_kv = p->heads_kv; a.n_rep = p->heads_q / p->heads_kv;
    a.cache_len = p->cache_len; a.window = p->window_left; a.n_splits = p->n_splits;
    a.kv_offset = p->kv_offset;
    a.total_len = p->total_len > 0 ? p->total_len : p->cache_len;
    a.c2 = p->qk_scale * kLog2e;
    a.kv_sb = p->kv_stride_b; a.kv_st = p->kv_stride_t; a.kv_sh = p->kv_stride_h;
    if (xch) {
        if ((st = make_exchange_args(xch, a.xch)) != PLX_OK) return st;
        if (xch->n_records != p->batch * p->heads_q || xch->head_dim != p->head_dim || xch->dtype != p->dtype) return PLX_ERR_BAD_ARG;
        if (!decode_fused_exchange_supported(a)) return PLX_ERR_UNSUPPORTED;
        const ErrorWords ew = sm100_error_words();
        if (!ew.word) return PLX_ERR_LAUNCH;
        a.xch.err_word = ew.word;
        a.xch.err_mirror = ew.mirror;
    }
    if (step) {
        a.q_copy = step->q;
        a.r_copy = step->r;
        a.lens_copy = step->lens_src ? step->lens : nullptr;
        a.n_lens = step->lens_src ? p->batch : 0;
        for (int i = 0; i < a.n_lens; ++i) a.lens[i] = step->lens_src[i];
    }
    a.page_table = p->page_table;
    if (p->page_table) {
        a.pages_per_seq = p->pages_per_seq;
        a.last_page = p->n_pages > 0 ? static_cast<uint32_t>(p->n_pages) - 1u : INT32_MAX;
        a.page_mask = p->page_size - 1;
        a.page_shift = 0;
        while ((1 << a.page_shift) < p->page_size) ++a.page_shift;
    }
    return launch_decode(a, p->dtype, p->head_dim, stream);
}

static size_t prefix_part_bytes(const plx_decode_problem *p, const plx_prefix *x) {
    if (x->n_splits == 0) return 0;
    return static_cast<size_t>(p->batch) * p->heads_q * (x->n_splits + 1) * PLX_DECODE_PART_FLOATS(p->head_dim) * sizeof(float);
}

static int check_prefix(const plx_decode_problem *p, const plx_prefix *x) {
    if (!x || x->len <= 0 || x->n_splits < 0 || x->n_splits > PLX_PREFIX_MAX_SPLITS || p->window_left >= 0 || p->kv_offset != 0) return PLX_ERR_BAD_ARG;
    if (x->n_splits > (static_cast<int64_t>(x->len) + 63) / 64) return PLX_ERR_BAD_ARG;      // a part holds a tile of 64 keys at least
    if (!x->k)        // in the pages of the cache
        return p->page_table && p->n_pages > 0 && !x->v && x->len % p->page_size == 0 && x->len <= p->cache_len ? PLX_OK : PLX_ERR_BAD_ARG;
    if (!x->v || misaligned16(x->k) || misaligned16(x->v)) return PLX_ERR_BAD_ARG;
    if (p->page_table) return PLX_ERR_UNSUPPORTED;      // the kernels of kShared have no page table behind the prefix
    return x->stride_t >= 0 && x->stride_h >= 0 && (x->stride_t & 7) == 0 && (x->stride_h & 7) == 0 ? PLX_OK : PLX_ERR_BAD_ARG;
}

constexpr int kMostRows = 65535;      // rows of a shared launch are fewer: the sweep of own keys has one more CTA than they need

// a batch's rows against their prefix, but for pointers to q, r and keys
static TrainArgs make_prefix_args(const plx_decode_problem *p, const plx_prefix *x) {
    const bool in_cache = !x->k;                       // the rows' own page tables begin with the prefix
    TrainArgs a{};
    a.batch = p->batch; a.heads_q = p->heads_q; a.heads_kv = p->heads_kv; a.n_rep = p->heads_q / p->heads_kv;
    a.len_q = 1; a.len_k = x->len;
    a.window = -1;
    a.scale = p->qk_scale;
    a.c2 = p->qk_scale * kLog2e;
    a.q_st = p->head_dim; a.q_sh = static_cast<int64_t>(a.n_rep) * p->head_dim; a.q_sb = static_cast<int64_t>(p->heads_q) * p->head_dim;
    a.kv_sb = in_cache ? p->kv_stride_b : x->stride_t; a.kv_st = in_cache ? p->kv_stride_t : x->stride_t; a.kv_sh = in_cache ? p->kv_stride_h : x->stride_h;
    if (in_cache) {
        a.page_table = p->page_table;
        a.pages_per_seq = p->pages_per_seq;
        a.n_pages = p->n_pages;
        a.page_mask = p->page_size - 1;
        while ((1 << a.page_shift) < p->page_size) ++a.page_shift;
    }
    return a;
}

// the backward: the chosen stages (all of them with sinks)
static int run_train_bwd(const plx_train_problem *p, int32_t sink_tokens, int32_t stages, const void *q, const void *r, const void *k, const void *v,
                         const void *o, const void *barv, const float *d1, const float *bart, const float *m, const void *grad_o, void *dq, void *dr,
                         void *dk, void *dv, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    int st = check_train(p);
    if (st != PLX_OK) return st;
    if (sink_tokens < 0) return PLX_ERR_BAD_ARG;
    if (stages <= 0 || (stages & ~PLX_BWD_ALL) != 0) return PLX_ERR_BAD_ARG;
    if (!q || !r || !k || !v || !o || !barv || !d1 || !bart || !m || !grad_o || !dq || !dr || !dk || !dv)
        return PLX_ERR_BAD_ARG;
    const void *ptrs[] = {q, r, k, v, o, barv, grad_o, dq, dr, dk, dv};
    for (const void *x : ptrs)
        if (misaligned16(x)) return PLX_ERR_BAD_ARG;
    TrainArgs a = make_train_args(p);
    set_sinks(a, sink_tokens);
    if (!workspace || workspace_bytes < train_ws_bytes(p) + train_sink_bytes(a, p->head_dim) || misaligned16(workspace)) return PLX_ERR_WORKSPACE;
    if ((st = check_device()) != PLX_OK) return st;
    a.q = q; a.r = r; a.k = k; a.v = v; a.o_in = o; a.barv_in = barv; a.go = grad_o;
    a.d1 = const_cast<float *>(d1); a.bart = const_cast<float *>(bart); a.m = const_cast<float *>(m);
    a.dq = dq; a.dr = dr; a.dk = dk; a.dv = dv;
    a.bst = static_cast<float *>(workspace);
    a.cst = a.bst + train_stat_rows(p) * 8;
    a.parts = a.bst + train_stat_rows(p) * 12;
    cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
    const bool tc = train_bwd_sm100_supported(a, p->head_dim);
    // dk/dv before dq/dr: the two are independent, and the CTAs of the second start as those of the first, longer
    // one leave their SMs.  (The three kernels, B = 2, H = 8, L = 1024: 62.9 us one after the other, 43.5 so; at B = 4,
    // H = 16 174 against 145, at B = 8, H = 16, L = 4096 the same.)
    int before = 0;
    for (int stage : {PLX_BWD_STATS, PLX_BWD_DKV, PLX_BWD_DQR}) {
        if (!(stages & stage)) continue;
        const bool overlap = before == (stage == PLX_BWD_DKV ? PLX_BWD_STATS : PLX_BWD_DKV);
        st = (tc && stage != PLX_BWD_STATS) ? launch_train_bwd_sm100(a, p->dtype, p->head_dim, stage, overlap, cs)
                                            : launch_train_bwd_mma(a, p->dtype, p->head_dim, stage, cs);
        if (st != PLX_OK) return st;
        before = stage;
    }
    // (dq/dr waits for dk/dv at its end: what follows it follows both)
    if (tc && a.sink && a.sink_slots > 0) return launch_train_bwd_join(a, p->dtype, p->head_dim, cs);
    return PLX_OK;
}

// n_splits of plx_prefix and of the problem
static void plan_prefix(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t len, int32_t own_len, int32_t head_dim, int32_t sm_count,
                        int32_t *prefix_splits, int32_t *own_splits) {
    // A model of a call in units of 10 ns, its constants fitted at head_dim 128 to the times of 25 shapes at up to 90 pairs of splits each (4 to 200
    // rows, prefixes of 1000 to 32768 keys, 30 to 8000 own ones of uneven lengths): what it chooses is within 7% of the best pair for each of them.
    const bool grouped = heads_q > heads_kv;
    const int64_t rows = static_cast<int64_t>(batch) * heads_kv * (grouped ? (heads_q / heads_kv + 15) / 16 : 1);   // sweeps of own keys
    // own_len is the room that rows have; what they hold of it is on the device.  Up to 512 keys the plan is that for full rows; with more room
    // it has the least product of its times at 512 keys and at the room, counted up to 8192.  Measured over 19 shapes with rooms of 4096 and 65536 keys,
    // rows of 40 to 16384 in use, against the best way for each: 17% more time in the mean, the worst 1.9 times; the plan for full rows 62% and 10.8 times,
    // the one for 512 keys 46% and 12.1 times.  Device time with 512 keys in room for 512 / 8192 / 98304, us: 32 rows, 32 : 8 heads, 8192 keys in front
    // 29.9 / 31.6 / 31.4; 128 rows, 32768 keys 155 / 174 / 173; 16 rows, 8 : 1 heads, 16000 keys 24.2 / 30.8 / 29.7.
    const int64_t lens[2] = {std::min<int64_t>(own_len, 512), std::min<int64_t>(own_len, 8192)};
    const int n_lens = lens[1] > lens[0] ? 2 : 1;
    const int dim = n_lens > 1 ? 128 : head_dim;      // (64 takes 0.6 to 0.8 of the time, either way: its own figures in half the model are 29% off, those of 128 21%)
    // Shared.  The prefix: rounds of items over the SMs, 1.07 us a tile of 64 keys and about four tiles for start and end.  The own keys run beside
    // it, `k` times 16 of them in a CTA: one CTA on an SM of the prefix, which slows that one down, eight on an SM that the prefix leaves free; the
    // longest row's CTA may take longest.  So the best prefix may leave SMs free.  Then the merge.  (The two one after the other, each over all SMs: 32
    // rows, 32 : 8 heads, 8192 keys and 512 own ones 34.7 us against 29.2; 128 rows, 32768 keys 172 against 153.)
    const int64_t beside = grouped ? 80 : 460, free_start = grouped ? 300 : 380, free_step = grouped ? 140 : 240, tail_start = grouped ? 350 : 600,
                  tail_step = grouped ? 100 : 200;
    const int64_t units = static_cast<int64_t>(prefix_row_tiles(heads_q / heads_kv, batch)) * heads_kv, tiles = (static_cast<int64_t>(len) + 63) / 64;
    auto shared_time = [&](int n, int own, int64_t own_keys) {
        const int64_t rounds = (units * n + sm_count - 1) / sm_count, used = units * n / rounds, free = sm_count > used ? sm_count - used : 0;
        const int64_t prefix = 400 + rounds * (107 * ((tiles + n - 1) / n) + 400);
        const int64_t merge = 200 + static_cast<int64_t>(batch) * heads_q * (n + 1) * PLX_DECODE_PART_FLOATS(dim) * 4 / 40000;
        const int64_t k = (own_keys + 16 * own - 1) / (16 * own);
        const int64_t ctas = grouped || heads_q % 2 ? rows * own : rows * own / 2;
        int64_t cost = prefix;
        if (k > 0) {
            const double rate_beside = static_cast<double>(used) / (beside * k), rate = rate_beside + 8.0 * free / (free_start + free_step * k);
            const int64_t all = static_cast<int64_t>(ctas / rate), tail = tail_start + tail_step * k;
            cost += static_cast<int64_t>(0.75 * std::min(all, prefix) * rate_beside / rate);
            cost = std::max(cost, std::max(500 + all, tail) + std::min(all, tail) / 8);
        }
        return cost + merge;
    };
    // Every row sweeping the prefix in front of its own keys, one launch instead of three, its bytes at 4.4 TB/s with one q head per kv head and, the
    // rows meeting in L2, 9 with grouped ones.  Measured, device time of the call with 40 own keys, us, shared / every row: 8 : 8 heads, 4 rows, 500 keys
    // 11.4 / 7.2, 2000 12.6 / 11.4, 4000 14.7 / 17.4, 16000 25.0 / 66.1; 8 rows, 500 11.2 / 9.2, 1000 11.7 / 15.8; 16 rows, 500 11.3 / 14.3; 32 : 8 heads, 2 rows, 4000
    // 15.0 / 13.7, 16000 24.8 / 26.8; 4 rows, 4000 14.8 / 17.4; 16 rows, 500 12.8 / 12.0, 1000 13.3 / 16.3, 4000 16.4 / 38.8; 8 : 1 heads, 8 rows, 16000 19.8 / 20.0, 16 rows 21.0 / 28.2.
    auto every_row_time = [&](int64_t own_keys) {
        const int64_t kb = 4ll * batch * (len + own_keys) * heads_kv * dim / 1000;
        return grouped ? 1050 + kb / 90 : (static_cast<int64_t>(batch) * heads_q <= PLX_DECODE_SPLIT_GROUP_MAX_BH ? 450 : 900) + kb / 44;
    };
    int best = 1, best_own = 1;
    double shared = INFINITY, limit = 0, every_row = 1;      // (the model is 1/15 above the times of shared ones, where there are few own keys)
    for (int i = 0; i < n_lens; ++i) every_row *= static_cast<double>(every_row_time(lens[i]));
    for (int n = 1; n <= PLX_PREFIX_MAX_SPLITS && n <= tiles; ++n)
        for (int own = 1; own <= 32 && (own == 1 || 16 * own <= own_len); own *= 2) {
            double cost = 1, less = 1;
            for (int i = 0; i < n_lens; ++i) {
                const int64_t t = shared_time(n, own, lens[i]);
                cost *= static_cast<double>(t);
                less *= static_cast<double>(t * 15 / 16);
            }
            if (cost < shared) {
                shared = cost;
                limit = less;
                best = n;
                best_own = own;
            }
        }
    if (every_row < limit) {
        const int64_t keys = static_cast<int64_t>(len) + own_len;
        *prefix_splits = 0;
        *own_splits = plx_decode_choose_splits_gqa(batch, heads_q, heads_kv, static_cast<int32_t>(keys < INT32_MAX ? keys : INT32_MAX), sm_count);
        return;
    }
    *prefix_splits = best;
    *own_splits = best_own;
}

}  // namespace plx

using namespace plx;

extern "C" {

int plx_abi_version(void) { return PLX_ABI_VERSION; }

const char *plx_strerror(int status) {
    switch (status) {
        case PLX_OK: return "ok";
        case PLX_ERR_BAD_ARG: return "bad argument (null pointer, size, stride or alignment)";
        case PLX_ERR_UNSUPPORTED: return "unsupported dtype, head_dim or shape";
        case PLX_ERR_LAUNCH: return "CUDA kernel launch failed";
        case PLX_ERR_WORKSPACE: return "workspace missing, misaligned or too small";
        case PLX_ERR_DEVICE: return "current CUDA device is not sm_100 (B200)";
        case PLX_ERR_STATIC_SCRATCH:
            return "problem needs more split-KV scratch than the built-in array of plx_decode_static; lower n_splits "
                   "or call plx_decode with a caller-owned workspace";
        default: return "unknown status";
    }
}

uint64_t plx_kernel_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }

int plx_device_error(int32_t *value, int32_t clear) {
    if (!value) return PLX_ERR_BAD_ARG;
    int v = 0;
    int st = sm100_error_word(&v, clear != 0);
    *value = v;
    return st;
}

int plx_device_error_peek(int32_t *value, int32_t clear) {
    if (!value) return PLX_ERR_BAD_ARG;
    int v = 0;
    int st = sm100_error_peek(&v, clear != 0);
    *value = v;
    return st;
}

int plx_train_workspace_bytes(const plx_train_problem *p, size_t *bytes) {
    int st = check_train(p);
    if (st != PLX_OK) return st;
    if (!bytes) return PLX_ERR_BAD_ARG;
    *bytes = train_ws_bytes(p);
    return PLX_OK;
}

int plx_train_workspace_bytes_sink(const plx_train_problem *p, int32_t sink_tokens, size_t *bytes) {
    int st = check_train(p);
    if (st != PLX_OK) return st;
    if (!bytes || sink_tokens < 0) return PLX_ERR_BAD_ARG;
    TrainArgs a = make_train_args(p);
    set_sinks(a, sink_tokens);
    *bytes = train_ws_bytes(p) + train_sink_bytes(a, p->head_dim);
    return PLX_OK;
}

int plx_train_fwd(const plx_train_problem *p, const void *q, const void *r, const void *k, const void *v, void *o,
                  void *barv, float *d1, float *bart, float *m, plx_stream_t stream) {
    return plx_train_fwd_sink(p, 0, q, r, k, v, o, barv, d1, bart, m, stream);
}

int plx_train_fwd_sink(const plx_train_problem *p, int32_t sink_tokens, const void *q, const void *r, const void *k, const void *v, void *o,
                       void *barv, float *d1, float *bart, float *m, plx_stream_t stream) {
    int st = check_train(p);
    if (st != PLX_OK) return st;
    if (sink_tokens < 0) return PLX_ERR_BAD_ARG;
    if (!q || !r || !k || !v || !o || !barv || !d1 || !bart || !m) return PLX_ERR_BAD_ARG;
    if (misaligned16(q) || misaligned16(r) || misaligned16(k) || misaligned16(v) || misaligned16(o) || misaligned16(barv))
        return PLX_ERR_BAD_ARG;
    if ((st = check_device()) != PLX_OK) return st;
    TrainArgs a = make_train_args(p);
    set_sinks(a, sink_tokens);
    a.q = q; a.r = r; a.k = k; a.v = v; a.o = o; a.barv = barv; a.d1 = d1; a.bart = bart; a.m = m;
    if (train_fwd_sm100_supported(a, p->head_dim))
        return launch_train_fwd_sm100(a, p->dtype, p->head_dim, reinterpret_cast<cudaStream_t>(stream));
    return launch_train_fwd_mma(a, p->dtype, p->head_dim, reinterpret_cast<cudaStream_t>(stream));
}

int plx_train_extend(const plx_train_problem *p, const void *q, const void *r, const void *k, const void *v, void *o,
                     const int32_t *seqused_k, const int32_t *page_table, int32_t page_size, int32_t pages_per_seq,
                     int32_t n_pages, plx_stream_t stream) {
    return plx_train_extend_sink(p, 0, q, r, k, v, o, seqused_k, page_table, page_size, pages_per_seq, n_pages, stream);
}

int plx_train_extend_sink(const plx_train_problem *p, int32_t sink_tokens, const void *q, const void *r, const void *k, const void *v, void *o,
                          const int32_t *seqused_k, const int32_t *page_table, int32_t page_size, int32_t pages_per_seq,
                          int32_t n_pages, plx_stream_t stream) {
    int st = check_train(p);
    if (st != PLX_OK) return st;
    if (sink_tokens < 0) return PLX_ERR_BAD_ARG;
    if (!q || !r || !k || !v || !o || p->cu_seqlens || p->len_q > p->len_k) return PLX_ERR_BAD_ARG;
    if (misaligned16(q) || misaligned16(r) || misaligned16(k) || misaligned16(v) || misaligned16(o)) return PLX_ERR_BAD_ARG;
    TrainArgs a = make_train_args(p);
    set_sinks(a, sink_tokens);
    a.q = q; a.r = r; a.k = k; a.v = v; a.o = o;
    a.seqused = seqused_k;
    if (page_table) {
        if (page_size < 1 || (page_size & (page_size - 1)) != 0 || pages_per_seq < 1 || n_pages < 1) return PLX_ERR_BAD_ARG;
        if (static_cast<int64_t>(pages_per_seq) * page_size < p->len_k) return PLX_ERR_BAD_ARG;
        a.page_table = page_table;
        a.pages_per_seq = pages_per_seq;
        a.n_pages = n_pages;
        a.page_mask = page_size - 1;
        while ((1 << a.page_shift) < page_size) ++a.page_shift;
    }
    if ((st = check_device()) != PLX_OK) return st;
    if (!train_extend_sm100_supported(a, p->head_dim)) return PLX_ERR_UNSUPPORTED;
    return launch_train_extend_sm100(a, p->dtype, p->head_dim, reinterpret_cast<cudaStream_t>(stream));
}

int plx_train_bwd_stages(const plx_train_problem *p, int32_t stages, const void *q, const void *r, const void *k,
                         const void *v, const void *o, const void *barv, const float *d1, const float *bart,
                         const float *m, const void *grad_o, void *dq, void *dr, void *dk, void *dv, void *workspace,
                         size_t workspace_bytes, plx_stream_t stream) {
    return run_train_bwd(p, 0, stages, q, r, k, v, o, barv, d1, bart, m, grad_o, dq, dr, dk, dv, workspace, workspace_bytes, stream);
}

int plx_train_bwd_sink(const plx_train_problem *p, int32_t sink_tokens, const void *q, const void *r, const void *k, const void *v, const void *o,
                       const void *barv, const float *d1, const float *bart, const float *m, const void *grad_o, void *dq, void *dr, void *dk,
                       void *dv, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    return run_train_bwd(p, sink_tokens, PLX_BWD_ALL, q, r, k, v, o, barv, d1, bart, m, grad_o, dq, dr, dk, dv, workspace, workspace_bytes, stream);
}

int plx_train_bwd(const plx_train_problem *p, const void *q, const void *r, const void *k, const void *v, const void *o,
                  const void *barv, const float *d1, const float *bart, const float *m, const void *grad_o, void *dq,
                  void *dr, void *dk, void *dv, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    return plx_train_bwd_stages(p, PLX_BWD_ALL, q, r, k, v, o, barv, d1, bart, m, grad_o, dq, dr, dk, dv, workspace,
                                workspace_bytes, stream);
}

int plx_decode_choose_splits(int32_t batch, int32_t heads_q, int32_t n_keys, int32_t sm_count) {
    if (batch <= 0 || heads_q <= 0 || n_keys <= 0 || sm_count <= 0) return 1;
    // One warp per (batch, head, split).  Measured on B200: a launch is fastest when all its warps are
    // resident at once (16 per SM at this kernel's register count; one warp more starts a second wave
    // with a long tail, and more splits only add partial records to merge), unless that leaves more
    // than ~1024 keys to a warp, where several waves of smaller units balance better.  At least 32
    // keys per split.
    const int64_t bh = static_cast<int64_t>(batch) * heads_q;
    const int64_t resident = static_cast<int64_t>(sm_count) * 16;
    // Few (batch, head) pairs and not many keys: the launch is bound by latency.  Split groups (eight
    // splits per CTA, merged in shared memory): about 16 keys per warp, so that all of a warp's loads are
    // in flight at once, as long as every warp is resident; a multiple of 8, at most 256.
    if (bh <= PLX_DECODE_SPLIT_GROUP_MAX_BH && n_keys >= 128 && bh * n_keys <= (static_cast<int64_t>(1) << 19)) {
        if (n_keys <= 2048) {
            // at most eight CTAs per (batch, head): they form one thread-block cluster and merge through
            // distributed shared memory; 8, 16, 32 or 64 splits of at least 16 keys.  (Measured at B = 1,
            // H = 8: 4.8 / 6.1 us at 512 / 1024 keys.)
            int64_t g = 64;
            while (g > 8 && n_keys / g < 16) g /= 2;
            return static_cast<int>(g);
        }
        // Up to 6144 keys a cluster still wins where its CTAs are all resident at once and no warp walks
        // more than about 200 keys.  Measured (H = 8, cold K/V, us at 2560 / 3072 / 4096 / 6144 keys):
        // B = 1: 64 splits 7.9 / 7.9 / 9.4 / 11.8 against 9.6 / 10.2 / 11.0 / 12.2 for the rule below;
        // B = 4: 32 splits 12.4 / 13.8 / 16.5 / 21.7 against 14.5 / 16.2 / 19.2 / 24.1 (B = 3 alike);
        // B = 2, 6 and 8 are faster with the rule below.
        if (n_keys <= 6144) {
            if (bh <= 8) return 64;
            if (bh > 16 && bh <= 32) return 32;
        }
        int64_t g = (n_keys + 15) / 16;
        if (g > resident / bh) g = resident / bh;
        if (g > PLX_DECODE_MAX_SPLITS) g = PLX_DECODE_MAX_SPLITS;
        g -= g % 8;
        if (g >= 8) return static_cast<int>(g);
    }
    int64_t s = resident / bh;
    if (s < 1) s = 1;
    if (n_keys / s > 1024) s = (n_keys + 1023) / 1024;
    int64_t cap = n_keys / 32;
    if (cap < 1) cap = 1;
    if (s > cap) s = cap;
    if (s > PLX_DECODE_MAX_SPLITS) s = PLX_DECODE_MAX_SPLITS;
    return s < 1 ? 1 : static_cast<int>(s);
}

int plx_decode_choose_splits_gqa(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t n_keys, int32_t sm_count) {
    if (heads_kv <= 0 || heads_q <= heads_kv || heads_q % heads_kv != 0)
        return plx_decode_choose_splits(batch, heads_q, n_keys, sm_count);
    if (batch <= 0 || n_keys <= 0 || sm_count <= 0) return 1;
    // Grouped heads run one warp per (batch, kv head, 16-row head group, split), kDecodeGqaWarps
    // resident per SM (their K / V tiles fill the shared memory).  The warps of a launch run in waves of
    // that many: take the smallest split count whose last wave is at least 85 % full (or the fullest,
    // if none is), with at least 64 keys per split.
    const int64_t units = static_cast<int64_t>(batch) * heads_kv * ((heads_q / heads_kv + 15) / 16);
    const int64_t resident = static_cast<int64_t>(sm_count) * kDecodeGqaWarps;
    int64_t cap = n_keys / 64;
    if (cap < 1) cap = 1;
    if (cap > PLX_DECODE_MAX_SPLITS) cap = PLX_DECODE_MAX_SPLITS;
    int64_t best = 1;
    double best_fill = 0.0;
    for (int64_t s = 1; s <= cap; ++s) {
        const int64_t warps = units * s, waves = (warps + resident - 1) / resident;
        const double fill = static_cast<double>(warps) / static_cast<double>(waves * resident);
        if (fill > best_fill + 1e-9) {
            best_fill = fill;
            best = s;
        }
        if (fill >= 0.85) break;
    }
    // A warp sweeps whole tiles of 16 keys, so a part of 65 keys costs as much as one of 80 and leaves the last warps
    // without any: where that wastes more than 8 %, cut at a tile boundary instead if the warps still fit into as many
    // waves and the parts of a row into whole CTAs.  (B = 1, 8192 keys, 32 : 8 heads: 126 parts would be swept as 103 of 80
    // keys and 23 of none, waste 23 %; 128 parts of 64 keys, 16.4 -> 16.0 us.  Where rows then end inside a CTA it does not
    // pay: B = 2, 5200 keys, 16 %, 65 parts for 63 17.0 -> 20.8 us; B = 8, 1300 keys, 18 %, 17 for 16 16.4 -> 18.6.  Nor for a
    // waste of 2 %: 3 rows of 17104 keys in 90 parts took 35.6 us against 34.0 in 84.)
    const int64_t waves = (units * best + resident - 1) / resident, part = n_keys / best / 16 * 16;
    const int64_t swept = ((n_keys + best - 1) / best + 15) / 16 * 16;
    if (part >= 64 && 100 * swept * best > 108 * static_cast<int64_t>(n_keys)) {
        const int64_t even = (n_keys + part - 1) / part;
        if (even <= cap && even % kDecodeGqaWarps == 0 && units * even <= waves * resident) best = even;
    }
    return static_cast<int>(best);
}

int plx_decode_workspace_bytes(const plx_decode_problem *p, size_t *bytes) {
    int st = check_decode(p);
    if (st != PLX_OK) return st;
    if (!bytes) return PLX_ERR_BAD_ARG;
    *bytes = decode_ws_bytes(p);
    return PLX_OK;
}

// internal (not in plx_abi.h): lets plx_decode_static run plx_decode's checks before it enqueues its memset
int plx_decode_check_args(const plx_decode_problem *p, const void *q, const void *r, const void *k, const void *v,
                          const void *out) {
    if (!out) return PLX_ERR_BAD_ARG;
    return check_decode_args(p, q, r, k, v, out, nullptr);
}

int plx_decode_stage(void *q, const void *q_src, void *r, const void *r_src, size_t bytes, int32_t *seqused_k,
                     const int32_t *seqused_src, int32_t n, plx_stream_t stream) {
    if ((q_src && !q) || (r_src && !r) || (seqused_src && !seqused_k) || n < 0 || n > PLX_DECODE_STAGE_LENS || (bytes & 15u) != 0)
        return PLX_ERR_BAD_ARG;
    if (misaligned16(q) || misaligned16(q_src) || misaligned16(r) || misaligned16(r_src)) return PLX_ERR_BAD_ARG;
    // An element is copied to q, then to r, by one thread: a source may be the other buffer, but not a shifted part of one.
    for (const void *src : {q_src, r_src}) {
        if (q_src && src != q && overlap(src, bytes, q, bytes)) return PLX_ERR_UNSUPPORTED;
        if (r_src && src != r && overlap(src, bytes, r, bytes)) return PLX_ERR_UNSUPPORTED;
        if (seqused_src && overlap(src, bytes, seqused_k, n * sizeof(int32_t))) return PLX_ERR_UNSUPPORTED;
    }
    int st = check_device();
    if (st != PLX_OK) return st;
    return launch_decode_stage(q, q_src, r, r_src, bytes, seqused_k, seqused_src, n, reinterpret_cast<cudaStream_t>(stream));
}

int plx_decode_step(const plx_decode_problem *p, void *q, const void *q_src, void *r, const void *r_src, const void *k, const void *v, void *out,
                    int32_t *seqused_k, const int32_t *seqused_src, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    return plx_decode_step_sink(p, 0, q, q_src, r, r_src, k, v, out, seqused_k, seqused_src, workspace, workspace_bytes, stream);
}

int plx_decode_step_sink(const plx_decode_problem *p, int32_t sink_tokens, void *q, const void *q_src, void *r, const void *r_src, const void *k,
                         const void *v, void *out, int32_t *seqused_k, const int32_t *seqused_src, void *workspace, size_t workspace_bytes,
                         plx_stream_t stream) {
    if (!p || !out || !q || !r || (seqused_src && !seqused_k) || misaligned16(q) || misaligned16(r) || sink_tokens < 0) return PLX_ERR_BAD_ARG;
    if (p->batch > PLX_DECODE_STEP_ROWS) return PLX_ERR_UNSUPPORTED;
    const int st = check_decode(p);
    if (st != PLX_OK) return st;
    // The parts of a row read the sources while the first of them writes the copies: nothing that is written may lie in a source.
    const size_t bytes = static_cast<size_t>(p->batch) * p->heads_q * p->head_dim * 2;
    for (const void *src : {q_src, r_src}) {
        if ((q_src && overlap(src, bytes, q, bytes)) || (r_src && overlap(src, bytes, r, bytes)) || overlap(src, bytes, out, bytes) ||
            (seqused_src && overlap(src, bytes, seqused_k, p->batch * sizeof(int32_t))) ||
            (p->n_splits > 1 && overlap(src, bytes, workspace, decode_ws_bytes(p))))
            return PLX_ERR_UNSUPPORTED;
    }
    const StepCopies step{q_src ? q : nullptr, r_src ? r : nullptr, seqused_k, seqused_src};
    return run_decode(p, q_src ? q_src : q, r_src ? r_src : r, k, v, out, nullptr, seqused_src ? nullptr : seqused_k, nullptr, workspace,
                      workspace_bytes, reinterpret_cast<cudaStream_t>(stream), nullptr, &step, Sweep{sink_tokens});
}

int plx_decode(const plx_decode_problem *p, const void *q, const void *r, const void *k, const void *v, void *out,
               const int32_t *seqused_k, const int32_t *cache_start, void *workspace, size_t workspace_bytes,
               plx_stream_t stream) {
    if (!out) return PLX_ERR_BAD_ARG;
    return run_decode(p, q, r, k, v, out, nullptr, seqused_k, cache_start, workspace, workspace_bytes,
                      reinterpret_cast<cudaStream_t>(stream));
}

int plx_decode_sink(const plx_decode_problem *p, int32_t sink_tokens, const void *q, const void *r, const void *k, const void *v, void *out,
                    const int32_t *seqused_k, const int32_t *cache_start, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    if (!out) return PLX_ERR_BAD_ARG;
    return run_decode(p, q, r, k, v, out, nullptr, seqused_k, cache_start, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream), nullptr,
                      nullptr, Sweep{sink_tokens});
}

int plx_decode_prefix_plan(int32_t batch, int32_t heads_q, int32_t heads_kv, int32_t len, int32_t own_len, int32_t head_dim, int32_t sm_count,
                           int32_t *prefix_splits, int32_t *own_splits) {
    if (batch <= 0 || heads_kv <= 0 || heads_q < heads_kv || heads_q % heads_kv != 0 || len <= 0 || own_len < 0 || head_dim <= 0 || sm_count <= 0 ||
        !prefix_splits || !own_splits)
        return PLX_ERR_BAD_ARG;
    // Host arithmetic on these seven numbers, for up to 762 pairs, 20 to 50 us of a host core.  A decode loop asks the same for every
    // layer and step, so a thread keeps its last plans.
    struct Plan {
        std::array<int32_t, 7> key;
        int32_t prefix_splits, own_splits;
    };
    thread_local Plan plans[16] = {};                   // (a key of zeros is not valid)
    const std::array<int32_t, 7> key = {batch, heads_q, heads_kv, len, own_len, head_dim, sm_count};
    uint32_t h = 0;
    for (int32_t x : key) h = (h ^ static_cast<uint32_t>(x)) * 0x9E3779B1u;
    Plan &plan = plans[h >> 28];
    if (plan.key != key) {
        plan_prefix(batch, heads_q, heads_kv, len, own_len, head_dim, sm_count, &plan.prefix_splits, &plan.own_splits);
        plan.key = key;
    }
    *prefix_splits = plan.prefix_splits;
    *own_splits = plan.own_splits;
    return PLX_OK;
}

int plx_decode_prefix_plan_call(const plx_decode_problem *p, const plx_prefix *x, int32_t sm_count, int32_t *prefix_splits, int32_t *own_splits) {
    if (!p || !x || sm_count <= 0 || !prefix_splits || !own_splits) return PLX_ERR_BAD_ARG;
    plx_decode_problem problem = *p;
    plx_prefix prefix = *x;
    problem.n_splits = 1;
    prefix.n_splits = 0;
    int st = check_decode(&problem);
    if (st == PLX_OK) st = check_prefix(&problem, &prefix);
    if (st != PLX_OK) return st;
    const int64_t keys = x->k ? static_cast<int64_t>(x->len) + p->cache_len : p->cache_len;
    if (p->batch < kMostRows && train_extend_sm100_fits(make_prefix_args(p, x), p->head_dim))
        return plx_decode_prefix_plan(p->batch, p->heads_q, p->heads_kv, x->len, static_cast<int32_t>(keys - x->len), p->head_dim, sm_count, prefix_splits, own_splits);
    *prefix_splits = 0;
    *own_splits = plx_decode_choose_splits_gqa(p->batch, p->heads_q, p->heads_kv, static_cast<int32_t>(keys < INT32_MAX ? keys : INT32_MAX), sm_count);
    return PLX_OK;
}

int plx_decode_prefix_workspace_bytes(const plx_decode_problem *p, const plx_prefix *x, size_t *bytes) {
    int st = check_decode(p);
    if (st != PLX_OK) return st;
    if (!x || !bytes || x->n_splits < 0 || x->n_splits > PLX_PREFIX_MAX_SPLITS) return PLX_ERR_BAD_ARG;
    *bytes = prefix_part_bytes(p, x) + decode_ws_bytes(p);
    return PLX_OK;
}

int plx_decode_prefix(const plx_decode_problem *p, const plx_prefix *x, const void *q, const void *r, const void *k, const void *v, void *out,
                      const int32_t *seqused_k, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    int st = check_decode(p);
    if (st == PLX_OK) st = check_prefix(p, x);
    if (st == PLX_OK) st = check_decode_args(p, q, r, k, v, out, nullptr);
    if (st != PLX_OK) return st;
    const size_t part_bytes = prefix_part_bytes(p, x);
    if (!workspace || misaligned16(workspace) || workspace_bytes < part_bytes + decode_ws_bytes(p)) return PLX_ERR_WORKSPACE;
    const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
    float *parts = static_cast<float *>(workspace);
    unsigned char *rest = static_cast<unsigned char *>(workspace) + part_bytes;
    const size_t rest_bytes = workspace_bytes - part_bytes;
    const bool in_cache = !x->k;
    TrainArgs a = make_prefix_args(p, x);
    a.q = q; a.r = r;
    a.k = in_cache ? k : x->k;
    a.v = in_cache ? v : x->v;
    a.parts = parts;
    Sweep own;
    own.first_key = own.min_len = 0;
    if (x->n_splits == 0 || p->batch == kMostRows || !train_extend_sm100_supported(a, p->head_dim)) {
        // every row sweeps the prefix in front of its own keys, in one launch
        if (in_cache) own.min_len = x->len;
        else own.prefix = x;
        return run_decode(p, q, r, k, v, out, nullptr, seqused_k, nullptr, rest, rest_bytes, cs, nullptr, nullptr, own);
    }
    // The prefix, bound by the tensor pipe's tile period, takes a CTA per SM and lets the sweep of the rows' own keys in, bound by
    // memory, whose CTAs of a warp or two fit beside it.
    const int n_parts = x->n_splits + 1;
    a.n_splits = x->n_splits;
    a.n_parts = n_parts;
    if ((st = launch_prefix_sm100(a, p->dtype, p->head_dim, cs)) != PLX_OK) return st;
    if (in_cache) own.first_key = own.min_len = x->len;
    own.part_stride = n_parts;
    own.under = 1;
    st = run_decode(p, q, r, k, v, nullptr, parts + static_cast<size_t>(n_parts - 1) * PLX_DECODE_PART_FLOATS(p->head_dim), seqused_k, nullptr, rest, rest_bytes,
                    cs, nullptr, nullptr, own);
    if (st != PLX_OK) return st;
    return launch_prefix_merge(parts, n_parts, static_cast<int64_t>(p->batch) * p->heads_q, p->head_dim, p->dtype, out, cs);
}

int plx_decode_partial(const plx_decode_problem *p, const void *q, const void *r, const void *k, const void *v,
                       float *part, const int32_t *seqused_k, const int32_t *cache_start, void *workspace,
                       size_t workspace_bytes, plx_stream_t stream) {
    if (!part) return PLX_ERR_BAD_ARG;
    return run_decode(p, q, r, k, v, nullptr, part, seqused_k, cache_start, workspace, workspace_bytes,
                      reinterpret_cast<cudaStream_t>(stream));
}

int plx_decode_merge(const float *parts, int32_t n_parts, int32_t n_records, int32_t head_dim, int32_t dtype, void *out,
                     plx_stream_t stream) {
    if (!parts || !out || n_parts <= 0 || n_records <= 0) return PLX_ERR_BAD_ARG;
    int st = check_device();
    if (st != PLX_OK) return st;
    return launch_decode_merge(parts, n_parts, n_records, head_dim, dtype, out, reinterpret_cast<cudaStream_t>(stream));
}

size_t plx_decode_exchange_bytes(int32_t world, int32_t n_records, int32_t head_dim) {
    if (world <= 0 || n_records <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
    const size_t slots = static_cast<size_t>(2) * world * n_records;   // two parities
    return slots * PLX_DECODE_PART_FLOATS(head_dim) * sizeof(float) + slots * sizeof(uint32_t) +
           static_cast<size_t>(n_records) * sizeof(uint32_t);   // records, stamps, step counters
}

int plx_decode_partial_exchange(const plx_decode_problem *p, const plx_exchange *x, const void *q, const void *r,
                                const void *k, const void *v, void *out, const int32_t *seqused_k,
                                const int32_t *cache_start, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    if (!x || !out) return PLX_ERR_BAD_ARG;
    return run_decode(p, q, r, k, v, out, nullptr, seqused_k, cache_start, workspace, workspace_bytes,
                      reinterpret_cast<cudaStream_t>(stream), x);
}

int plx_decode_exchange_merge(const plx_exchange *x, const float *part, void *out, plx_stream_t stream) {
    if (!x || !part || !out) return PLX_ERR_BAD_ARG;
    if (misaligned16(part) || misaligned16(out)) return PLX_ERR_BAD_ARG;
    ExchangeArgs e{};
    int st = make_exchange_args(x, e);
    if (st != PLX_OK) return st;
    if ((st = check_device()) != PLX_OK) return st;
    const ErrorWords err = sm100_error_words();
    if (!err.word) return PLX_ERR_LAUNCH;
    return launch_decode_exchange_merge(e, part, x->head_dim, x->dtype, out, err, reinterpret_cast<cudaStream_t>(stream));
}

int plx_pages_copy(const plx_page_pool *p, const int32_t *src, const int32_t *dst, int32_t n, plx_stream_t stream) {
    return launch_pages_copy(p, src, dst, n, reinterpret_cast<cudaStream_t>(stream));
}

int plx_pages_workspace_bytes(int32_t n_pages, int32_t batch, int32_t n_forks, size_t *bytes) {
    return pages_workspace_bytes(n_pages, batch, n_forks, bytes);
}

int plx_pages_free_workspace_bytes(int32_t n_pages, size_t *bytes) { return pages_free_workspace_bytes(n_pages, bytes); }

int plx_pages_fork(const plx_page_pool *p, const int32_t *page_table, const int32_t *lens, int32_t batch, int32_t pages_per_seq,
                   const int32_t *parents, const int32_t *children, int32_t n, int32_t *new_page_table, int32_t *new_lens,
                   int32_t *missing, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    return launch_pages_fork(p, page_table, lens, batch, pages_per_seq, parents, children, n, new_page_table, new_lens, missing,
           workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

int plx_pages_compact(const plx_page_pool *p, const int32_t *page_table, const int32_t *lens, int32_t batch, int32_t pages_per_seq,
                      int32_t *new_page_table, int32_t *n_live, void *workspace, size_t workspace_bytes, plx_stream_t stream) {
    return launch_pages_compact(p, page_table, lens, batch, pages_per_seq, new_page_table, n_live, workspace, workspace_bytes,
           reinterpret_cast<cudaStream_t>(stream));
}

int plx_pages_free(const int32_t *page_table, const int32_t *lens, int32_t batch, int32_t pages_per_seq, const int32_t *rows, int32_t n_rows,
                   int32_t n_pages, int32_t page_size, int32_t *new_lens, int32_t *free_list, int32_t *n_free, void *workspace,
                   size_t workspace_bytes, plx_stream_t stream) {
    return launch_pages_free(page_table, lens, batch, pages_per_seq, rows, n_rows, n_pages, page_size, new_lens, free_list, n_free,
           workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
