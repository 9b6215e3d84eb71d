// Pages of a paged key/value cache forked, copied, given back and compacted (no
// counterpart in the reference, whose caches are contiguous): mi_paged_fork,
// mi_paged_compact.
//
// Which pages are in use follows from the block table and the lengths alone; there is
// no count of a page's holders that could go wrong beside them. A page is in use if some
// request's live entries (the first ceil(len / page)) name it.
//
// Fork: before and after are the sets of pages in use by the old rows and by the rows
// that the sources name, as bitmaps; before without after goes back to the free list, in
// the order of ids. A source whose last page is part-filled leaves it to one child (itself,
// else its first); each other child takes a page, from the end of the list, and a copy.
// Compact: the n pages in use with ids from n on move, in order, into the free ids below n.
//
// Two launches each: one marks, a workgroup a request, and its last workgroup to finish
// does the bookkeeping for all; the second writes the table's rows and moves the data of
// all layers, a wave a head of a page of a pool, however many copies there are. (The
// rows are written in a second launch since others are still read in the first; no page
// that is written is read: free and freed pages are no source of a copy.)
//
// Bound by HBM where pages are moved (figures at pages_move_kernel); else by two launches and
// the trips to memory in the first, one after another: lengths, rows, marks, ticket, bitmaps,
// lists (four beams 11 to 12 us, of which the first launch takes 8.5).
#include "mi_common.h"

namespace mi {
namespace {

constexpr int PG_MAX_R = 4096, PG_THREADS = 512;
constexpr int64_t PG_MAX_PAGES = (int64_t)1 << 20, PG_MAX_W = 131072;
constexpr int64_t PG_BITMAP = PG_MAX_PAGES / 8;  // bytes
static_assert(MI_PAGES_ZERO_BYTES == 64 + 2 * PG_BITMAP, "a ticket and two bitmaps");

struct PagesArgs {
    int *table, *lens;
    const int *sources;
    int *free_pages, *free_count, *result;
    void *const *pools;
    int R, W, page_log2, pages, n_free, n_pools, HK, row_bytes;
    // the workspace
    unsigned *ticket, *before, *after;
    int *head;  // [0]: moves, -1: nothing changes; [1]: pages in use (compact)
    int *moves;     // (from, to, rows, -) each
    int *new_len;   // fork, a request: its new length,
    int *new_last;  //   and its copy of its last page (-1: none)
    int *rows;      //   and the table as it was
    int *to;        // compact, a page: where it moves
};

// Live pages of a request of `len` keys, whose length is held to its row of the table.
__device__ __forceinline__ int held(const PagesArgs &a, int len) {
    return min(max(len, 0), a.W << a.page_log2);
}
__device__ __forceinline__ int pages_of(const PagesArgs &a, int len) {
    return (held(a, len) + (1 << a.page_log2) - 1) >> a.page_log2;
}
__device__ __forceinline__ void mark(unsigned *map, int id, int pages) {
    if ((unsigned)id < (unsigned)pages)
        __hip_atomic_fetch_or(map + (id >> 5), 1u << (id & 31), __ATOMIC_RELAXED,
                              __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T> __device__ __forceinline__ T get_agent(const T *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T> __device__ __forceinline__ void put_agent(T *p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// What the workgroup's threads have stored with agent scope is read by others of it.
__device__ __forceinline__ void settled() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
}

// The sum of v over the workgroup's threads before this one, and over all.
__device__ __forceinline__ int wg_before(int v, int *total) {
    __shared__ int waves[PG_THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int upto = wave_scan(v);
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    int at = upto - v, all = 0;
    for (int w = 0; w < PG_THREADS / 64; ++w) {
        if (w < wave) at += waves[w];
        all += waves[w];
    }
    __syncthreads();
    *total = all;
    return at;
}

// A bitmap's words of this thread, [w0, w1) of `words`, each read once where there are at
// most KEPT of them (65536 pages).
template <typename F> struct Words {
    static constexpr int KEPT = 4;
    F get;
    int w0, w1;
    unsigned kept[KEPT];
    __device__ __forceinline__ Words(int words, F get_) : get(get_) {
        const int per = (words + PG_THREADS - 1) / PG_THREADS;
        w0 = min((int)threadIdx.x * per, words), w1 = min(w0 + per, words);
#pragma unroll
        for (int i = 0; i < KEPT; ++i) kept[i] = w0 + i < w1 ? get(w0 + i) : 0;
    }
    template <typename G> __device__ __forceinline__ void each(G f) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i)
            if (w0 + i < w1) f(w0 + i, kept[i]);
        for (int w = w0 + KEPT; w < w1; ++w) f(w, get(w));
    }
};
template <typename F> __device__ __forceinline__ Words<F> words_of(int pages, F get) {
    return Words<F>((pages + 31) >> 5, get);
}

__device__ __forceinline__ void fork_books(const PagesArgs &a) {
    __shared__ int keeper[PG_MAX_R], source[PG_MAX_R], length[PG_MAX_R];  // length: the source's
    const int each = (a.R + PG_THREADS - 1) / PG_THREADS;
    const int r0 = min((int)threadIdx.x * each, a.R), r1 = min(r0 + each, a.R);
    const int mask = (1 << a.page_log2) - 1;
    const int count = min(max(*a.free_count, 0), a.n_free);
    int wrong = 0;
    for (int r = r0; r < r1; ++r) {
        const int s = a.sources[r];
        wrong += s >= a.R;
        source[r] = (unsigned)s < (unsigned)a.R ? s : -1;
        keeper[r] = 0x7fffffff;
    }
    auto gone = words_of(a.pages, [&](int w) { return get_agent(a.before + w) & ~get_agent(a.after + w); });
    int mine = 0;
    gone.each([&](int, unsigned g) { mine += __popc(g); });
    for (int r = r0; r < r1; ++r) length[r] = source[r] < 0 ? 0 : a.lens[source[r]];
    __syncthreads();
    for (int r = r0; r < r1; ++r)
        if (source[r] >= 0) atomicMin(&keeper[source[r]], source[r] == r ? -1 : r);
    __syncthreads();
    auto copies = [&](int r) {
        const int s = source[r];
        return s >= 0 && (held(a, length[r]) & mask) && keeper[s] != (s == r ? -1 : r);
    };
    int need = 0;
    for (int r = r0; r < r1; ++r) need += copies(r);
    int freed, needed, wrongs;
    const int at = wg_before(mine, &freed);
    const int taken = wg_before(need, &needed);
    wg_before(wrong, &wrongs);
    const int have = min(count + freed, a.n_free);
    const int lacking = max(needed - have, 0) + wrongs;
    const bool ok = lacking == 0;
    // pages back to the list; the bitmaps zero again
    int i = count + at;
    gone.each([&](int w, unsigned g) {
        put_agent(a.before + w, 0u);
        put_agent(a.after + w, 0u);
        for (; ok && g; g &= g - 1, ++i)
            if (i < a.n_free) put_agent(a.free_pages + i, 32 * w + __builtin_ctz(g));
    });
    settled();
    for (int r = r0, j = taken; ok && r < r1; ++r) {
        int page = -1;
        if (copies(r)) {
            page = get_agent(a.free_pages + (have - 1 - j));
            const int n = held(a, length[r]);
            int *m = a.moves + 4 * j++;
            m[0] = a.table[(int64_t)source[r] * a.W + (n >> a.page_log2)];
            m[1] = page;
            m[2] = n & mask;
        }
        a.new_len[r] = length[r];
        a.new_last[r] = page;
    }
    if (threadIdx.x == 0) {
        a.head[0] = ok ? needed : -1;
        *a.result = lacking;
        if (ok) *a.free_count = have - needed;  // (every thread has read it: barriers since)
    }
}

__device__ __forceinline__ void compact_books(const PagesArgs &a) {
    auto used = words_of(a.pages, [&](int w) { return get_agent(a.before + w); });
    int mine = 0, live, n, holes = 0, movers = 0;
    used.each([&](int, unsigned u) { mine += __popc(u); });
    wg_before(mine, &live);
    // the bits of word w that lie below page `live`
    auto below = [&](int w) {
        const int d = live - 32 * w;
        return d >= 32 ? ~0u : d <= 0 ? 0u : (1u << d) - 1;
    };
    used.each([&](int w, unsigned u) {
        const unsigned b = below(w);
        holes += __popc(~u & b);
        movers += __popc(u & ~b);
    });
    int h = wg_before(holes, &n), m = wg_before(movers, &n);
    used.each([&](int w, unsigned u) {
        const unsigned b = below(w);
        put_agent(a.before + w, 0u);
        for (unsigned g = ~u & b; g; g &= g - 1)
            put_agent(a.moves + 4 * h++ + 1, 32 * w + __builtin_ctz(g));
        for (unsigned g = u & ~b; g; g &= g - 1, ++m) {
            put_agent(a.moves + 4 * m, 32 * w + __builtin_ctz(g));
            a.moves[4 * m + 2] = 1 << a.page_log2;
        }
    });
    settled();
    for (int i = threadIdx.x; i < n; i += PG_THREADS)
        a.to[get_agent(a.moves + 4 * i)] = get_agent(a.moves + 4 * i + 1);
    if (threadIdx.x == 0) {
        a.head[0] = n;
        a.head[1] = live;
        *a.result = live;
        *a.free_count = a.pages - live;
    }
}

// A workgroup a request.
template <bool FORK> __global__ __launch_bounds__(PG_THREADS) void pages_mark_kernel(PagesArgs a) {
    const int r = blockIdx.x;
    const int n = pages_of(a, a.lens[r]);
    const int *row = a.table + (int64_t)r * a.W;
    for (int w = threadIdx.x; w < n; w += PG_THREADS) {
        const int id = row[w];
        mark(a.before, id, a.pages);
        if (FORK) a.rows[(int64_t)r * a.W + w] = id;
    }
    if (FORK) {
        const int s = a.sources[r];
        if ((unsigned)s < (unsigned)a.R) {
            const int m = pages_of(a, a.lens[s]);
            for (int w = threadIdx.x; w < m; w += PG_THREADS)
                mark(a.after, a.table[(int64_t)s * a.W + w], a.pages);
        }
    }
    if (!last_of(a.ticket, a.R)) return;
    if (FORK)
        fork_books(a);
    else
        compact_books(a);
}

// Rows of the table, lengths and the free list, then the moves' data: a wave a head of
// a page of a pool, past the caches, but for the part-filled pages that a fork copies, which
// are few and were written by the last step (64 beams of twelve layers, 40 MB moved, both
// launches: 20.2 us, with ordinary stores 22.5, loads past the caches 26; compaction of 538
// MB 217 us, 5.2 TB/s, a copy's rate; with ordinary loads and stores 238).
template <bool FORK> __global__ __launch_bounds__(256) void pages_move_kernel(PagesArgs a) {
    const int n = a.head[0];
    if (n < 0) return;
    for (int r = blockIdx.x; r < a.R; r += gridDim.x) {
        int *row = a.table + (int64_t)r * a.W;
        if (FORK) {
            const int s = a.sources[r], len = a.new_len[r], last = a.new_last[r];
            if (s == r) continue;
            const int m = pages_of(a, len);
            for (int w = threadIdx.x; w < m; w += 256)
                row[w] = w == m - 1 && last >= 0 ? last : a.rows[(int64_t)s * a.W + w];
            if (threadIdx.x == 0) a.lens[r] = len;
        } else {
            const int live = a.head[1], m = pages_of(a, a.lens[r]);
            for (int w = threadIdx.x; w < m; w += 256) {
                const int id = row[w];
                if (id >= live && id < a.pages) row[w] = a.to[id];
            }
        }
    }
    if (!FORK) {
        const int free = a.pages - a.head[1];
        for (int i = blockIdx.x * 256 + threadIdx.x; i < free; i += gridDim.x * 256)
            a.free_pages[i] = a.pages - 1 - i;
    }
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t jobs = (int64_t)n * a.n_pools * a.HK;
    const int64_t head_bytes = (int64_t)a.row_bytes << a.page_log2;
    for (int64_t j = (int64_t)blockIdx.x * 4 + wave; j < jobs; j += (int64_t)gridDim.x * 4) {
        const int64_t mp = j / a.HK;
        const int h = (int)(j - mp * a.HK), move = (int)(mp / a.n_pools);
        const int *m = a.moves + 4 * move;
        const int from = m[0], to = m[1], bytes = m[2] * a.row_bytes;
        if ((unsigned)from >= (unsigned)a.pages || (unsigned)to >= (unsigned)a.pages) continue;
        char *pool = (char *)a.pools[mp - (int64_t)move * a.n_pools];
        const char *src = pool + ((int64_t)from * a.HK + h) * head_bytes;
        char *dst = pool + ((int64_t)to * a.HK + h) * head_bytes;
        constexpr int IN_FLIGHT = 8;
        for (int i = 16 * lane; i < bytes; i += 1024 * IN_FLIGHT) {
            uint4 v[IN_FLIGHT];
#pragma unroll
            for (int k = 0; k < IN_FLIGHT; ++k)
                if (i + 1024 * k < bytes)
                    v[k] = FORK ? ld16(src + i + 1024 * k) : ld16_nt(src + i + 1024 * k);
#pragma unroll
            for (int k = 0; k < IN_FLIGHT; ++k)
                if (i + 1024 * k < bytes) st16_nt(dst + i + 1024 * k, v[k]);
        }
    }
}

// The workspace behind the zeroed prefix.
inline int64_t pages_bytes(bool fork, int64_t R, int64_t W, int64_t pages) {
    const int64_t ints = fork ? 16 + 4 * R + 2 * R + R * W : 16 + 4 * (pages / 2 + 1) + pages;
    return MI_PAGES_ZERO_BYTES + 4 * ints;
}

int check_pages(const char *what, int64_t R, int64_t W, int64_t page_size, int64_t n_pages,
                int64_t n_free, int64_t n_pools, int64_t HK, int64_t row_bytes, int &lp) {
    for (lp = 4; lp <= 8 && page_size != (1 << lp); ++lp) {}
    if (lp > 8)
        return fail(MI_ERR_UNSUPPORTED, "page size %lld; this build covers 16, 32, 64, 128, 256",
                    (long long)page_size);
    if (R < 0 || R > PG_MAX_R || W < 1 || W > PG_MAX_W || n_pages < 1 || n_pages > PG_MAX_PAGES ||
        n_free < n_pages || n_free > 0x3fffffff)
        return fail(MI_ERR_ARG, "%s R=%lld (to %d) table width %lld (to %lld) pages=%lld (to 2^20) "
                    "free list of %lld (all pages)", what, (long long)R, PG_MAX_R, (long long)W,
                    (long long)PG_MAX_W, (long long)n_pages, (long long)n_free);
    if (n_pools < 0 || n_pools > 65536 || HK < 1 || HK > 65536 || row_bytes < 16 ||
        row_bytes % 16 || row_bytes > 65536)
        return fail(MI_ERR_ARG, "%s pools=%lld (to 65536) heads=%lld rows of %lld bytes (a multiple "
                    "of 16)", what, (long long)n_pools, (long long)HK, (long long)row_bytes);
    return MI_OK;
}

template <bool FORK>
int launch_pages(PagesArgs a, int64_t workspace_bytes, void *workspace, hipStream_t st) {
    const int64_t need = pages_bytes(FORK, a.R, a.W, a.pages);
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return fail(MI_ERR_ARG, "a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
    char *ws = (char *)workspace;
    a.ticket = (unsigned *)ws;
    a.before = (unsigned *)(ws + 64);
    a.after = (unsigned *)(ws + 64 + PG_BITMAP);
    a.head = (int *)(ws + MI_PAGES_ZERO_BYTES);
    a.moves = a.head + 16;
    if (FORK) {
        a.new_len = a.moves + 4 * a.R;
        a.new_last = a.new_len + a.R;
        a.rows = a.new_last + a.R;
    } else {
        a.to = a.moves + 4 * (a.pages / 2 + 1);
    }
    pages_mark_kernel<FORK><<<(unsigned)a.R, PG_THREADS, 0, st>>>(a);
    // (waves for as many heads of pages as there can be, at most so many workgroups)
    const int64_t jobs = (FORK ? a.R : a.pages / 2) * (int64_t)a.n_pools * a.HK;
    int64_t grid = ceil_div(jobs, 4);
    if (grid < a.R) grid = a.R;
    if (grid > (FORK ? 2048 : 8192)) grid = FORK ? 2048 : 8192;
    pages_move_kernel<FORK><<<(unsigned)grid, 256, 0, st>>>(a);
    return launch_status(FORK ? "paged fork" : "paged compact");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_paged_fork_workspace_bytes(int64_t R, int64_t table_width) {
    return R < 0 || table_width < 1 ? 0 : pages_bytes(true, R, table_width, 0);
}
extern "C" int64_t mi_paged_compact_workspace_bytes(int64_t n_pages) {
    return n_pages < 1 ? 0 : pages_bytes(false, 0, 0, n_pages);
}

extern "C" int mi_paged_fork(int32_t *block_table, int64_t table_width, int32_t *kv_lens,
                             const int32_t *sources, int64_t R, int32_t *free_pages, int64_t n_free,
                             int32_t *free_count, int32_t *refused, void *const *pools,
                             int64_t n_pools, int64_t n_pages, int64_t Hkv, int64_t page_size,
                             int64_t row_bytes, void *workspace, int64_t workspace_bytes,
                             void *stream) {
    int lp;
    if (const int e = check_pages("paged fork", R, table_width, page_size, n_pages, n_free, n_pools,
                                  Hkv, row_bytes, lp))
        return e;
    if (R == 0) return fail(MI_ERR_ARG, "paged fork R=0");
    if (!block_table || !kv_lens || !sources || !free_pages || !free_count || !refused ||
        (n_pools && !pools))
        return fail(MI_ERR_ARG, "null pointer");
    PagesArgs a = {};
    a.table = block_table, a.lens = kv_lens, a.sources = sources, a.free_pages = free_pages;
    a.free_count = free_count, a.result = refused, a.pools = pools;
    a.R = (int)R, a.W = (int)table_width, a.page_log2 = lp, a.pages = (int)n_pages;
    a.n_free = (int)n_free, a.n_pools = (int)n_pools, a.HK = (int)Hkv, a.row_bytes = (int)row_bytes;
    return launch_pages<true>(a, workspace_bytes, workspace, as_stream(stream));
}

extern "C" int mi_paged_compact(int32_t *block_table, int64_t table_width, const int32_t *kv_lens,
                                int64_t R, int32_t *free_pages, int64_t n_free, int32_t *free_count,
                                int32_t *live, void *const *pools, int64_t n_pools, int64_t n_pages,
                                int64_t Hkv, int64_t page_size, int64_t row_bytes, void *workspace,
                                int64_t workspace_bytes, void *stream) {
    int lp;
    if (const int e = check_pages("paged compact", R, table_width, page_size, n_pages, n_free,
                                  n_pools, Hkv, row_bytes, lp))
        return e;
    if (R == 0) return fail(MI_ERR_ARG, "paged compact R=0");
    if (!block_table || !kv_lens || !free_pages || !free_count || !live || (n_pools && !pools))
        return fail(MI_ERR_ARG, "null pointer");
    PagesArgs a = {};
    a.table = block_table, a.lens = const_cast<int *>(kv_lens), a.free_pages = free_pages;
    a.free_count = free_count, a.result = live, a.pools = pools;
    a.R = (int)R, a.W = (int)table_width, a.page_log2 = lp, a.pages = (int)n_pages;
    a.n_free = (int)n_free, a.n_pools = (int)n_pools, a.HK = (int)Hkv, a.row_bytes = (int)row_bytes;
    return launch_pages<false>(a, workspace_bytes, workspace, as_stream(stream));
}
