// Causal GQA attention of requests that share a prefix, over a paged key/value cache (no
// counterpart in the reference, whose caches are contiguous): mi_paged_shared_plan,
// mi_paged_shared_attention.
//
// Requests come in groups; the first S keys of a group's requests lie in the same pages.
// For a row (token i of request r, q head h over kv head h / G), with s_j = scale log2(e)
// q . k_j over the keys j <= len - n + i that it sees:
//   o = (sum_c w_c O_c) / (sum_c w_c l_c),  w_c = 2^(m_c - max m),
// where the parts c cut the keys: some over [0, S), in which the rows of all the group's
// requests are columns of one block, so that these K and V are read once a group (or once
// for 128 columns of it), and some over [S, len) of the request alone; of each part m_c is
// the largest s_j, l_c = sum 2^(s_j - m_c), O_c = sum 2^(s_j - m_c) v_j.
//
// The plan is made once a step, for the attention of every layer: the keys that each group
// shares, from the table's rows, and a list of the parts. The attention is a workgroup a
// part and kv head, then a kernel that joins a row's parts. A block whose keys are not cut
// and that has no prefix writes its rows itself.
//
// What bounds it, on MI355X (32 q / 8 kv heads; calls back to back): four beams behind 960
// keys 13 us, of which a graph takes 9.3, two launches and a chain of trips to memory; 64
// requests in five groups, heads of 64, 94 MB, 27 us, HBM at 4.0 TB/s while the parts are read
// (24 us, of which about 6 are their starts and ends); 96 requests of up to four tokens behind
// 16256 keys, 359 MB and 61 GFLOP (92 with the rests' product), 133 us: the matrix cores over
// the prefix, busy 49% of the cycles, then HBM over the requests' own keys (43 us by
// themselves at 7 TB/s), which overlap little, since two workgroups a CU is all that its
// registers and LDS hold. The paged attention, which reads the prefix once a request, takes
// 12.1, 54 and 588 us in graphs, where these take 9.3, 27.5 and 137.
//
// Probabilities enter the second product as T, and the product of what that rounding left is
// taken too: over prefixes in groups of any size, over a request's own keys up to REST_COLS
// columns. What is off is then the result's own rounding (bf16 1.66e-3 of the norm, fp16
// 2.1e-4). Prompts, bound by these products, keep one rounding (2.1e-3 to 2.3e-3, 2.8e-4), as
// in the paged attention, which takes the rests of requests of at most 32 columns.
#include <type_traits>

#include "mi_paged_common.h"

namespace mi {
namespace {

// ---------------------------------------------------------------------------
// the plan

constexpr int SP_MAX_R = 4096;
constexpr int SP_THREADS = 1024;
// Keys that a group has to share, and the columns (rows of a kv head) that each of its
// requests may have, for it to be worth parts of its own. (us with / without: 16 groups of
// four sharing 64 keys 20.4 / 18.6, 128 21.0 / 22.3, 512 23.2 / 29.7, 1024 29.0 / 40.8; 16
// requests behind 2048, in fours, of 64 columns each 32.4 / 35.8, of 128 47.7 / 45.0; eight
// behind 4096 of 64 31.3 / 35.1, of 128 43.8 / 43.2.)
constexpr int SP_MIN_KEYS = 128, SP_MAX_COLS = 64;
// Columns up to which a request takes the probabilities' rests over its own keys: four wide
// blocks, steps of some tokens and short questions. (us with / without: 16 requests of 40
// tokens over 1000 keys 42 / 35, of 128 over 500 39 / 33, over 2000 109 / 86. Prompts, which
// nothing but the products bounds, would take half as many MFMAs again.)
constexpr int REST_COLS = 512;

// A part of the work, for one kv head.
enum { NARROW, WIDE_REST, WIDE };  // a block of 32 columns, or of 128
struct SharedItem {
    int r;       // the request whose pages hold the keys
    int t0;      // the first token of the columns' rows
    int cols;    // columns in all: token after token, in a token its G q heads
    int c0;      // the block's first
    int k0, k1;  // its keys
    int state;   // its first column's state, -1: the block writes its rows itself
    int kind;
};
// What a token's rows are joined from.
struct SharedToken {
    int seen;    // keys that it sees
    int prefix;  // the first state of its group's prefix, -1: none
    int prefix_parts;  // parts | columns of a block << 16
    int prefix_col;    // the token's first column there
    int own, own_parts, own_col;  // and of its own keys (own -1 and prefix -1: nothing to join)
    int unused;
};
struct SharedGroup {
    int lead;      // the request whose pages are read
    int keys;      // keys shared, 0 where they are not worth it
    int t0, cols;  // its tokens' first and their columns
};

struct PlanArgs {
    const int *table, *cu_q, *kv_lens, *cu_groups;
    int *keys;
    // the schedule
    int *head;  // [0]: items, [1]: the key of the sizes it is for
    SharedGroup *groups;
    int *group_of;  // a request
    SharedItem *items;
    SharedToken *tokens;
    int R, W, T, G, NG, page_log2;
    int max_items, slots, key;
    int64_t states;
};

// Request r's first token, tokens and keys, held to what there is.
struct Span {
    int q0, n, len;
};
__device__ __forceinline__ Span span_of(const PlanArgs &a, int r) {
    const int from = a.cu_q[r], to = a.cu_q[r + 1], len = a.kv_lens[r];
    Span s;
    s.q0 = min(max(from, 0), a.T);
    s.n = min(max(to, s.q0), a.T) - s.q0;
    s.len = min(max(len, 0), a.W << a.page_log2);
    return s;
}

// A workgroup a group: the leading entries of the table that all of its requests have
// alike, as far as each one's keys from before the step fill them. Requests without
// tokens or keys do not count.
__global__ __launch_bounds__(SP_THREADS) void shared_keys_kernel(PlanArgs a) {
    __shared__ int lead, limit, most, others;
    __shared__ bool part[SP_MAX_R];  // whether the request counts
    const int g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int first = min(max(a.cu_groups[g], 0), a.R);
    const int end = min(max(a.cu_groups[g + 1], first), a.R);
    if (threadIdx.x == 0) lead = a.R, limit = a.W, most = 0, others = 0;
    __syncthreads();
    for (int r = first + (int)threadIdx.x; r < end; r += SP_THREADS) {
        const Span s = span_of(a, r);
        a.group_of[r] = g;
        part[r] = s.n > 0 && s.len > 0;
        atomicMax(&most, s.n);  // (of all: their rows are columns of the prefix's blocks)
        if (!part[r]) continue;
        atomicMin(&lead, r);
        atomicMin(&limit, max(s.len - s.n, 0) >> a.page_log2);
        atomicAdd(&others, 1);
    }
    // requests outside the groups are in none
    if (g == 0)
        for (int r = threadIdx.x; r < first; r += SP_THREADS) a.group_of[r] = -1;
    if (g == a.NG - 1)
        for (int r = end + (int)threadIdx.x; r < a.R; r += SP_THREADS) a.group_of[r] = -1;
    __syncthreads();
    const int l = lead;
    if (l < end) {
        const int *with = a.table + (int64_t)l * a.W;
        // a wave compares four requests' rows with the lead's, 256 entries a step
        constexpr int ROWS = 4, AHEAD = 4, WAVES = SP_THREADS / 64;
        for (int r0 = l + 1 + wave; r0 < end; r0 += ROWS * WAVES) {
            const int *row[ROWS];
#pragma unroll
            for (int j = 0; j < ROWS; ++j) {
                const int r = r0 + j * WAVES;
                row[j] = r < end && part[r] ? a.table + (int64_t)r * a.W : with;
            }
            for (int w0 = 0; w0 < *(volatile int *)&limit; w0 += 64 * AHEAD) {
                int x[AHEAD], y[ROWS][AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int w = min(w0 + 64 * i + lane, a.W - 1);
                    x[i] = with[w];
#pragma unroll
                    for (int j = 0; j < ROWS; ++j) y[j][i] = row[j][w];
                }
                int first_other = a.W;  // (entries past the limit may differ: it stands)
#pragma unroll
                for (int i = AHEAD - 1; i >= 0; --i) {
                    bool other = false;
#pragma unroll
                    for (int j = 0; j < ROWS; ++j) other |= x[i] != y[j][i];
                    const uint64_t b = __builtin_amdgcn_ballot_w64(other);
                    if (b) first_other = w0 + 64 * i + (int)__builtin_ctzll(b);
                }
                if (first_other < a.W) {
                    if (lane == 0) atomicMin(&limit, first_other);
                    break;
                }
            }
        }
    }
    __syncthreads();
    if (threadIdx.x) return;
    const int keys = l < end ? limit << a.page_log2 : 0;
    a.keys[g] = keys;
    SharedGroup o = {l < end ? l : 0, 0, 0, 0};
    if (first < end) {
        const Span s = span_of(a, first), e = span_of(a, end - 1);
        o.t0 = s.q0;
        o.cols = max(e.q0 + e.n - s.q0, 0) * a.G;
    }
    if (others > 1 && keys >= SP_MIN_KEYS && most * a.G <= SP_MAX_COLS) o.keys = keys;
    a.groups[g] = o;
}

// Blocks of `cols` columns and the runs of CHUNK_KEYS keys that each reads: a group's
// prefix (s < NG) or the rest of a request's keys.
struct Segment {
    int r, t0, cols, from, to;  // keys [from, to)
    int blocks, runs;
    bool alone;  // nothing else is joined with it
    bool rest;   // whether wide blocks take the probabilities' rests
};
// Runs a part that are wanted, of narrow and of wide blocks (parts_wanted).
struct Each {
    int narrow, wide;
};
__device__ __forceinline__ Segment segment_of(const PlanArgs &a, int s) {
    Segment g;
    if (s < a.NG) {
        const SharedGroup o = a.groups[s];
        g = {o.lead, o.t0, o.keys ? o.cols : 0, 0, o.keys, 0, 0, false, true};
    } else {
        const int r = s - a.NG, of = a.group_of[r];
        const Span p = span_of(a, r);
        const int shared = (unsigned)of < (unsigned)a.NG ? a.groups[of].keys : 0;
        g = {r, p.q0, p.n * a.G, min(shared, p.len), p.len, 0, 0, shared == 0,
             p.n * a.G <= REST_COLS};
        // (of a group's request without keys behind the prefix nothing is to be done)
        if (shared && g.from >= g.to) g.cols = 0;
    }
    g.blocks = g.cols <= 32 ? (g.cols + 31) >> 5 : (g.cols + WIDE_COLS - 1) / WIDE_COLS;
    g.runs = (g.to - g.from + CHUNK_KEYS - 1) / CHUNK_KEYS;
    return g;
}
// Parts of each of its blocks, and runs a part: parts of one length, and none for a quarter
// of one (16 prompts of 128 tokens behind 2048 keys, a round of whole blocks, 146 -> 90 us).
__device__ __forceinline__ int parts_of(const Segment &g, const Each &each, int &per) {
    const int want = g.cols > 32 ? each.wide : each.narrow;
    const int ns = min(max(1, (g.runs - want / 4 + want - 1) / want), MAX_CHUNKS);
    per = max(1, (g.runs + ns - 1) / ns);
    return ns;
}
// One round of workgroups for all blocks' runs; where it would be a long one, narrow blocks,
// whose parts' states are small, are cut for one and a half: what waits for HBM at a part's
// start and end is then hidden by others. (us, one round / one and a half: 32 pairs behind
// 1984 60.8 / 59.1; but 8 requests behind 8192, a short round, 16.4 / 21.7, and with the wide
// blocks too 96 requests behind 16256 136 / 146.)
__device__ __forceinline__ Each parts_wanted(unsigned long long runs, int slots) {
    const unsigned long long one = (runs + slots - 1) / slots;
    const unsigned long long more = (2 * runs + 3 * slots - 1) / (3 * slots);
    Each e;
    e.wide = one < 1 ? 1 : one < (1u << 30) ? (int)one : 1 << 30;
    e.narrow = one < 8 ? e.wide : more < (1u << 30) ? (int)more : 1 << 30;
    return e;
}
__device__ __forceinline__ int width_of(const Segment &g) { return min(g.cols, WIDE_COLS); }

// The list. Every workgroup sums over all segments by itself, then makes its share of the
// items and tokens, each finding its segment by bisection.
__global__ __launch_bounds__(SP_THREADS) void shared_plan_kernel(PlanArgs a) {
    __shared__ int item_end[2 * SP_MAX_R], state_end[2 * SP_MAX_R], cu[SP_MAX_R + 1];
    __shared__ int waves[2][SP_THREADS / 64];
    __shared__ unsigned long long total;
    __shared__ int wrong;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int segments = a.NG + a.R, own = (segments + SP_THREADS - 1) / SP_THREADS;
    const int s0 = min((int)threadIdx.x * own, segments), s1 = min(s0 + own, segments);
    if (threadIdx.x == 0) total = 0, wrong = 0;
    __syncthreads();
    // offsets that fall: nothing is taken (their rows could be those of others)
    bool falls = false;
    for (int r = threadIdx.x; r <= a.R; r += SP_THREADS) {
        cu[r] = a.cu_q[r];
        falls |= r < a.R && a.cu_q[r + 1] < cu[r];
    }
    for (int g = threadIdx.x; g < a.NG; g += SP_THREADS)
        falls |= a.cu_groups[g + 1] < a.cu_groups[g];
    if (falls) wrong = 1;
    // (the thread's first segment, as a rule its only one, is kept)
    Segment kept = {};
    if (s0 < s1) kept = segment_of(a, s0);
    auto segment = [&](int s) { return s == s0 ? kept : segment_of(a, s); };
    unsigned long long runs = 0;
    for (int s = s0; s < s1; ++s) {
        const Segment g = segment(s);
        runs += (unsigned long long)g.blocks * g.runs;
    }
    if (runs) atomicAdd(&total, runs);
    __syncthreads();
    const Each each = parts_wanted(total, a.slots);
    int items = 0, states = 0;
    for (int s = s0; s < s1; ++s) {
        const Segment g = segment(s);
        int per;
        const int ns = parts_of(g, each, per);
        items += g.blocks * ns;
        if (!g.alone || ns > 1) states += g.blocks * ns * width_of(g);
    }
    const int iu = wave_scan(items), su = wave_scan(states);
    if (lane == 63) waves[0][wave] = iu, waves[1][wave] = su;
    __syncthreads();
    int ia = iu - items, sa = su - states;
    for (int w = 0; w < wave; ++w) ia += waves[0][w], sa += waves[1][w];
    for (int s = s0; s < s1; ++s) {
        const Segment g = segment(s);
        int per;
        const int ns = parts_of(g, each, per);
        ia += g.blocks * ns;
        if (!g.alone || ns > 1) sa += g.blocks * ns * width_of(g);
        item_end[s] = ia;
        state_end[s] = sa;
    }
    __syncthreads();
    const int all = item_end[segments - 1];
    const bool ok = !wrong && all <= a.max_items && state_end[segments - 1] <= a.states;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.head[0] = ok ? all : 0;
        a.head[1] = a.key;
    }
    // every other workgroup makes items, every other one tokens
    const int step = gridDim.x / 2 * SP_THREADS;
    const int at = blockIdx.x / 2 * SP_THREADS + threadIdx.x;
    for (int u = at; ok && blockIdx.x % 2 == 0 && u < all; u += step) {
        int lo = -1, hi = segments - 1;  // item_end[lo] <= u < item_end[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (item_end[mid] <= u)
                lo = mid;
            else
                hi = mid;
        }
        const Segment g = segment_of(a, hi);
        int per;
        const int ns = parts_of(g, each, per), width = width_of(g);
        const int i = u - (hi ? item_end[hi - 1] : 0), part = i % ns;
        // (wide blocks from the last, which sees the most keys)
        const int block = g.blocks - 1 - i / ns;
        SharedItem it;
        it.r = g.r;
        it.t0 = g.t0;
        it.cols = g.cols;
        it.c0 = block * width;
        it.kind = g.cols <= 32 ? NARROW : g.rest ? WIDE_REST : WIDE;
        // keys that the block's last token sees
        int to = g.to;
        if (hi >= a.NG) {
            const Span p = span_of(a, g.r);
            const int last = (min(it.c0 + width, g.cols) - 1) / a.G;
            to = min(max(p.len - p.n + last + 1, g.from), g.to);
        }
        it.k0 = min(g.from + part * per * CHUNK_KEYS, to);
        it.k1 = min(g.from + (part + 1) * per * CHUNK_KEYS, to);
        it.state = g.alone && ns == 1
                       ? -1 : (hi ? state_end[hi - 1] : 0) + (block * ns + part) * width;
        a.items[u] = it;
    }
    for (int t = at; blockIdx.x % 2 && t < a.T; t += step) {
        SharedToken o = {0, -1, 0, 0, -1, 0, 0, 0};
        int lo = 0, hi = a.R;  // cu[lo] <= t < cu[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (cu[mid] <= t)
                lo = mid;
            else
                hi = mid;
        }
        const Span p = span_of(a, lo);
        if (ok && t >= p.q0 && t < p.q0 + p.n) {
            o.seen = min(max(p.len - p.n + t - p.q0 + 1, 0), p.len);
            int per;
            const Segment g = segment_of(a, a.NG + lo);
            const int ns = parts_of(g, each, per), s = a.NG + lo;
            if (g.cols && (!g.alone || ns > 1)) {
                o.own = s ? state_end[s - 1] : 0;
                o.own_parts = ns | width_of(g) << 16;
                o.own_col = (t - g.t0) * a.G;
            }
            if (!g.alone) {
                const int of = a.group_of[lo];
                const Segment f = segment_of(a, of);
                o.prefix = of ? state_end[of - 1] : 0;
                o.prefix_parts = parts_of(f, each, per) | width_of(f) << 16;
                o.prefix_col = (t - f.t0) * a.G;
            }
        }
        a.tokens[t] = o;
    }
}

// ---------------------------------------------------------------------------
// the attention

struct SharedArgs {
    const void *q, *k, *v;
    void *out;
    const int *table, *head;
    const SharedItem *items;
    const SharedToken *tokens;
    float *o;    // states by kv head and column: D sums each,
    float2 *lm;  // (l, m)
    int64_t states;
    int T, W, H, HK, G, pages, page_log2, key;
    float scale;    // > 0, log2 units
    uint32_t flip;  // sign bits of a negative scale, for Q
};

#if defined(__HIP_DEVICE_COMPILE__)
// Column c's row of q and out, and the keys below k1 that it sees; c < cols.
template <int D>
__device__ __forceinline__ int64_t row_of(const SharedArgs &a, const SharedItem &it, int hk, int c,
                                          int &seen) {
    const int tok = min(it.t0 + c / a.G, a.T - 1), g = c - c / a.G * a.G;
    seen = min(a.tokens[tok].seen, it.k1);
    return (int64_t)tok * a.H + hk * a.G + g;
}
__device__ __forceinline__ int wave_min(int v) {
    for (int o = 1; o < 64; o <<= 1) v = min(v, __shfl_xor(v, o, 64));
    return __builtin_amdgcn_readfirstlane(v);
}

// A block of 32 columns: wave w takes the key tiles w, w + 4, ... into LDS of its own (a
// K and a V slot, refilled as soon as their reads are in registers: no barrier), and the
// four states are folded at the end.
template <typename T, int D>
__device__ __forceinline__ void shared_narrow(const SharedArgs &a, const SharedItem &it, int hk,
                                              char *lds) {
    typedef Tile<D> Tl;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h2 = lane >> 5, r = lane & 31;
    const bool ok = it.c0 + r < it.cols;
    int end;
    const int64_t qrow = row_of<D>(a, it, hk, ok ? it.c0 + r : it.c0, end);
    const int full = wave_min(end);
    const int ntiles = (it.k1 - it.k0 + ATT_KT - 1) / ATT_KT, t0 = wave;
    char *kslot = lds + wave * 2 * Tl::BYTES, *vslot = kslot + Tl::BYTES;
    const T *k = (const T *)a.k, *v = (const T *)a.v;
    AttnState<D> st;
    attn_init(st);
    uint4 qf[D / 16];
    uint32_t flip = a.flip;
    auto run = [&](char *__restrict__ ks, char *__restrict__ vs, auto with_rest)
                   __attribute__((always_inline)) {
        read_q<D>((const T *)a.q + qrow * D, h2, qf);
        TilePages<PA_WAVES> pg(a, it.r, hk);
        if (t0 < ntiles) {
            pg.load(t0, lane, it.k0);
            int64_t lo, hi;
            const int key = it.k0 + t0 * ATT_KT;
            pg.rows(0, key, lo, hi);
            dma_paged_tile<T, D, false, true, true>(k + lo * D, k + hi * D, it.k1 - key, ks, lane);
            dma_paged_tile<T, D, true, true, true>(v + lo * D, v + hi * D, it.k1 - key, vs, lane);
        }
        for (int kt = t0; kt < ntiles; kt += PA_WAVES) {  // wave-uniform
            const int nx = kt + PA_WAVES, key = it.k0 + nx * ATT_KT;
            const bool more = nx < ntiles;
            int64_t lo = 0, hi = 0;
            if (more) {
                const int at = (nx - t0) / PA_WAVES;
                if ((at & 63) == 0) pg.load(nx, lane, it.k0);
                pg.rows(at, key, lo, hi);
            }
            // K (and, the first time, q) has landed once only V's loads, issued
            // after it, are in flight
            att_wait_vmcnt<Tl::NI>();
            flip_q<D>(qf, flip);
            uint4 kf[D / 16];
            read_k<D>(ks, kf, r, h2);
#pragma unroll
            for (int s = 0; s < D / 16; ++s) launder(kf[s]);  // the reads have returned
            __builtin_amdgcn_sched_barrier(0);
            if (more) dma_paged_tile<T, D, false, true, true>(k + lo * D, k + hi * D, it.k1 - key, ks, lane);
            f32x16 s = attn_scores<T, D>(kf, qf);
            const int k0 = it.k0 + kt * ATT_KT;
            if (k0 + ATT_KT > full) attn_mask(s, end - k0, h2);
            uint32_t p[8], rest[8];
            attn_softmax<T, D, with_rest.value>(st, s, p, a.scale, rest);
            if (more)
                att_wait_vmcnt<Tl::NI>();
            else
                att_wait_vmcnt<0>();
            VFrag<T, D> vf;
            read_v<T, D>(vs, vf, lane);
            attn_pv<T, D>(st, p, vf);
            if constexpr (with_rest.value) attn_pv<T, D>(st, rest, vf);
            __builtin_amdgcn_sched_barrier(0);
            att_wait_lds();  // V's reads have returned
            if (more) dma_paged_tile<T, D, true, true, true>(v + lo * D, v + hi * D, it.k1 - key, vs, lane);
        }
    };
    run(kslot, vslot, std::true_type{});
    // an infinite value times a rest of 0, or below it, leaves NaN: once more, without
    // the rests
    if (not_a_number(st)) {
        flip = a.flip;
        attn_init(st);
        run(kslot, vslot, std::false_type{});
    }

    // fold (0 + 1) + (2 + 3): wave t folds O^T tile t
    __syncthreads();
    float4 *part = (float4 *)lds;
    float4 *mine = part + (size_t)wave * Part<D>::WORDS;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) part_put<D>(mine, st, t, lane);
    part_lm<D>(mine)[lane] = make_float2(st.l, st.m);
    __syncthreads();
    if (wave >= D / 32) return;
    const Fold f = fold_streams<D>(part, wave, lane);
    if (it.state < 0) {
        const float inv = row_inv(f.l);
        if (ok) store_fold<T>(f, inv, (T *)a.out + qrow * D, wave, h2);
        return;
    }
    const int64_t at = hk * a.states + it.state + r;
    const float l = f.l + __shfl_xor(f.l, 32, 64);
    if (!ok) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *(float4 *)(a.o + at * D + 32 * wave + 8 * j + 4 * h2) = f.o[j];
    if (wave == 0 && h2 == 0) a.lm[at] = make_float2(l, f.m);
}

// A block of 128 columns: wave w has the columns 32 w .. 32 w + 31, and all four share
// each stage of two key tiles, staged by DMA into one of two buffers while the other is
// read. REST: with the product of what rounding the probabilities left.
template <typename T, int D, bool REST>
__device__ __forceinline__ void shared_wide(const SharedArgs &a, const SharedItem &it, int hk,
                                            char *lds) {
    typedef Tile<D> Tl;
    constexpr int STAGE = 4 * Tl::BYTES;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h2 = lane >> 5, r = lane & 31;
    const int c = it.c0 + 32 * wave + r;
    const bool ok = c < it.cols;
    int end;
    const int64_t qrow = row_of<D>(a, it, hk, ok ? c : it.c0, end);
    if (!ok) end = 0;
    const int full = wave_min(ok ? end : 0x7fffffff), most = -wave_min(-end);
    const int ntiles = (it.k1 - it.k0 + ATT_KT - 1) / ATT_KT;
    const int mine = most > it.k0 ? (most - it.k0 + ATT_KT - 1) / ATT_KT : 0;

    AttnState<D> st;
    uint4 qf[D / 16];
    uint32_t flip = a.flip;
    // stage s: key tiles 2 s, 2 s + 1; waves 0 and 1 stage K, 2 and 3 V
    TilePages<2> pg(a, it.r, hk);
    const T *pool = (const T *)(wave < 2 ? a.k : a.v);
    auto issue = [&](int s, char *dst) __attribute__((always_inline)) {
        const int kt = 2 * s + (wave & 1), key = it.k0 + kt * ATT_KT;
        if ((s & 63) == 0) pg.load(kt, lane, it.k0);
        int64_t lo, hi;
        pg.rows(s, key, lo, hi);
        if (wave < 2)
            dma_paged_tile<T, D, false, false, true>(pool + lo * D, pool + hi * D, it.k1 - key,
                                               dst + wave * Tl::BYTES, lane);
        else
            dma_paged_tile<T, D, true, false, true>(pool + lo * D, pool + hi * D, it.k1 - key,
                                              dst + wave * Tl::BYTES, lane);
    };
    auto step = [&](const char *__restrict__ cb, char *__restrict__ nb, int s, bool more,
                    auto with_rest) __attribute__((always_inline)) {
        // every wave's DMAs of stage s have landed, and every wave is done with
        // the buffer the next ones go to
        att_wait_vmcnt<0>();
        __syncthreads();
        flip_q<D>(qf, flip);
        if (more) issue(s + 1, nb);
        const int kt = 2 * s;
        if (kt >= mine) return;  // (wave-uniform)
        f32x16 sc[2];
        {
            uint4 kf[D / 16];
            read_k<D>(cb, kf, r, h2);
            sc[0] = attn_scores<T, D>(kf, qf);
            read_k<D>(cb + Tl::BYTES, kf, r, h2);
            sc[1] = attn_scores<T, D>(kf, qf);
        }
        VFrag<T, D> vf;
        read_v<T, D>(cb + 2 * Tl::BYTES, vf, lane);
        const int k0 = it.k0 + kt * ATT_KT;
        if (k0 + 2 * ATT_KT > full) {
            attn_mask(sc[0], end - k0, h2);
            attn_mask(sc[1], end - k0 - ATT_KT, h2);
        }
        uint32_t p[2][8], rest[2][8];
        softmax_pair<T, D, with_rest.value>(st, sc, p, a.scale, rest);
        attn_pv<T, D>(st, p[0], vf);
        if constexpr (with_rest.value) attn_pv<T, D>(st, rest[0], vf);
        read_v<T, D>(cb + 3 * Tl::BYTES, vf, lane);
        attn_pv<T, D>(st, p[1], vf);
        if constexpr (with_rest.value) attn_pv<T, D>(st, rest[1], vf);
    };
    const int stages = (ntiles + 1) / 2;
    char *b0 = lds, *b1 = lds + STAGE;
    auto run = [&](auto with_rest) __attribute__((always_inline)) {
        attn_init(st);
        read_q<D>((const T *)a.q + qrow * D, h2, qf);
        if (stages) issue(0, b0);
        for (int s = 0; s < stages; s += 2) {  // workgroup-uniform
            step(b0, b1, s, s + 1 < stages, with_rest);
            if (s + 1 < stages) step(b1, b0, s + 1, s + 2 < stages, with_rest);
        }
    };
    run(std::integral_constant<bool, REST>{});
    // (as in the narrow block; here all four waves, which share the stages)
    if (REST && __syncthreads_or(not_a_number(st))) {
        flip = a.flip;
        run(std::false_type{});
    }
    if (it.state < 0) {
        const float inv = row_inv(st.l);
        T *orow = (T *)a.out + qrow * D;
        if (ok)
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float e[4] = {st.o[t][4 * j] * inv, st.o[t][4 * j + 1] * inv,
                                        st.o[t][4 * j + 2] * inv, st.o[t][4 * j + 3] * inv};
                    st8(orow + 32 * t + 8 * j + 4 * h2, pack4<T>(e));
                }
        return;
    }
    const int64_t at = hk * a.states + it.state + 32 * wave + r;
    const float l = st.l + __shfl_xor(st.l, 32, 64);
    if (!ok) return;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *(float4 *)(a.o + at * D + 32 * t + 8 * j + 4 * h2) =
                make_float4(st.o[t][4 * j], st.o[t][4 * j + 1], st.o[t][4 * j + 2],
                            st.o[t][4 * j + 3]);
    if (h2 == 0) a.lm[at] = make_float2(l, st.m);
}
#endif

// One workgroup an item and kv head.
template <int D> constexpr int shared_per_cu() { return D == 128 ? 2 : 3; }
template <typename T, int D>
__global__ __launch_bounds__(64 * PA_WAVES)
__attribute__((amdgpu_waves_per_eu(shared_per_cu<D>())))
void shared_attn_kernel(SharedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __attribute__((aligned(1024))) char lds[PagedLds<D>::BYTES];
    const int *p = (const int *)(a.items + blockIdx.y);
    int f[sizeof(SharedItem) / 4];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(SharedItem) / 4); ++i) f[i] = p[i];
    const int items = a.head[0], key = a.head[1];  // (asked for together)
    if (key != a.key || (int)blockIdx.y >= items) return;  // (workgroup-uniform)
#pragma unroll
    for (int i = 0; i < (int)(sizeof(SharedItem) / 4); ++i)
        f[i] = __builtin_amdgcn_readfirstlane(f[i]);
    const SharedItem it = __builtin_bit_cast(SharedItem, f);
    if (it.kind == WIDE_REST)
        shared_wide<T, D, true>(a, it, blockIdx.x, lds);
    else if (it.kind == WIDE)
        shared_wide<T, D, false>(a, it, blockIdx.x, lds);
    else
        shared_narrow<T, D>(a, it, blockIdx.x, lds);
#endif
}

// A row's parts joined: D / 4 lanes a row, of four values each. GROUPS such lanes take
// every so manyth part, in order, and are added in order.
template <typename T, int D, int GROUPS>
__global__ __launch_bounds__(256) void shared_join_kernel(SharedArgs a) {
#pragma clang fp contract(off)
    constexpr int LANES = D / 4, ROWS = 256 / (LANES * GROUPS);
    __shared__ float4 sums[GROUPS > 1 ? GROUPS * ROWS * LANES : 1];
    __shared__ float2 lms[GROUPS > 1 ? GROUPS * ROWS : 1];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int at_row = sub % ROWS, group = sub / ROWS;
    const int64_t row = (int64_t)blockIdx.x * ROWS + at_row;
    const int64_t at_most = min(row, (int64_t)a.T * a.H - 1);
    const int t = (int)(at_most / a.H), h = (int)(at_most - (int64_t)t * a.H);
    const int hk = h / a.G, g = h - hk * a.G;
    SharedToken k = a.tokens[t];
    const int key = a.head[1];  // (asked for together)
    if (row != at_most || key != a.key) k.prefix = k.own = -1;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f, m = -INFINITY;
    auto add = [&](const float4 &v, const float2 &w) {
        // (a part that saw no key of the row, whatever its sums; of one whose scores are all
        // NaN l is NaN, and so are they)
        if (w.y == -INFINITY && w.x == 0.0f) return;
        const MergeCoef c = merge_coef(m, w.y);
        o.x = merge_one(o.x, v.x, c);
        o.y = merge_one(o.y, v.y, c);
        o.z = merge_one(o.z, v.z, c);
        o.w = merge_one(o.w, v.w, c);
        l = merge_one(l, w.x, c);
        m = c.m_new;
    };
    // the prefix's parts, then the row's own, as one list
    auto place = [&](int first, int parts, int col, int &n, int &width) -> int64_t {
        n = first < 0 ? 0 : parts & 0xffff;
        width = first < 0 ? 1 : parts >> 16;
        const int b = col / width;
        return hk * a.states + first + (int64_t)b * n * width + (col - b * width);
    };
    int np, wp, no, wo;
    const int64_t pa = place(k.prefix, k.prefix_parts, k.prefix_col + g, np, wp);
    const int64_t oa = place(k.own, k.own_parts, k.own_col + g, no, wo) - (int64_t)np * wo;
    const int n = np + no;
    constexpr int IN_FLIGHT = 8;
    for (int s0 = group; s0 < n; s0 += GROUPS * IN_FLIGHT) {
        float4 v[IN_FLIGHT];
        float2 w[IN_FLIGHT];
#pragma unroll
        for (int i = 0; i < IN_FLIGHT; ++i) {
            const int s = min(s0 + GROUPS * i, n - 1);
            const int64_t c = s < np ? pa + (int64_t)s * wp : oa + (int64_t)s * wo;
            v[i] = *(const float4 *)(a.o + c * D + 4 * lane);
            w[i] = a.lm[c];
        }
#pragma unroll
        for (int i = 0; i < IN_FLIGHT; ++i)
            if (s0 + GROUPS * i < n) add(v[i], w[i]);
    }
    if constexpr (GROUPS > 1) {
        sums[threadIdx.x] = o;
        if (lane == 0) lms[sub] = make_float2(l, m);
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int i = 1; i < GROUPS; ++i)
            add(sums[threadIdx.x + i * ROWS * LANES], lms[sub + i * ROWS]);
    }
    if (k.prefix < 0 && k.own < 0) return;  // (nothing to join)
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const float e[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    st8((T *)a.out + row * D + 4 * lane, pack4<T>(e));
}

// ---------------------------------------------------------------------------
// dispatch

// What bounds a plan, from the sizes alone. Blocks: a column is in one of its group's and
// in one of its request's, of 128 (or the last, shorter one of each). Parts: one and a
// half rounds of workgroups, beside one a block. States, of a block's columns one a part:
// where a prefix is shared (requests of at most SP_MAX_COLS columns) one of the prefix, whose
// blocks are filled up to 128, so at most two, and one of the request's own keys; of other
// blocks that are cut, filled up as well, at most two a column; and all parts beyond those.
struct SharedGrid {
    int64_t items, states, slots, ints;
    int64_t at_groups, at_group_of, at_items, at_tokens;  // in the schedule, ints
    int key;
};
inline SharedGrid shared_grid(int64_t T, int64_t R, int64_t NG, int64_t W, int64_t H, int64_t HK,
                              int64_t D, int64_t page) {
    SharedGrid g;
    const int64_t G = H / HK, cols = T * G;
    const int64_t some = (R < T ? R : T) + (NG < T ? NG : T);
    // workgroups that the chip holds, for each kv head
    g.slots = 256 * (D == 128 ? shared_per_cu<128>() : shared_per_cu<64>()) / HK;
    if (g.slots < 1) g.slots = 1;
    const int64_t target = 3 * g.slots / 2 + 1;
    const int64_t blocks = 2 * (cols / WIDE_COLS) + some;
    const int64_t runs = ceil_div(W * page, CHUNK_KEYS);
    const int64_t extra = target < blocks * runs ? target : blocks * runs;
    g.items = blocks + extra;
    const int64_t joined = cols < R * SP_MAX_COLS ? cols : R * SP_MAX_COLS;
    const int64_t more = extra * (cols < WIDE_COLS ? cols : WIDE_COLS);
    g.states = 3 * joined + more + (2 * cols < more ? 2 * cols : more);
    g.at_groups = 16;
    g.at_group_of = g.at_groups + NG * (int64_t)(sizeof(SharedGroup) / 4);
    g.at_items = ceil_div(g.at_group_of + R, 8) * 8;
    g.at_tokens = g.at_items + g.items * (int64_t)(sizeof(SharedItem) / 4);
    g.ints = g.at_tokens + T * (int64_t)(sizeof(SharedToken) / 4);
    uint32_t key = 0x9e3779b9u;
    for (const int64_t v : {T, R, NG, W, H, HK, D, page}) key = (key ^ (uint32_t)v) * 0x01000193u;
    g.key = (int)key;
    return g;
}

int check_shared(const char *what, int64_t T, int64_t R, int64_t NG, int64_t W, int64_t H,
                 int64_t HK, int64_t D, int64_t page, int &lp) {
    if (D != 64 && D != 128) return fail(MI_ERR_UNSUPPORTED, "%s head dim %lld", what, (long long)D);
    if (!page_log2_of(page, lp))
        return fail(MI_ERR_UNSUPPORTED, "page size %lld; this build covers 16, 32, 64, 128, 256",
                    (long long)page);
    if (T < 0 || T > (1 << 18) || R < 1 || R > SP_MAX_R || NG < 1 || NG > R || W < 1 ||
        W > (0x3fffffff >> lp) || H < 1 || HK < 1 || H % HK || HK > 65535 ||
        T * (H / HK) > 0x3fffff || H > 0x3fffffff / (T + 1))
        return fail(MI_ERR_ARG, "%s T=%lld (to 2^18) R=%lld (1 to %d) groups=%lld (1 to R) table "
                    "width %lld H=%lld HK=%lld", what, (long long)T, (long long)R, SP_MAX_R,
                    (long long)NG, (long long)W, (long long)H, (long long)HK);
    const SharedGrid g = shared_grid(T, R, NG, W, H, HK, D, page);
    if (g.items > 65535)
        return fail(MI_ERR_ARG, "%s: %lld blocks of query rows, at most 65535", what,
                    (long long)g.items);
    return MI_OK;
}

template <typename T, int D>
int launch_shared(const SharedArgs &a, const SharedGrid &g, hipStream_t st) {
    shared_attn_kernel<T, D><<<dim3((unsigned)a.HK, (unsigned)g.items), 64 * PA_WAVES, 0, st>>>(a);
    // few rows: eight groups of lanes a row, whose parts are then read together (8 requests
    // behind 8192 keys 28 -> 22 us in all; 128 of them 52 with, 46 without)
    const int64_t rows = (int64_t)a.T * a.H, lanes = rows * (D / 4);
    if (rows <= 1024)
        shared_join_kernel<T, D, 8><<<(unsigned)ceil_div(8 * lanes, 256), 256, 0, st>>>(a);
    else
        shared_join_kernel<T, D, 1><<<(unsigned)ceil_div(lanes, 256), 256, 0, st>>>(a);
    return launch_status("shared attention");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_paged_shared_plan_ints(int64_t T, int64_t R, int64_t n_groups,
                                             int64_t table_width, int64_t H, int64_t HK, int64_t D,
                                             int64_t page_size) {
    int lp;
    if (check_shared("shared plan", T, R, n_groups, table_width, H, HK, D, page_size, lp)) return 0;
    return shared_grid(T, R, n_groups, table_width, H, HK, D, page_size).ints;
}

extern "C" int mi_paged_shared_plan(const int32_t *block_table, int64_t table_width,
                                    const int32_t *cu_q, const int32_t *kv_lens, int64_t R,
                                    const int32_t *cu_groups, int64_t n_groups, int64_t T, int64_t H,
                                    int64_t HK, int64_t D, int64_t page_size, int32_t *keys,
                                    int32_t *schedule, int64_t schedule_ints, void *stream) {
    int lp;
    if (const int e = check_shared("shared plan", T, R, n_groups, table_width, H, HK, D, page_size,
                                   lp))
        return e;
    if (!block_table || !cu_q || !kv_lens || !cu_groups || !keys || !schedule)
        return fail(MI_ERR_ARG, "null pointer");
    const SharedGrid g = shared_grid(T, R, n_groups, table_width, H, HK, D, page_size);
    if (schedule_ints < g.ints || !aligned(schedule, 16))
        return fail(MI_ERR_ARG, "shared plan needs a 16-byte aligned schedule of %lld ints",
                    (long long)g.ints);
    const PlanArgs a = {block_table, cu_q, kv_lens, cu_groups, keys, schedule,
                        (SharedGroup *)(schedule + g.at_groups), schedule + g.at_group_of,
                        (SharedItem *)(schedule + g.at_items),
                        (SharedToken *)(schedule + g.at_tokens), (int)R, (int)table_width, (int)T,
                        (int)(H / HK), (int)n_groups, lp, (int)g.items, (int)g.slots,
                        g.key, g.states};
    hipStream_t st = as_stream(stream);
    shared_keys_kernel<<<(unsigned)n_groups, SP_THREADS, 0, st>>>(a);
    int64_t grid = ceil_div(T > g.items ? T : g.items, SP_THREADS);
    grid = grid < 1 ? 1 : grid > 32 ? 32 : grid;
    shared_plan_kernel<<<(unsigned)(2 * grid), SP_THREADS, 0, st>>>(a);
    return launch_status("shared plan");
}

extern "C" int64_t mi_paged_shared_attention_workspace_bytes(int64_t T, int64_t R, int64_t n_groups,
                                                             int64_t table_width, int64_t H,
                                                             int64_t HK, int64_t D,
                                                             int64_t page_size) {
    int lp;
    if (check_shared("shared attention", T, R, n_groups, table_width, H, HK, D, page_size, lp))
        return 0;
    return shared_grid(T, R, n_groups, table_width, H, HK, D, page_size).states * HK * (D + 2) * 4;
}

extern "C" int mi_paged_shared_attention(const void *q, const void *k_pages, const void *v_pages,
                                         void *out, const int32_t *block_table,
                                         const int32_t *schedule, int64_t T, int64_t R,
                                         int64_t n_groups, int64_t table_width, int64_t H, int64_t HK,
                                         int64_t D, int64_t n_pages, int64_t page_size, float scale,
                                         int dtype, void *workspace, int64_t workspace_bytes,
                                         void *stream) {
    if (dtype != MI_BF16 && dtype != MI_F16)
        return fail(MI_ERR_UNSUPPORTED, "shared attention covers bf16 and fp16 (dtype code %d)",
                    dtype);
    int lp;
    if (const int e = check_shared("shared attention", T, R, n_groups, table_width, H, HK, D,
                                   page_size, lp))
        return e;
    if (n_pages < 1 || n_pages > (0x7fffffff >> lp))
        return fail(MI_ERR_ARG, "shared attention pages=%lld", (long long)n_pages);
    if (T == 0) return MI_OK;
    if (!q || !k_pages || !v_pages || !out || !block_table || !schedule)
        return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 8) ||
        !aligned(schedule, 16))
        return fail(MI_ERR_ARG, "q, the pages and the schedule must be 16-byte aligned, out 8-byte "
                    "aligned");
    const SharedGrid g = shared_grid(T, R, n_groups, table_width, H, HK, D, page_size);
    const int64_t need = g.states * HK * (D + 2) * 4;
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return fail(MI_ERR_ARG, "shared attention needs a 16-byte aligned workspace of %lld bytes",
                    (long long)need);
    const float sl = scale * 1.4426950408889634f;
    // (a scale of 0 as the smallest normal: masked scores stay -inf; NaN stays NaN)
    const float mag = fabsf(sl) < 1.17549435e-38f ? 1.17549435e-38f : fabsf(sl);
    float *o = (float *)workspace;
    const SharedArgs a = {q, k_pages, v_pages, out, block_table, schedule,
                          (const SharedItem *)(schedule + g.at_items),
                          (const SharedToken *)(schedule + g.at_tokens), o,
                          (float2 *)(o + g.states * HK * D), g.states, (int)T, (int)table_width,
                          (int)H, (int)HK, (int)(H / HK), (int)n_pages, lp, g.key, mag,
                          sl < 0.0f ? 0x80008000u : 0u};
    hipStream_t st = as_stream(stream);
    if (dtype == MI_BF16)
        return D == 128 ? launch_shared<bf16, 128>(a, g, st) : launch_shared<bf16, 64>(a, g, st);
    return D == 128 ? launch_shared<f16, 128>(a, g, st) : launch_shared<f16, 64>(a, g, st);
}
