// Causal GQA attention of requests of different lengths over a paged key/value
// cache (no counterpart in the reference, whose caches are contiguous):
// mi_paged_attention.
//
// For request r with n new tokens and len keys, token i, q head h over kv head
// h / G:  o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),
// s_j = scale log2(e) q . k_j,  j <= len - n + i;  0 where no key is seen.
// Key j sits in row j % page_size of page block_table[r][j / page_size].
//
// What bounds it, on MI355X: decode (narrow blocks) HBM, 5.8 TB/s of K and V for 48
// requests of 64 to 8191 keys (136 us; the rest is the chunks' starts and ends), 6.3
// for 64 of 4096 (170 us); one request of 1001 keys 9.5 us (8.4 at least), a chain of
// trips to memory. Prompts (wide blocks) the matrix cores beside the softmax VALU, at
// the clock that the card's power leaves: 1.0 PFLOP/s over 8192 keys (526 to 552 us from
// card to card), where a plain matrix product of 8192 reaches 1.2; MFMAs are busy 52% of
// the cycles, and the clock falls to 1.5-1.9 GHz. Dealing the next tile's score MFMAs
// between this one's exponentials, or eight waves a stage, changed nothing there.
//
// Probabilities enter the second product as T. Narrow blocks, whose MFMAs wait for HBM,
// take the product of what that rounding left too: what is off is then the result's own
// rounding (one row over 4096 keys: 2.0e-3 -> 1.67e-3 of the norm in bf16, 2.6e-4 ->
// 2.1e-4 in fp16; 48 requests 136.8 -> 137.5 us). Wide blocks do not (2.2e-3 and
// 2.8e-4): they are bound by these products (8192 tokens 526 -> 694 us with it, four
// prompts of 2048 161 -> 203).
//
// The tile, the softmax and the folds are the contiguous attention's
// (mi_attn_common.h). A kv head's query rows, token after token and in a token
// its G q heads, are the columns of 32-wide blocks, so K and V are read once per
// block and kv head and a block sees nearly one causal range.
//
// Requests differ in length, and only the GPU knows the lengths. The keys of
// every block are therefore cut into chunks of one size, chosen on the GPU from
// the lengths of all requests so that the chunks fill the chip, and a workgroup
// finds its chunk by summing over the requests (find_item). A block of one chunk
// writes its rows; the others' states go to a workspace, and the last workgroup of
// a block to finish folds them, in order. The chunk size, so a row's last bits,
// depends on the lengths of the whole batch.
#include <type_traits>

#include "mi_attn_common.h"

namespace mi {
namespace {

constexpr int PA_WAVES = ATT_STREAMS;

// The work of one workgroup beside its kv head.
struct PagedItem {
    int r;           // request, < 0: none
    int wide;
    int q0, n, len;  // its first token, its tokens, its keys
    int cb;          // column block
    int split, ns;   // chunk of the block's keys, chunks (a request's earlier wide
                     // blocks have fewer than its last: split >= ns is no work)
    int runs;        // CHUNK_KEYS runs a chunk
    int first;       // the block's first state in the workspace (of 32 columns each),
                     // where it is cut
};

struct PagedArgs {
    const void *q, *k, *v;
    void *out;
    const int *table, *cu_q, *kv_lens;
    PagedItem *items;   // made by paged_items_kernel; null: each workgroup finds its own
    unsigned *tickets;  // by a block's first state and kv head
    float *part;  // partial states, by state and kv head; null: no block is cut
    int T, R, W, H, HK, G, pages, page_log2;
    int target;     // chunks wanted for a kv head
    int wide_runs;  // the least runs of a wide block's chunk
    float scale;    // > 0, log2 units
    uint32_t flip;  // sign bits of a negative scale, for Q
};

constexpr int CHUNK_KEYS = ATT_KT * PA_WAVES;  // keys are cut in multiples of this
constexpr int MAX_CHUNKS = 128;  // of a block: one workgroup adds them

// One request a lane: its first token, tokens, keys, column blocks (wide: of
// WIDE_COLS columns) and CHUNK_KEYS runs of keys. (Offsets and lengths are held
// to the rows and the table that there are.)
constexpr int WIDE_COLS = 128;
struct Req {
    int q0, n, len, wide, narrow, runs;
    int falls;  // whether it ends before it starts
};
template <bool WIDE> __device__ __forceinline__ Req load_req(const PagedArgs &a, int r) {
    Req q;
    const bool in = r < a.R;
    const int at = min(r, a.R - 1);  // (loads in flight together, no branch)
    const int from = a.cu_q[at], to = a.cu_q[at + 1], len = a.kv_lens[at];
    q.falls = to < from;
    q.q0 = min(max(from, 0), a.T);
    q.n = in ? min(max(to, q.q0), a.T) - q.q0 : 0;
    q.len = in ? min(max(len, 0), a.W << a.page_log2) : 0;
    const int cols = q.n * a.G;
    const bool wide = WIDE && cols > 32;
    q.wide = wide ? (cols + WIDE_COLS - 1) / WIDE_COLS : 0;
    q.narrow = wide ? 0 : (cols + 31) >> 5;
    q.runs = (q.len + CHUNK_KEYS - 1) / CHUNK_KEYS;
    return q;
}

// Runs that the lane's request's blocks read on average (a wide request's first
// block sees fewer keys than its last).
__device__ __forceinline__ int mean_runs(const PagedArgs &a, const Req &q) {
    const int first = q.len - q.n + min(WIDE_COLS / a.G + 1, q.n);
    return q.wide ? (q.runs + (max(first, 0) + CHUNK_KEYS - 1) / CHUNK_KEYS + 1) / 2 : q.runs;
}

// The wide blocks of a lane's request that see at least L runs of keys, its last
// ones: block cb's last token is min((128 cb + 127) / G, n - 1), which sees len - n
// keys and those up to its own.
__device__ __forceinline__ int blocks_from(const PagedArgs &a, const Req &q, int L) {
    const int y = (L - 1) * CHUNK_KEYS - (q.len - q.n);  // the first token that does
    if (q.wide == 0 || (y >= q.n && L > 0)) return 0;
    return y <= 0 || L == 0 ? q.wide : q.wide - min(y * a.G / WIDE_COLS, q.wide - 1);
}

// Item u: the wide blocks' chunks, then the narrow ones' whole chunks, then what is
// left of them, each in the order of requests, of their blocks, of their chunks;
// but the wide ones of at most 64 requests from those that see the most keys to
// those that see the fewest: what starts last should be short. Every wave finds
// its item by itself, 64 requests a step: first the runs of all blocks, which give
// the size of a chunk, then the chunks up to its own.
template <bool WIDE>
__device__ __forceinline__ PagedItem find_item(const PagedArgs &a, int u, int lane) {
    Req q = load_req<WIDE>(a, lane);
    int runs = 1 << 30, longest = 0;
    if (a.part) {
        // (blocks < 2^16 and runs < 2^23: summed in two halves)
        uint64_t total = 0, falls = 0;
        for (int r0 = 0;;) {
            const Req next = a.R > r0 + 64 ? load_req<WIDE>(a, r0 + 64 + lane) : q;
            longest = max(longest, q.runs);
            falls |= __builtin_amdgcn_ballot_w64(q.falls != 0);
            const uint64_t mine =
                (uint64_t)(unsigned)(q.wide + q.narrow) * (unsigned)mean_runs(a, q);
            const int lo = wave_scan((int)(mine & 0xFFFFFF)), hi = wave_scan((int)(mine >> 24));
            total += (uint64_t)(unsigned)__builtin_amdgcn_readlane(lo, 63) +
                     ((uint64_t)(unsigned)__builtin_amdgcn_readlane(hi, 63) << 24);
            r0 += 64;
            if (r0 >= a.R) break;
            q = next;
        }
        // requests that overlap could be more blocks than there are items and tickets:
        // none is taken
        if (falls) u = 0x7fffffff;
        total += a.target - 1;
        const uint64_t each = total >> 32 ? total / (unsigned)a.target
                                          : (unsigned)total / (unsigned)a.target;
        runs = each < 1 ? 1 : each < (1u << 30) ? (int)each : 1 << 30;
    }
    PagedItem it;
    it.r = -1;
    int before = 0, states = 0, narrow_states = 0;  // items, and cut blocks' states
#pragma unroll
    for (int kind = WIDE ? 0 : 1; kind < 3; ++kind) {
        const bool wide = kind == 0;
        const int scale = wide ? WIDE_COLS / 32 : 1;
        if (wide && a.R <= 64) {
            const int per = max(max(runs, a.wide_runs), (q.runs + MAX_CHUNKS - 1) / MAX_CHUNKS);
            const int ns = max(1, (q.runs + per - 1) / per);
            const int end = wave_scan(q.wide * ns);
            const int state_items = ns > 1 ? q.wide * ns : 0, state_end = wave_scan(state_items);
            before = __builtin_amdgcn_readlane(end, 63);
            states = scale * __builtin_amdgcn_readlane(state_end, 63);
            if (u >= before) continue;
            // the largest L of which more than u items see at least L runs
            int lo = 0, hi = ((a.W << a.page_log2) + CHUNK_KEYS - 1) / CHUNK_KEYS + 1, above = 0;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                const int n = __builtin_amdgcn_readlane(wave_scan(blocks_from(a, q, mid) * ns), 63);
                if (n > u)
                    lo = mid;
                else
                    hi = mid, above = n;
            }
            const int have = blocks_from(a, q, lo), at = (have - blocks_from(a, q, lo + 1)) * ns;
            const int upto = above + wave_scan(at);
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > u));
            it.r = l;
            it.wide = true;
            it.q0 = __builtin_amdgcn_readlane(q.q0, l);
            it.n = __builtin_amdgcn_readlane(q.n, l);
            it.len = __builtin_amdgcn_readlane(q.len, l);
            it.ns = __builtin_amdgcn_readlane(ns, l);
            it.runs = __builtin_amdgcn_readlane(per, l);
            const int p = u - __builtin_amdgcn_readlane(upto - at, l), b = p / it.ns;
            it.split = p - b * it.ns;
            it.cb = __builtin_amdgcn_readlane(q.wide - have, l) + b;
            it.first =
                scale * (__builtin_amdgcn_readlane(state_end - state_items, l) + it.cb * it.ns);
            return it;
        }
        if (kind == 1) {
            narrow_states = states;
            if (!__builtin_amdgcn_ballot_w64(longest >= runs)) continue;  // none is cut
        }
        if (kind == 2) states = narrow_states;
        if (a.R > 64) q = load_req<WIDE>(a, lane);
        for (int r0 = 0;;) {
            const Req next = a.R > r0 + 64 ? load_req<WIDE>(a, r0 + 64 + lane) : q;
            const int per = max(max(runs, wide ? a.wide_runs : 1),
                                (q.runs + MAX_CHUNKS - 1) / MAX_CHUNKS);
            const int ns = max(1, (q.runs + per - 1) / per), whole = q.runs / per;
            const int blocks = wide ? q.wide : q.narrow;
            const int some = wide ? ns : kind == 1 ? whole : ns - whole, items = blocks * some;
            const int end = before + wave_scan(items);
            const int state_items = ns > 1 ? scale * blocks * ns : 0;
            const int state_end = states + wave_scan(state_items);
            const uint64_t past = __builtin_amdgcn_ballot_w64(end > u);
            if (past) {
                const int l = __builtin_ctzll(past);
                it.r = r0 + l;
                it.wide = wide;
                it.q0 = __builtin_amdgcn_readlane(q.q0, l);
                it.n = __builtin_amdgcn_readlane(q.n, l);
                it.len = __builtin_amdgcn_readlane(q.len, l);
                it.ns = __builtin_amdgcn_readlane(ns, l);
                it.runs = __builtin_amdgcn_readlane(per, l);
                const int at = u - __builtin_amdgcn_readlane(end - items, l);
                const int each = __builtin_amdgcn_readlane(some, l), b = at / each;
                it.split = at - b * each + (kind == 2 ? __builtin_amdgcn_readlane(whole, l) : 0);
                it.cb = wide ? __builtin_amdgcn_readlane(blocks, l) - 1 - b : b;
                it.first =
                    __builtin_amdgcn_readlane(state_end - state_items, l) + scale * b * it.ns;
                return it;
            }
            before = __builtin_amdgcn_readlane(end, 63);
            states = __builtin_amdgcn_readlane(state_end, 63);
            r0 += 64;
            if (r0 >= a.R) break;
            q = next;
        }
    }
    return it;
}

#if defined(__HIP_DEVICE_COMPILE__)
// The DMA of one key tile of K or V: rows [0, left) of it (at most 32) lie at
// lo (rows 0..15) and hi (rows 16..31, its own 16 rows); the rest arrive as zeros.
// NT: non-temporal, for what is read once (decode: 48 requests of 64 to 8191 keys
// 152 -> 136 us; wide blocks, which share keys through the L2, 97 -> 105 with it).
template <typename T, int D, bool ISV, bool NT>
__device__ __forceinline__ void dma_paged_tile(const T *lo, const T *hi, int left, char *dst,
                                               int lane) {
    typedef Tile<D> Tl;
    const int n0 = left < 0 ? 0 : (left < 16 ? left : 16);
    const int n1 = left < 16 ? 0 : (left < 32 ? left - 16 : 16);
    const __amdgpu_buffer_rsrc_t r0 = att_rsrc(lo, (uint32_t)(n0 * D * 2));
    const __amdgpu_buffer_rsrc_t r1 = att_rsrc(hi, (uint32_t)(n1 * D * 2));
#pragma unroll
    for (int i = 0; i < Tl::NI; ++i) {
        const int row = i * Tl::RPI + lane / Tl::CPR, pos = lane % Tl::CPR;
        const int c = pos ^ (ISV ? swz_v<D>(row) : swz_k<D>(row));
        const bool second = i * Tl::RPI >= 16;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(second ? r1 : r0, (lds_ptr)(dst + i * 1024), 16,
                                                 ((row & 15) * D + 8 * c) * 2, 0, 0, NT ? 2 : 0);
    }
}
#endif

template <int D> struct PagedLds {
    static constexpr int SLOTS = PA_WAVES * 2 * Tile<D>::BYTES;  // = two wide stages
    static constexpr int FOLD = PA_WAVES * Part<D>::BYTES;
    static constexpr int BYTES = SLOTS > FOLD ? SLOTS : FOLD;
};

// A chunk's state in the workspace, of 32 columns, in whole lines of a wave's
// stores (written past the caches, pieces of a line cost a line each): a narrow
// block's is columns of D sums, then of (l, m); a wide one's is the registers' pairs
// by lane, then (l, m) by lane.
template <int D> struct PartState {
    static constexpr int WORDS = 32 * D + 128;
};

template <int D> __device__ __forceinline__ float *part_at(const PagedArgs &a, int state, int hk) {
    return a.part + ((int64_t)state * a.HK + hk) * PartState<D>::WORDS;
}

// A narrow block's chunk has been put: the last workgroup of it to come here adds
// the chunks, out = sum_s w_s O_s / sum_s w_s l_s with w_s = 2^(m_s - max m). A
// column takes D / 4 lanes of four values; four columns at a time, the 256 / D
// groups of lanes take every so manyth chunk, in order, and are added in order.
constexpr int JOIN_COLS = 4;
template <typename T, int D>
__device__ __forceinline__ void join_narrow(const PagedArgs &a, const PagedItem &it, int hk,
                                            int have, char *lds) {
#pragma clang fp contract(off)
    constexpr int LANES = D / 4, GROUPS = 256 / (LANES * JOIN_COLS), IN_FLIGHT = D == 64 ? 8 : 16;
    if (!last_of(a.tickets + (int64_t)it.first * a.HK + hk, it.ns)) return;
    float4 *acc = (float4 *)lds;                                    // [GROUPS][JOIN_COLS][LANES]
    float2 *lm = (float2 *)(acc + GROUPS * JOIN_COLS * LANES);      // [GROUPS][JOIN_COLS]
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int jc = sub % JOIN_COLS, g = sub / JOIN_COLS;
    const int64_t step = (int64_t)a.HK * PartState<D>::WORDS;
    for (int c0 = 0; c0 < have; c0 += JOIN_COLS) {  // (workgroup-uniform)
        const int col = c0 + jc, c = col < have ? col : 0;
        const float *base = part_at<D>(a, it.first, hk);
        const float *po = base + c * D + 4 * lane, *pl = base + 32 * D + 2 * c;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.0f, m = -INFINITY;
        auto add = [&](const float4 &v, const float2 &w) {
            const MergeCoef k = merge_coef(m, w.y);
            o.x = merge_one(o.x, v.x, k);
            o.y = merge_one(o.y, v.y, k);
            o.z = merge_one(o.z, v.z, k);
            o.w = merge_one(o.w, v.w, k);
            l = merge_one(l, w.x, k);
            m = k.m_new;
        };
        for (int s0 = g; s0 < it.ns; s0 += GROUPS * IN_FLIGHT) {
            float4 v[IN_FLIGHT];
            float2 w[IN_FLIGHT];
#pragma unroll
            for (int i = 0; i < IN_FLIGHT; ++i) {
                const int s = s0 + GROUPS * i;
                const int64_t at = (s < it.ns ? s : g) * step;
                const float2 a0 = get_part((const float2 *)(po + at));
                const float2 a1 = get_part((const float2 *)(po + at + 2));
                v[i] = make_float4(a0.x, a0.y, a1.x, a1.y);
                w[i] = get_part((const float2 *)(pl + at));
            }
#pragma unroll
            for (int i = 0; i < IN_FLIGHT; ++i)
                if (s0 + GROUPS * i < it.ns) add(v[i], w[i]);
        }
        __syncthreads();
        acc[(g * JOIN_COLS + jc) * LANES + lane] = o;
        if (lane == 0) lm[g * JOIN_COLS + jc] = make_float2(l, m);
        __syncthreads();
        if (g == 0 && col < have) {
#pragma unroll
            for (int i = 1; i < GROUPS; ++i)
                add(acc[(i * JOIN_COLS + jc) * LANES + lane], lm[i * JOIN_COLS + jc]);
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            const int idx = it.cb * 32 + col, tok = idx / a.G;
            T *orow = (T *)a.out +
                      ((int64_t)(it.q0 + tok) * a.H + hk * a.G + (idx - tok * a.G)) * D;
            const float e[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
            st8(orow + 4 * lane, pack4<T>(e));
        }
    }
}

#if defined(__HIP_DEVICE_COMPILE__)
// The pages of a wave's next 64 tiles kt, kt + STEP, ..., one a lane (a tile of
// 16-row pages has two), and a tile's first and second 16 rows of the kv head in
// the pools.
template <int STEP> struct TilePages {
    const int *row;
    int64_t hk;
    int W, pages, lp, HK;
    int id0, id1;
    __device__ __forceinline__ TilePages(const PagedArgs &a, int r, int hk_)
        : row(a.table + (int64_t)r * a.W), hk(hk_), W(a.W), pages(a.pages), lp(a.page_log2),
          HK(a.HK), id0(0), id1(0) {}
    __device__ __forceinline__ void load(int kt, int lane) {
        const int key = (kt + STEP * lane) * ATT_KT;
        id0 = min(max(row[min(key >> lp, W - 1)], 0), pages - 1);
        id1 = min(max(row[min((key + 16) >> lp, W - 1)], 0), pages - 1);
    }
    // the tile `at` steps (mod 64) behind the loaded one, of first key `key`
    __device__ __forceinline__ void rows(int at, int key, int64_t &lo, int64_t &hi) const {
        const int64_t mask = ((int64_t)1 << lp) - 1;
        lo = (((int64_t)__builtin_amdgcn_readlane(id0, at & 63) * HK + hk) << lp) + (key & mask);
        hi = (((int64_t)__builtin_amdgcn_readlane(id1, at & 63) * HK + hk) << lp) +
             ((key + 16) & mask);
    }
};

// Whether a wave's sums have a NaN (or infinities of both signs).
template <int D> __device__ __forceinline__ bool not_a_number(const AttnState<D> &st) {
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[i & 3] += st.o[t][i];
    const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    return __builtin_amdgcn_ballot_w64(all != all) != 0;
}

// A narrow block: wave w takes the key tiles w, w + 4, ... of the chunk into LDS of
// its own (a K and a V slot, refilled as soon as their reads are in registers: no
// barrier), and the four states are folded at the end. Bound by HBM: K and V are
// read once.
template <typename T, int D>
__device__ __forceinline__ void narrow_block(const PagedArgs &a, const PagedItem &it, int hk,
                                             char *lds) {
    typedef Tile<D> Tl;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h2 = lane >> 5, r = lane & 31;
    const int idx = it.cb * 32 + r, cols = it.n * a.G;
    const bool ok = idx < cols;
    const int tok = (ok ? idx : 0) / a.G, g = (ok ? idx : 0) - tok * a.G;
    const int64_t qrow = (int64_t)(it.q0 + tok) * a.H + hk * a.G + g;
    // keys [0, end) are seen by the lane's row, [0, full) by every row, [0, last)
    // by the block's last
    const int off = it.len - it.n;
    const int end = off + tok + 1;
    const int full = off + (it.cb * 32) / a.G + 1;
    const int bottom = min(it.cb * 32 + 31, cols - 1);
    const int last = min(off + bottom / a.G + 1, it.len);
    // the chunk's key tiles
    const int all = last > 0 ? (last + ATT_KT - 1) / ATT_KT : 0;
    const int t0 = it.split * it.runs * PA_WAVES + wave;
    const int ntiles = it.ns > 1 ? min(all, (it.split + 1) * it.runs * PA_WAVES) : all;
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
            pg.load(t0, lane);
            int64_t lo, hi;
            pg.rows(0, t0 * ATT_KT, lo, hi);
            const int left = it.len - t0 * ATT_KT;
            dma_paged_tile<T, D, false, true>(k + lo * D, k + hi * D, left, ks, lane);
            dma_paged_tile<T, D, true, true>(v + lo * D, v + hi * D, left, vs, lane);
        }
        for (int kt = t0; kt < ntiles; kt += PA_WAVES) {  // wave-uniform
            const int nx = kt + PA_WAVES;
            const bool more = nx < ntiles;
            int64_t lo = 0, hi = 0;
            if (more) {
                const int at = (nx - t0) / PA_WAVES;
                if ((at & 63) == 0) pg.load(nx, lane);
                pg.rows(at, nx * ATT_KT, lo, hi);
            }
            const int left = it.len - nx * ATT_KT;
            // K (and, the first time, q) has landed once only V's loads, issued
            // after it, are in flight
            att_wait_vmcnt<Tl::NI>();
            flip_q<D>(qf, flip);
            uint4 kf[D / 16];
            read_k<D>(ks, kf, r, h2);
#pragma unroll
            for (int s = 0; s < D / 16; ++s) launder(kf[s]);  // the reads have returned
            __builtin_amdgcn_sched_barrier(0);
            if (more)
                dma_paged_tile<T, D, false, true>(k + lo * D, k + hi * D, left, ks, lane);
            f32x16 s = attn_scores<T, D>(kf, qf);
            const int k0 = kt * ATT_KT;
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
            if (more)
                dma_paged_tile<T, D, true, true>(v + lo * D, v + hi * D, left, vs, lane);
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
    Fold f;
    if (wave < D / 32) f = fold_streams<D>(part, wave, lane);
    if (it.ns == 1) {  // (workgroup-uniform)
        if (wave >= D / 32) return;
        const float inv = row_inv(f.l);
        if (ok) store_fold<T>(f, inv, (T *)a.out + qrow * D, wave, h2);
        return;
    }
    __syncthreads();  // every wave has folded; the state by columns, then out
    float *cols_at = (float *)lds;  // [32][D], [32] (l, m)
    if (wave < D / 32) {
        const float l = f.l + __shfl_xor(f.l, 32, 64);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *(float4 *)(cols_at + r * D + 32 * wave + 8 * j + 4 * h2) = f.o[j];
        if (wave == 0 && h2 == 0) *(float2 *)(cols_at + 32 * D + 2 * r) = make_float2(l, f.m);
    }
    __syncthreads();
    float *o = part_at<D>(a, it.first + it.split, hk);
    const int have = min(cols - it.cb * 32, 32);
    for (int i = 2 * threadIdx.x; i < have * D; i += 128 * PA_WAVES)
        put_part((float2 *)(o + i), *(float2 *)(cols_at + i));
    if ((int)threadIdx.x < have)
        put_part((float2 *)(o + 32 * D) + threadIdx.x,
                 *(float2 *)(cols_at + 32 * D + 2 * threadIdx.x));
    join_narrow<T, D>(a, it, hk, have, lds);
}

// attn_softmax over two key tiles.
template <typename T, int D>
__device__ __forceinline__ void softmax_pair(AttnState<D> &st, const f32x16 (&s)[2],
                                             uint32_t (&pk)[2][8], float scale) {
#pragma clang fp contract(off)
    float mt[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        mt[j] = fmaxf(s[j][0], s[j][1]);
#pragma unroll
        for (int i = 2; i < 16; i += 2) mt[j] = fmaxf(fmaxf(mt[j], s[j][i]), s[j][i + 1]);
    }
    const float m = max_halves(fmaxf(mt[0], mt[1])) * scale;
    const bool grow = m > st.m + 8.0f;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float m_new = grow ? m : st.m;
        const float corr = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - m_new);
        st.l *= corr;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) st.o[t][i] *= corr;
        st.m = m_new;
    }
    const float nm = st.m == -INFINITY ? 0.0f : -st.m;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][2 * i], scale, nm));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][2 * i + 1], scale, nm));
            pk[j][i] = pk2<T>(p0, p1);
            sum[2 * (i & 1)] += p0;
            sum[2 * (i & 1) + 1] += p1;
        }
    st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// A wide block: wave w has the columns 32 w .. 32 w + 31 of the block's 128, and
// all four share each stage of two key tiles, staged by DMA into one of two
// buffers while the other is read: K and V pass through LDS once for 128 columns
// where a narrow block's pass for 32.
template <typename T, int D>
__device__ __forceinline__ void wide_block(const PagedArgs &a, const PagedItem &it, int hk,
                                           char *lds) {
    typedef Tile<D> Tl;
    constexpr int STAGE = 4 * Tl::BYTES;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h2 = lane >> 5, r = lane & 31;
    const int cols = it.n * a.G, c0 = it.cb * WIDE_COLS + 32 * wave, idx = c0 + r;
    const bool ok = idx < cols;
    const int tok = (ok ? idx : 0) / a.G, g = (ok ? idx : 0) - tok * a.G;
    const int64_t qrow = (int64_t)(it.q0 + tok) * a.H + hk * a.G + g;
    const int off = it.len - it.n, end = off + tok + 1, full = off + c0 / a.G + 1;
    // key tiles that the wave's columns see, and the block's
    auto tiles_to = [&](int col) {
        const int last = min(off + min(col, cols - 1) / a.G + 1, it.len);
        return last > 0 ? (last + ATT_KT - 1) / ATT_KT : 0;
    };
    const int t0 = it.split * it.runs * PA_WAVES;
    const int stop = it.ns > 1 ? (it.split + 1) * it.runs * PA_WAVES : 1 << 30;
    const int t1 = min(tiles_to(it.cb * WIDE_COLS + WIDE_COLS - 1), stop);
    const int mine = c0 < cols ? min(tiles_to(c0 + 31), stop) : 0;

    AttnState<D> st;
    attn_init(st);
    uint4 qf[D / 16];
    uint32_t flip = a.flip;
    read_q<D>((const T *)a.q + qrow * D, h2, qf);
    // stage s: key tiles t0 + 2 s, t0 + 2 s + 1; waves 0 and 1 stage K, 2 and 3 V
    TilePages<2> pg(a, it.r, hk);
    const T *pool = (const T *)(wave < 2 ? a.k : a.v);
    auto issue = [&](int s, char *dst) __attribute__((always_inline)) {
        const int kt = t0 + 2 * s + (wave & 1);
        if ((s & 63) == 0) pg.load(kt, lane);
        int64_t lo, hi;
        pg.rows(s, kt * ATT_KT, lo, hi);
        const int left = it.len - kt * ATT_KT;
        if (wave < 2)
            dma_paged_tile<T, D, false, false>(pool + lo * D, pool + hi * D, left,
                                               dst + wave * Tl::BYTES, lane);
        else
            dma_paged_tile<T, D, true, false>(pool + lo * D, pool + hi * D, left,
                                              dst + wave * Tl::BYTES, lane);
    };
    auto step = [&](const char *__restrict__ cb, char *__restrict__ nb, int s, bool more)
                    __attribute__((always_inline)) {
        // every wave's DMAs of stage s have landed, and every wave is done with
        // the buffer the next ones go to
        att_wait_vmcnt<0>();
        __syncthreads();
        flip_q<D>(qf, flip);
        if (more) issue(s + 1, nb);
        const int kt = t0 + 2 * s;
        if (kt >= mine) return;  // (wave-uniform)
        // both tiles: two chains of score MFMAs, one running maximum
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
        const int k0 = kt * ATT_KT;
        if (k0 + 2 * ATT_KT > full) {
            attn_mask(sc[0], end - k0, h2);
            attn_mask(sc[1], end - k0 - ATT_KT, h2);
        }
        uint32_t p[2][8];
        softmax_pair<T, D>(st, sc, p, a.scale);
        attn_pv<T, D>(st, p[0], vf);
        read_v<T, D>(cb + 3 * Tl::BYTES, vf, lane);
        attn_pv<T, D>(st, p[1], vf);
    };
    const int stages = t1 > t0 ? (t1 - t0 + 1) / 2 : 0;
    char *b0 = lds, *b1 = lds + STAGE;
    if (stages) issue(0, b0);
    for (int s = 0; s < stages; s += 2) {  // workgroup-uniform
        step(b0, b1, s, s + 1 < stages);
        if (s + 1 < stages) step(b1, b0, s + 1, s + 2 < stages);
    }
    if (it.ns > 1) {
        // the state out; the last workgroup of the block to come here folds all of
        // them, in order, each wave its own columns'
        constexpr int PAIRS = D / 32 * 8;
        float2 *o =
            (float2 *)part_at<D>(a, it.first + it.split * (WIDE_COLS / 32) + wave, hk) + lane;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
            put_part(o + 64 * i,
                     make_float2(st.o[i / 8][2 * (i % 8)], st.o[i / 8][2 * (i % 8) + 1]));
        put_part(o + 64 * PAIRS, make_float2(st.l, st.m));
        if (!last_of(a.tickets + (int64_t)it.first * a.HK + hk, it.ns)) return;
        attn_init(st);
        for (int s = 0; s < it.ns; ++s) {
            const float2 *p =
                (const float2 *)part_at<D>(a, it.first + s * (WIDE_COLS / 32) + wave, hk) + lane;
            float2 v[PAIRS + 1];
#pragma unroll
            for (int i = 0; i <= PAIRS; ++i) v[i] = get_part(p + 64 * i);
            const MergeCoef c = merge_coef(st.m, v[PAIRS].y);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const int t = i / 8, e = 2 * (i % 8);
                st.o[t][e] = merge_one(st.o[t][e], v[i].x, c);
                st.o[t][e + 1] = merge_one(st.o[t][e + 1], v[i].y, c);
            }
            st.l = merge_one(st.l, v[PAIRS].x, c);
            st.m = c.m_new;
        }
    }
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
}
#endif

// Workgroups a CU holds, a wave a SIMD each (four of the wide form with heads of 64
// would spill).
template <int D, bool WIDE> constexpr int paged_per_cu() { return D == 128 ? 2 : (WIDE ? 3 : 4); }

// A wave an item: found once for all kv heads.
template <bool WIDE>
__global__ __launch_bounds__(256) void paged_items_kernel(PagedArgs a, int items) {
    const int u = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (u >= items) return;
    const PagedItem it = find_item<WIDE>(a, u, threadIdx.x & 63);
    if ((threadIdx.x & 63) == 0) a.items[u] = it;
}

// One workgroup an item and kv head. WIDE: requests of more than 32 columns are in
// wide blocks; without it (decode) every block is narrow.
template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(64 * PA_WAVES)
__attribute__((amdgpu_waves_per_eu(paged_per_cu<D, WIDE>())))
void paged_attn_kernel(PagedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __attribute__((aligned(1024))) char lds[PagedLds<D>::BYTES];
    PagedItem it;
    if (a.items) {
        const int *p = (const int *)(a.items + blockIdx.y);
        int f[sizeof(PagedItem) / 4];
#pragma unroll
        for (int i = 0; i < (int)(sizeof(PagedItem) / 4); ++i) f[i] = p[i];
#pragma unroll
        for (int i = 0; i < (int)(sizeof(PagedItem) / 4); ++i)
            f[i] = __builtin_amdgcn_readfirstlane(f[i]);
        it = __builtin_bit_cast(PagedItem, f);
    } else {
        it = find_item<WIDE>(a, blockIdx.y, threadIdx.x & 63);
    }
    if (it.r < 0) return;  // (workgroup-uniform)
    if (WIDE && it.wide) {
        if (it.ns > 1) {
            // the block's own chunks, of equal sizes
            const int last = min((it.cb * WIDE_COLS + WIDE_COLS - 1) / a.G, it.n - 1);
            const int keys = max(it.len - it.n + last + 1, 1);
            const int runs = (keys + CHUNK_KEYS - 1) / CHUNK_KEYS;
            it.ns = (runs + it.runs - 1) / it.runs;
            it.runs = (runs + it.ns - 1) / it.ns;
            if (it.split >= it.ns) return;
        }
        wide_block<T, D>(a, it, blockIdx.x, lds);
    } else {
        narrow_block<T, D>(a, it, blockIdx.x, lds);
    }
#endif
}

// ---------------------------------------------------------------------------
// dispatch

// Workgroups of a launch. wide and narrow bound the blocks of each kind (n G / 128
// or n G / 32 of a request, rounded up). A chunk is one run or more, so there are
// at most `target` chunks and the last, shorter one of every block, and no more
// than a row of the table has. Few blocks: as many chunks as one round of
// workgroups takes with those last ones; many: one and a half rounds' worth, the
// shorter ones last (64 requests of 4096 keys: 171 us, with four rounds' 183).
// Wide blocks, whose parts cost 66 KB written and read, are then cut only where
// they fill less than two rounds, past 32 runs (20 requests, four of 256 to 512
// tokens and up to 4096 keys: 89 us; from 8 runs on, 97). Past two rounds the longest
// block's chain is mostly hidden (8192 tokens of one prompt 542 us; cut past 32 runs as
// well, 554), but not where one request's keys outgrow the others' by far: 512 tokens
// behind 32256 keys beside eight prompts of 1024 take 777 us, and cut 397.
struct PagedGrid {
    int64_t wide, narrow, items, states, target, wide_runs;
    bool cut, cut_wide, listed;
};
inline PagedGrid paged_grid(int64_t T, int64_t R, int64_t W, int64_t G, int64_t HK, int64_t D,
                            int64_t page, int64_t max_q) {
    PagedGrid g;
    const int64_t some = R < T ? R : T;
    if (max_q * G > 32) {
        const int64_t most = T * G / 33 < some ? T * G / 33 : some;  // requests that can be wide
        g.wide = T * G / WIDE_COLS + most;
        g.narrow = some;
    } else {
        g.wide = 0;
        g.narrow = T * G / 32 + some;
    }
    const int64_t slots = 256 * (D == 128 ? paged_per_cu<128, true>()
                                          : g.wide ? paged_per_cu<64, true>()
                                                   : paged_per_cu<64, false>());
    const int64_t runs = ceil_div(W * page, CHUNK_KEYS);
    const int64_t few = slots - (g.wide + g.narrow) * HK;
    g.target = (few >= slots / 2 ? few : 3 * slots / 2) / HK;
    if (g.target < 1) g.target = 1;
    g.wide_runs = few >= slots / 2 ? 1 : g.wide * HK < 2 * slots ? 32 : 1 << 23;
    g.cut = runs > 1;
    g.cut_wide = g.wide && runs > g.wide_runs;
    // Chunks of each kind, and those of cut blocks, which have states: a block cut
    // in two or more has at most twice its runs over a chunk's.
    int64_t wide = g.wide, narrow = g.narrow, wide_states = 0, narrow_states = 0;
    if (g.cut_wide) {
        // (the chunks are counted by a request's last block, their size comes from
        // the mean: up to twice as many)
        const int64_t most = g.wide * ceil_div(runs, g.wide_runs), some = g.wide + 2 * g.target;
        wide = some < most ? some : most;
        wide_states = wide < 4 * g.target ? wide : 4 * g.target;
    }
    if (g.cut) {
        const int64_t most = g.narrow * runs;
        narrow = g.narrow + g.target < most ? g.narrow + g.target : most;
        narrow_states = narrow < 2 * g.target ? narrow : 2 * g.target;
    }
    g.items = wide + narrow;
    // Past 192 requests a workgroup would sum over them for longer than a launch
    // takes that lists the items once (1000 requests of 300 keys: 222 us, without
    // 423; 300 of 600: 128, 140; 129 of 1000: 96, 90).
    g.listed = R > 192;
    g.states = wide_states * (WIDE_COLS / 32) + narrow_states;
    return g;
}
// The tickets take a fixed prefix of the workspace, so that calls of any sizes can
// share one whose prefix is zero.
constexpr int64_t PAGED_TICKETS = MI_PAGED_ZERO_BYTES / 4;
inline int64_t paged_list_bytes(const PagedGrid &g) {
    return g.listed ? ceil_div(g.items * (int64_t)sizeof(PagedItem), 256) * 256 : 0;
}
inline bool paged_cuts(const PagedGrid &g, int64_t HK) {
    return g.cut && g.states * HK <= PAGED_TICKETS;
}
inline int64_t paged_bytes(const PagedGrid &g, int64_t HK, int64_t D) {
    const int64_t states =
        paged_cuts(g, HK) ? g.states * HK * (32 * D + 128) * (int64_t)sizeof(float) : 0;
    return states || g.listed ? MI_PAGED_ZERO_BYTES + paged_list_bytes(g) + states : 0;
}

template <typename T, int D, bool WIDE>
int launch_paged_w(const PagedArgs &a, const PagedGrid &g, hipStream_t st) {
    const int64_t items = a.part ? g.items : g.wide + g.narrow;
    if (a.items)
        paged_items_kernel<WIDE><<<(unsigned)ceil_div(items, 4), 256, 0, st>>>(a, (int)items);
    paged_attn_kernel<T, D, WIDE><<<dim3((unsigned)a.HK, (unsigned)items),
                                    64 * PA_WAVES, 0, st>>>(a);
    return launch_status("paged attention");
}
template <typename T, int D>
int launch_paged(const PagedArgs &a, const PagedGrid &g, hipStream_t st) {
    return g.wide ? launch_paged_w<T, D, true>(a, g, st) : launch_paged_w<T, D, false>(a, g, st);
}

bool page_log2_of(int64_t page, int &lp) {
    for (lp = 4; lp <= 8; ++lp)
        if (page == (1 << lp)) return true;
    return false;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_paged_attention_workspace_bytes(int64_t T, int64_t R, int64_t table_width,
                                                      int64_t H, int64_t HK, int64_t D,
                                                      int64_t page_size, int64_t max_q_len) {
    if (T <= 0 || R <= 0 || table_width <= 0 || H <= 0 || HK <= 0 || H % HK ||
        (D != 64 && D != 128) || page_size <= 0)
        return 0;
    return paged_bytes(paged_grid(T, R, table_width, H / HK, HK, D, page_size,
                                  max_q_len > 0 && max_q_len < T ? max_q_len : T), HK, D);
}

extern "C" int mi_paged_attention(const void *q, const void *k_pages, const void *v_pages,
                                  void *out, const int32_t *block_table, const int32_t *cu_q,
                                  const int32_t *kv_lens, int64_t T, int64_t R,
                                  int64_t table_width, int64_t H, int64_t HK, int64_t D,
                                  int64_t n_pages, int64_t page_size, int64_t max_q_len,
                                  float scale, int dtype, void *workspace,
                                  int64_t workspace_bytes, void *stream) {
    if (dtype != MI_BF16 && dtype != MI_F16)
        return fail(MI_ERR_UNSUPPORTED, "paged attention covers bf16 and fp16 (dtype code %d)",
                    dtype);
    if (D != 64 && D != 128)
        return fail(MI_ERR_UNSUPPORTED, "paged attention head dim %lld", (long long)D);
    int lp;
    if (!page_log2_of(page_size, lp))
        return fail(MI_ERR_UNSUPPORTED, "page size %lld; this build covers 16, 32, 64, 128, 256",
                    (long long)page_size);
    if (T < 0 || R < 0 || H < 1 || HK < 1 || H % HK || HK > 65535 || table_width < 1 ||
        n_pages < 1 || n_pages > (0x7fffffff >> lp) || table_width > (0x3fffffff >> lp) ||
        T > 0x3fffffff || T * (H / HK) > 0x3fffffff || R > 0x3fffffff)
        return fail(MI_ERR_ARG, "paged attention shape T=%lld R=%lld table width %lld H=%lld "
                    "HK=%lld pages=%lld", (long long)T, (long long)R, (long long)table_width, (long long)H,
                    (long long)HK, (long long)n_pages);
    if (T == 0 || R == 0) return MI_OK;
    if (!q || !k_pages || !v_pages || !out || !block_table || !cu_q || !kv_lens)
        return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 8))
        return fail(MI_ERR_ARG, "q and the pages must be 16-byte aligned, out 8-byte aligned");
    const PagedGrid g = paged_grid(T, R, table_width, H / HK, HK, D, page_size,
                                   max_q_len > 0 && max_q_len < T ? max_q_len : T);
    if (g.items > 65535)
        return fail(MI_ERR_ARG, "paged attention: %lld blocks of query rows, at most 65535",
                    (long long)g.items);
    const int64_t need = paged_bytes(g, HK, D);
    char *ws = need && workspace && workspace_bytes >= need && aligned(workspace, 16)
                   ? (char *)workspace : nullptr;
    const float sl = scale * 1.4426950408889634f;
    // (a scale of 0 as the smallest normal: masked scores stay -inf; NaN stays NaN)
    const float mag = fabsf(sl) < 1.17549435e-38f ? 1.17549435e-38f : fabsf(sl);
    char *lists = ws ? ws + MI_PAGED_ZERO_BYTES : nullptr;
    const PagedArgs a = {q, k_pages, v_pages, out, block_table, cu_q, kv_lens,
                         ws && g.listed ? (PagedItem *)lists : nullptr, (unsigned *)ws,
                         ws && paged_cuts(g, HK) ? (float *)(lists + paged_list_bytes(g)) : nullptr,
                         (int)T, (int)R, (int)table_width, (int)H, (int)HK, (int)(H / HK),
                         (int)n_pages, lp,
                         (int)g.target, (int)g.wide_runs, mag, sl < 0.0f ? 0x80008000u : 0u};
    hipStream_t st = as_stream(stream);
    if (dtype == MI_BF16)
        return D == 128 ? launch_paged<bf16, 128>(a, g, st) : launch_paged<bf16, 64>(a, g, st);
    return D == 128 ? launch_paged<f16, 128>(a, g, st) : launch_paged<f16, 64>(a, g, st);
}
