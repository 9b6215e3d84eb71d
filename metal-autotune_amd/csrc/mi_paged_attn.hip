// Causal GQA attention of requests of different lengths over a paged key/value
// cache (no counterpart in the reference, whose caches are contiguous):
// mi_paged_attention.
//
// For request r with n new tokens and len keys, token i, q head h over kv head
// h / G:  o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),
// s_j = scale log2(e) q . k_j,  j <= len - n + i;  0 where no key is seen.
// Key j sits in row j % page_size of page block_table[r][j / page_size].
//
// The tile, the softmax and the folds are the contiguous attention's
// (mi_attn_common.h). A kv head's query rows, token after token and in a token
// its G q heads, are the columns of 32-wide blocks, so K and V are read once per
// block and kv head and a block sees nearly one causal range.
//
// Requests differ in length, and only the GPU knows the lengths. The keys of
// every block are therefore cut into chunks of one size, chosen on the GPU from
// the lengths of all requests so that the chunks fill the chip (chunk_of), and a
// workgroup finds its chunk by summing over the requests. A block of one chunk
// writes its rows; the others' states go to a workspace and
// paged_combine_kernel folds them. The chunk size, so a row's last bits, depends
// on the lengths of the whole batch.
#include "mi_attn_common.h"

namespace mi {
namespace {

constexpr int PA_WAVES = ATT_STREAMS;

struct PagedArgs {
    const void *q, *k, *v;
    void *out;
    const int *table, *cu_q, *kv_lens;
    float *part;  // partial states, by item and kv head; null: no block is cut
    int T, R, W, H, HK, G, pages, page_log2;
    int target;     // chunks wanted for a kv head
    float scale;    // > 0, log2 units
    uint32_t flip;  // sign bits of a negative scale, for Q
};

// The sum of v over the wave's lanes up to and including this one (see
// paged_plan_kernel's).
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    v = dpp_add<0x118, 0xF>(v);
    v = dpp_add<0x142, 0xA>(v);
    v = dpp_add<0x143, 0xC>(v);
    return v;
}

constexpr int CHUNK_KEYS = ATT_KT * PA_WAVES;  // keys are cut in multiples of this

// One request a lane: its first token, tokens, keys, column blocks and
// CHUNK_KEYS runs of keys. (Offsets and lengths are held to the rows and the
// table that there are.)
struct Req {
    int q0, n, len, blocks, runs;
};
__device__ __forceinline__ Req load_req(const PagedArgs &a, int r) {
    Req q;
    const bool in = r < a.R;
    q.q0 = in ? min(max(a.cu_q[r], 0), a.T) : 0;
    q.n = in ? min(max(a.cu_q[r + 1], q.q0), a.T) - q.q0 : 0;
    q.len = in ? min(max(a.kv_lens[r], 0), a.W << a.page_log2) : 0;
    q.blocks = (q.n * a.G + 31) >> 5;
    q.runs = (q.len + CHUNK_KEYS - 1) / CHUNK_KEYS;
    return q;
}

// The work of one workgroup beside its kv head.
struct PagedItem {
    int r;           // request, < 0: none
    int q0, n, len;  // its first token, its tokens, its keys
    int cb;          // column block
    int split, ns;   // chunk of the block's keys, chunks
    int runs;        // CHUNK_KEYS runs a chunk
    int first;       // the block's first item
};

// Item u (BLOCK: the first item of column block u) in the order of requests, of
// their blocks, of their chunks. Every wave finds it by itself, 64 requests a
// step: first the runs of all blocks, which give the size of a chunk, then the
// chunks up to its own.
template <bool BLOCK>
__device__ __forceinline__ PagedItem find_item(const PagedArgs &a, int u, int lane) {
    Req q = load_req(a, lane);
    int runs = 1 << 30;
    if (a.part) {
        // (blocks < 2^16 and runs < 2^23: summed in two halves)
        uint64_t total = 0;
        for (int r0 = 0;;) {
            const uint64_t mine = (uint64_t)(unsigned)q.blocks * (unsigned)q.runs;
            const int lo = wave_scan((int)(mine & 0xFFFFFF)), hi = wave_scan((int)(mine >> 24));
            total += (uint64_t)(unsigned)__builtin_amdgcn_readlane(lo, 63) +
                     ((uint64_t)(unsigned)__builtin_amdgcn_readlane(hi, 63) << 24);
            r0 += 64;
            if (r0 >= a.R) break;
            q = load_req(a, r0 + lane);
        }
        total += a.target - 1;
        runs = total >> 32 ? (int)(total / (unsigned)a.target)
                           : (int)((unsigned)total / (unsigned)a.target);
        runs = max(1, runs);
        if (a.R > 64) q = load_req(a, lane);
    }
    int before = 0, items = 0;
    for (int r0 = 0;;) {
        const int ns = max(1, (q.runs + runs - 1) / runs);
        const int mine = q.blocks * ns;
        const int count = BLOCK ? q.blocks : mine;
        const int end = before + wave_scan(count);
        const int item_end = BLOCK ? items + wave_scan(mine) : end;
        const uint64_t past = __builtin_amdgcn_ballot_w64(end > u);
        if (past) {
            const int l = __builtin_ctzll(past);
            PagedItem it;
            it.r = r0 + l;
            it.q0 = __builtin_amdgcn_readlane(q.q0, l);
            it.n = __builtin_amdgcn_readlane(q.n, l);
            it.len = __builtin_amdgcn_readlane(q.len, l);
            it.ns = __builtin_amdgcn_readlane(ns, l);
            it.runs = runs;
            const int at = u - __builtin_amdgcn_readlane(end - count, l);
            it.cb = BLOCK ? at : at / it.ns;
            it.split = BLOCK ? 0 : at - it.cb * it.ns;
            it.first = __builtin_amdgcn_readlane(item_end - mine, l) + it.cb * it.ns;
            return it;
        }
        before = __builtin_amdgcn_readlane(end, 63);
        if (BLOCK) items = __builtin_amdgcn_readlane(item_end, 63);
        r0 += 64;
        if (r0 >= a.R) break;
        q = load_req(a, r0 + lane);
    }
    PagedItem none;
    none.r = -1;
    return none;
}

#if defined(__HIP_DEVICE_COMPILE__)
// The DMA of one key tile of K or V: rows [0, left) of it (at most 32) lie at
// lo (rows 0..15) and hi (rows 16..31, its own 16 rows); the rest arrive as zeros.
template <typename T, int D, bool ISV>
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
                                                 ((row & 15) * D + 8 * c) * 2, 0, 0, 0);
    }
}
#endif

template <int D> struct PagedLds {
    static constexpr int SLOTS = PA_WAVES * 2 * Tile<D>::BYTES;
    static constexpr int FOLD = PA_WAVES * Part<D>::BYTES;
    static constexpr int BYTES = SLOTS > FOLD ? SLOTS : FOLD;
};

// A chunk's state in the workspace: 32 columns of D sums, then of (l, m).
template <int D> struct PartState {
    static constexpr int WORDS = 32 * (D + 2);
};

// Four waves a workgroup, a column block of one kv head; wave w takes the key
// tiles w, w + 4, ... into LDS of its own (a K and a V slot, refilled as soon as
// their reads are in registers), and the four states are folded at the end.
template <typename T, int D>
__global__ __launch_bounds__(64 * PA_WAVES) void paged_wave_kernel(PagedArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Tile<D> Tl;
    __shared__ __attribute__((aligned(1024))) char lds[PagedLds<D>::BYTES];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h2 = lane >> 5, r = lane & 31;
    const int hk = blockIdx.x;
    const PagedItem it = find_item<false>(a, blockIdx.y, lane);
    if (it.r < 0) return;  // (workgroup-uniform)
    const int lp = a.page_log2, idx = it.cb * 32 + r, cols = it.n * a.G;
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
    const int *row_of = a.table + (int64_t)it.r * a.W;
    const int64_t head_rows = (int64_t)1 << lp;

    char *kslot = lds + wave * 2 * Tl::BYTES, *vslot = kslot + Tl::BYTES;
    AttnState<D> st;
    attn_init(st);
    uint4 qf[D / 16];
    uint32_t flip = a.flip;
    auto run = [&](char *__restrict__ ks, char *__restrict__ vs) __attribute__((always_inline)) {
        read_q<D>((const T *)a.q + qrow * D, h2, qf);
        // pages of the wave's next 64 tiles, one a lane (a tile of 16-row pages
        // has two)
        int id0 = 0, id1 = 0;
        auto pages_from = [&](int kt) __attribute__((always_inline)) {
            const int key = (kt + PA_WAVES * lane) * ATT_KT;
            const int p0 = min(key >> lp, a.W - 1), p1 = min((key + 16) >> lp, a.W - 1);
            id0 = min(max(row_of[p0], 0), a.pages - 1);
            id1 = min(max(row_of[p1], 0), a.pages - 1);
        };
        // the tile's first and second 16 rows of the kv head, as row numbers
        auto rows_of = [&](int kt, int64_t &lo, int64_t &hi) __attribute__((always_inline)) {
            const int l = ((kt - t0) / PA_WAVES) & 63, key = kt * ATT_KT;
            const int64_t mask = head_rows - 1;
            lo = (((int64_t)__builtin_amdgcn_readlane(id0, l) * a.HK + hk) << lp) + (key & mask);
            hi = (((int64_t)__builtin_amdgcn_readlane(id1, l) * a.HK + hk) << lp) +
                 ((key + 16) & mask);
        };
        if (t0 < ntiles) {
            pages_from(t0);
            int64_t lo, hi;
            rows_of(t0, lo, hi);
            const int left = it.len - t0 * ATT_KT;
            dma_paged_tile<T, D, false>((const T *)a.k + lo * D, (const T *)a.k + hi * D, left, ks, lane);
            dma_paged_tile<T, D, true>((const T *)a.v + lo * D, (const T *)a.v + hi * D, left, vs, lane);
        }
        for (int kt = t0; kt < ntiles; kt += PA_WAVES) {  // wave-uniform
            const int nx = kt + PA_WAVES;
            const bool more = nx < ntiles;
            int64_t lo = 0, hi = 0;
            if (more) {
                if ((((nx - t0) / PA_WAVES) & 63) == 0) pages_from(nx);
                rows_of(nx, lo, hi);
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
                dma_paged_tile<T, D, false>((const T *)a.k + lo * D, (const T *)a.k + hi * D, left,
                                            ks, lane);
            f32x16 s = attn_scores<T, D>(kf, qf);
            const int k0 = kt * ATT_KT;
            if (k0 + ATT_KT > full) attn_mask(s, end - k0, h2);
            uint32_t p[8];
            attn_softmax<T, D>(st, s, p, a.scale);
            if (more)
                att_wait_vmcnt<Tl::NI>();
            else
                att_wait_vmcnt<0>();
            VFrag<T, D> vf;
            read_v<T, D>(vs, vf, lane);
            attn_pv<T, D>(st, p, vf);
            __builtin_amdgcn_sched_barrier(0);
            att_wait_lds();  // V's reads have returned
            if (more)
                dma_paged_tile<T, D, true>((const T *)a.v + lo * D, (const T *)a.v + hi * D, left,
                                           vs, lane);
        }
    };
    run(kslot, vslot);

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
    if (it.ns > 1) {  // (workgroup-uniform)
        const float l = f.l + __shfl_xor(f.l, 32, 64);
        float *o = a.part + ((int64_t)blockIdx.y * a.HK + hk) * PartState<D>::WORDS;
        if (!ok) return;
        float *oc = o + r * D + 32 * wave + 4 * h2;
#pragma unroll
        for (int j = 0; j < 4; ++j) *(float4 *)(oc + 8 * j) = f.o[j];
        if (wave == 0 && h2 == 0) *(float2 *)(o + 32 * D + 2 * r) = make_float2(l, f.m);
        return;
    }
    const float inv = row_inv(f.l);
    if (ok) store_fold<T>(f, inv, (T *)a.out + qrow * D, wave, h2);
#endif
}

// The chunks of four columns of a block: out = sum_s w_s O_s / sum_s w_s l_s
// with w_s = 2^(m_s - max m). A column takes D / 4 lanes of four values; the
// workgroup's groups of four columns take every so manyth chunk, in order, and
// the groups are added in order.
constexpr int COMBINE_COLS = 4;
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedArgs a) {
#pragma clang fp contract(off)
    constexpr int LANES = D / 4, GROUPS = 256 / (LANES * COMBINE_COLS), IN_FLIGHT = 4;
    __shared__ float4 acc[GROUPS][COMBINE_COLS][LANES];
    __shared__ float2 lm[GROUPS][COMBINE_COLS];
    const int hk = blockIdx.x;
    const PagedItem it = find_item<true>(a, blockIdx.y, threadIdx.x & 63);
    if (it.r < 0 || it.ns == 1) return;
    const int left = it.n * a.G - it.cb * 32;
    if ((int)blockIdx.z * COMBINE_COLS >= left) return;
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const int col = blockIdx.z * COMBINE_COLS + sub % COMBINE_COLS, g = sub / COMBINE_COLS;
    const bool ok = col < left;
    const float *base = a.part + ((int64_t)it.first * a.HK + hk) * PartState<D>::WORDS;
    const int64_t step = (int64_t)a.HK * PartState<D>::WORDS;
    const float *po = base + (ok ? col : 0) * D + 4 * lane;
    const float *pl = base + 32 * D + 2 * (ok ? col : 0);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f, m = -INFINITY;
    for (int s0 = g; s0 < it.ns; s0 += GROUPS * IN_FLIGHT) {
        float4 v[IN_FLIGHT];
        float2 w[IN_FLIGHT];
#pragma unroll
        for (int i = 0; i < IN_FLIGHT; ++i) {
            const int s = s0 + GROUPS * i;
            v[i] = *(const float4 *)(po + (s < it.ns ? s : g) * step);
            w[i] = *(const float2 *)(pl + (s < it.ns ? s : g) * step);
        }
#pragma unroll
        for (int i = 0; i < IN_FLIGHT; ++i) {
            if (s0 + GROUPS * i < it.ns) {
                const MergeCoef c = merge_coef(m, w[i].y);
                o.x = merge_one(o.x, v[i].x, c);
                o.y = merge_one(o.y, v[i].y, c);
                o.z = merge_one(o.z, v[i].z, c);
                o.w = merge_one(o.w, v[i].w, c);
                l = merge_one(l, w[i].x, c);
                m = c.m_new;
            }
        }
    }
    acc[g][sub % COMBINE_COLS][lane] = o;
    if (lane == 0) lm[g][sub % COMBINE_COLS] = make_float2(l, m);
    __syncthreads();
    if (g || !ok) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
        const float4 b = acc[i][sub][lane];
        const float2 w = lm[i][sub];
        const MergeCoef c = merge_coef(m, w.y);
        o.x = merge_one(o.x, b.x, c);
        o.y = merge_one(o.y, b.y, c);
        o.z = merge_one(o.z, b.z, c);
        o.w = merge_one(o.w, b.w, c);
        l = merge_one(l, w.x, c);
        m = c.m_new;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int idx = it.cb * 32 + col, tok = idx / a.G;
    T *orow = (T *)a.out + ((int64_t)(it.q0 + tok) * a.H + hk * a.G + (idx - tok * a.G)) * D;
    const float e[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    st8(orow + 4 * lane, pack4<T>(e));
}

// ---------------------------------------------------------------------------
// dispatch

// Workgroups of a launch. blocks: a bound on the column blocks (n G / 32 of a
// request, rounded up); a chunk is one run or more, so there are at most
// `target` chunks and the last, shorter one of every block, and no more than
// runs of the table's rows. Few blocks: as many chunks as one round of
// workgroups takes with those last ones; many: four rounds' worth, so that what
// the last round leaves idle is small.
struct PagedGrid {
    int64_t blocks, items, target;
    bool cut;
};
inline PagedGrid paged_grid(int64_t T, int64_t R, int64_t W, int64_t G, int64_t HK, int64_t D,
                            int64_t page) {
    PagedGrid g;
    g.blocks = T * G / 32 + (R < T ? R : T);
    const int64_t slots = D == 128 ? 512 : 1024;  // workgroups the chip holds
    const int64_t runs = ceil_div(W * page, CHUNK_KEYS);
    const int64_t few = slots - g.blocks * HK;
    g.target = (few >= slots / 2 ? few : 4 * slots) / HK;
    if (g.target < 1) g.target = 1;
    g.cut = runs > 1;
    g.items = g.cut ? g.blocks + g.target : g.blocks;
    if (g.items > g.blocks * runs) g.items = g.blocks * runs;
    return g;
}

template <typename T, int D>
int launch_paged(PagedArgs a, const PagedGrid &g, hipStream_t st) {
    paged_wave_kernel<T, D><<<dim3((unsigned)a.HK, (unsigned)(a.part ? g.items : g.blocks)),
                              64 * PA_WAVES, 0, st>>>(a);
    if (a.part) {
        const int64_t cols = (int64_t)a.T * a.G < 32 ? (int64_t)a.T * a.G : 32;
        paged_combine_kernel<T, D><<<dim3((unsigned)a.HK, (unsigned)g.blocks,
                                          (unsigned)ceil_div(cols, COMBINE_COLS)),
                                     256, 0, st>>>(a);
    }
    return launch_status("paged attention");
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
                                                      int64_t page_size) {
    if (T <= 0 || R <= 0 || table_width <= 0 || H <= 0 || HK <= 0 || H % HK ||
        (D != 64 && D != 128) || page_size <= 0)
        return 0;
    const PagedGrid g = paged_grid(T, R, table_width, H / HK, HK, D, page_size);
    return g.cut ? g.items * HK * 32 * (D + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int mi_paged_attention(const void *q, const void *k_pages, const void *v_pages,
                                  void *out, const int32_t *block_table, const int32_t *cu_q,
                                  const int32_t *kv_lens, int64_t T, int64_t R,
                                  int64_t table_width, int64_t H, int64_t HK, int64_t D,
                                  int64_t n_pages, int64_t page_size, float scale, int dtype,
                                  void *workspace, int64_t workspace_bytes, void *stream) {
    if (dtype != MI_BF16 && dtype != MI_F16)
        return fail(MI_ERR_UNSUPPORTED, "paged attention covers bf16 and fp16 (dtype code %d)", dtype);
    if (D != 64 && D != 128)
        return fail(MI_ERR_UNSUPPORTED, "paged attention head dim %lld", (long long)D);
    int lp;
    if (!page_log2_of(page_size, lp))
        return fail(MI_ERR_UNSUPPORTED, "page size %lld; this build covers 16, 32, 64, 128, 256",
                    (long long)page_size);
    if (T < 0 || R < 0 || H < 1 || HK < 1 || H % HK || HK > 65535 || table_width < 1 ||
        n_pages < 1 || n_pages > (0x7fffffff >> lp) || table_width > (0x3fffffff >> lp) ||
        T > 0x3fffffff || T * (H / HK) > 0x3fffffff || R > 0x3fffffff)
        return fail(MI_ERR_ARG, "paged attention shape T=%lld R=%lld table width %lld H=%lld HK=%lld "
                    "pages=%lld", (long long)T, (long long)R, (long long)table_width, (long long)H,
                    (long long)HK, (long long)n_pages);
    if (T == 0 || R == 0) return MI_OK;
    if (!q || !k_pages || !v_pages || !out || !block_table || !cu_q || !kv_lens)
        return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 8))
        return fail(MI_ERR_ARG, "q and the pages must be 16-byte aligned, out 8-byte aligned");
    const PagedGrid g = paged_grid(T, R, table_width, H / HK, HK, D, page_size);
    if (g.items > 65535 || g.blocks > 65535)
        return fail(MI_ERR_ARG, "paged attention: %lld column blocks (tokens x q heads of a kv head "
                    "/ 32, and requests), at most 65535", (long long)g.blocks);
    const int64_t need = g.cut ? g.items * HK * 32 * (D + 2) * (int64_t)sizeof(float) : 0;
    float *ws = need && workspace && workspace_bytes >= need && aligned(workspace, 16)
                    ? (float *)workspace : nullptr;
    const float sl = scale * 1.4426950408889634f;
    // (a scale of 0 as the smallest normal: masked scores stay -inf; NaN stays NaN)
    const float mag = fabsf(sl) < 1.17549435e-38f ? 1.17549435e-38f : fabsf(sl);
    const PagedArgs a = {q, k_pages, v_pages, out, block_table, cu_q, kv_lens, ws, (int)T, (int)R,
                         (int)table_width, (int)H, (int)HK, (int)(H / HK), (int)n_pages, lp,
                         (int)g.target, mag, sl < 0.0f ? 0x80008000u : 0u};
    hipStream_t st = as_stream(stream);
    if (dtype == MI_BF16)
        return D == 128 ? launch_paged<bf16, 128>(a, g, st) : launch_paged<bf16, 64>(a, g, st);
    return D == 128 ? launch_paged<f16, 128>(a, g, st) : launch_paged<f16, 64>(a, g, st);
}
