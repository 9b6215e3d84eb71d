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
#include "mi_attn_common.h"

namespace mi {
namespace {

constexpr int PA_WAVES = ATT_STREAMS;

// The work of one workgroup beside its kv head.
struct PagedItem {
    int r;       // request, < 0: none
    int q0, n;   // its first token, its tokens
    int len;     // its keys
    int cb;      // column block
};

struct PagedArgs {
    const void *q, *k, *v;
    void *out;
    const int *table, *cu_q, *kv_lens;
    int T, R, W, H, HK, G, pages, page_log2;
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

// Item u of the column blocks of all requests in order; every wave finds it by
// itself, 64 requests a step.
__device__ __forceinline__ PagedItem find_item(const PagedArgs &a, int u, int lane) {
    int before = 0;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
        const int r = r0 + lane;
        const bool in = r < a.R;
        // (offsets held to the rows that there are)
        const int c0 = in ? min(max(a.cu_q[r], 0), a.T) : 0;
        const int c1 = in ? min(max(a.cu_q[r + 1], c0), a.T) : 0;
        const int len = in ? min(max(a.kv_lens[r], 0), a.W << a.page_log2) : 0;
        const int blocks = ((c1 - c0) * a.G + 31) >> 5;
        const int end = before + wave_scan(blocks);
        const uint64_t mine = __builtin_amdgcn_ballot_w64(end > u);
        if (mine) {
            const int l = __builtin_ctzll(mine);
            const int q0 = __builtin_amdgcn_readlane(c0, l);
            return {r0 + l, q0, __builtin_amdgcn_readlane(c1, l) - q0,
                    __builtin_amdgcn_readlane(len, l),
                    u - __builtin_amdgcn_readlane(end - blocks, l)};
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return {-1, 0, 0, 0, 0};
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
    const PagedItem it = find_item(a, blockIdx.y, lane);
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
    const int ntiles = last > 0 ? (last + ATT_KT - 1) / ATT_KT : 0;
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
            const int l = ((kt - wave) / PA_WAVES) & 63, key = kt * ATT_KT;
            const int64_t mask = head_rows - 1;
            lo = (((int64_t)__builtin_amdgcn_readlane(id0, l) * a.HK + hk) << lp) + (key & mask);
            hi = (((int64_t)__builtin_amdgcn_readlane(id1, l) * a.HK + hk) << lp) +
                 ((key + 16) & mask);
        };
        if (wave < ntiles) {
            pages_from(wave);
            int64_t lo, hi;
            rows_of(wave, lo, hi);
            const int left = it.len - wave * ATT_KT;
            dma_paged_tile<T, D, false>((const T *)a.k + lo * D, (const T *)a.k + hi * D, left, ks, lane);
            dma_paged_tile<T, D, true>((const T *)a.v + lo * D, (const T *)a.v + hi * D, left, vs, lane);
        }
        for (int kt = wave; kt < ntiles; kt += PA_WAVES) {  // wave-uniform
            const int nx = kt + PA_WAVES;
            const bool more = nx < ntiles;
            int64_t lo = 0, hi = 0;
            if (more) {
                if ((((nx - wave) / PA_WAVES) & 63) == 0) pages_from(nx);
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
    const float inv = row_inv(f.l);
    if (ok) store_fold<T>(f, inv, (T *)a.out + qrow * D, wave, h2);
#endif
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_paged_attention(const void *q, const void *k_pages, const void *v_pages,
                                  void *out, const int32_t *block_table, const int32_t *cu_q,
                                  const int32_t *kv_lens, int64_t T, int64_t R,
                                  int64_t table_width, int64_t H, int64_t HK, int64_t D,
                                  int64_t n_pages, int64_t page_size, float scale, int dtype,
                                  void *stream) {
    if (dtype != MI_BF16 && dtype != MI_F16)
        return fail(MI_ERR_UNSUPPORTED, "paged attention covers bf16 and fp16 (dtype code %d)", dtype);
    if (D != 64 && D != 128)
        return fail(MI_ERR_UNSUPPORTED, "paged attention head dim %lld", (long long)D);
    int lp = -1;
    for (int l = 4; l <= 8; ++l)
        if (page_size == (1 << l)) lp = l;
    if (lp < 0)
        return fail(MI_ERR_UNSUPPORTED, "page size %lld; this build covers 16, 32, 64, 128, 256",
                    (long long)page_size);
    if (T < 0 || R < 0 || H < 1 || HK < 1 || H % HK || HK > 65535 || table_width < 1 ||
        n_pages < 1 || n_pages > (0x7fffffff >> lp) || table_width > (0x3fffffff >> lp) ||
        T * (H / HK) > 0x3fffffff || R > 0x3fffffff)
        return fail(MI_ERR_ARG, "paged attention shape T=%lld R=%lld table width %lld H=%lld HK=%lld "
                    "pages=%lld", (long long)T, (long long)R, (long long)table_width, (long long)H,
                    (long long)HK, (long long)n_pages);
    if (T == 0 || R == 0) return MI_OK;
    if (!q || !k_pages || !v_pages || !out || !block_table || !cu_q || !kv_lens)
        return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(q, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 8))
        return fail(MI_ERR_ARG, "q and the pages must be 16-byte aligned, out 8-byte aligned");
    const int64_t G = H / HK;
    const int64_t items = T * G / 32 + (R < T ? R : T);  // a bound on the column blocks
    if (items > 65535)
        return fail(MI_ERR_ARG, "paged attention: %lld column blocks", (long long)items);
    const float sl = scale * 1.4426950408889634f;
    // (a scale of 0 as the smallest normal: masked scores stay -inf; NaN stays NaN)
    const float mag = fabsf(sl) < 1.17549435e-38f ? 1.17549435e-38f : fabsf(sl);
    const PagedArgs a = {q, k_pages, v_pages, out, block_table, cu_q, kv_lens, (int)T, (int)R,
                         (int)table_width, (int)H, (int)HK, (int)G, (int)n_pages, lp, mag,
                         sl < 0.0f ? 0x80008000u : 0u};
    hipStream_t st = as_stream(stream);
    const dim3 grid((unsigned)HK, (unsigned)items);
    if (dtype == MI_BF16) {
        if (D == 128)
            paged_wave_kernel<bf16, 128><<<grid, 64 * PA_WAVES, 0, st>>>(a);
        else
            paged_wave_kernel<bf16, 64><<<grid, 64 * PA_WAVES, 0, st>>>(a);
    } else {
        if (D == 128)
            paged_wave_kernel<f16, 128><<<grid, 64 * PA_WAVES, 0, st>>>(a);
        else
            paged_wave_kernel<f16, 64><<<grid, 64 * PA_WAVES, 0, st>>>(a);
    }
    return launch_status("paged attention");
}
