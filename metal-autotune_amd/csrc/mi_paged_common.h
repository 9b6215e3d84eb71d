// Device helpers shared by the attention kernels over a paged cache (mi_paged_attn.hip,
// mi_shared_attn.hip): pages of key tiles, their DMA, the softmax of a wide block's two
// tiles, LDS sizes.
#pragma once

#include "mi_attn_common.h"

namespace mi {
namespace {

constexpr int PA_WAVES = ATT_STREAMS;
constexpr int CHUNK_KEYS = ATT_KT * PA_WAVES;  // keys are cut in multiples of this
constexpr int MAX_CHUNKS = 128;  // of a block: one workgroup adds them
constexpr int WIDE_COLS = 128;

#if defined(__HIP_DEVICE_COMPILE__)
// The DMA of one key tile of K or V: rows [0, left) of it (at most 32) lie at
// lo (rows 0..15) and hi (rows 16..31, its own 16 rows); the rest arrive as zeros.
// NT: non-temporal, for what is read once (decode: 48 requests of 64 to 8191 keys
// 152 -> 136 us; wide blocks, which share keys through the L2, 97 -> 105 with it).
// SCALAR: `left` clamped in scalar registers; else it is vector work, and each of the first
// rows' loads a loop over lanes (96 requests behind 16256 keys 125 -> 120 us; but decode
// with heads of 64, which four waves a SIMD leave 128 registers, would spill).
template <typename T, int D, bool ISV, bool NT, bool SCALAR = false>
__device__ __forceinline__ void dma_paged_tile(const T *lo, const T *hi, int left, char *dst,
                                               int lane) {
    typedef Tile<D> Tl;
    int n0 = left < 0 ? 0 : (left < 16 ? left : 16);
    int n1 = left < 16 ? 0 : (left < 32 ? left - 16 : 16);
    if constexpr (SCALAR) {
        n0 = __builtin_amdgcn_readfirstlane(n0);
        n1 = __builtin_amdgcn_readfirstlane(n1);
    }
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

// The pages of a wave's next 64 tiles kt, kt + STEP, ..., one a lane (a tile of
// 16-row pages has two), and a tile's first and second 16 rows of the kv head in
// the pools.
template <int STEP> struct TilePages {
    const int *row;
    int64_t hk;
    int W, pages, lp, HK;
    int id0, id1;
    template <typename Args>
    __device__ __forceinline__ TilePages(const Args &a, int r, int hk_)
        : row(a.table + (int64_t)r * a.W), hk(hk_), W(a.W), pages(a.pages), lp(a.page_log2),
          HK(a.HK), id0(0), id1(0) {}
    // (from: the key that tile 0 begins with, a multiple of 16)
    __device__ __forceinline__ void load(int kt, int lane, int from = 0) {
        const int key = from + (kt + STEP * lane) * ATT_KT;
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
#endif

// attn_softmax over two key tiles.
template <typename T, int D, bool REST = false>
__device__ __forceinline__ void softmax_pair(AttnState<D> &st, const f32x16 (&s)[2],
                                             uint32_t (&pk)[2][8], float scale,
                                             uint32_t (*rest)[8] = nullptr) {
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
            if constexpr (REST) rest[j][i] = rest2<T>(p0, p1, pk[j][i]);
            sum[2 * (i & 1)] += p0;
            sum[2 * (i & 1) + 1] += p1;
        }
    st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <int D> struct PagedLds {
    static constexpr int SLOTS = PA_WAVES * 2 * Tile<D>::BYTES;  // = two wide stages
    static constexpr int FOLD = PA_WAVES * Part<D>::BYTES;
    static constexpr int BYTES = SLOTS > FOLD ? SLOTS : FOLD;
};

inline bool page_log2_of(int64_t page, int &lp) {
    for (lp = 4; lp <= 8; ++lp)
        if (page == (1 << lp)) return true;
    return false;
}

}  // namespace
}  // namespace mi
