// Device helpers shared by the attention kernels (mi_attn.hip: contiguous caches,
// mi_paged_attn.hip: paged ones): the 32-key tile, its LDS layout and swizzles,
// the online softmax of a wave, and the folding of partial states.
#pragma once

#include <math.h>

#include "mi_common.h"

namespace mi {
namespace {

template <typename T> struct AMfma;
template <> struct AMfma<bf16> {
    static __device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct AMfma<f16> {
    static __device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

constexpr int ATT_KT = 32;       // keys per tile
constexpr int ATT_STREAMS = 4;   // key-tile streams per query row

// Online-softmax state of one wave: O^T tiles (lane = query column r, half
// h2), the row's reference maximum m (log2 units) and this lane's half of the
// row sum l.
template <int D> struct AttnState {
    f32x16 o[D / 32];
    float m, l;
};

template <int D> __device__ __forceinline__ void attn_init(AttnState<D> &st) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[t][i] = 0.0f;
    st.m = -INFINITY;
    st.l = 0.0f;
}

// The larger of a lane's value and that of the lane 32 away, in both. (The pair's
// members are copied out first: a bit cast of a vector's subscript reads its first
// element, whatever the subscript.)
__device__ __forceinline__ float max_halves(float v) {
    typedef unsigned U2 __attribute__((ext_vector_type(2)));
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const U2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned lo = r[0], hi = r[1];
    return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

// Scores of keys from `vis` on (of the tile's 32) set to -inf.
__device__ __forceinline__ void attn_mask(f32x16 &s, int vis, int h2) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
        s[i] = 8 * (i / 4) + 4 * h2 + (i % 4) < vis ? s[i] : -INFINITY;
}

// What rounding to T took from two values, in T.
template <typename T> __device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t pk) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    const T2 v = __builtin_bit_cast(T2, pk);
    return pk2<T>(a - (float)v[0], b - (float)v[1]);
}

// Scores to probabilities of one key tile: s[i] = S^T (key 8*(i/4) + 4*h2 +
// i%4 of the tile, the lane's query row; -inf where the row does not see the
// key), pk gets 2^(s scale - m) in pairs of T, in register order. The row sum
// adds the fp32 values, in four chains (rounded to T first, the denominator
// would carry T's error of a probability, up to 2^-9 in bf16). The pairs are
// operands of the second product's MFMAs, hence in T: of a result's norm that rounding
// costs about what the result's own does (300 rows over 1000 keys 2.2e-3 in bf16, where
// 1.7e-3 is the least that bf16 can hold). REST: rest gets what it took, for a
// product of its own. scale > 0 (a negative scale was moved into Q's sign).
template <typename T, int D, bool REST = false>
__device__ __forceinline__ void attn_softmax(AttnState<D> &st, const f32x16 &s, uint32_t (&pk)[8],
                                             float scale, uint32_t *rest = nullptr) {
#pragma clang fp contract(off)
    float mt = fmaxf(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) mt = fmaxf(fmaxf(mt, s[i]), s[i + 1]);
    mt = max_halves(mt) * scale;
    // Lazy rescale: the exponents are taken against a running reference m
    // that moves only when a row's maximum passes it by more than 8 (log2
    // units). p then stays below 2^8, where fp32 sums and the bf16/fp16 P
    // operand keep their relative precision, and the accumulator rescales run
    // only on those (wave-uniform) steps.
    const bool grow = mt > st.m + 8.0f;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float m_new = grow ? mt : st.m;
        const float corr = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m - m_new);
        st.l *= corr;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) st.o[t][i] *= corr;
        st.m = m_new;
    }
    // (a row that has seen no key yet: every score is -inf, and p is 0)
    const float nm = st.m == -INFINITY ? 0.0f : -st.m;
    float sum[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i], scale, nm));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + 1], scale, nm));
        pk[i] = pk2<T>(p0, p1);
        if constexpr (REST) rest[i] = rest2<T>(p0, p1, pk[i]);
        float &a = sum[2 * (i & 1)], &b = sum[2 * (i & 1) + 1];
        a = i < 2 ? p0 : a + p0;
        b = i < 2 ? p1 : b + p1;
    }
    st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Swizzles of a staged tile: 16-byte chunk c of key row r sits at chunk
// position c ^ swz(r). K: the 32 rows' ds_read_b128 of one chunk spread over
// the banks. V: the four rows one transposing read covers (64 bytes of each)
// take four distinct 64-byte windows.
template <int D> __device__ __forceinline__ int swz_k(int r) {
    return D == 128 ? (r & 15) : ((r >> 1) & 7);
}
template <int D> __device__ __forceinline__ int swz_v(int r) {
    return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
}

template <int D> struct Tile {
    static constexpr int BYTES = ATT_KT * D * 2;      // a K or V tile in LDS
    static constexpr int CPR = D / 8;                 // 16-byte chunks per row
    static constexpr int RPI = 64 / CPR;              // rows per DMA instruction
    static constexpr int NI = ATT_KT / RPI;           // DMA instructions per tile
};

typedef __attribute__((address_space(3))) void *lds_ptr;

// Division of a block or unit index by a launch constant: a multiply by
// ceil(2^32 / d), exact for n d < 2^32 (the host checks the largest n; else m =
// 0 and the quotient is computed), where a division costs a workgroup tens of
// dependent scalar instructions before its first load.
struct Div {
    unsigned d, m;
    __device__ __forceinline__ unsigned of(unsigned n) const {
        if (d == 1) return n;
        return m ? __umulhi(n, m) : n / d;
    }
};
inline Div make_div(int64_t d, int64_t n_max) {
    const bool exact = d > 1 && n_max * d < ((int64_t)1 << 32);
    return {(unsigned)d, exact ? (unsigned)((((uint64_t)1 << 32) + d - 1) / d) : 0u};
}

#if defined(__HIP_DEVICE_COMPILE__)
// A raw buffer resource over [base, base + bytes): reads past the end return
// zero instead of touching memory.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t att_rsrc(const void *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes,
                                             0x00020000);
}

// DMA instructions [i0, i0 + n) of key tile kt of one kv head's K or V (base:
// its row 0) into the tile's LDS. Rows past Lk, whole tiles too, arrive as
// zeros without a memory access (the resource ends at row Lk).
template <typename T, int D, bool ISV>
__device__ __forceinline__ void dma_tile(const T *base, int64_t kt, int64_t Lk, char *dst, int i0,
                                         int n, int lane) {
    typedef Tile<D> Tl;
    const int64_t left = Lk - kt * ATT_KT;
    const int rows = left < 0 ? 0 : (left < ATT_KT ? (int)left : ATT_KT);
    const __amdgpu_buffer_rsrc_t rs =
        att_rsrc(base + (rows ? kt * ATT_KT * D : 0), (uint32_t)(rows * D * 2));
#pragma unroll
    for (int i = 0; i < n; ++i) {
        const int row = (i0 + i) * Tl::RPI + lane / Tl::CPR, pos = lane % Tl::CPR;
        const int c = pos ^ (ISV ? swz_v<D>(row) : swz_k<D>(row));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(dst + (i0 + i) * 1024), 16,
                                                 (row * D + 8 * c) * 2, 0, 0, 0);
    }
}
#endif

// s_waitcnt with vmcnt = N and no wait on the other counters.
template <int N> __device__ __forceinline__ void att_wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt is a 6-bit count");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
// s_waitcnt lgkmcnt(0) alone.
__device__ __forceinline__ void att_wait_lds() {
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));
}

// K fragments of the lane: row r, head-dim chunk 16 s + 8 h2 of MFMA step s.
template <int D>
__device__ __forceinline__ void read_k(const char *ks, uint4 (&kf)[D / 16], int r, int h2) {
    const int a = r * (D * 2) + ((h2 ^ swz_k<D>(r)) << 4);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) kf[s] = *(const uint4 *)(ks + (a ^ (s << 5)));
}

template <typename T, int D>
__device__ __forceinline__ f32x16 attn_scores(const uint4 (&kf)[D / 16], const uint4 (&qf)[D / 16]) {
    typedef typename Vec<T>::x8 V8;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
        s = AMfma<T>::mma(__builtin_bit_cast(V8, kf[ks]), __builtin_bit_cast(V8, qf[ks]), s);
    return s;
}

// Four 16-bit values by ds_read_b64_tr_b16. Within each 16-lane group, with
// lane s addressing four consecutive values E[s][0..3], lane 4a + b receives
// (E[a][b], E[a + 4][b], E[a + 8][b], E[a + 12][b]) (probed on gfx950: LDS
// filled with each value's index, lanes addressing rows of 4 and of 16).
template <typename T>
__device__ __forceinline__ typename Vec<T>::x4 lds_read_tr4(const char *p) {
    typedef short S4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) S4 *LP;
    return __builtin_bit_cast(typename Vec<T>::x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LP)p));
}

// O^T += V^T . P^T over one tile, in two steps: read_v fetches the A fragments
// (before the softmax, whose arithmetic then covers the LDS latency: read at
// their MFMAs, each pair of reads was waited for in turn), attn_pv runs the
// MFMAs. The fragment of lane (r, h2), MFMA k2 of head-dim tile t, is
// V^T[32 t + r][keys 16 k2 + 4 h2 + (0..3), then the same + 8]. Lane s of
// 16-lane group G addresses key row 16 k2 + 4 (G / 2) + s / 4 at column 32 t +
// 16 (G % 2) + 4 (s % 4); by the rule above lane 4a + b of the group (r = 16
// (G % 2) + 4a + b) then receives column 32 t + r of the key rows 16 k2 + 4 h2
// + 0..3.
template <typename T, int D> struct VFrag {
    typename Vec<T>::x4 v[D / 32][2][2];
};
template <typename T, int D>
__device__ __forceinline__ void read_v(const char *vs, VFrag<T, D> &f, int lane) {
    const int s = lane & 15, g = lane >> 4;
    const int row = 4 * (g >> 1) + (s >> 2);  // + 16 k2 (+ 8): the same swizzle
    const int low = ((2 * (g & 1) + ((s & 3) >> 1)) << 4) + 8 * (s & 1);
    const int a0 = row * (D * 2) + low, z = swz_v<D>(row) << 4;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
        const char *vr = vs + a0 + ((t << 6) ^ z);
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
            f.v[t][k2][0] = lds_read_tr4<T>(vr + (16 * k2) * (D * 2));
            f.v[t][k2][1] = lds_read_tr4<T>(vr + (16 * k2 + 8) * (D * 2));
        }
    }
}
template <typename T, int D>
__device__ __forceinline__ void attn_pv(AttnState<D> &st, const uint32_t (&pk)[8],
                                        const VFrag<T, D> &f) {
    typedef typename Vec<T>::x8 V8;
    const V8 pb[2] = {__builtin_bit_cast(V8, (uint4){pk[0], pk[1], pk[2], pk[3]}),
                      __builtin_bit_cast(V8, (uint4){pk[4], pk[5], pk[6], pk[7]})};
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int t = 0; t < D / 32; ++t) {
            V8 a;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = f.v[t][k2][0][e];
                a[4 + e] = f.v[t][k2][1][e];
            }
            st.o[t] = AMfma<T>::mma(a, pb[k2], st.o[t]);
        }
}

// Folding a later state (mw, lw, o_w) into an earlier (m, l, o):
// m' = max(m, mw); o' = o c0 + o_w cw and l' = l c0 + lw cw with
// c0 = 2^(m - m'), cw = 2^(mw - m'); a state that saw no visible key of the
// row (m = -inf) has coefficient 0.
struct MergeCoef {
    float c0, cw, m_new;
};
__device__ __forceinline__ MergeCoef merge_coef(float m, float mw) {
#pragma clang fp contract(off)
    const float m_new = fmaxf(m, mw);
    return {m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - m_new),
            mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - m_new), m_new};
}
__device__ __forceinline__ float merge_one(float o, float ow, const MergeCoef &c) {
#pragma clang fp contract(off)
    return __builtin_fmaf(o, c.c0, ow * c.cw);
}

// 1 / the row's sum (both halves), 0 for a row that saw no key.
__device__ __forceinline__ float row_inv(float l) {
#pragma clang fp contract(off)
    const float l_tot = l + __shfl_xor(l, 32, 64);
    return l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
}

// The Q fragments of a row.
template <int D>
__device__ __forceinline__ void read_q(const void *row, int h2, uint4 (&qf)[D / 16]) {
    const char *qp = (const char *)row + 16 * h2;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = ld16(qp + 32 * s);
}
// The sign of a negative scale moved into them (exact), once: called where they
// have landed, so that the loads in flight behind them are not waited for.
template <int D> __device__ __forceinline__ void flip_q(uint4 (&qf)[D / 16], uint32_t &flip) {
    if (flip == 0) return;  // (uniform)
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
        qf[s].x ^= flip, qf[s].y ^= flip, qf[s].z ^= flip, qf[s].w ^= flip;
    flip = 0;
}

// A wave's state in LDS for the last fold: float4 [D / 32 * 4][64] (registers
// 4j .. 4j + 3 of tile t at t * 4 + j), then float2 (l, m) [64].
template <int D> struct Part {
    static constexpr int WORDS = D / 32 * 4 * 64 + 32;  // 16-byte words
    static constexpr int BYTES = WORDS * 16;
};
template <int D>
__device__ __forceinline__ void part_put(float4 *pp, const AttnState<D> &st, int t, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        pp[(t * 4 + j) * 64 + lane] = make_float4(st.o[t][4 * j], st.o[t][4 * j + 1],
                                                  st.o[t][4 * j + 2], st.o[t][4 * j + 3]);
}
template <int D> __device__ __forceinline__ float2 *part_lm(float4 *pp) {
    return (float2 *)(pp + D / 32 * 4 * 64);
}
struct Fold {  // one O^T tile of a state
    float4 o[4];
    float l, m;
};
__device__ __forceinline__ void fold(Fold &a, const Fold &b) {
    const MergeCoef c = merge_coef(a.m, b.m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        a.o[j].x = merge_one(a.o[j].x, b.o[j].x, c);
        a.o[j].y = merge_one(a.o[j].y, b.o[j].y, c);
        a.o[j].z = merge_one(a.o[j].z, b.o[j].z, c);
        a.o[j].w = merge_one(a.o[j].w, b.o[j].w, c);
    }
    a.l = merge_one(a.l, b.l, c);
    a.m = c.m_new;
}
template <int D>
__device__ __forceinline__ Fold part_get(float4 *pp, int t, int lane) {
    Fold f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.o[j] = pp[(t * 4 + j) * 64 + lane];
    const float2 lm = part_lm<D>(pp)[lane];
    f.l = lm.x;
    f.m = lm.y;
    return f;
}

// O^T tile t of the four streams' states at part, folded (0 + 1) + (2 + 3).
template <int D> __device__ __forceinline__ Fold fold_streams(float4 *part, int t, int lane) {
    Fold f = part_get<D>(part, t, lane);
    fold(f, part_get<D>(part + Part<D>::WORDS, t, lane));
    Fold g = part_get<D>(part + 2 * Part<D>::WORDS, t, lane);
    fold(g, part_get<D>(part + 3 * Part<D>::WORDS, t, lane));
    fold(f, g);
    return f;
}
template <typename T>
__device__ __forceinline__ void store_fold(const Fold &f, float inv, T *orow, int t, int h2) {
#pragma clang fp contract(off)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float e[4] = {f.o[j].x * inv, f.o[j].y * inv, f.o[j].z * inv, f.o[j].w * inv};
        st8(orow + 32 * t + 8 * j + 4 * h2, pack4<T>(e));
    }
}

}  // namespace
}  // namespace mi
