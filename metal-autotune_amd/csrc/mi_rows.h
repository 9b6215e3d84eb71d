// Device helpers shared by the kernels that read rows of logits (mi_logprob.hip,
// mi_beam.hip): a row in 16-byte pieces and chunks of 1024 values, reductions of a
// wave, and the k largest values of a row from the maxima of its chunks.
//
// The k largest values need no list during the pass over a row, only the maximum of
// every chunk: ordered by (value descending, index ascending) they lie in the k chunks
// whose maxima come first in that order, since a value outside these has k maxima before
// it. So the pass leaves the maxima; rank_chunks ranks them, and top_of reads the k best
// chunks again and keeps what reaches the k-th maximum (as good as k values in all, but
// for ties) in a list, a lane an entry.
#pragma once

#include <math.h>

#include "mi_common.h"

namespace mi {
namespace {

constexpr int LP_MAX_TOP = 64;   // a lane an entry
constexpr int LP_WAVES = 4, LP_SPLIT_WAVES = 8;  // of a workgroup that has a row, a part of one
constexpr int LP_CHUNK = 1024;   // values a chunk, 2 (16 bits) or 4 (fp32) 16-byte pieces a lane
constexpr int64_t LP_MAX_V = (int64_t)1 << 20;
// (the first may begin before the row)
constexpr int LP_MAX_CHUNKS = (int)(LP_MAX_V / LP_CHUNK) + 1;
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;

// A 16-byte piece of a row as floats.
template <typename T> struct Piece {
    static constexpr int N = 16 / (int)sizeof(T);
    float f[N];
};
template <typename T> __device__ __forceinline__ Piece<T> open_piece(uint4 raw) {
    Piece<T> p;
    if constexpr (sizeof(T) == 2) {
        unpack8<T>(raw, p.f);
    } else {
        p.f[0] = __builtin_bit_cast(float, raw.x);
        p.f[1] = __builtin_bit_cast(float, raw.y);
        p.f[2] = __builtin_bit_cast(float, raw.z);
        p.f[3] = __builtin_bit_cast(float, raw.w);
    }
    return p;
}

__device__ __forceinline__ float readlane_f(float v, int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
// Over a wave, by DPP moves within its rows of 16 and their lane 0 (no trip
// through the LDS unit).
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));
    v = fmaxf(v, dpp_f32<0x4E>(v));
    v = fmaxf(v, dpp_f32<0x141>(v));
    v = fmaxf(v, dpp_f32<0x140>(v));
    return fmaxf(fmaxf(readlane_f(v, 0), readlane_f(v, 16)),
                 fmaxf(readlane_f(v, 32), readlane_f(v, 48)));
}
__device__ __forceinline__ float wave_add(float v) {
    v = row16_sum(v);
    return (readlane_f(v, 0) + readlane_f(v, 16)) + (readlane_f(v, 32) + readlane_f(v, 48));
}
// The same in 64 bits, two moves a value.
template <int CTRL> __device__ __forceinline__ double dpp_f64(double v) {
    const uint2 b = __builtin_bit_cast(uint2, v);
    const uint2 m = {(unsigned)__builtin_amdgcn_update_dpp(0, (int)b.x, CTRL, 0xF, 0xF, false),
                     (unsigned)__builtin_amdgcn_update_dpp(0, (int)b.y, CTRL, 0xF, 0xF, false)};
    return __builtin_bit_cast(double, m);
}
__device__ __forceinline__ double readlane_d(double v, int l) {
    const uint2 b = __builtin_bit_cast(uint2, v);
    const uint2 m = {(unsigned)__builtin_amdgcn_readlane((int)b.x, l),
                     (unsigned)__builtin_amdgcn_readlane((int)b.y, l)};
    return __builtin_bit_cast(double, m);
}
__device__ __forceinline__ double wave_add(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    v += dpp_f64<0x140>(v);
    return (readlane_d(v, 0) + readlane_d(v, 16)) + (readlane_d(v, 32) + readlane_d(v, 48));
}

// What a wave sums is in units of log2: t = x log2 e - C with C = rint(ref log2 e) an
// integer, p = 2^t, S = sum p, E = sum p t: one fma a value, rounded as finely as t
// is small, and a step from one C to another scales by a power of two. From 2^23 on
// no rounding to an integer is left in fp32 and C misses ref log2 e by more than 1/2,
// past 2e9 by more than 2^t can take (a mask of -1e10). References beyond 2^20 (such
// masks; -FLT_MAX before the first value) take t = (x - ref) log2 e instead.
__device__ __forceinline__ bool far(float ref) { return !(fabsf(ref) <= 1048576.0f); }
__device__ __forceinline__ float units(float ref) { return __builtin_rintf(ref * LP_LOG2E); }
// By how much the sums' zero lies above ref log2 e.
__device__ __forceinline__ float excess(float ref) {
    return far(ref) ? 0.0f : __builtin_fmaf(-ref, LP_LOG2E, units(ref));
}

// The order of floats as the order of ints (-0 as 0); what is no value is NONE.
constexpr int NONE = (int)0x80000000;
__device__ __forceinline__ int key_of(float x) {
    const int b = __builtin_bit_cast(int, x + 0.0f);
    return x != x ? NONE : b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float of_key(int k) {
    return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff));
}

// A wave's list: lane i < k holds the i-th best (key, index).
struct TopList {
    int key, id;
    int last_key, last_id;  // what a value has to come before (uniform)
    float floor;            // a value that it has to reach
};
__device__ __forceinline__ bool before(int ka, int ia, int kb, int ib) {
    return ka > kb || (ka == kb && ia < ib);
}
__device__ __forceinline__ void top_insert(TopList &l, int key, int id, int k, int lane) {
    const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before(l.key, l.id, key, id)));
    const int pk = __shfl_up(l.key, 1, 64), pi = __shfl_up(l.id, 1, 64);
    l.key = lane < at ? l.key : (lane == at ? key : pk);
    l.id = lane < at ? l.id : (lane == at ? id : pi);
    const int lk = __builtin_amdgcn_readlane(l.key, k - 1);
    if (lk != NONE) {
        l.last_key = lk;
        l.last_id = __builtin_amdgcn_readlane(l.id, k - 1);
        l.floor = of_key(lk);
    }
}

// 16 bytes at any address.
struct __attribute__((packed, aligned(2))) Bytes16 {
    unsigned v[4];
};
__device__ __forceinline__ uint4 ld16_any(const void *p) {
    const Bytes16 b = *(const Bytes16 *)p;
    return make_uint4(b.v[0], b.v[1], b.v[2], b.v[3]);
}
__device__ __forceinline__ uint4 ld16_any_nt(const void *p) {
    typedef unsigned U4 __attribute__((ext_vector_type(4), aligned(2)));
    const U4 v = __builtin_nontemporal_load((const U4 *)p);
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// A row as 16-byte pieces from the one that holds its first value; value i of
// piece p is row element p N + i - skew. What lies outside the row reads as -inf.
// ANY: pieces from the first value on, at whatever address, so that a row's parts
// (and the order of its sums) are the same wherever it lies.
template <typename T, bool ANY = false> struct Row {
    static constexpr int N = Piece<T>::N, PER = LP_CHUNK / (64 * N);  // pieces a lane and chunk
    const T *x;
    const char *base;
    int skew, V;
    __device__ __forceinline__ Row(const T *x_, int V_) : x(x_), V(V_) {
        skew = ANY ? 0 : (int)(((uintptr_t)x & 15) / sizeof(T));
        base = (const char *)x - skew * (int)sizeof(T);
    }
    __device__ __forceinline__ int chunks() const { return (V + skew + LP_CHUNK - 1) / LP_CHUNK; }
    __device__ __forceinline__ int first(int chunk, int i, int lane) const {
        return chunk * LP_CHUNK + (64 * i + lane) * N - skew;
    }
    // whether every value of the chunk's pieces is the row's
    __device__ __forceinline__ bool whole(int chunk) const {
        return (chunk > 0 || skew == 0) && (chunk + 1) * LP_CHUNK - skew <= V;
    }
    // a whole chunk; NT: a row read once, past the caches
    template <bool NT>
    __device__ __forceinline__ void load(int chunk, int lane, uint4 (&raw)[PER]) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const char *at =
                base + ((int64_t)chunk * LP_CHUNK + (64 * i + lane) * N) * (int)sizeof(T);
            raw[i] = ANY ? (NT ? ld16_any_nt(at) : ld16_any(at)) : NT ? ld16_nt(at) : ld16(at);
        }
    }
    __device__ __forceinline__ void open(const uint4 (&raw)[PER], Piece<T> (&pc)[PER]) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) pc[i] = open_piece<T>(raw[i]);
    }
    // the row's ends: the pieces within it as 16 bytes, the one across an end value by
    // value (all of these loads in flight together)
    __device__ __forceinline__ void get_end(int chunk, int lane, Piece<T> (&pc)[PER]) const {
        uint4 raw[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int f = first(chunk, i, lane);
            const char *at = base + (int64_t)(f + skew) * (int)sizeof(T);
            if (f >= 0 && f + N <= V) raw[i] = ANY ? ld16_any(at) : ld16(at);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int f = first(chunk, i, lane);
            if (f >= 0 && f + N <= V) {
                pc[i] = open_piece<T>(raw[i]);
                continue;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) pc[i].f[e] = -INFINITY;
            if (f + N > 0 && f < V) {
                T v[N];
#pragma unroll
                for (int e = 0; e < N; ++e) v[e] = x[min(max(f + e, 0), V - 1)];
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (f + e >= 0 && f + e < V) pc[i].f[e] = (float)v[e];
            }
        }
    }
};

// By a workgroup of WAVES, from the keys of a row's chunks' maxima in LDS.
template <int WAVES> struct TopLds {
    int rank[LP_MAX_CHUNKS], sel[LP_MAX_TOP];
    int key[WAVES * LP_MAX_TOP], id[WAVES * LP_MAX_TOP];
    int bkey[LP_MAX_TOP], bid[LP_MAX_TOP];
    int count[WAVES];
    int floor;
};
template <int WAVES>
__device__ __forceinline__ void rank_chunks(const int *maxima, int nc, int k, TopLds<WAVES> *t) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int need = k < nc ? k : nc;
    // the chunks' ranks: a wave compares every chunk, a lane each, with eight
    // others at a time (maxima: padded by NONE to a multiple of 8; rank: zero)
    for (int i = 8 * wave; i < nc; i += 8 * WAVES) {
        const int4 u = *(const int4 *)(maxima + i), v = *(const int4 *)(maxima + i + 4);
        const int e[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        for (int c = lane; c < nc; c += 64) {
            const int key = maxima[c];
            int rank = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) rank += before(e[j], i + j, key, c);
            atomicAdd(&t->rank[c], rank);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < nc; c += 64 * WAVES) {
        const int rank = t->rank[c];
        if (rank < need) t->sel[rank] = c;
        if (rank == need - 1) t->floor = need == k ? maxima[c] : NONE + 1;
    }
}
// The k best (key, index) into t->bkey, t->bid (key NONE, index 0 where there are fewer);
// a barrier lies between rank_chunks and this.
template <typename T, bool ANY, int WAVES>
__device__ __forceinline__ void top_of(const Row<T, ANY> &row, int k, TopLds<WAVES> *t) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nc = row.chunks(), need = k < nc ? k : nc;
    // (a floor of NONE + 1, every value: its float is a NaN)
    const int floor = t->floor;
    TopList l = {NONE, 0x7fffffff, floor - 1, 0, floor == NONE + 1 ? -INFINITY : of_key(floor)};
    constexpr int PER = Row<T>::PER, BATCH = 4;  // chunks asked for together
    for (int j0 = wave; j0 < need; j0 += BATCH * WAVES) {
        uint4 raw[BATCH][PER];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int j = j0 + b * WAVES;
            if (j < need && row.whole(t->sel[j]))
                row.template load<false>(t->sel[j], lane, raw[b]);
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int j = j0 + b * WAVES;
            if (j >= need) break;
            const int c = __builtin_amdgcn_readfirstlane(t->sel[j]);
            Piece<T> pc[PER];
            if (row.whole(c))
                row.open(raw[b], pc);
            else
                row.get_end(c, lane, pc);
#pragma unroll
            for (int i = 0; i < PER; ++i)
#pragma unroll
                for (int e = 0; e < Row<T>::N; ++e) {
                    // (most values of a chunk: nothing reaches the list's end)
                    if (!__builtin_amdgcn_ballot_w64(pc[i].f[e] >= l.floor)) continue;
                    const int id = row.first(c, i, lane) + e;
                    const int key = id >= 0 && id < row.V ? key_of(pc[i].f[e]) : NONE;
                    uint64_t in =
                        __builtin_amdgcn_ballot_w64(before(key, id, l.last_key, l.last_id));
                    while (in) {
                        const int from = __builtin_ctzll(in);
                        in &= in - 1;
                        const int ki = __builtin_amdgcn_readlane(key, from);
                        const int ii = __builtin_amdgcn_readlane(id, from);
                        if (before(ki, ii, l.last_key, l.last_id))
                            top_insert(l, ki, ii, k, lane);
                    }
                }
        }
    }
    // the best k of the waves' lists, by counting what comes before each entry
    const bool mine = lane < k && l.key != NONE;
    const int entries = __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine));
    if (lane == 0) t->count[wave] = entries;
    if (threadIdx.x < k) t->bkey[threadIdx.x] = NONE, t->bid[threadIdx.x] = 0;
    __syncthreads();
    int at = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) at += t->count[w];
        total += t->count[w];
    }
    if (mine) t->key[at + lane] = l.key, t->id[at + lane] = l.id;
    __syncthreads();
    for (int j = threadIdx.x; j < total; j += 64 * WAVES) {
        const int key = t->key[j], id = t->id[j];
        int rank = 0;
#pragma unroll 4
        for (int i = 0; i < total; ++i) rank += before(t->key[i], t->id[i], key, id);
        if (rank < k) t->bkey[rank] = key, t->bid[rank] = id;
    }
    __syncthreads();
}

}  // namespace
}  // namespace mi
