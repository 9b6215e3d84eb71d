// Log probabilities of given tokens, row entropies and the most probable tokens
// of a batch of logits (no counterpart in the reference, which samples greedily):
// mi_token_logprobs.
//
// With m the row's maximum, d_i = x_i - m, S = sum e^d_i:
//   log p(i) = d_i - log S,   H = log S - (sum e^d_i d_i) / S.
// One pass over the row. A wave keeps S and E = sum e^d d against a reference
// that all its lanes share and that moves only when a value passes it by 30: the
// sums are fp32 and keep their relative precision at any offset, and moving the
// reference by c turns E into (E + c S) e^c. The last step refers them to the
// row's true maximum.
//
// The k likeliest tokens need no list during the pass, only the maximum of every
// chunk of 1024 values: ordered by (value descending, index ascending) they lie
// in the k chunks whose maxima come first in that order, since a value outside
// these has k maxima before it. So the pass leaves the maxima, and its end ranks
// them, reads the k best chunks again and keeps what reaches the k-th maximum
// (as good as k values in all, but for ties) in a list, a lane an entry.
//
// Bound by HBM at many rows (the row's one read, 8.7 VALU instructions a value of
// the 13 that fit beside it: 1024 rows of 151936 bf16, 311 MB, 57.4 us back to back,
// 5.4 TB/s; fp32, 622 MB, 97 us, 6.4); by the launch and its trips to memory, one after
// another, at few, where a row is split over workgroups (one row of as many, with its
// 5 likeliest: 10.0 us).
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

// What a wave sums is in units of log2: t = x log2 e - C with C = rint(ref log2 e) an
// integer, p = 2^t, S = sum p, E = sum p t: one fma a value, rounded as finely as t
// is small, and a step from one C to another scales by a power of two. From 2^23 on
// no rounding to an integer is left in fp32 and C misses ref log2 e by more than 1/2,
// past 2e9 by more than 2^t can take (a mask of -1e10). References beyond 2^20 (such
// masks; -FLT_MAX before the first value) take t = (x - ref) log2 e instead.
struct Sums {
    float ref;   // shared by the wave
    float top;   // the lane's largest value
    float s, e;  // the lane's sums against ref
};
__device__ __forceinline__ bool far(float ref) { return !(fabsf(ref) <= 1048576.0f); }
__device__ __forceinline__ float units(float ref) { return __builtin_rintf(ref * LP_LOG2E); }
// By how much the sums' zero lies above ref log2 e.
__device__ __forceinline__ float excess(float ref) {
    return far(ref) ? 0.0f : __builtin_fmaf(-ref, LP_LOG2E, units(ref));
}
// (2^t = 0 for t below -150: the floor keeps a forbidden token's -inf out of 0 * t;
// NaN reaches s.)
__device__ __forceinline__ void add_value(float &s, float &e, float t) {
    const float p = __builtin_amdgcn_exp2f(t);
    s += p;
    e = __builtin_fmaf(p, fmaxf(t, -300.0f), e);
}
// Sums against a reference c units higher.
__device__ __forceinline__ void move_sums(float &s, float &e, float c) {
    const float f = __builtin_amdgcn_exp2f(c);
    // (c s may overflow where what it is weighted with has vanished)
    e = f == 0.0f ? 0.0f : __builtin_fmaf(c, s, e) * f;
    s *= f;
}
__device__ __forceinline__ void move_ref(float &s, float &e, float from, float to) {
    move_sums(s, e, far(from) || far(to) ? (from - to) * LP_LOG2E + (excess(from) - excess(to))
                                         : units(from) - units(to));
}
// ... against the row's maximum itself.
__device__ __forceinline__ void move_to(float &s, float &e, float from, float m) {
    move_sums(s, e, far(from) ? (from - m) * LP_LOG2E
                              : __builtin_fmaf(-m, LP_LOG2E, units(from)));
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

// A row as 16-byte pieces from the one that holds its first value; value i of
// piece p is row element p N + i - skew. What lies outside the row reads as -inf.
template <typename T> struct Row {
    static constexpr int N = Piece<T>::N, PER = LP_CHUNK / (64 * N);  // pieces a lane and chunk
    const T *x;
    const char *base;
    int skew, V;
    __device__ __forceinline__ Row(const T *x_, int V_) : x(x_), V(V_) {
        skew = (int)(((uintptr_t)x & 15) / sizeof(T));
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
            raw[i] = NT ? ld16_nt(at) : ld16(at);
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
            if (f >= 0 && f + N <= V) raw[i] = ld16(base + (int64_t)(f + skew) * (int)sizeof(T));
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

// One chunk added to a wave's sums; (TOP) the key of its maximum at maxima[c].
template <typename T, bool TOP>
__device__ __forceinline__ void add_chunk(Sums &a, const Piece<T> (&pc)[Row<T>::PER], int c,
                                          int *maxima, int lane) {
    constexpr int N = Row<T>::N, PER = Row<T>::PER;
    float pm = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int e = 0; e < N; e += 2) pm = fmaxf(fmaxf(pm, pc[i].f[e]), pc[i].f[e + 1]);
    a.top = fmaxf(a.top, pm);
    if (TOP) {
        const float cm = wave_max(pm);
        if (lane == 0) maxima[c] = key_of(cm);
    }
    if (__builtin_amdgcn_ballot_w64(pm > a.ref + 30.0f)) {
        const float to = fmaxf(a.ref, wave_max(pm));
        move_ref(a.s, a.e, a.ref, to);
        a.ref = to;
    }
    // a chunk's values by themselves first: two short chains of roundings, not one
    // through the row's values
    float s = 0.0f, e = 0.0f;
    if (far(a.ref)) {  // (uniform)
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) add_value(s, e, (pc[i].f[j] - a.ref) * LP_LOG2E);
    } else {
        const float c2 = units(a.ref);
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j)
                add_value(s, e, __builtin_fmaf(pc[i].f[j], LP_LOG2E, -c2));
    }
    a.s += s;
    a.e += e;
}

// The chunks c0, c0 + STEP, ... below c1 of a row, by one wave. The row's ends come
// after the whole chunks, in a loop of their own: among them, the waits for their
// loads would stop the next chunk's, which are on their way while one is added.
template <typename T, bool TOP, bool NT, int STEP>
__device__ __forceinline__ float4 pass(const Row<T> &row, int c0, int c1, int *maxima, int lane) {
    constexpr int PER = Row<T>::PER;
    Sums a = {-3.4028235e38f, -INFINITY, 0.0f, 0.0f};
    const int w0 = c0 + (row.skew && c0 == 0 ? STEP : 0);
    const int w1 = min(c1, (row.V + row.skew) / LP_CHUNK);
    uint4 raw[PER];
    if (w0 < w1) row.template load<NT>(w0, lane, raw);
    for (int c = w0; c < w1; c += STEP) {
        Piece<T> pc[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) launder(raw[i]);
        row.open(raw, pc);
        if (c + STEP < w1) row.template load<NT>(c + STEP, lane, raw);
        add_chunk<T, TOP>(a, pc, c, maxima, lane);
    }
    for (int j = 0; j < 2; ++j) {
        const int c = j ? row.chunks() - 1 : 0;
        if (c < c0 || c >= c1 || (c - c0) % STEP || row.whole(c) || (j && c == 0)) continue;
        Piece<T> pc[PER];
        row.get_end(c, lane, pc);
        add_chunk<T, TOP>(a, pc, c, maxima, lane);
    }
    return make_float4(a.ref, wave_max(a.top), wave_add(a.s), wave_add(a.e));
}

struct LpArgs {
    const void *x;
    int64_t row_stride;
    const void *tokens;
    int wide, V, k;
    float *logprob, *entropy;
    int *top_ids;
    float *top_logprobs;
    // rows split over workgroups: of each row its segments' sums and its chunks'
    // maxima, nc a row
    unsigned *tickets;  // a row
    float4 *part;
    int *maxima;
    int nc, per;  // chunks a segment
};

// What follows the pass, by a workgroup of WAVES, from the row's n partial sums (ref,
// top, s, e) and, in LDS, the keys of its chunks' maxima.
template <int WAVES> struct TopLds {
    int rank[LP_MAX_CHUNKS], sel[LP_MAX_TOP];
    int key[WAVES * LP_MAX_TOP], id[WAVES * LP_MAX_TOP];
    int bkey[LP_MAX_TOP], bid[LP_MAX_TOP];
    int count[WAVES];
    int floor;
};
// The logit of row r's token, asked for before the pass.
template <typename T> __device__ __forceinline__ float token_logit(const Row<T> &row, int64_t r,
                                                                   const LpArgs &a) {
    const int64_t tok = a.wide ? ((const int64_t *)a.tokens)[r] : ((const int *)a.tokens)[r];
    return tok >= 0 && tok < row.V ? (float)row.x[tok] : NAN;
}
__device__ __forceinline__ float4 get_sums(const float4 *at) {
    const float2 a = get_part((const float2 *)at), b = get_part((const float2 *)at + 1);
    return make_float4(a.x, a.y, b.x, b.y);
}
// p0: partial sum `lane` (any where there is none; past 64 they are in part)
template <typename T, bool TOP, int WAVES>
__device__ __forceinline__ void finish(const Row<T> &row, int64_t r, float logit, float4 p0,
                                       const float4 *part, int n, const int *maxima,
                                       TopLds<WAVES> *t, const LpArgs &a) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (TOP) {
        // the chunks' ranks: a wave compares every chunk, a lane each, with eight
        // others at a time (maxima: padded by NONE to a multiple of 8; rank: zero)
        const int k = a.k, nc = row.chunks(), need = k < nc ? k : nc;
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
    // every wave adds the partial sums, 64 a step, in one order
    float m = lane < n ? p0.y : -INFINITY;
    for (int i = lane + 64; i < n; i += 64) m = fmaxf(m, get_sums(part + i).y);
    m = wave_max(m);
    float S = 0.0f, E = 0.0f;
    for (int i = lane; i < n; i += 64) {
        const float4 p = i == lane ? p0 : get_sums(part + i);
        float s = p.z, e = p.w;
        move_to(s, e, p.x, m);
        S += s;
        E += e;
    }
    S = wave_add(S);
    E = wave_add(E);
    const float ls = logf(S);
    if (threadIdx.x == 0) {
        a.logprob[r] = (logit - m) - ls;
        a.entropy[r] = ls - LP_LN2 * (E / S);
    }
    if constexpr (TOP) {
        const int k = a.k, nc = row.chunks(), need = k < nc ? k : nc;
        __syncthreads();
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
        if (threadIdx.x < k) {
            const int key = t->bkey[threadIdx.x];
            a.top_ids[r * k + threadIdx.x] = t->bid[threadIdx.x];
            a.top_logprobs[r * k + threadIdx.x] = key == NONE ? NAN : (of_key(key) - m) - ls;
        }
    }
}

// SPLIT: a workgroup a segment of a row, whose sums and maxima go to the workspace;
// the row's last workgroup to finish goes on with them. Else a workgroup a row.
template <typename T, bool TOP, bool SPLIT>
__global__ __launch_bounds__(64 * (SPLIT ? LP_SPLIT_WAVES : LP_WAVES))
void logprob_kernel(LpArgs a) {
    constexpr int WAVES = SPLIT ? LP_SPLIT_WAVES : LP_WAVES;
    __shared__ float4 part[WAVES];
    __shared__ __attribute__((aligned(16))) int maxima[TOP ? LP_MAX_CHUNKS + 8 : 1];
    __shared__ TopLds<WAVES> top[1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t r = SPLIT ? blockIdx.y : blockIdx.x;
    const Row<T> row((const T *)a.x + r * a.row_stride, a.V);
    const int nc = row.chunks();
    const float logit = token_logit(row, r, a);
    if (TOP) {
        if (threadIdx.x < 8) maxima[nc + threadIdx.x] = NONE;
        for (int c = threadIdx.x; c < nc; c += 64 * WAVES) top->rank[c] = 0;
    }
    if constexpr (!SPLIT) {
        const float4 p = pass<T, TOP, true, WAVES>(row, wave, nc, maxima, lane);
        if (lane == 0) part[wave] = p;
        __syncthreads();
        finish<T, TOP, WAVES>(row, r, logit, part[lane % WAVES], part, WAVES, maxima, top, a);
        return;
    }
    const int c0 = blockIdx.x * a.per, c1 = min(c0 + a.per, nc), segments = gridDim.x;
    const float4 p = pass<T, TOP, false, WAVES>(row, c0 + wave, c1, maxima, lane);
    if (lane == 0) part[wave] = p;
    __syncthreads();
    int *all = a.maxima + r * a.nc;
    float4 *sums = a.part + r * segments;
    if (TOP)
        for (int c = c0 + threadIdx.x; c < c1; c += 64 * WAVES)
            __hip_atomic_store(all + c, maxima[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (threadIdx.x == 0) {
        // to the largest reference (each is finite, a segment of -inf alone too)
        float ref = part[0].x, best = part[0].y, s = 0.0f, e = 0.0f;
        for (int w = 1; w < WAVES; ++w) ref = fmaxf(ref, part[w].x), best = fmaxf(best, part[w].y);
        for (int w = 0; w < WAVES; ++w) {
            float sw = part[w].z, ew = part[w].w;
            move_ref(sw, ew, part[w].x, ref);
            s += sw;
            e += ew;
        }
        put_part((float2 *)(sums + blockIdx.x), make_float2(ref, best));
        put_part((float2 *)(sums + blockIdx.x) + 1, make_float2(s, e));
    }
    if (!last_of(a.tickets + r, segments)) return;
    const float4 p0 = get_sums(sums + (lane < segments ? lane : 0));
    if (TOP) {
        for (int c = threadIdx.x; c < nc; c += 64 * WAVES)
            maxima[c] = __hip_atomic_load(all + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
    }
    finish<T, TOP, WAVES>(row, r, logit, p0, sums, segments, maxima, top, a);
}

// Segments of a row: none from 512 rows on (two workgroups a CU by themselves);
// below, about 512 workgroups in all, of at least a chunk a wave.
constexpr int64_t LP_SPLIT_ROWS = 512;
static_assert(LP_SPLIT_ROWS * 4 <= MI_LOGPROBS_ZERO_BYTES, "a ticket a row");
struct LpSplit {
    int64_t nc, segments, per;
};
inline LpSplit lp_split(int64_t rows, int64_t V, int dtype) {
    LpSplit s;
    s.nc = (V + (dtype == MI_F32 ? 3 : 7) + LP_CHUNK - 1) / LP_CHUNK;
    const int64_t most = ceil_div(s.nc, LP_SPLIT_WAVES);
    const int64_t want = rows < LP_SPLIT_ROWS ? ceil_div(512, rows) : 1;
    s.per = ceil_div(s.nc, want < most ? want : most);
    s.segments = ceil_div(s.nc, s.per);
    return s;
}
inline int64_t lp_bytes(const LpSplit &s, int64_t rows, int top) {
    return s.segments > 1
               ? MI_LOGPROBS_ZERO_BYTES + rows * (s.segments * 16 + (top ? s.nc * 4 : 0)) : 0;
}

template <typename T, bool TOP>
int launch_logprobs(LpArgs a, int64_t rows, const LpSplit &s, char *ws, hipStream_t st) {
    if (!ws) {
        logprob_kernel<T, TOP, false><<<(unsigned)rows, 64 * LP_WAVES, 0, st>>>(a);
        return launch_status("token logprobs");
    }
    a.tickets = (unsigned *)ws;
    a.part = (float4 *)(ws + MI_LOGPROBS_ZERO_BYTES);
    a.maxima = (int *)(a.part + rows * s.segments);
    a.nc = (int)s.nc;
    a.per = (int)s.per;
    logprob_kernel<T, TOP, true>
        <<<dim3((unsigned)s.segments, (unsigned)rows), 64 * LP_SPLIT_WAVES, 0, st>>>(a);
    return launch_status("token logprobs");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_token_logprobs_workspace_bytes(int64_t rows, int64_t V, int top, int dtype) {
    if (rows <= 0 || V <= 0 || V > LP_MAX_V || top < 0) return 0;
    return lp_bytes(lp_split(rows, V, dtype), rows, top);
}

extern "C" int mi_token_logprobs(const void *logits, int64_t rows, int64_t V, int64_t row_stride,
                                 const void *tokens, int tokens_are_64, int top, float *logprobs,
                                 float *entropy, int32_t *top_ids, float *top_logprobs, int dtype,
                                 void *workspace, int64_t workspace_bytes, void *stream) {
    if (!valid_dtype(dtype)) return fail(MI_ERR_UNSUPPORTED, "dtype code %d", dtype);
    if (rows < 0 || rows > 0x7fffffff || V < 1 || V > LP_MAX_V || row_stride < 0)
        return fail(MI_ERR_ARG, "token logprobs rows=%lld V=%lld (1 to 2^20) row stride %lld",
                    (long long)rows, (long long)V, (long long)row_stride);
    if (top < 0 || top > LP_MAX_TOP || top > V)
        return fail(MI_ERR_ARG, "token logprobs top=%d: 0 to %d, at most V=%lld", top, LP_MAX_TOP,
                    (long long)V);
    if (rows == 0) return MI_OK;
    if (!logits || !tokens || !logprobs || !entropy || (top && (!top_ids || !top_logprobs)))
        return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(logits, dtype == MI_F32 ? 4 : 2))
        return fail(MI_ERR_ARG, "logits are not aligned to their type");
    const LpSplit s = lp_split(rows, V, dtype);
    const int64_t need = lp_bytes(s, rows, top);
    char *ws = need && workspace && workspace_bytes >= need && aligned(workspace, 16)
                   ? (char *)workspace : nullptr;
    const LpArgs a = {logits, row_stride, tokens, tokens_are_64, (int)V, top, logprobs, entropy,
                      top_ids, top_logprobs, nullptr, nullptr, nullptr, 0, 0};
    hipStream_t st = as_stream(stream);
    auto run = [&](auto tag) {
        typedef decltype(tag) T;
        return top ? launch_logprobs<T, true>(a, rows, s, ws, st)
                   : launch_logprobs<T, false>(a, rows, s, ws, st);
    };
    return dtype == MI_BF16 ? run(bf16{}) : dtype == MI_F16 ? run(f16{}) : run(float{});
}
