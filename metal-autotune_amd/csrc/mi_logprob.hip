// Log probabilities of given tokens, row entropies and the most probable tokens
// of a batch of logits (no counterpart in the reference, which samples greedily):
// mi_token_logprobs.
//
// With m the row's maximum, d_i = x_i - m, S = sum e^d_i:
//   log p(i) = d_i - log S,   H = log S - (sum e^d_i d_i) / S.
// One pass over the row. A wave keeps S and E = sum e^d d against a reference
// that all its lanes share and that moves only when a value passes it by 30: the
// sums are fp32 and keep their relative precision at any offset, and moving the
// reference by c turns E into (E - c S) e^-c. The last step refers them to the
// row's true maximum.
//
// The likeliest tokens: lane i of a wave holds the wave's i-th best value and
// index. Values reach the list in index order and only if strictly larger than
// its last entry, so equal values keep the lowest indices. NaN never enters; a
// row with a NaN has NaN sums.
#include <math.h>

#include "mi_common.h"

namespace mi {
namespace {

constexpr int LP_MAX_TOP = 64;   // a lane an entry
constexpr int LP_WAVES = 4;
constexpr float LP_LOG2E = 1.4426950408889634f;

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
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

struct Sums {
    float ref;   // shared by the wave
    float top;   // the lane's largest value
    float s, e;  // the lane's sums against ref
};

// d and e^d of one value against a reference, added. (e^d = 0 for d below -104:
// the floor keeps a forbidden token's -inf out of 0 * d; NaN reaches s.)
__device__ __forceinline__ void add_value(Sums &a, float x) {
    const float d = x - a.ref;
    const float p = __builtin_amdgcn_exp2f(d * LP_LOG2E);
    a.s += p;
    a.e = __builtin_fmaf(p, fmaxf(d, -200.0f), a.e);
}
__device__ __forceinline__ void move_ref(float &s, float &e, float from, float to) {
    const float c = from - to;
    const float f = __builtin_amdgcn_exp2f(c * LP_LOG2E);
    // (a reference at a mask's lowest value, or -FLT_MAX before the first: c s may
    // overflow, and what it is weighted with has vanished)
    e = f == 0.0f ? 0.0f : __builtin_fmaf(c, s, e) * f;
    s *= f;
}

struct TopList {
    float v;  // lane i: the i-th best value
    int id;
    float last;  // the k-th best value (uniform)
};
__device__ __forceinline__ void top_insert(TopList &l, float v, int id, int k, int lane) {
    const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(l.v >= v));
    const float pv = __shfl_up(l.v, 1, 64);
    const int pi = __shfl_up(l.id, 1, 64);
    l.v = lane < at ? l.v : (lane == at ? v : pv);
    l.id = lane < at ? l.id : (lane == at ? id : pi);
    l.last = readlane_f(l.v, k - 1);
}

// One piece a lane (first: the index of its first value; lanes in index order).
template <typename T, bool TOP>
__device__ __forceinline__ void add_piece(Sums &a, TopList &l, const Piece<T> &p, int first, int k,
                                          int lane) {
    constexpr int N = Piece<T>::N;
    float pm = fmaxf(p.f[0], p.f[1]);
#pragma unroll
    for (int i = 2; i < N; i += 2) pm = fmaxf(fmaxf(pm, p.f[i]), p.f[i + 1]);
    a.top = fmaxf(a.top, pm);
    if (__builtin_amdgcn_ballot_w64(pm > a.ref + 30.0f)) {
        const float to = fmaxf(a.ref, wave_max(pm));
        move_ref(a.s, a.e, a.ref, to);
        a.ref = to;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) add_value(a, p.f[i]);
    if constexpr (TOP) {
        uint64_t mask = __builtin_amdgcn_ballot_w64(pm > l.last);
        while (mask) {
            const int from = __builtin_ctzll(mask);
            float v = 0.0f;  // lane i < N: value i of that lane's piece
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float w = readlane_f(p.f[i], from);
                v = lane == i ? w : v;
            }
            const int base = __builtin_amdgcn_readlane(first, from);
            uint64_t in = __builtin_amdgcn_ballot_w64(lane < N && v > l.last);
            while (in) {
                const int i = __builtin_ctzll(in);
                top_insert(l, readlane_f(v, i), base + i, k, lane);
                in &= in - 1;
                in &= __builtin_amdgcn_ballot_w64(lane < N && v > l.last);
            }
            mask &= mask - 1;
            mask &= __builtin_amdgcn_ballot_w64(pm > l.last);
        }
    }
}

// One workgroup a row.
template <typename T, bool TOP>
__global__ __launch_bounds__(64 * LP_WAVES) void logprob_kernel(
    const T *__restrict__ x, int64_t row_stride, const void *__restrict__ tokens, int wide,
    int V, int k, float *__restrict__ logprob, float *__restrict__ entropy,
    int *__restrict__ top_ids, float *__restrict__ top_logprobs) {
    constexpr int N = Piece<T>::N;
    __shared__ float4 part[LP_WAVES];
    __shared__ float lv[LP_WAVES * LP_MAX_TOP];
    __shared__ int li[LP_WAVES * LP_MAX_TOP];
    __shared__ float bv[LP_MAX_TOP];
    __shared__ int bi[LP_MAX_TOP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x;
    const T *xr = x + row * row_stride;
    // 16-byte pieces from the one that holds the row's first value; value i of
    // piece p is row element p N + i - skew
    const int skew = (int)(((uintptr_t)xr & 15) / sizeof(T));
    const char *base = (const char *)xr - skew * (int)sizeof(T);
    const int np = (V + skew + N - 1) / N;
    Sums a = {-3.4028235e38f, -INFINITY, 0.0f, 0.0f};
    TopList l = {-INFINITY, 0x7fffffff, -INFINITY};
    for (int p0 = wave * 64; p0 < np; p0 += 64 * LP_WAVES) {
        const int p = p0 + lane, first = p * N - skew;
        Piece<T> pc;
        if (p > 0 && first + N <= V) {
            pc = open_piece<T>(ld16(base + (int64_t)p * 16));
        } else {  // the row's ends, and lanes past it
#pragma unroll
            for (int i = 0; i < N; ++i)
                pc.f[i] = first + i >= 0 && first + i < V ? (float)xr[first + i] : -INFINITY;
        }
        add_piece<T, TOP>(a, l, pc, first, k, lane);
    }
    const float top = wave_max(a.top);
    const float s = wave_add(a.s), e = wave_add(a.e);
    if (lane == 0) part[wave] = make_float4(a.ref, top, s, e);
    if constexpr (TOP) {
        if (lane < k) lv[wave * k + lane] = l.v, li[wave * k + lane] = l.id;
        if (threadIdx.x < k) bv[threadIdx.x] = -INFINITY, bi[threadIdx.x] = 0x7fffffff;
    }
    __syncthreads();
    float m = part[0].y;
#pragma unroll
    for (int w = 1; w < LP_WAVES; ++w) m = fmaxf(m, part[w].y);
    float S = 0.0f, E = 0.0f;
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w) {
        float sw = part[w].z, ew = part[w].w;
        move_ref(sw, ew, part[w].x, m);
        S += sw;
        E += ew;
    }
    const float ls = logf(S);
    if (threadIdx.x == 0) {
        const int64_t t = wide ? ((const int64_t *)tokens)[row] : ((const int *)tokens)[row];
        logprob[row] = t >= 0 && t < V ? ((float)xr[t] - m) - ls : NAN;
        entropy[row] = ls - E / S;
    }
    if constexpr (TOP) {
        // the best k of the waves' lists, by counting what comes before each
        const int n = LP_WAVES * k;
        if (threadIdx.x < n) {
            const float v = lv[threadIdx.x];
            const int id = li[threadIdx.x];
            int rank = 0;
            for (int i = 0; i < n; ++i)
                rank += lv[i] > v || (lv[i] == v && (li[i] < id || (li[i] == id && i < threadIdx.x)));
            if (rank < k) bv[rank] = v, bi[rank] = id;
        }
        __syncthreads();
        if (wave == 0) {
            // fewer than k values above -inf: the lowest indices of -inf fill up
            int have = __builtin_popcountll(
                __builtin_amdgcn_ballot_w64(lane < k && bi[lane] != 0x7fffffff));
            float v = lane < k ? bv[lane] : 0.0f;
            int id = lane < k ? bi[lane] : 0;
            for (int i0 = 0; have < k && i0 < V; i0 += 64) {
                const int i = i0 + lane;
                uint64_t in = __builtin_amdgcn_ballot_w64(i < V && (float)xr[i < V ? i : 0] == -INFINITY);
                while (in && have < k) {
                    if (lane == have) id = i0 + __builtin_ctzll(in);
                    in &= in - 1;
                    ++have;
                }
            }
            if (lane < k) {
                top_ids[row * k + lane] = id < V ? id : 0;
                top_logprobs[row * k + lane] = (v - m) - ls;
            }
        }
    }
}

template <typename T>
int launch_logprobs(const void *x, int64_t rows, int64_t V, int64_t stride, const void *tokens,
                    int wide, int top, float *lp, float *ent, int32_t *ids, float *tlp,
                    hipStream_t st) {
    if (top)
        logprob_kernel<T, true><<<(unsigned)rows, 64 * LP_WAVES, 0, st>>>(
            (const T *)x, stride, tokens, wide, (int)V, top, lp, ent, ids, tlp);
    else
        logprob_kernel<T, false><<<(unsigned)rows, 64 * LP_WAVES, 0, st>>>(
            (const T *)x, stride, tokens, wide, (int)V, 0, lp, ent, ids, tlp);
    return launch_status("token logprobs");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_token_logprobs(const void *logits, int64_t rows, int64_t V, int64_t row_stride,
                                 const void *tokens, int tokens_are_64, int top, float *logprobs,
                                 float *entropy, int32_t *top_ids, float *top_logprobs, int dtype,
                                 void *stream) {
    if (!valid_dtype(dtype)) return fail(MI_ERR_UNSUPPORTED, "dtype code %d", dtype);
    if (rows < 0 || rows > 0x7fffffff || V < 1 || V > (1 << 30) || row_stride < 0)
        return fail(MI_ERR_ARG, "token logprobs rows=%lld V=%lld row stride %lld", (long long)rows,
                    (long long)V, (long long)row_stride);
    if (top < 0 || top > LP_MAX_TOP || top > V)
        return fail(MI_ERR_ARG, "token logprobs top=%d: 0 to %d, at most V=%lld", top, LP_MAX_TOP,
                    (long long)V);
    if (rows == 0) return MI_OK;
    if (!logits || !tokens || !logprobs || !entropy || (top && (!top_ids || !top_logprobs)))
        return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(logits, dtype == MI_F32 ? 4 : 2))
        return fail(MI_ERR_ARG, "logits are not aligned to their type");
    hipStream_t st = as_stream(stream);
    auto run = [&](auto tag) {
        return launch_logprobs<decltype(tag)>(logits, rows, V, row_stride, tokens, tokens_are_64,
                                              top, logprobs, entropy, top_ids, top_logprobs, st);
    };
    return dtype == MI_BF16 ? run(bf16{}) : dtype == MI_F16 ? run(f16{}) : run(float{});
}
