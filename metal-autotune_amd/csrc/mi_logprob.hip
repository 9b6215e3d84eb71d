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
// The k likeliest tokens are found from the maxima of the row's chunks (mi_rows.h).
//
// Bound by HBM at many rows (the row's one read, 8.7 VALU instructions a value of
// the 13 that fit beside it: 1024 rows of 151936 bf16, 311 MB, 57.4 us back to back,
// 5.4 TB/s; fp32, 622 MB, 97 us, 6.4); by the launch and its trips to memory, one after
// another, at few, where a row is split over workgroups (one row of as many, with its
// 5 likeliest: 10.0 us).
#include <math.h>

#include "mi_rows.h"

namespace mi {
namespace {

// A wave's sums, in units of log2 (mi_rows.h).
struct Sums {
    float ref;   // shared by the wave
    float top;   // the lane's largest value
    float s, e;  // the lane's sums against ref
};
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
        rank_chunks<WAVES>(maxima, row.chunks(), a.k, t);
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
        const int k = a.k;
        __syncthreads();
        top_of<T, false, WAVES>(row, k, t);
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
