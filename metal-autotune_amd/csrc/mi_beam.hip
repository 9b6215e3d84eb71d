// Beam search's selection over beams and vocabulary (no counterpart in the reference,
// which samples greedily): mi_beam_select.
//
// Candidate (b, v) of a prompt: c = (x[b, v] - lse_b) + score_b, with
// lse_b = log sum_v e^x[b, v]; a finished beam has one, (b, eos), at its own score. The
// K best, lowest b and then lowest v first among equals.
//
// Within a beam the order is the logits'. So each row gives its K best (mi_rows.h: one
// pass over the row, then its K best chunks again) and its lse, and the K best of a
// prompt are among these B K: an entry's place in the end is its own in its list plus, by
// bisection, what comes before it in every other (the lists are sorted).
//
// Beams are compared in 64 bits, since candidates of different beams lie close together
// (fp32 scores near -100 are 8e-6 apart, and two beams' candidates that often): lse_b is
// the sum of a row's 2^t in fp32, against a reference within 2 of the row's maximum so that
// t is rounded finely, 16 terms of a lane in pairs and their sums, chunk after chunk, in 64
// bits, and freed of what log2 e lost in fp32. In 2^-24 it is off by at most 2 of the
// exponential, 4 of the pairs, 0.7 |t| for t's rounding and 0.16 |t| for what log2 e lacks
// at terms below the maximum, |t| on average at most log2 V + 4: 26 2^-24 = 1.6e-6 (one
// token over a long constant tail, whose roundings go the same way; random rows 1e-7, rows
// of one value below 2e-7). Rows are cut the same wherever they lie, so that rows of equal
// logits have equal lse, and equal candidates stay equal.
//
// Bound at many rows by HBM beside the VALU (exponentials; 2000 rows of 151936 bf16, 608 MB,
// 131 us, 4.6 TB/s; 256 rows of fp32, 156 MB, 37), at few by launch and trips to memory, one
// after another: pass, the row's ticket, ranks, second reading, the prompt's ticket, the
// lists (four rows 13.2 us, 240 rows, 73 MB, 24).
#include "mi_rows.h"

namespace mi {
namespace {

constexpr int BS_MAX_R = 4096, BS_MAX_B = 64, BS_MAX_K = LP_MAX_TOP;
constexpr int64_t BS_SPLIT_ROWS = 160;  // rows from which on none is split
static_assert((BS_SPLIT_ROWS + BS_MAX_R) * 4 <= MI_BEAM_ZERO_BYTES, "a ticket a row and a prompt");

// A part of a row's sum: the reference, the largest value, sum 2^(x log2 e - zero).
struct Part3 {
    float ref, top;
    double s;
};

// By how much, in units, sums against `from` have to be scaled for `to`: an integer where
// both are near, so that nothing is lost.
__device__ __forceinline__ float moved(float from, float to) {
    return far(from) || far(to) ? (from - to) * LP_LOG2E + (excess(from) - excess(to))
                                : units(from) - units(to);
}

// The sum of 2^t(x) over a lane's 16 values, by pairs of pairs.
template <typename T, typename F>
__device__ __forceinline__ float sum_pairs(const Piece<T> (&pc)[Row<T>::PER], F t) {
    constexpr int N = Row<T>::N;
    static_assert(N * Row<T>::PER == 16, "a lane's values of a chunk");
    float level[4];  // of 1, 2, 4, 8 terms each, until there are two
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float s = __builtin_amdgcn_exp2f(t(pc[i / N].f[i % N]));
        int at = 0;
#pragma unroll
        for (; at < 4 && (i >> at & 1); ++at) s = level[at] + s;
        if (i == 15) return s;
        level[at] = s;
    }
    return 0.0f;  // (not reached)
}

// One chunk added to a wave's sum; the key of its maximum at maxima[c].
template <typename T>
__device__ __forceinline__ void add_beam_chunk(Part3 &a, const Piece<T> (&pc)[Row<T>::PER], int c,
                                               int *maxima, int lane) {
    constexpr int N = Row<T>::N, PER = Row<T>::PER;
    float pm = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int e = 0; e < N; e += 2) pm = fmaxf(fmaxf(pm, pc[i].f[e]), pc[i].f[e + 1]);
    const float cm = wave_max(pm);
    if (lane == 0) maxima[c] = key_of(cm);
    a.top = fmaxf(a.top, cm);
    if (cm > a.ref + 2.0f) {  // (uniform)
        a.s *= __builtin_amdgcn_exp2f(moved(a.ref, cm));
        a.ref = cm;
    }
    if (far(a.ref)) {
        a.s += sum_pairs<T>(pc, [&](float x) { return (x - a.ref) * LP_LOG2E; });
    } else {
        const float zero = units(a.ref);
        a.s += sum_pairs<T>(pc, [&](float x) { return __builtin_fmaf(x, LP_LOG2E, -zero); });
    }
}

// The chunks c0, c0 + STEP, ... below c1 of a row, by one wave; the row's end last.
template <typename T, int STEP>
__device__ __forceinline__ Part3 beam_pass(const Row<T, true> &row, int c0, int c1, int *maxima,
                                           int lane) {
    constexpr int PER = Row<T>::PER;
    Part3 a = {-3.4028235e38f, -INFINITY, 0.0};
    const int w1 = min(c1, row.V / LP_CHUNK);
    uint4 raw[PER];
    if (c0 < w1) row.template load<true>(c0, lane, raw);
    for (int c = c0; c < w1; c += STEP) {
        Piece<T> pc[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) launder(raw[i]);
        row.open(raw, pc);
        if (c + STEP < w1) row.template load<true>(c + STEP, lane, raw);
        add_beam_chunk<T>(a, pc, c, maxima, lane);
    }
    const int end = row.V / LP_CHUNK;  // the chunk that the row fills in part
    if (end >= c0 && end < c1 && (end - c0) % STEP == 0) {
        Piece<T> pc[PER];
        row.get_end(end, lane, pc);
        add_beam_chunk<T>(a, pc, end, maxima, lane);
    }
    a.s = wave_add(a.s);
    return a;
}

// Parts joined, one a lane (n of them; the others' are of no matter), in every lane.
struct Joined {
    float ref, top;
    double s;
};
__device__ __forceinline__ Joined join_parts(Part3 p, int n, int lane) {
    if (lane >= n) p = {-3.4028235e38f, -INFINITY, 0.0};
    Joined j;
    j.ref = wave_max(p.ref);
    j.top = wave_max(p.top);
    j.s = wave_add(p.s * (double)__builtin_amdgcn_exp2f(moved(p.ref, j.ref)));
    return j;
}
// log sum e^x of what was joined, in 64 bits; NaN where there was a NaN or +inf, or no
// value above -inf. Where the zero is an integer number of units, t was x times log2 e's
// fp32 value; what that lacks is put back at the largest value (the others weigh less the
// farther they lie from it).
__device__ __forceinline__ double joined_log(const Joined &j) {
    constexpr double LN2 = 0.69314718055994530942, LACKS = 1.44269504088896340736 - (double)LP_LOG2E;
    if (!(j.s > 0.0)) return NAN;
    const double ls = log(j.s);
    return far(j.ref) ? (double)j.ref + ls
                      : LN2 * ((double)units(j.ref) + (double)j.top * LACKS) + ls;
}

struct BeamArgs {
    const void *x;
    int64_t row_stride;
    const float *scores;
    const uint8_t *finished;  // or null
    int eos, B, K, V;
    float *out_scores;
    int *parents, *tokens;
    uint8_t *out_finished;
    // the workspace: tickets of rows and prompts; of each row its segments' sums and its
    // chunks' maxima (nc a row), then its K best (logit, token) and lse
    unsigned *row_tickets, *prompt_tickets;
    float4 *part;
    int *maxima;
    float2 *best;
    double *lse;
    int nc, per;  // chunks a segment
};

// The prompt's K best from its rows' lists, by the last workgroup to come here.
template <int WAVES>
__device__ __forceinline__ void join_beams(int64_t r, const BeamArgs &a, char *lds) {
    const int B = a.B, K = a.K;
    const int64_t row0 = r * B;
    double *cand = (double *)lds;          // [B][K]
    int *ids = (int *)(cand + B * K);      // [B][K]
    int *counts = ids + B * K;             // [B]
    for (int b = threadIdx.x; b < B; b += 64 * WAVES) counts[b] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < B * K; i += 64 * WAVES) {
        const int b = i / K, j = i - b * K;
        const float score = a.scores[row0 + b];
        double c = -INFINITY;
        int id = 0;
        if (!(score > -INFINITY)) {
            // (a dead beam, NaN too: nothing)
        } else if (a.finished && a.finished[row0 + b]) {
            if (j == 0) c = score, id = a.eos;
        } else {
            const float2 e = get_part(a.best + (row0 + b) * K + j);
            const double lse = __builtin_bit_cast(
                double, __hip_atomic_load((const uint64_t *)(a.lse + row0 + b), __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT));
            c = ((double)e.x - lse) + (double)score;
            id = __builtin_bit_cast(int, e.y);
            if (!(c > -INFINITY)) c = -INFINITY;  // (a row with NaN or +inf: nothing)
        }
        cand[i] = c;
        ids[i] = id;
        if (c > -INFINITY) atomicAdd(&counts[b], 1);
    }
    __syncthreads();
    int total = 0;
    for (int b = 0; b < B; ++b) total += counts[b];
    for (int i = threadIdx.x; i < B * K; i += 64 * WAVES) {
        const int b = i / K, j = i - b * K;
        if (j >= counts[b]) continue;
        const double c = cand[i];
        int rank = j;
        for (int o = 0; o < B && rank < K; ++o) {
            if (o == b) continue;
            // entries of list o before (c, b): larger ones, equal ones of a lower beam
            int lo = 0, hi = min(counts[o], K);
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                const double m = cand[o * K + mid];
                if (m > c || (m == c && o < b))
                    lo = mid + 1;
                else
                    hi = mid;
            }
            rank += lo;
        }
        if (rank < K) {
            const int64_t at = r * K + rank;
            const int id = ids[i];
            a.out_scores[at] = (float)c;
            a.parents[at] = (int)(row0 + b);
            a.tokens[at] = id;
            a.out_finished[at] = (a.finished && a.finished[row0 + b]) || id == a.eos;
        }
    }
    for (int j = total + threadIdx.x; j < K; j += 64 * WAVES) {
        const int64_t at = r * K + j;
        a.out_scores[at] = -INFINITY;
        a.parents[at] = (int)row0;
        a.tokens[at] = 0;
        a.out_finished[at] = 0;
    }
}

// SPLIT: a workgroup a segment of a row, the row's last to finish goes on with it; else
// a workgroup a row. The prompt's last row to finish goes on with the prompt.
template <int WAVES> struct BeamLds {
    int maxima[(LP_MAX_CHUNKS + 8 + 3) / 4 * 4];
    TopLds<WAVES> top;
};
template <int WAVES> inline size_t beam_lds(int64_t B, int64_t K) {
    const size_t join = (size_t)(B * K * 12 + B * 4);
    return join > sizeof(BeamLds<WAVES>) ? join : sizeof(BeamLds<WAVES>);
}
template <typename T, bool SPLIT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void beam_kernel(BeamArgs a) {
    __shared__ Part3 part[WAVES];
    // the row's, then the prompt's (beam_lds)
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t r = SPLIT ? blockIdx.y : blockIdx.x;
    const bool offers = a.scores[r] > -INFINITY && !(a.finished && a.finished[r]);
    if (offers) {  // (workgroup-uniform)
        const Row<T, true> row((const T *)a.x + r * a.row_stride, a.V);
        const int nc = row.chunks(), segments = SPLIT ? gridDim.x : 1;
        BeamLds<WAVES> *l = (BeamLds<WAVES> *)lds;
        int *maxima = l->maxima;
        const int c0 = SPLIT ? blockIdx.x * a.per : 0, c1 = SPLIT ? min(c0 + a.per, nc) : nc;
        const Part3 p = beam_pass<T, WAVES>(row, c0 + wave, c1, maxima, lane);
        if (lane == 0) part[wave] = p;
        __syncthreads();
        Part3 mine;
        if constexpr (SPLIT) {
            int *all = a.maxima + r * a.nc;
            for (int c = c0 + threadIdx.x; c < c1; c += 64 * WAVES)
                __hip_atomic_store(all + c, maxima[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (wave == 0) {
                const Joined j = join_parts(part[lane % WAVES], WAVES, lane);
                float4 *sums = a.part + r * segments + blockIdx.x;
                if (lane == 0) {
                    put_part((float2 *)sums, make_float2(j.ref, j.top));
                    put_part((float2 *)sums + 1, __builtin_bit_cast(float2, j.s));
                }
            }
            if (!last_of(a.row_tickets + r, segments)) return;
            const float2 *sums = (const float2 *)(a.part + r * segments + min(lane, segments - 1));
            const float2 u = get_part(sums);
            mine = {u.x, u.y, __builtin_bit_cast(double, get_part(sums + 1))};
            for (int c = threadIdx.x; c < nc; c += 64 * WAVES)
                maxima[c] = __hip_atomic_load(all + c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        TopLds<WAVES> *t = &l->top;
        if (threadIdx.x < 8) maxima[nc + threadIdx.x] = NONE;
        for (int c = threadIdx.x; c < nc; c += 64 * WAVES) t->rank[c] = 0;
        __syncthreads();
        rank_chunks<WAVES>(maxima, nc, a.K, t);
        if (wave == 0) {
            Part3 p = part[lane % WAVES];
            if constexpr (SPLIT) p = mine;
            const double lse = joined_log(join_parts(p, SPLIT ? segments : WAVES, lane));
            if (lane == 0)
                __hip_atomic_store((uint64_t *)(a.lse + r), __builtin_bit_cast(uint64_t, lse),
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        top_of<T, true, WAVES>(row, a.K, t);
        if (threadIdx.x < a.K) {
            const int key = t->bkey[threadIdx.x];
            put_part(a.best + r * a.K + threadIdx.x,
                     make_float2(key == NONE ? -INFINITY : of_key(key),
                                 __builtin_bit_cast(float, t->bid[threadIdx.x])));
        }
    } else if (SPLIT && blockIdx.x > 0) {
        return;
    }
    const int64_t prompt = r / a.B;
    if (!last_of(a.prompt_tickets + prompt, a.B)) return;
    join_beams<WAVES>(prompt, a, lds);
}

// Segments of a row, and a workgroup's waves. Few rows are split, about 512 workgroups of
// eight waves in all, of at least a chunk a wave and at most 64 a row (a lane a segment joins
// them): 64 rows of 151936 17.3 us, in one workgroup of 16 waves each 19.3. From 160 rows
// on none is, which spares the row's ticket (240 rows 27.7 -> 24; 480 47 -> 35), of 16
// waves as long as there is hardly more than one a CU (240 rows 24, of eight 25.4; 480 44,
// of eight 36).
struct BeamSplit {
    int64_t nc, segments, per, waves;
};
inline BeamSplit beam_split(int64_t rows, int64_t V) {
    BeamSplit s;
    s.nc = ceil_div(V, LP_CHUNK);
    int64_t want = rows < BS_SPLIT_ROWS ? ceil_div(512, rows) : 1;
    if (want > ceil_div(s.nc, 8)) want = ceil_div(s.nc, 8);
    if (want > 64) want = 64;
    s.per = ceil_div(s.nc, want);
    s.segments = ceil_div(s.nc, s.per);
    s.waves = s.segments == 1 && rows <= 320 ? 16 : 8;
    return s;
}
inline int64_t beam_bytes(const BeamSplit &s, int64_t rows, int64_t K) {
    const int64_t split =
        s.segments > 1 ? rows * (s.segments * 16 + ceil_div(s.nc, 2) * 8) : 0;
    return MI_BEAM_ZERO_BYTES + split + rows * (8 + 8 * K);
}

template <typename T>
int launch_beam(BeamArgs a, int64_t rows, const BeamSplit &s, char *ws, hipStream_t st) {
    const bool split = s.segments > 1;
    a.row_tickets = (unsigned *)ws;
    a.prompt_tickets = a.row_tickets + BS_SPLIT_ROWS;
    a.nc = (int)(ceil_div(s.nc, 2) * 2);
    a.per = (int)s.per;
    a.part = (float4 *)(ws + MI_BEAM_ZERO_BYTES);
    a.maxima = (int *)(a.part + (split ? rows * s.segments : 0));
    a.lse = (double *)(a.maxima + (split ? rows * a.nc : 0));
    a.best = (float2 *)(a.lse + rows);
    if (split)
        beam_kernel<T, true, 8><<<dim3((unsigned)s.segments, (unsigned)rows), 64 * 8,
                               beam_lds<8>(a.B, a.K), st>>>(a);
    else if (s.waves == 16)
        beam_kernel<T, false, 16><<<(unsigned)rows, 64 * 16, beam_lds<16>(a.B, a.K), st>>>(a);
    else
        beam_kernel<T, false, 8><<<(unsigned)rows, 64 * 8, beam_lds<8>(a.B, a.K), st>>>(a);
    return launch_status("beam select");
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_beam_select_workspace_bytes(int64_t R, int64_t B, int64_t V, int64_t K) {
    if (R <= 0 || B <= 0 || V <= 0 || V > LP_MAX_V || K <= 0) return 0;
    return beam_bytes(beam_split(R * B, V), R * B, K);
}

extern "C" int mi_beam_select(const void *logits, int64_t row_stride, const float *scores,
                              const uint8_t *finished, int64_t eos, int64_t R, int64_t B, int64_t V,
                              int64_t K, float *out_scores, int32_t *parents, int32_t *tokens,
                              uint8_t *out_finished, int dtype, void *workspace,
                              int64_t workspace_bytes, void *stream) {
    if (!valid_dtype(dtype)) return fail(MI_ERR_UNSUPPORTED, "dtype code %d", dtype);
    if (R < 0 || R > BS_MAX_R || B < 1 || B > BS_MAX_B || V < 1 || V > LP_MAX_V || row_stride < 0)
        return fail(MI_ERR_ARG, "beam select R=%lld (to %d) B=%lld (1 to %d) V=%lld (1 to 2^20) row "
                    "stride %lld", (long long)R, BS_MAX_R, (long long)B, BS_MAX_B, (long long)V,
                    (long long)row_stride);
    if (K < 1 || K > BS_MAX_K || K > V * B)
        return fail(MI_ERR_ARG, "beam select K=%lld: 1 to %d, at most B V", (long long)K, BS_MAX_K);
    if (eos < -1 || eos >= V || (finished && eos < 0))
        return fail(MI_ERR_ARG, "beam select eos=%lld: a token of V=%lld (-1: none, without finished "
                    "beams)", (long long)eos, (long long)V);
    if (R == 0) return MI_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens || !out_finished)
        return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(logits, dtype == MI_F32 ? 4 : 2))
        return fail(MI_ERR_ARG, "logits are not aligned to their type");
    const int64_t rows = R * B;
    const BeamSplit s = beam_split(rows, V);
    if (!workspace || workspace_bytes < beam_bytes(s, rows, K) || !aligned(workspace, 16))
        return fail(MI_ERR_ARG, "beam select needs a 16-byte aligned workspace of %lld bytes",
                    (long long)beam_bytes(s, rows, K));
    const BeamArgs a = {logits, row_stride, scores, finished, (int)eos, (int)B, (int)K, (int)V,
                        out_scores, parents, tokens, out_finished, nullptr, nullptr, nullptr,
                        nullptr, nullptr, nullptr, 0, 0};
    hipStream_t st = as_stream(stream);
    if (dtype == MI_BF16) return launch_beam<bf16>(a, rows, s, (char *)workspace, st);
    if (dtype == MI_F16) return launch_beam<f16>(a, rows, s, (char *)workspace, st);
    return launch_beam<float>(a, rows, s, (char *)workspace, st);
}
