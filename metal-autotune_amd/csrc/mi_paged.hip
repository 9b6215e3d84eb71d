// Bookkeeping and attention prologue of a step over a paged key/value cache
// (no counterpart in the reference, whose caches are contiguous): mi_paged_plan
// and mi_norm_rope_paged.
#include <math.h>

#include <type_traits>

#include "mi_common.h"

namespace mi {
namespace {

// ---------------------------------------------------------------------------
// mi_paged_plan. With p the page size and, for request r, kv cached keys and q
// new tokens: old = ceil(kv / p), new = ceil((kv + q) / p), need = new - old.
// cu is the running sum of q, end that of need; the request gets its pages if it
// needs none or end <= free_count, page w of it (old <= w < new) being
// free_pages[free_count - 1 - (end - need + w - old)].
//
// Nothing here is large: the call is bounded by one launch and two trips to
// memory (32 requests 2.9 us, 256 requests of 8000 tokens 6.7). So one launch does
// all of it: every workgroup sums the (at most 4096) requests' lengths for itself,
// which costs less than a second launch would, then serves 1024 tokens, each
// finding its request by bisection in LDS. The table entry of a new page is written
// by the token at its first row: such a token exists for every new page (a request
// whose tokens pass the T rows is refused), and no other workgroup reads that entry.
// Refused requests leave no gap in the pages: once one lacks pages or rows, so does
// every later one that needs a page.
constexpr int PLAN_MAX_R = 4096, PLAN_MAX_T = 1 << 18;  // (lengths held to T + 1: sums below 2^31)
constexpr int PLAN_TOKENS = 1024;  // tokens a workgroup

struct PlanArgs {
    int *table;
    const int *kv, *q, *free_pages, *free_count;
    int *cu_q, *kv_after, *positions, *slots, *free_left, *refused;
    int R, W, T, n_free, page_log2;
};

__global__ __launch_bounds__(256) void paged_plan_kernel(PlanArgs a, int per) {
    __shared__ int cu[PLAN_MAX_R + 1];
    __shared__ int first[PLAN_MAX_R];  // end - need, or -1: refused
    __shared__ int wq[4], wn[4], wrefused[4], wtaken[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int lp = a.page_log2;
    const int count = min(max(*a.free_count, 0), a.n_free);
    // this thread's requests [r0, r1)
    const int r0 = min((int)threadIdx.x * per, a.R), r1 = min(r0 + per, a.R);
    // (need is at most W <= 2^17 a request and a query at most T + 1 tokens, a
    // length at least 0: what lies outside is not a length, and would only
    // reach past the arrays)
    auto load = [&](int r, int &kv, int &q, int &old, int &need, bool &fits) {
        kv = max(a.kv[r], 0);
        q = min(max(a.q[r], 0), a.T + 1);
        const int64_t pages = ((int64_t)kv + q + (1 << lp) - 1) >> lp;
        old = (int)(((int64_t)kv + (1 << lp) - 1) >> lp);
        fits = pages <= a.W;
        need = fits ? (int)pages - old : 0;
    };
    int sq = 0, sn = 0;
    for (int r = r0; r < r1; ++r) {
        int kv, q, old, need;
        bool fits;
        load(r, kv, q, old, need, fits);
        sq += q;
        sn += need;
    }
    const int iq = wave_scan(sq), in = wave_scan(sn);
    if (lane == 63) wq[wave] = iq, wn[wave] = in;
    __syncthreads();
    int bq = iq - sq, bn = in - sn;
    for (int w = 0; w < wave; ++w) bq += wq[w], bn += wn[w];
    int nrefused = 0, taken = 0;
    for (int r = r0; r < r1; ++r) {
        int kv, q, old, need;
        bool fits;
        load(r, kv, q, old, need, fits);
        const bool ok = fits && (q == 0 || bq + q <= a.T) && (need == 0 || bn + need <= count);
        cu[r] = bq;
        first[r] = ok ? bn : -1;
        if (blockIdx.x == 0) {
            a.cu_q[r] = bq;
            a.kv_after[r] = ok ? kv + q : 0;
        }
        nrefused += !ok;
        if (ok && need) taken = bn + need;
        bq += q;
        bn += need;
    }
    if (threadIdx.x == 255) cu[a.R] = bq;  // (thread 255's requests are the last, or none)
    if (blockIdx.x == 0) {
        const int nr = wave_scan(nrefused);
        for (int o = 32; o > 0; o >>= 1) taken = max(taken, __shfl_xor(taken, o, 64));
        if (lane == 63) wrefused[wave] = nr, wtaken[wave] = taken;
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.cu_q[a.R] = cu[a.R];
        *a.free_left = count - max(max(wtaken[0], wtaken[1]), max(wtaken[2], wtaken[3]));
        *a.refused = (wrefused[0] + wrefused[1]) + (wrefused[2] + wrefused[3]);
    }

    const int total = cu[a.R];
#pragma unroll
    for (int i = 0; i < PLAN_TOKENS / 256; ++i) {
        const int t = blockIdx.x * PLAN_TOKENS + i * 256 + threadIdx.x;
        if (t >= a.T) return;
        int pos = 0, slot = -1;
        if (t < total) {
            int lo = 0, hi = a.R;  // cu[lo] <= t < cu[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cu[mid] <= t)
                    lo = mid;
                else
                    hi = mid;
            }
            const int kv = max(a.kv[lo], 0), f = first[lo];
            pos = kv + t - cu[lo];
            const int w = pos >> lp, row = pos & ((1 << lp) - 1);
            if (f >= 0) {
                const int old = (int)(((int64_t)kv + (1 << lp) - 1) >> lp);
                int page;
                if (w < old) {
                    page = a.table[(int64_t)lo * a.W + w];
                } else {
                    page = a.free_pages[count - 1 - (f + w - old)];
                    if (row == 0) a.table[(int64_t)lo * a.W + w] = page;
                }
                slot = (page << lp) + row;
            }
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
}

// ---------------------------------------------------------------------------
// mi_norm_rope_paged. For a head x of D values, with weight w and angle
// pos * inv_freq[i] of rotation pair i:
//   y = x / sqrt(mean(x^2) + eps) * w,  (y_a, y_b) -> (y_a cos - y_b sin,
//   y_a sin + y_b cos),
// computed in fp32 and rounded once (the contiguous prologue rounds after each
// of its three steps, as the op stream that it replaces does). The angle is
// taken in turns in 64 bits and reduced to [-1/2, 1/2] before it becomes fp32:
// at position 10^5 an fp32 angle is off by up to 4e-3 rad.
//
// Bound by HBM: every row is read once (past the caches: 45.2 -> 40.4 us) and
// written once; 8192 tokens, 32/8 heads of 128, bf16, 201 MB: 39.8 us, 5.1 TB/s,
// what a plain copy reaches. A head takes D / 8 lanes of eight values (four
// rotation pairs), a workgroup one token, whose angles its lanes compute once for
// all the heads they take.
__device__ __forceinline__ uint2 ld8_nt(const void *p) {
    typedef unsigned U2 __attribute__((ext_vector_type(2)));
    const U2 v = __builtin_nontemporal_load((const U2 *)p);
    return make_uint2(v[0], v[1]);
}
template <typename T, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void norm_rope_paged_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, int64_t q_stride,
    int64_t k_stride, int64_t v_stride, const T *__restrict__ q_norm,
    const T *__restrict__ k_norm, T *__restrict__ q_out, T *__restrict__ k_pages,
    T *__restrict__ v_pages, const double *__restrict__ inv_freq, const int *__restrict__ positions,
    const int *__restrict__ slots, int Hq, int Hkv, float eps, int dims, int page_log2,
    unsigned n_slots) {
    constexpr int LPH = D / 8, HPW = 64 / LPH;  // lanes a head, heads a wave
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = lane % LPH, sub = lane / LPH;
    const int slot = slots[t], pos = positions[t];
    const bool keep = (unsigned)slot < n_slots;
    // element offsets of the lane's two groups of four: rotation pairs
    // (e0 + e, e1 + e), or interleaved pairs within eight neighbours
    const int half = dims / 2;
    const bool rot = 8 * j < dims;
    const int e0 = INTERLEAVED || !rot ? 8 * j : 4 * j;
    const int e1 = INTERLEAVED || !rot ? 8 * j + 4 : half + 4 * j;
    float cs[4], sn[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        cs[e] = 1.0f;
        sn[e] = 0.0f;
        if (rot) {
            const double turns = (double)pos * inv_freq[4 * j + e] * 0.15915494309189535;
            const float r = (float)(turns - __builtin_rint(turns));
            cs[e] = __builtin_amdgcn_cosf(r);
            sn[e] = __builtin_amdgcn_sinf(r);
        }
    }
    const int64_t page = slot >> page_log2, row = slot & ((1 << page_log2) - 1);
    const int heads = Hq + 2 * Hkv;
    // the lane's share of head h: its row and its two groups
    auto row_of = [&](int h) -> const T * {
        return h < Hq ? q + t * q_stride + (int64_t)h * D
               : h < Hq + Hkv ? k + t * k_stride + (int64_t)(h - Hq) * D
                              : v + t * v_stride + (int64_t)(h - Hq - Hkv) * D;
    };
    constexpr int BATCH = 3;  // heads of a lane whose loads are in flight together
    for (int h0 = wave * HPW + sub; h0 < heads; h0 += 4 * HPW * BATCH) {
        uint2 ra[BATCH], rb[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int h = h0 + 4 * HPW * i;
            if (h < heads) {
                const T *src = row_of(h);
                const bool is_v = h >= Hq + Hkv;
                ra[i] = ld8_nt(src + (is_v ? 8 * j : e0));
                rb[i] = ld8_nt(src + (is_v ? 8 * j + 4 : e1));
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int h = h0 + 4 * HPW * i;
            if (h >= heads) break;
            const bool is_q = h < Hq, is_v = h >= Hq + Hkv;
            const int hk = is_q ? 0 : (is_v ? h - Hq - Hkv : h - Hq);
            const int64_t at = ((page * Hkv + hk) << page_log2) + row;
            T *dst = is_q ? q_out + (t * Hq + h) * D : (is_v ? v_pages : k_pages) + at * D;
            if (is_v) {
                if (keep) st16(dst + 8 * j, make_uint4(ra[i].x, ra[i].y, rb[i].x, rb[i].y));
                continue;
            }
            const T *w = is_q ? q_norm : k_norm;
            float a[4], b[4];
            unpack4<T>(ra[i], a);
            unpack4<T>(rb[i], b);
            if (w) {  // (uniform over the head's lanes)
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = __builtin_fmaf(a[e], a[e], ss);
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = __builtin_fmaf(b[e], b[e], ss);
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
                const float inv = 1.0f / __fsqrt_rn(ss * (1.0f / D) + eps);
                float wa[4], wb[4];
                unpack4<T>(ld8(w + e0), wa);
                unpack4<T>(ld8(w + e1), wb);
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] *= inv * wa[e], b[e] *= inv * wb[e];
            }
            if (rot) {
                if constexpr (INTERLEAVED) {
                    float f[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = f[2 * e], y = f[2 * e + 1];
                        f[2 * e] = rope_first(x, y, cs[e], sn[e]);
                        f[2 * e + 1] = rope_second(x, y, cs[e], sn[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = f[e], b[e] = f[4 + e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = a[e], y = b[e];
                        a[e] = rope_first(x, y, cs[e], sn[e]);
                        b[e] = rope_second(x, y, cs[e], sn[e]);
                    }
                }
            }
            if (is_q || keep) {
                st8(dst + e0, pack4<T>(a));
                st8(dst + e1, pack4<T>(b));
            }
        }
    }
}

int page_log2_of(int64_t page) {  // -1: not a page size of this build
    for (int l = 4; l <= 8; ++l)
        if (page == (1 << l)) return l;
    return -1;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int mi_paged_plan(int32_t *block_table, int64_t table_width, const int32_t *kv_lens,
                             const int32_t *q_lens, const int32_t *free_pages, int64_t n_free,
                             const int32_t *free_count, int64_t R, int64_t T, int64_t page_size,
                             int32_t *cu_q, int32_t *kv_after, int32_t *positions, int32_t *slots,
                             int32_t *free_left, int32_t *refused, void *stream) {
    const int lp = page_log2_of(page_size);
    if (lp < 0)
        return fail(MI_ERR_UNSUPPORTED, "page size %lld; this build covers 16, 32, 64, 128, 256",
                    (long long)page_size);
    if (R < 1 || R > PLAN_MAX_R || table_width < 1 || table_width > (1 << 17) || T < 0 ||
        T > PLAN_MAX_T || n_free < 0 || n_free > (1 << 30))
        return fail(MI_ERR_ARG, "paged plan: R=%lld (1..%d) table width %lld (1..131072) T=%lld "
                    "(0..%d) free pages %lld", (long long)R, PLAN_MAX_R, (long long)table_width,
                    (long long)T, PLAN_MAX_T, (long long)n_free);
    if (!block_table || !kv_lens || !q_lens || !free_count || !cu_q || !kv_after || !free_left ||
        !refused || (T && (!positions || !slots)) || (n_free && !free_pages))
        return fail(MI_ERR_ARG, "null pointer");
    const PlanArgs a = {block_table, kv_lens, q_lens, free_pages, free_count, cu_q, kv_after,
                        positions, slots, free_left, refused, (int)R, (int)table_width, (int)T,
                        (int)n_free, lp};
    const int64_t blocks = T ? ceil_div(T, PLAN_TOKENS) : 1;
    paged_plan_kernel<<<(unsigned)blocks, 256, 0, as_stream(stream)>>>(a, (int)ceil_div(R, 256));
    return launch_status("paged plan");
}

extern "C" int mi_norm_rope_paged(const void *q, const void *k, const void *v,
                                  int64_t q_row_stride, int64_t k_row_stride,
                                  int64_t v_row_stride, const void *q_norm, const void *k_norm,
                                  void *q_out, void *k_pages, void *v_pages,
                                  const double *inv_freq, int rope_dims, int traditional,
                                  const int32_t *positions, const int32_t *slots, int64_t T,
                                  int64_t Hq, int64_t Hkv, int64_t D, int64_t n_pages,
                                  int64_t page_size, float eps, int dtype, void *stream) {
    if (dtype != MI_BF16 && dtype != MI_F16)
        return fail(MI_ERR_UNSUPPORTED, "norm_rope_paged covers bf16 and fp16 (dtype code %d)",
                    dtype);
    const int lp = page_log2_of(page_size);
    if (lp < 0)
        return fail(MI_ERR_UNSUPPORTED, "page size %lld; this build covers 16, 32, 64, 128, 256",
                    (long long)page_size);
    if (D != 64 && D != 128) return fail(MI_ERR_UNSUPPORTED, "head dim %lld", (long long)D);
    if (rope_dims < 0 || rope_dims > D || rope_dims % 8)
        return fail(MI_ERR_ARG, "rope dims %d: a multiple of 8 up to the head dim", rope_dims);
    if (T < 0 || T > 0x7fffffff || Hq < 1 || Hkv < 1 || Hq > (1 << 20) || Hkv > (1 << 20) ||
        n_pages < 1 || n_pages > (0x7fffffff >> lp))
        return fail(MI_ERR_ARG, "norm_rope_paged shape T=%lld Hq=%lld Hkv=%lld pages=%lld (pages x "
                    "page size < 2^31)", (long long)T, (long long)Hq, (long long)Hkv,
                    (long long)n_pages);
    if (q_row_stride % 8 || k_row_stride % 8 || v_row_stride % 8 || !aligned(q, 16) ||
        !aligned(k, 16) || !aligned(v, 16) || !aligned(q_norm, 8) || !aligned(k_norm, 8) ||
        !aligned(q_out, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
        !aligned(inv_freq, 8))
        return fail(MI_ERR_ARG, "norm_rope_paged rows must be 16-byte aligned");
    if (T == 0) return MI_OK;
    if (!q || !k || !v || !q_out || !k_pages || !v_pages || !positions || !slots ||
        (rope_dims && !inv_freq))
        return fail(MI_ERR_ARG, "null pointer");
    hipStream_t st = as_stream(stream);
    auto run = [&](auto tag, auto dim, auto inter) {
        typedef decltype(tag) TT;
        norm_rope_paged_kernel<TT, dim.value, inter.value><<<(unsigned)T, 256, 0, st>>>(
            (const TT *)q, (const TT *)k, (const TT *)v, q_row_stride, k_row_stride, v_row_stride,
            (const TT *)q_norm, (const TT *)k_norm, (TT *)q_out, (TT *)k_pages, (TT *)v_pages,
            inv_freq, positions, slots, (int)Hq, (int)Hkv, eps, rope_dims, lp,
            (unsigned)(n_pages << lp));
    };
    auto by_dim = [&](auto tag) {
        auto by_pairs = [&](auto dim) {
            traditional ? run(tag, dim, std::true_type{}) : run(tag, dim, std::false_type{});
        };
        D == 128 ? by_pairs(std::integral_constant<int, 128>{})
                 : by_pairs(std::integral_constant<int, 64>{});
    };
    dtype == MI_BF16 ? by_dim(bf16{}) : by_dim(f16{});
    return launch_status("norm_rope_paged");
}
