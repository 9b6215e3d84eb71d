// Row A7: causal GQA scaled-dot-product attention (mx.fast.scaled_dot_product_attention
// with mask='causal' or none), flash-style over 32-key tiles.
//
// The arithmetic of one query row is fixed: its key tiles of 32 (from key 0)
// are dealt to four streams by tile index (stream w: tiles w, w + 4, ...);
// each stream runs its own online softmax from scratch; the streams' states
// are then folded as (0 + 1) + (2 + 3). Two kernels carry it out, bit for bit
// alike (same tile-update and merge functions, no floating-point contraction
// in them), whatever their work split:
//   attn_prefill_kernel  many query rows. A workgroup is two units (a unit: one
//                        q head's 32-row block; the units of one kv head are
//                        its q heads' blocks) of four waves, a wave a stream;
//                        the units share each stage of four key tiles in LDS.
//   attn_wave_kernel     few query rows. A workgroup is one unit, or (at most
//                        DEC_MAX_LQ rows: decode) the rows of all q heads of
//                        one kv head as the columns of one tile, so K and V
//                        are read once per kv head. A wave a stream, each with
//                        LDS of its own: no barrier before the fold.
// Past DEC_SPLIT_MIN_LK keys a decode call's key tiles are also cut into
// contiguous splits, one workgroup each, whose states attn_combine_kernel folds
// in split order (with a caller's workspace; without one a single workgroup
// runs all of them): the one case where a row's last bits depend on the call's
// shape.
// Per wave and tile:
//   S^T[key][q] = K . Q^T   32x32x16 MFMA, A = K rows, B = Q^T held in
//                           registers for the whole kernel;
//   lane (q = lane%32, half) then holds 16 of the 32 keys of its query row, so
//   the row max/sum needs one exchange between the wave's halves;
//   O^T[d][q] += V^T . P^T  A = V^T, read by transposing LDS loads from the
//                           V tile staged key-major as it sits in memory,
//                           B = P^T straight from the S^T registers
//                           (bf16/fp16): the k order inside each MFMA is
//                           permuted to match the S^T register layout, for
//                           both operands.
// K and V tiles go from memory to LDS by direct DMA (buffer_load ... lds), the
// 16-byte chunks of a row XOR-swizzled so the fragment reads hit distinct
// banks. Online softmax in the log2 domain, fp32 running max/sum, one division
// at the end. Causal masking is bottom-right aligned (query i sees keys
// j <= i + Lk - Lq) and key tiles past the last visible key are skipped.
// A row's result depends only on its global position and the keys, so a
// chunked prefill whose chunks start at multiples of 32 reproduces the whole
// prefill bit for bit, and a decode call the last prefill row; except that split
// calls (at most DEC_MAX_LQ rows over more than DEC_SPLIT_MIN_LK keys, with a
// workspace), a short last chunk among them, agree within rounding.
//
// What bounds it: at long prompts the softmax VALU, some 60 instructions and 16
// v_exp (a quarter-rate unit) for the 16 MFMAs of a tile at D = 128, 8 at D = 64
// (143 VALU a tile counted with everything in), and its waves' turns (two a SIMD at D = 128); for decode one memory round
// trip and the launches. Measured on MI355X in a graph, 32 q / 8 kv heads (in
// brackets: a form that masked and rescaled every score with 360 VALU a tile,
// staged tiles through registers, and ran decode on one workgroup per q head):
// 2048 tokens D = 128 61 us (85), D = 64 30 (60); 501 behind 777, D = 128, 19
// (54); 128 tokens 5.6 (6.5); decode over 129 keys 5.2 (7.6), 1001 9.6 (18.8),
// 8191 11.5 us, 2.9 TB/s of K and V (115).
#include <math.h>

#include "mi_attn_common.h"

namespace mi {
namespace {

constexpr int DEC_MAX_LQ = 8;    // query rows of a decode call (the GEMV row limit)
constexpr int64_t DEC_SPLIT_MIN_LK = 1024;  // keys past which decode calls are split

// Key tiles visible to a q block (causal: up to its last row).
__device__ __forceinline__ int attn_ntiles(int64_t q0, int64_t off, int64_t Lk, int causal) {
    int64_t kend = Lk;
    if (causal) {
        const int64_t last = q0 + 31 + off + 1;
        kend = last < Lk ? last : Lk;
    }
    return kend > 0 ? (int)ceil_div(kend, ATT_KT) : 0;
}

// ---------------------------------------------------------------------------
// attn_prefill_kernel

// LDS: two stages (a key tile of K, then of V, per stream), reused for the fold.
template <int D, int HW> struct PrefillLds {
    static constexpr int STAGE = 2 * ATT_STREAMS * Tile<D>::BYTES;
    static constexpr int FOLD = HW * ATT_STREAMS * Part<D>::BYTES;
    static constexpr int BYTES = 2 * STAGE > FOLD ? 2 * STAGE : FOLD;
};
// (64-value heads fit four waves a SIMD, two workgroups of eight a CU)
template <int D> constexpr int prefill_waves_per_eu() { return D == 64 ? 4 : 2; }

template <typename T, int D, int HW>
__global__ __launch_bounds__(256 * HW)
__attribute__((amdgpu_waves_per_eu(prefill_waves_per_eu<D>()))) void attn_prefill_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ out, int64_t H, int64_t Lq, int64_t Lk, int64_t cap, float scale,
    uint32_t flip, int causal, int out_layout, Div nbk, Div HK, Div rep, unsigned units,
    unsigned nub) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Tile<D> Tl;
    typedef PrefillLds<D, HW> L;
    constexpr int SW = ATT_STREAMS;
    constexpr int NI = Tl::NI / HW;  // DMA instructions of a tile a wave issues
    static_assert(Tl::NI % HW == 0, "a tile's DMA splits over the units' waves");
    __shared__ __attribute__((aligned(1024))) char lds[L::BYTES];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hw = wave / SW, ws = wave % SW;  // unit slot, stream
    const int h2 = lane >> 5, r = lane & 31;
    // Blocks: kv heads fastest (consecutive blocks go to the XCDs in turn, so
    // with 8 kv heads each XCD's L2 holds one head's K and V), the units with
    // the most key tiles first (the grid then drains evenly). nbk = B HK.
    const unsigned bid = blockIdx.x, bq = nbk.of(bid), bk = bid - bq * nbk.d, ub = nub - 1 - bq;
    const unsigned bb = HK.d == nbk.d ? 0u : HK.of(bk);
    const int64_t b = bb, hk = bk - bb * HK.d;
    const unsigned u = ub * HW + hw;
    const bool active = u < units;
    const unsigned uc = active ? u : units - 1, uq = rep.of(uc);
    const int64_t hq = hk * rep.d + (uc - uq * rep.d), q0 = (int64_t)uq * 32;
    const int64_t off = Lk - Lq, qrow = q0 + r;
    const bool qok = active && qrow < Lq;
    const int nt = active ? attn_ntiles(q0, off, Lk, causal) : 0;
    // the workgroup's last unit has the most tiles
    const unsigned ul = ub * HW + HW - 1 < units ? ub * HW + HW - 1 : units - 1;
    const int total = (attn_ntiles((int64_t)rep.of(ul) * 32, off, Lk, causal) + SW - 1) / SW;
    const T *kb = k + (int64_t)bk * cap * D;
    const T *vb = v + (int64_t)bk * cap * D;

    // Stage i holds key tiles 4 i .. 4 i + 3; the waves of one stream share
    // its tile's DMA.
    auto issue = [&](int i, char *dst) {
        const int kt = SW * i + ws;
        dma_tile<T, D, false>(kb, kt, Lk, dst + ws * Tl::BYTES, hw * NI, NI, lane);
        dma_tile<T, D, true>(vb, kt, Lk, dst + (SW + ws) * Tl::BYTES, hw * NI, NI, lane);
    };
    AttnState<D> st;
    attn_init(st);
    uint4 qf[D / 16];
    // tiles before nfull: every row of the block sees all 32 keys
    const int64_t seen = causal && q0 + off + 1 < Lk ? q0 + off + 1 : Lk;
    const int nfull = (int)(seen / ATT_KT);
    const int64_t end = causal && qrow + off + 1 < Lk ? qrow + off + 1 : Lk;
    // One stage: cb is read, the next stage's DMAs land in nb. (restrict:
    // the waits the compiler adds before LDS reads then leave those DMAs in
    // flight.)
    auto step = [&](const char *__restrict__ cb, char *__restrict__ nb, int i)
                    __attribute__((always_inline)) {
        // every wave's DMAs of stage i have landed, and every wave is done with
        // the buffer the next ones go to
        att_wait_vmcnt<0>();
        __syncthreads();
        flip_q<D>(qf, flip);
        if (i + 1 < total) issue(i + 1, nb);
        const int kt = SW * i + ws;
        if (kt < nt) {  // wave-uniform
            uint4 kf[D / 16];
            read_k<D>(cb + ws * Tl::BYTES, kf, r, h2);
            VFrag<T, D> vf;
            read_v<T, D>(cb + (SW + ws) * Tl::BYTES, vf, lane);
            __builtin_amdgcn_sched_barrier(0);  // (not sunk to the PV MFMAs)
            f32x16 s = attn_scores<T, D>(kf, qf);
            if (kt >= nfull) attn_mask(s, (int)(end - (int64_t)kt * ATT_KT), h2);
            uint32_t p[8];
            attn_softmax<T, D>(st, s, p, scale);
            attn_pv<T, D>(st, p, vf);
        }
    };
    char *buf0 = lds, *buf1 = lds + L::STAGE;
    if (total > 0) issue(0, buf0);
    // (a row past the last reads the first: its results are not stored)
    read_q<D>(q + ((b * H + hq) * Lq + (qok ? qrow : 0)) * D, h2, qf);
    for (int i = 0; i < total; i += 2) {  // workgroup-uniform
        step(buf0, buf1, i);
        if (i + 1 < total) step(buf1, buf0, i + 1);
    }

    // The fold, (0 + 1) + (2 + 3): the states pass through LDS, and wave t of
    // a unit folds and stores its O^T tile t.
    __syncthreads();  // every wave is done with the stages
    float4 *part = (float4 *)lds + (size_t)(hw * SW) * Part<D>::WORDS;
    float4 *mine = part + (size_t)ws * Part<D>::WORDS;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) part_put<D>(mine, st, t, lane);
    part_lm<D>(mine)[lane] = make_float2(st.l, st.m);
    __syncthreads();
    if (ws >= D / 32) return;
    const Fold f = fold_streams<D>(part, ws, lane);
    const float inv = row_inv(f.l);
    T *orow = out_layout ? out + ((b * Lq + qrow) * H + hq) * D
                         : out + ((b * H + hq) * Lq + qrow) * D;
    if (qok) store_fold<T>(f, inv, orow, ws, h2);
#endif
}

// ---------------------------------------------------------------------------
// attn_wave_kernel: four waves, a stream each; a wave owns its tiles' LDS: no
// barrier until the fold. One K and one V slot a wave; each is refilled with
// the wave's next tile as soon as its reads are in registers, so K's next tile
// flies under the softmax and the PV MFMAs, V's under the next scores.
// PACK (decode): grid (column block, split). Column c of block cb is row idx =
// 32 cb + c of the kv head's rep Lq query rows (q head idx / Lq, query row idx
// % Lq: contiguous in q). Otherwise the grid is attn_prefill_kernel's with one
// unit a workgroup.
constexpr int DEC_WAVES = ATT_STREAMS;
template <int D> struct DecodeLds {
    static constexpr int SLOTS = DEC_WAVES * 2 * Tile<D>::BYTES;
    static constexpr int FOLD = DEC_WAVES * Part<D>::BYTES;
    static constexpr int BYTES = SLOTS > FOLD ? SLOTS : FOLD;
};

template <typename T, int D, bool PACK>
__global__ __launch_bounds__(64 * DEC_WAVES) void attn_wave_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ out, float *__restrict__ part_o, float2 *__restrict__ part_lm_out, int64_t H,
    int64_t Lq, int64_t Lk, int64_t cap, float scale, uint32_t flip, int causal, int out_layout,
    Div ncb, Div nbk, Div HK, Div rep, int cols, int tps) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Tile<D> Tl;
    __shared__ __attribute__((aligned(1024))) char lds[DecodeLds<D>::BYTES];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h2 = lane >> 5, r = lane & 31;
    const unsigned bid = blockIdx.x, split = PACK ? blockIdx.y : 0u;
    // causal: query row i sees keys j <= i + off
    const int64_t off = Lk - Lq;
    unsigned bk, bb;
    int idx = 0, ntiles;
    int64_t hq, hk, qrow, full_end;
    bool ok;
    if constexpr (PACK) {
        bk = ncb.of(bid);
        bb = HK.d == nbk.d ? 0u : HK.of(bk);
        hk = bk - bb * HK.d;
        idx = (int)(bid - bk * ncb.d) * 32 + r;
        ok = idx < cols;
        const int hrow = Lq == 1 ? idx : (int)((unsigned)idx / (unsigned)Lq);
        qrow = idx - hrow * (int)Lq;
        hq = hk * rep.d + hrow;
        full_end = causal ? off + 1 : Lk;  // every row sees the keys before it
        ntiles = (int)ceil_div(Lk, ATT_KT);
    } else {
        // the units with the most key tiles first; nbk blocks a unit
        const unsigned bq = nbk.of(bid), u = (unsigned)cols - 1 - bq;  // cols: units
        bk = bid - bq * nbk.d;
        bb = HK.d == nbk.d ? 0u : HK.of(bk);
        hk = bk - bb * HK.d;
        const unsigned uq = rep.of(u);
        hq = hk * rep.d + (u - uq * rep.d);
        const int64_t q0 = (int64_t)uq * 32;
        qrow = q0 + r;
        ok = qrow < Lq;
        full_end = causal && q0 + off + 1 < Lk ? q0 + off + 1 : Lk;
        ntiles = attn_ntiles(q0, off, Lk, causal);
    }
    const int64_t b = bb, end = causal && qrow + off + 1 < Lk ? qrow + off + 1 : Lk;
    const T *kb = k + (int64_t)bk * cap * D;
    const T *vb = v + (int64_t)bk * cap * D;
    const int t0 = (int)split * tps, t1 = !PACK || t0 + tps > ntiles ? ntiles : t0 + tps;

    char *kslot = lds + wave * 2 * Tl::BYTES, *vslot = kslot + Tl::BYTES;
    const int first = t0 + wave;  // tps is a multiple of four: stream = wave
    AttnState<D> st;
    attn_init(st);
    uint4 qf[D / 16];
    auto run = [&](char *__restrict__ ks, char *__restrict__ vs) __attribute__((always_inline)) {
        // (a column without a row reads the first: its results are not stored)
        read_q<D>(q + ((b * H + (ok ? hq : 0)) * Lq + (ok ? qrow : 0)) * D, h2, qf);
        if (first < t1) {
            dma_tile<T, D, false>(kb, first, Lk, ks, 0, Tl::NI, lane);
            dma_tile<T, D, true>(vb, first, Lk, vs, 0, Tl::NI, lane);
        }
        for (int kt = first; kt < t1; kt += DEC_WAVES) {  // wave-uniform
            const bool more = kt + DEC_WAVES < t1;
            // K (and, the first time, q) has landed once only V's loads, issued
            // after it, are in flight
            att_wait_vmcnt<Tl::NI>();
            flip_q<D>(qf, flip);
            uint4 kf[D / 16];
            read_k<D>(ks, kf, r, h2);
#pragma unroll
            for (int s = 0; s < D / 16; ++s) launder(kf[s]);  // the reads have returned
            __builtin_amdgcn_sched_barrier(0);
            if (more) dma_tile<T, D, false>(kb, kt + DEC_WAVES, Lk, ks, 0, Tl::NI, lane);
            f32x16 s = attn_scores<T, D>(kf, qf);
            const int64_t k0 = (int64_t)kt * ATT_KT;
            if (k0 + ATT_KT > full_end) attn_mask(s, (int)(end - k0), h2);
            uint32_t p[8];
            attn_softmax<T, D>(st, s, p, scale);
            if (more)
                att_wait_vmcnt<Tl::NI>();
            else
                att_wait_vmcnt<0>();
            VFrag<T, D> vf;
            read_v<T, D>(vs, vf, lane);
            attn_pv<T, D>(st, p, vf);
            __builtin_amdgcn_sched_barrier(0);
            att_wait_lds();  // V's reads have returned
            if (more) dma_tile<T, D, true>(vb, kt + DEC_WAVES, Lk, vs, 0, Tl::NI, lane);
        }
    };
    run(kslot, vslot);

    // fold (0 + 1) + (2 + 3), as in the prefill kernel: wave t folds O^T tile t
    __syncthreads();
    float4 *part = (float4 *)lds;
    float4 *mine = part + (size_t)wave * Part<D>::WORDS;
    if (ok) {
#pragma unroll
        for (int t = 0; t < D / 32; ++t) part_put<D>(mine, st, t, lane);
        part_lm<D>(mine)[lane] = make_float2(st.l, st.m);
    }
    __syncthreads();
    if (wave >= D / 32) return;
    const int t = wave;
    const Fold f = fold_streams<D>(part, t, lane);  // (lanes without a column: unused)
    if (PACK && part_o) {  // one split's state, for attn_combine_kernel
        const int64_t rows = (int64_t)ncb.of(gridDim.x) * cols;
        const int64_t row = (int64_t)bk * cols + idx;
        const float l_tot = f.l + __shfl_xor(f.l, 32, 64);
        if (!ok) return;
        float *o = part_o + ((int64_t)split * rows + row) * D + 32 * t + 4 * h2;
#pragma unroll
        for (int j = 0; j < 4; ++j) *(float4 *)(o + 8 * j) = f.o[j];
        if (t == 0 && h2 == 0) part_lm_out[(int64_t)split * rows + row] = make_float2(l_tot, f.m);
        return;
    }
    const float inv = row_inv(f.l);
    if (!ok) return;
    T *orow = out_layout ? out + ((b * Lq + qrow) * H + hq) * D
                         : out + ((b * H + hq) * Lq + qrow) * D;
    store_fold<T>(f, inv, orow, t, h2);
#endif
}

// One query row (b, q head, query row) per workgroup: out = sum_s w_s O_s /
// sum_s w_s l_s with w_s = 2^(m_s - max m), s over the splits. The weights
// first (a lane a split), then 256 / (D / 4) thread groups take every so manyth
// split, in order, and the groups are added in order.
constexpr int DEC_MAX_SPLITS = 512;
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_combine_kernel(const float *__restrict__ part_o,
                                                           const float2 *__restrict__ part_lm_in,
                                                           T *__restrict__ out, int64_t H,
                                                           int64_t Lq, int nsplit,
                                                           int out_layout) {
#pragma clang fp contract(off)
    constexpr int LANES = D / 4, GROUPS = 256 / LANES, IN_FLIGHT = 8;
    __shared__ float wt[DEC_MAX_SPLITS];
    __shared__ float4 acc[GROUPS][LANES];
    __shared__ float lw[4];
    const int64_t rows = gridDim.x, row = blockIdx.x;
    const int c = threadIdx.x % LANES, g = threadIdx.x / LANES;
    // this thread's first partial sums, requested before the weights are known
    const float *po = part_o + row * D + 4 * c;
    float4 v[IN_FLIGHT];
#pragma unroll
    for (int i = 0; i < IN_FLIGHT; ++i) {
        const int s = g + GROUPS * i;
        v[i] = *(const float4 *)(po + (s < nsplit ? s : 0) * rows * D);
    }
    float m = -INFINITY;
    for (int s = threadIdx.x & 63; s < nsplit; s += 64) m = fmaxf(m, part_lm_in[s * rows + row].y);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    float l = 0.0f;
    for (int s = threadIdx.x; s < nsplit; s += 256) {
        const float2 lm = part_lm_in[s * rows + row];
        const float w = lm.y == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lm.y - m);
        wt[s] = w;
        l = __builtin_fmaf(w, lm.x, l);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
    if ((threadIdx.x & 63) == 0) lw[threadIdx.x >> 6] = l;
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = g; s0 < nsplit; s0 += GROUPS * IN_FLIGHT) {
        if (s0 != g) {
#pragma unroll
            for (int i = 0; i < IN_FLIGHT; ++i) {
                const int s = s0 + GROUPS * i;
                v[i] = *(const float4 *)(po + (s < nsplit ? s : 0) * rows * D);
            }
        }
#pragma unroll
        for (int i = 0; i < IN_FLIGHT; ++i) {
            const int s = s0 + GROUPS * i;
            if (s < nsplit) {
                const float w = wt[s];
                o.x = __builtin_fmaf(w, v[i].x, o.x);
                o.y = __builtin_fmaf(w, v[i].y, o.y);
                o.z = __builtin_fmaf(w, v[i].z, o.z);
                o.w = __builtin_fmaf(w, v[i].w, o.w);
            }
        }
    }
    acc[g][c] = o;
    __syncthreads();
    if (g) return;
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) {
        const float4 a = acc[i][c];
        o.x += a.x;
        o.y += a.y;
        o.z += a.z;
        o.w += a.w;
    }
    l = ((lw[0] + lw[1]) + lw[2]) + lw[3];
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int64_t bh = row / Lq, lq = row % Lq, b = bh / H, h = bh % H;
    T *orow = out_layout ? out + ((b * Lq + lq) * H + h) * D : out + row * D;
    const float e[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    st8(orow + 4 * c, pack4<T>(e));
}

// ---------------------------------------------------------------------------
// dispatch

struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    int64_t B, H, HK, Lq, Lk, cap;
    float scale;    // > 0, log2 units
    uint32_t flip;  // sign bits of a negative scale, for Q
    int causal, out_layout;
};

// Splits of a decode call and key tiles per split (a multiple of four: the
// streams keep their tiles). One workgroup per split and column block; past
// DEC_SPLIT_MIN_LK keys as many as put two workgroups on every CU (256), each
// wave at least one tile. Up to that line one workgroup a kv head, so that a
// decode row keeps the bits of the prefill's there (by time alone the line would
// lie lower: 1001 keys unsplit take 9.6 us, 1025 split 8.1).
struct DecSplit {
    int ncb, nsplit, tps;
};
inline DecSplit decode_split(int64_t B, int64_t H, int64_t HK, int64_t Lq, int64_t Lk) {
    const int ncb = (int)ceil_div(H / HK * Lq, 32);
    const int64_t quads = ceil_div(ceil_div(Lk, ATT_KT), ATT_STREAMS);
    int64_t n = 1;
    if (Lk > DEC_SPLIT_MIN_LK) {
        n = DEC_MAX_SPLITS / (B * HK * ncb);
        n = n < 1 ? 1 : (n > quads ? quads : n);
    }
    const int64_t tps = ceil_div(quads, n) * ATT_STREAMS;
    return {ncb, (int)ceil_div(quads * ATT_STREAMS, tps), (int)tps};
}

template <typename T, int D>
int launch_decode(const AttnArgs &a, float *ws, hipStream_t st) {
    DecSplit d = decode_split(a.B, a.H, a.HK, a.Lq, a.Lk);
    if (!ws) {
        d.tps = (int)(ceil_div(ceil_div(a.Lk, ATT_KT), ATT_STREAMS) * ATT_STREAMS);
        d.nsplit = 1;
    }
    const int64_t rows = a.B * a.H * a.Lq, nbk = a.B * a.HK, rep = a.H / a.HK;
    float *po = d.nsplit > 1 ? ws : nullptr;
    float2 *plm = d.nsplit > 1 ? (float2 *)(ws + d.nsplit * rows * D) : nullptr;
    const dim3 grid((unsigned)(nbk * d.ncb), (unsigned)d.nsplit);
    attn_wave_kernel<T, D, true><<<grid, 64 * DEC_WAVES, 0, st>>>(
        (const T *)a.q, (const T *)a.k, (const T *)a.v, (T *)a.out, po, plm, a.H, a.Lq, a.Lk,
        a.cap, a.scale, a.flip, a.causal, a.out_layout, make_div(d.ncb, nbk * d.ncb),
        make_div(nbk, nbk), make_div(a.HK, nbk), make_div(rep, rep), (int)(rep * a.Lq), d.tps);
    if (d.nsplit > 1)
        attn_combine_kernel<T, D><<<(unsigned)rows, 256, 0, st>>>(po, plm, (T *)a.out, a.H, a.Lq,
                                                                  d.nsplit, a.out_layout);
    return launch_status("sdpa (decode)");
}

// Two units (q heads' 32-row blocks) share each staged K/V tile where that leaves
// a workgroup for most CUs and the rows are long (half the K/V traffic, two waves a
// SIMD); else one unit a workgroup, of which a CU holds two and whose waves wait
// for no barrier (64 tokens 5.05 us against 6.2 for one unit through the shared
// stages, 16 behind 4080 26.6 against 35). Short rows fill few of the stages: 205
// tokens, 64/8 heads of 64 5.2 / 6.4; 265 tokens, 64/8 of 128 10.1 / 14.4; 16 x 289
// tokens 114 / 150. Past 256 keys only while K and V of all heads (a unit reads
// its own copy) stay in the caches: 8 x 436 tokens, 64/32 heads of 128 (57 MB) 226
// / 161. Same results.
template <typename T, int D>
int launch_attn_d(const AttnArgs &a, float *ws, hipStream_t st) {
    if (a.Lq <= DEC_MAX_LQ) return launch_decode<T, D>(a, ws, st);
    const int64_t rep = a.H / a.HK, units = rep * ceil_div(a.Lq, 32), nbk = a.B * a.HK;
    const int64_t nub = ceil_div(units, 2);
    const bool short_rows =
        a.Lk <= 256 || (a.Lk <= 640 && nbk * a.Lk * D * 4 <= ((int64_t)40 << 20));
    if (nbk * nub >= 192 && !short_rows)
        attn_prefill_kernel<T, D, 2><<<(unsigned)(nbk * nub), 512, 0, st>>>(
            (const T *)a.q, (const T *)a.k, (const T *)a.v, (T *)a.out, a.H, a.Lq, a.Lk, a.cap,
            a.scale, a.flip, a.causal, a.out_layout, make_div(nbk, nbk * nub),
            make_div(a.HK, nbk), make_div(rep, units), (unsigned)units, (unsigned)nub);
    else
        attn_wave_kernel<T, D, false><<<(unsigned)(nbk * units), 64 * DEC_WAVES, 0, st>>>(
            (const T *)a.q, (const T *)a.k, (const T *)a.v, (T *)a.out, nullptr, nullptr, a.H,
            a.Lq, a.Lk, a.cap, a.scale, a.flip, a.causal, a.out_layout, make_div(1, 1),
            make_div(nbk, nbk * units), make_div(a.HK, nbk), make_div(rep, units), (int)units, 0);
    return launch_status("sdpa");
}

int run_sdpa(const void *q, const void *k, const void *v, void *out, int64_t B, int64_t H,
             int64_t HK, int64_t Lq, int64_t Lk, int64_t D, int64_t kv_cap, float scale,
             int causal, int out_layout, int dtype, void *ws, int64_t ws_bytes, void *stream) {
    if (dtype != MI_BF16 && dtype != MI_F16)
        return fail(MI_ERR_UNSUPPORTED, "sdpa covers bf16 and fp16 (dtype code %d)", dtype);
    if (D != 64 && D != 128) return fail(MI_ERR_UNSUPPORTED, "sdpa head dim %lld", (long long)D);
    if (B < 0 || H <= 0 || HK <= 0 || H % HK || Lq < 0 || Lk <= 0 || kv_cap < Lk)
        return fail(MI_ERR_ARG, "sdpa shape B=%lld H=%lld HK=%lld Lq=%lld Lk=%lld cap=%lld",
                    (long long)B, (long long)H, (long long)HK, (long long)Lq, (long long)Lk,
                    (long long)kv_cap);
    if (causal && Lq > Lk) return fail(MI_ERR_ARG, "causal sdpa needs Lq <= Lk");
    if (B * Lq && (!q || !k || !v || !out)) return fail(MI_ERR_ARG, "null pointer");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 8))
        return fail(MI_ERR_ARG, "q/k/v must be 16-byte aligned, out 8-byte aligned");
    if (B * Lq == 0) return MI_OK;
    const int64_t need = mi_sdpa_workspace_bytes(B, H, HK, Lq, Lk, D);
    float *w = need > 0 && ws && ws_bytes >= need && aligned(ws, 16) ? (float *)ws : nullptr;
    const float sl = scale * 1.4426950408889634f;
    // (a scale of 0 as the smallest normal: masked scores stay -inf; NaN stays
    // NaN)
    const float mag = fabsf(sl) < 1.17549435e-38f ? 1.17549435e-38f : fabsf(sl);
    const AttnArgs a = {q, k, v, out, B, H, HK, Lq, Lk, kv_cap, mag,
                        sl < 0.0f ? 0x80008000u : 0u, causal, out_layout};
    hipStream_t st = as_stream(stream);
    if (dtype == MI_BF16)
        return D == 128 ? launch_attn_d<bf16, 128>(a, w, st) : launch_attn_d<bf16, 64>(a, w, st);
    return D == 128 ? launch_attn_d<f16, 128>(a, w, st) : launch_attn_d<f16, 64>(a, w, st);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_sdpa_workspace_bytes(int64_t B, int64_t H, int64_t HK, int64_t Lq,
                                           int64_t Lk, int64_t D) {
    if (B <= 0 || H <= 0 || HK <= 0 || H % HK || Lq <= 0 || Lq > DEC_MAX_LQ || Lk <= 0 ||
        (D != 64 && D != 128))
        return 0;
    const DecSplit d = decode_split(B, H, HK, Lq, Lk);
    return d.nsplit > 1 ? d.nsplit * B * H * Lq * (D + 2) * (int64_t)sizeof(float) : 0;
}

extern "C" int mi_sdpa(const void *q, const void *k, const void *v, void *out, int64_t B,
                       int64_t H, int64_t HK, int64_t Lq, int64_t Lk, int64_t D, int64_t kv_cap,
                       float scale, int causal, int out_layout, int dtype, void *stream) {
    return run_sdpa(q, k, v, out, B, H, HK, Lq, Lk, D, kv_cap, scale, causal, out_layout, dtype,
                    nullptr, 0, stream);
}

extern "C" int mi_sdpa_ws(const void *q, const void *k, const void *v, void *out, int64_t B,
                          int64_t H, int64_t HK, int64_t Lq, int64_t Lk, int64_t D,
                          int64_t kv_cap, float scale, int causal, int out_layout, int dtype,
                          void *workspace, int64_t workspace_bytes, void *stream) {
    return run_sdpa(q, k, v, out, B, H, HK, Lq, Lk, D, kv_cap, scale, causal, out_layout, dtype,
                    workspace, workspace_bytes, stream);
}
