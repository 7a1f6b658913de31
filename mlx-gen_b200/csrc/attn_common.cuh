// attn_common.cuh -- what the paged-attention kernels share: the parameter block, the view
// of one sequence, the division of the work, and the join of partial results.
//
//     o_i = sum_j softmax_j(scale q_i . k_j) v_j   over the positions j that token i sees
//
// Token i of a sequence with q_len new tokens and kv_len cached positions (the new ones
// included) stands at position p = kv_len - q_len + i; it sees j < kv_len, with `causal` only
// j <= p, with a window only j > p - window.  A token that sees nothing gets zeros.
//
// The q heads of one kv head are packed: row r of a (sequence, kv head) is token r / G, head
// r % G of the group (G = Hq / Hkv), so a group's heads read each key and value together.
#pragma once

#include "pdl.cuh"

namespace ql {
namespace attn {

constexpr int kSMs = 148;         // B200; used for planning only
constexpr int ROWS_TILE = 16;     // rows of the small-row kernel (one m16 tile)
constexpr int MAX_CLUSTER = 8;    // splits of the small-row kernel that can join inside a cluster
constexpr float NEG_INF = -INFINITY;

struct Params {
    const void *q;
    int64_t q_token, q_head;      // strides of q, elements
    int64_t T;                    // tokens of all sequences
    int Hq, Hkv, G;
    const void *k_cache, *v_cache;  // [pages, Hkv, page_size, D], inner three contiguous
    int64_t page_stride;          // elements between pages
    int num_pages, page_shift;
    const int32_t *table;         // [B, >= ceil(max_kv / page_size)]
    int64_t table_stride;
    const int32_t *q_starts, *kv_lens;
    int max_q, max_kv;
    float scale_log2;             // scale * log2(e)
    int causal, window;
    void *out;                    // [T, Hq, D]
    float *part_o, *part_lse;     // [T * Hq, nsplit, D], [T * Hq, nsplit]; nsplit > 1 only
    int nsplit, chunk;            // most splits of a row's positions; positions of one (tile kernel: whole steps)
    bool adapt;                   // small-row kernel: the chunk follows from the sequences' lengths (adapted_chunk)
    bool cluster;                 // small-row kernel: the splits join inside a cluster, part_* unused
    int rows_kernel_most;         // sequences with up to so many rows go to the small-row kernel
};

struct Seq {
    int q0, q_len, kv_len, ctx;
    bool ok;
};

__device__ __forceinline__ Seq load_seq(const Params &p, int b) {
    Seq s;
    s.q0 = p.q_starts[b];
    const int q1 = p.q_starts[b + 1];
    s.kv_len = p.kv_lens[b];
    s.q_len = q1 - s.q0;
    s.ctx = s.kv_len - s.q_len;
    // sizes that contradict what the launch was planned for: nothing is read or written
    s.ok = s.q0 >= 0 && q1 >= s.q0 && q1 <= p.T && s.q_len <= p.max_q && s.kv_len >= 0 && s.kv_len <= p.max_kv;
    return s;
}

// [lo, hi): the positions that token `tok` sees
__device__ __forceinline__ void visible(const Params &p, const Seq &s, int tok, int &lo, int &hi) {
    hi = p.causal ? min(s.kv_len, max(0, s.ctx + tok + 1)) : s.kv_len;
    lo = p.window ? max(0, s.ctx + tok + 1 - p.window) : 0;
}

// [lo, hi): the positions that some of the packed rows [r0, r1) sees
__device__ __forceinline__ void visible_rows(const Params &p, const Seq &s, int r0, int r1, int &lo, int &hi) {
    int unused;
    visible(p, s, r0 / p.G, lo, unused);
    visible(p, s, (r1 - 1) / p.G, unused, hi);
}

// The splits divide what the CTA's rows see, [lo, hi), from lo's 128-boundary on.
__device__ __forceinline__ void take_split(const Params &p, int split, int chunk, int &lo, int &hi) {
    if (p.nsplit == 1) return;
    const int64_t from = (lo & ~127) + (int64_t)split * chunk;
    lo = (int)max((int64_t)lo, min(from, (int64_t)hi));
    hi = (int)min((int64_t)hi, from + chunk);
}

// The page that holds position pos; an index outside the cache is reported and reads page 0.
__device__ __forceinline__ int page_of(const Params &p, int b, int pos) {
    int pg = p.table[b * p.table_stride + (pos >> p.page_shift)];
    if ((unsigned)pg >= (unsigned)p.num_pages) {
        raise_dev_error(DEV_ERR_BAD_INDEX);
        pg = 0;
    }
    return pg;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
    const int n = valid ? 16 : 0;  // 0: sixteen zero bytes, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// Two fp32 lanes in one register pair (one instruction for both).
__device__ __forceinline__ uint64_t f2_make(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float &x, float &y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// log2 of the factor on the softmax's weights, which are at most 2^BOUND without it.  f16 holds 2^15 at
// most and loses bits below 2^-14: with the factor that is 2^-(14 + shift), so a long tail that the sum
// (fp32) counts in full is not rounded away before the second product (half a million weights of
// 2^-24.9: the result 0.5 % off without it).  Sums and products carry the factor, which the division
// cancels.  bf16 has fp32's range.
template <typename T, int BOUND>
constexpr float kWeightShift = __is_same(T, __half) ? 15.f - BOUND : 0.f;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Joins the partial results of the splits: o = sum_s 2^(lse_s - max) o_s / sum_s 2^(lse_s - max)
// with each o_s normalised and lse_s in base 2.  A split that a row sees nothing of has lse
// -inf and an unwritten o_s, which is not read; one whose scores hold a NaN has lse NaN (which the
// maximum leaves out) and makes the row NaN.  One warp per row.
template <typename T, int D>
__global__ void __launch_bounds__(128) join_kernel(const float *part_o, const float *part_lse, int64_t rows, int nsplit,
                                                   T *out) {
    pdl_trigger();
    pdl_wait();
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    const float *lse = part_lse + row * nsplit;
    float mx = NEG_INF;
    for (int s = lane; s < nsplit; s += 32) mx = fmaxf(mx, lse[s]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    constexpr int PER = D / 32;
    float acc[PER] = {}, total = 0.f;
    const float base = mx == NEG_INF ? 0.f : mx;
    for (int s = 0; s < nsplit; ++s) {
        const float l = lse[s];
        if (l == NEG_INF) continue;
        const float w = ex2(l - base);
        total += w;
        const float *o = part_o + (row * nsplit + s) * D;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] += w * o[e * 32 + lane];
    }
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const uint32_t v = pack2<T>(acc[e] * inv, 0.f);
        reinterpret_cast<uint16_t *>(out)[row * D + e * 32 + lane] = (uint16_t)v;
    }
}

template <typename T, int D>
static int launch_join(const Params &p, cudaStream_t st) {
    const int64_t rows = p.T * p.Hq;
    QL_CUDA_TRY(launch_pdl(join_kernel<T, D>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, 1, (const float *)p.part_o,
                           (const float *)p.part_lse, rows, p.nsplit, (T *)p.out));
    return QL_OK;
}

}  // namespace attn
}  // namespace ql
