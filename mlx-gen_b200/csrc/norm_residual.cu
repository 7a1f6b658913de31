// norm_residual.cu -- the norms around a block, fused with its gate and residual scale:
//     u = post ? rms(y) * (offset + post) : y
//     r = residual + alpha * gate * u
//     h = rms(r) * (offset + weight) * (1 + scale),      rms(x) = x / sqrt(mean(x^2) + eps)
// One pass: the row of y and of the residual is read once, r and h are written once, and
// everything between stays in fp32 registers (h is taken from r before r's rounding; each
// output is rounded once, at its store).
//
// Bound: HBM for many rows (2 reads + 2 writes per element), launch latency for a few.
// Split: one CTA per row; a thread owns NCH chunks of VEC consecutive elements, so the row
// is held in registers whatever D is (up to 32 elements for each of 1024 threads).  The two
// sums of squares are block reductions; rows of up to 32 vectors run a warp each, eight to a CTA.
// Measured: 4608 x 3840 bf16 with post norm, gate and modulation 31.4 us = 4.51 TB/s (issue slots
// 78 % busy; without the reductions 27 us), 4 x 3072 1.8 us (a graph's replay; back to back 32.0, 4.7).  Rings of rows filled by bulk copies
// with the factors kept in registers took 31.5 us at best and were left out.
#include <string.h>

#include "pdl.cuh"

namespace ql {
namespace normres {

constexpr int MAX_D = 32768;

template <typename T, int V>
struct alignas(sizeof(T) * V >= 16 ? 16 : sizeof(T) * V) Pack {
    T v[V];
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(float &d, float v) { d = v; }
__device__ __forceinline__ void from_f(__nv_bfloat16 &d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(__half &d, float v) { d = __float2half_rn(v); }

// v[e] = x[e] rounded to T (two at a time where T is 16 bits wide)
template <typename T, int V>
__device__ __forceinline__ void round_to_pack(Pack<T, V> &o, const float (&x)[V]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        uint32_t w[V / 2];
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            if constexpr (__is_same(T, __half))
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(x[2 * e + 1]), "f"(x[2 * e]));
            else w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
        }
        memcpy(&o, w, sizeof(o));
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) from_f(o.v[e], x[e]);
    }
}

struct Params {
    const void *y, *residual;
    int64_t y_stride, r_stride;  // elements between rows
    int D;
    float inv_d, alpha, offset, eps;
    const void *post, *weight, *gate, *scale;
    int64_t gate_period, scale_period;
    void *h, *r_out;
};

// Sum over the threads of a row (a warp or the block); `red` holds one float per warp and is
// not reused within a row.
template <bool WARP_ROW>
__device__ __forceinline__ float row_sum(float v, float *red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (WARP_ROW) return v;
    const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < nw ? red[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename Y, typename R, int VEC, int NCH, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? 256 : 1024) norm_residual_kernel(const Params p, int64_t M) {
    __shared__ float red[2][32];
    pdl_trigger();
    pdl_wait();
    using PY = Pack<Y, VEC>;
    using PR = Pack<R, VEC>;
    const int nt = WARP_ROW ? 32 : blockDim.x, tid = WARP_ROW ? threadIdx.x & 31 : threadIdx.x;
    const int64_t m = WARP_ROW ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP_ROW && m >= M) return;
    const int n = p.D / VEC;
    const PY *yp = reinterpret_cast<const PY *>(reinterpret_cast<const Y *>(p.y) + m * p.y_stride);
    const PR *rp = reinterpret_cast<const PR *>(reinterpret_cast<const R *>(p.residual) + m * p.r_stride);
    const PY *postp = reinterpret_cast<const PY *>(p.post);
    const PY *wp = reinterpret_cast<const PY *>(p.weight);
    const PY *gp = reinterpret_cast<const PY *>(p.gate);
    const PY *sp = reinterpret_cast<const PY *>(p.scale);
    if (gp && p.gate_period) gp += m / p.gate_period * n;
    if (sp && p.scale_period) sp += m / p.scale_period * n;

    PY yv[NCH];
    PR rv[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int i = c * nt + tid;
        if (i < n) {
            yv[c] = yp[i];
            rv[c] = rp[i];
        }
    }
    // the sums first touch, then the weights: their loads overlap the reductions
    float post_factor = p.alpha;  // of y: alpha, and 1 / rms(y) with a post norm
    if (postp) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if (c * nt + tid < n)
#pragma unroll
                for (int e = 0; e < VEC; ++e) ss += to_f(yv[c].v[e]) * to_f(yv[c].v[e]);
        post_factor *= rsqrtf(row_sum<WARP_ROW>(ss, red[0]) * p.inv_d + p.eps);
    }
    float r[NCH][VEC], ss = 0.f;
    PR *ro = reinterpret_cast<PR *>(reinterpret_cast<R *>(p.r_out) + m * p.D);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int i = c * nt + tid;
        if (i >= n) continue;
        float u[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[e] = to_f(yv[c].v[e]) * post_factor;
        if (postp) {
            const PY w = postp[i];
            if (p.offset != 0.f) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[e] *= p.offset + to_f(w.v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[e] *= to_f(w.v[e]);
            }
        }
        if (gp) {
            const PY g = gp[i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[c][e] = fmaf(u[e], to_f(g.v[e]), to_f(rv[c].v[e]));
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[c][e] = u[e] + to_f(rv[c].v[e]);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += r[c][e] * r[c][e];
        PR o;
        round_to_pack(o, r[c]);
        ro[i] = o;
    }
    const float inv = rsqrtf(row_sum<WARP_ROW>(ss, red[1]) * p.inv_d + p.eps);
    PY *ho = reinterpret_cast<PY *>(reinterpret_cast<Y *>(p.h) + m * p.D);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int i = c * nt + tid;
        if (i >= n) continue;
        const PY w = wp[i];
        if (p.offset != 0.f) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[c][e] *= inv * (p.offset + to_f(w.v[e]));
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[c][e] *= inv * to_f(w.v[e]);
        }
        if (sp) {
            const PY s = sp[i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[c][e] = fmaf(r[c][e], to_f(s.v[e]), r[c][e]);
        }
        PY o;
        round_to_pack(o, r[c]);
        ho[i] = o;
    }
}

template <typename Y, typename R, int VEC, int NCH>
static cudaError_t launch_n(const Params &p, int64_t M, int nt, cudaStream_t st) {
    if (NCH == 1 && nt == 32)
        return launch_pdl(norm_residual_kernel<Y, R, VEC, 1, true>, dim3((unsigned)((M + 7) / 8)), dim3(256), 0, st, 1, p, M);
    return launch_pdl(norm_residual_kernel<Y, R, VEC, NCH, false>, dim3((unsigned)M), dim3(nt), 0, st, 1, p, M);
}

template <typename Y, typename R, int VEC>
static int launch(const Params &p, int64_t M, cudaStream_t st) {
    const int n = p.D / VEC;  // vectors of a row
    // chunks of a thread: the fewest that a block of 1024 threads needs.  Rows of one warp's
    // width (up to 32 vectors) run eight to a CTA.
    constexpr int MAXC = 32 / VEC;
    int nch = 1;
    while (nch < MAXC && (int64_t)nch * 1024 < n) nch *= 2;
    const int nt = ((n + nch - 1) / nch + 31) / 32 * 32;
    cudaError_t rc = cudaErrorInvalidValue;
    switch (nch) {
        case 1: rc = launch_n<Y, R, VEC, 1>(p, M, nt, st); break;
        case 2: rc = launch_n<Y, R, VEC, 2>(p, M, nt, st); break;
        case 4: rc = launch_n<Y, R, VEC, 4>(p, M, nt, st); break;
        default:
            if constexpr (VEC == 1) {
                if (nch == 8) rc = launch_n<Y, R, VEC, 8>(p, M, nt, st);
                else if (nch == 16) rc = launch_n<Y, R, VEC, 16>(p, M, nt, st);
                else rc = launch_n<Y, R, VEC, 32>(p, M, nt, st);
            }
    }
    QL_CUDA_TRY(rc);
    return QL_OK;
}

template <typename Y, typename R>
static int launch_types(const Params &p, int64_t M, bool vec, cudaStream_t st) {
    return vec ? launch<Y, R, 8>(p, M, st) : launch<Y, R, 1>(p, M, st);
}

}  // namespace normres

// vec: 16-byte loads (every row and vector 16-byte aligned, D a multiple of 8); the scalar
// form takes any D and alignment.
int launch_norm_residual(const normres::Params &p, int y_dtype, int r_dtype, int64_t M, bool vec, cudaStream_t st) {
    using namespace normres;
    if (y_dtype == QL_F32) return launch_types<float, float>(p, M, vec, st);
    if (y_dtype == QL_BF16)
        return r_dtype == QL_F32 ? launch_types<__nv_bfloat16, float>(p, M, vec, st)
                                 : launch_types<__nv_bfloat16, __nv_bfloat16>(p, M, vec, st);
    return r_dtype == QL_F32 ? launch_types<__half, float>(p, M, vec, st) : launch_types<__half, __half>(p, M, vec, st);
}

}  // namespace ql
