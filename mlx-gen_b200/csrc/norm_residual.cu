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
// sums of squares are block reductions.
#include "ql_common.cuh"

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

struct Params {
    const void *y, *residual;
    int64_t y_stride, r_stride;  // elements between rows
    int D;
    float inv_d, alpha, offset, eps;
    const void *post, *weight, *gate, *scale;
    int64_t gate_period, scale_period;
    void *h, *r_out;
};

// Sum over the block; `red` holds one float per warp and is not reused within a row.
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int nw = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (nw == 1) return v;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < nw ? red[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename Y, typename R, int VEC, int NCH>
__global__ void __launch_bounds__(1024) norm_residual_kernel(const Params p) {
    __shared__ float red[2][32];
    using PY = Pack<Y, VEC>;
    using PR = Pack<R, VEC>;
    const int64_t m = blockIdx.x;
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
        const int i = c * blockDim.x + threadIdx.x;
        if (i < n) {
            yv[c] = yp[i];
            rv[c] = rp[i];
        }
    }
    float inv_post = 1.f;
    if (postp) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c)
            if (c * blockDim.x + threadIdx.x < n)
#pragma unroll
                for (int e = 0; e < VEC; ++e) ss += to_f(yv[c].v[e]) * to_f(yv[c].v[e]);
        inv_post = rsqrtf(block_sum(ss, red[0]) * p.inv_d + p.eps);
    }
    float r[NCH][VEC], ss = 0.f;
    PR *ro = reinterpret_cast<PR *>(reinterpret_cast<R *>(p.r_out) + m * p.D);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        if (i >= n) continue;
        float u[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[e] = to_f(yv[c].v[e]);
        if (postp) {
            const PY w = postp[i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[e] = u[e] * inv_post * (p.offset + to_f(w.v[e]));
        }
        if (gp) {
            const PY g = gp[i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[e] *= to_f(g.v[e]);
        }
        PR o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            r[c][e] = fmaf(p.alpha, u[e], to_f(rv[c].v[e]));
            ss += r[c][e] * r[c][e];
            from_f(o.v[e], r[c][e]);
        }
        ro[i] = o;
    }
    const float inv = rsqrtf(block_sum(ss, red[1]) * p.inv_d + p.eps);
    PY *ho = reinterpret_cast<PY *>(reinterpret_cast<Y *>(p.h) + m * p.D);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int i = c * blockDim.x + threadIdx.x;
        if (i >= n) continue;
        const PY w = wp[i];
        PY o;
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = inv * (p.offset + to_f(w.v[e]));
        if (sp) {
            const PY s = sp[i];
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] *= 1.f + to_f(s.v[e]);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) from_f(o.v[e], r[c][e] * f[e]);
        ho[i] = o;
    }
}

template <typename Y, typename R, int VEC>
static int launch(const Params &p, int64_t M, cudaStream_t st) {
    const int n = p.D / VEC;  // vectors of a row
    // chunks of a thread: the fewest that a block of 1024 threads needs
    constexpr int MAXC = 32 / VEC;
    int nch = 1;
    while (nch < MAXC && (int64_t)nch * 1024 < n) nch *= 2;
    const int nt = ((n + nch - 1) / nch + 31) / 32 * 32;
    switch (nch) {
        case 1: norm_residual_kernel<Y, R, VEC, 1><<<(unsigned)M, nt, 0, st>>>(p); break;
        case 2: norm_residual_kernel<Y, R, VEC, 2><<<(unsigned)M, nt, 0, st>>>(p); break;
        case 4: norm_residual_kernel<Y, R, VEC, 4><<<(unsigned)M, nt, 0, st>>>(p); break;
        default:
            if constexpr (VEC == 1) {
                if (nch == 8) norm_residual_kernel<Y, R, VEC, 8><<<(unsigned)M, nt, 0, st>>>(p);
                else if (nch == 16) norm_residual_kernel<Y, R, VEC, 16><<<(unsigned)M, nt, 0, st>>>(p);
                else norm_residual_kernel<Y, R, VEC, 32><<<(unsigned)M, nt, 0, st>>>(p);
            }
    }
    QL_CUDA_TRY(cudaGetLastError());
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
