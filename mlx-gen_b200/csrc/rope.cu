// rope.cu -- rotary positions on q and k, and the append of k and v to a paged cache.
//     (a, b) -> (a cos - b sin, b cos + a sin)
// for the pairs (i, i + rot/2) of a head (half layout) or (2i, 2i + 1) (interleaved), i <
// rot/2; elements past rot are copied.  The angles come from a table of fp32 rows [cos | sin],
// one per position, so any scaling of the frequencies and any axis split is a table and long
// positions keep the accuracy the table was computed with.  fp32 arithmetic, one rounding.
//
// Bound: HBM (q, k, v read once, q and the cache lines written once).  Split: one CTA per
// token; a thread owns one chunk of pairs and walks over the heads with it, so it reads its
// cosines and sines once.  VEC = 8 moves 16 or 32 bytes per access; VEC = 1 takes any
// alignment and any even rot.
#include "ql_common.cuh"

namespace ql {
namespace ropek {

using normres::from_f;
using normres::Pack;
using normres::to_f;

struct Params {
    const void *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides, elements
    int Hq, Hk, D, rot;
    const float *table;  // [P, rot]
    int64_t P;
    const int64_t *positions, *slots;
    void *q_out, *k_out;        // [T, Hq, D], [T, Hk, D]; k_out NULL with a cache
    void *k_cache, *v_cache;    // [pages, Hk, page_size, D], page stride given; NULL: no cache
    int64_t page_stride, num_slots;
    int page_shift;
};

template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(1024) rope_kernel(const Params p) {
    using PT = Pack<T, VEC>;
    using PF = Pack<float, VEC>;
    const int64_t t = blockIdx.x;
    const int64_t pos = p.positions[t];
    const bool bad = pos < 0 || pos >= p.P;
    int64_t slot = -1;
    if (p.k_cache) {
        slot = p.slots[t];
        if (slot >= p.num_slots || bad) {
            if (slot >= p.num_slots && threadIdx.x == 0) raise_dev_error(DEV_ERR_BAD_INDEX);
            slot = -1;  // the token is not cached
        }
    }
    if (bad && threadIdx.x == 0) raise_dev_error(DEV_ERR_BAD_INDEX);
    const int64_t ps = (int64_t)1 << p.page_shift;
    const int64_t cache_at = slot < 0 ? 0 : (slot >> p.page_shift) * p.page_stride + (slot & (ps - 1)) * p.D;
    const int64_t cache_head = ps * p.D;

    const int half = p.rot / 2;
    const int U = half / VEC, C = U + (p.D - p.rot) / VEC;  // pair chunks, then copied chunks
    const int c = threadIdx.x % C, h0 = threadIdx.x / C, HG = blockDim.x / C;
    if (h0 < HG) {
        const bool pair = c < U;
        // elements of the thread's first and second access within a head
        const int e0 = !pair ? p.rot + (c - U) * VEC : HALF ? c * VEC : 2 * c * VEC;
        const int e1 = !pair ? e0 : HALF ? half + c * VEC : 2 * c * VEC + VEC;
        PF cs, sn;
        if (pair && !bad) {
            cs = *reinterpret_cast<const PF *>(p.table + pos * p.rot + c * VEC);
            sn = *reinterpret_cast<const PF *>(p.table + pos * p.rot + half + c * VEC);
        }
        for (int h = h0; h < p.Hq + p.Hk; h += HG) {
            const bool isq = h < p.Hq;
            const T *src = isq ? reinterpret_cast<const T *>(p.q) + t * p.q_token + h * p.q_head
                               : reinterpret_cast<const T *>(p.k) + t * p.k_token + (h - p.Hq) * p.k_head;
            T *dst;
            if (isq) dst = reinterpret_cast<T *>(p.q_out) + (t * p.Hq + h) * p.D;
            else if (p.k_cache) dst = reinterpret_cast<T *>(p.k_cache) + cache_at + (h - p.Hq) * cache_head;
            else dst = reinterpret_cast<T *>(p.k_out) + (t * p.Hk + (h - p.Hq)) * p.D;
            if (!isq && p.k_cache && slot < 0) continue;
            PT a, b;
            if (bad) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    from_f(a.v[e], 0.f);
                    from_f(b.v[e], 0.f);
                }
            } else {
                a = *reinterpret_cast<const PT *>(src + e0);
                if (pair) b = *reinterpret_cast<const PT *>(src + e1);
            }
            if (pair && !bad) {
                if (HALF || VEC == 1) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float x = to_f(a.v[e]), y = to_f(b.v[e]);
                        from_f(a.v[e], x * cs.v[e] - y * sn.v[e]);
                        from_f(b.v[e], y * cs.v[e] + x * sn.v[e]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        PT &w = e < VEC / 2 ? a : b;
                        const int i = 2 * e % VEC;
                        const float x = to_f(w.v[i]), y = to_f(w.v[i + 1]);
                        from_f(w.v[i], x * cs.v[e] - y * sn.v[e]);
                        from_f(w.v[i + 1], y * cs.v[e] + x * sn.v[e]);
                    }
                }
            }
            *reinterpret_cast<PT *>(dst + e0) = a;
            if (pair) *reinterpret_cast<PT *>(dst + e1) = b;
        }
    }
    if (slot >= 0) {
        const int per = p.D / VEC;
        for (int i = threadIdx.x; i < p.Hk * per; i += blockDim.x) {
            const int h = i / per, e = (i - h * per) * VEC;
            *reinterpret_cast<PT *>(reinterpret_cast<T *>(p.v_cache) + cache_at + h * cache_head + e) =
                *reinterpret_cast<const PT *>(reinterpret_cast<const T *>(p.v) + t * p.v_token + h * p.v_head + e);
        }
    }
}

template <typename T>
static int launch(const Params &p, int64_t tokens, bool half, bool vec, cudaStream_t st) {
    const int VEC = vec ? 8 : 1;
    const int C = p.rot / 2 / VEC + (p.D - p.rot) / VEC;
    int nt = C * (p.Hq + p.Hk);
    if (nt > 256) nt = 256;
    if (nt < C) nt = C;
    nt = (nt + 31) / 32 * 32;
    const unsigned grid = (unsigned)tokens;
    if (vec && half) rope_kernel<T, 8, true><<<grid, nt, 0, st>>>(p);
    else if (vec) rope_kernel<T, 8, false><<<grid, nt, 0, st>>>(p);
    else if (half) rope_kernel<T, 1, true><<<grid, nt, 0, st>>>(p);
    else rope_kernel<T, 1, false><<<grid, nt, 0, st>>>(p);
    QL_CUDA_TRY(cudaGetLastError());
    return QL_OK;
}

}  // namespace ropek

int launch_rope(const ropek::Params &p, int dtype, int64_t tokens, bool half, bool vec, cudaStream_t st) {
    if (dtype == QL_F32) return ropek::launch<float>(p, tokens, half, vec, st);
    if (dtype == QL_BF16) return ropek::launch<__nv_bfloat16>(p, tokens, half, vec, st);
    return ropek::launch<__half>(p, tokens, half, vec, st);
}

}  // namespace ql
