// rope.cu -- rotary positions on q and k, and the append of k and v to a paged cache.
//     (a, b) -> (a cos - b sin, b cos + a sin)
// for the pairs (i, i + rot/2) of a head (half layout) or (2i, 2i + 1) (interleaved), i <
// rot/2; elements past rot are copied.  The angles come from a table of fp32 rows [cos | sin],
// one per position, so any scaling of the frequencies and any axis split is a table and long
// positions keep the accuracy the table was computed with.  fp32 arithmetic, one rounding.
//
// Bound: HBM (q, k, v read once, q and the cache lines written once).  Split: one CTA per
// token; a thread owns one chunk of pairs and walks over the heads with it, so it reads its
// cosines and sines once; its first chunks are loaded before the position is known.  Measured: 4096
// tokens, 24 / 8 heads of 128, with the append 19.1 us = 4.51 TB/s (128 threads; 256 threads 24 us;
// CTAs that walk over tokens with positions fetched ahead 25 - 27 us).  Bound then: latency, 7 CTAs of
// 128 threads an SM (68 registers in bf16).  VEC = 8 moves 16 or 32 bytes per access; VEC = 1 takes
// any alignment and any even rot.
#include "pdl.cuh"

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
__global__ void __launch_bounds__(VEC == 8 ? 256 : 1024) rope_kernel(const Params p) {
    using PT = Pack<T, VEC>;
    using PF = Pack<float, VEC>;
    pdl_trigger();
    pdl_wait();
    const int64_t t = blockIdx.x;
    const int half = p.rot / 2;
    const int U = half / VEC, C = U + (p.D - p.rot) / VEC;  // pair chunks, then copied chunks
    const int c = threadIdx.x % C, h0 = threadIdx.x / C, HG = blockDim.x / C, heads = p.Hq + p.Hk;
    const bool pair = c < U;
    // elements of the thread's first and second access within a head
    const int e0 = !pair ? p.rot + (c - U) * VEC : HALF ? c * VEC : 2 * c * VEC;
    const int e1 = HALF ? half + c * VEC : 2 * c * VEC + VEC;
    auto load = [&](int h, PT &a, PT &b) {
        const T *src = h < p.Hq ? reinterpret_cast<const T *>(p.q) + t * p.q_token + h * p.q_head
                                : reinterpret_cast<const T *>(p.k) + t * p.k_token + (h - p.Hq) * p.k_head;
        a = *reinterpret_cast<const PT *>(src + e0);
        if (pair) b = *reinterpret_cast<const PT *>(src + e1);
    };
    const int v_per = p.D / VEC, v_all = p.k_cache ? p.Hk * v_per : 0;
    auto load_v = [&](int i) {
        const int h = i / v_per;
        return *reinterpret_cast<const PT *>(reinterpret_cast<const T *>(p.v) + t * p.v_token + h * p.v_head + (i - h * v_per) * VEC);
    };
    // the first chunks are in flight while the position and its table row are fetched
    const bool busy = h0 < HG && h0 < heads;
    PT a, b, w;
    if (busy) load(h0, a, b);
    if ((int)threadIdx.x < v_all) w = load_v(threadIdx.x);

    const int64_t pos = p.positions[t];
    int64_t slot = p.k_cache ? p.slots[t] : -1;
    const bool bad = pos < 0 || pos >= p.P;
    if ((bad || slot >= p.num_slots) && threadIdx.x == 0 && (bad || p.k_cache)) raise_dev_error(DEV_ERR_BAD_INDEX);
    if (bad || slot >= p.num_slots) slot = -1;  // the token is not cached
    const int64_t ps = (int64_t)1 << p.page_shift;
    const int64_t cache_at = slot < 0 ? 0 : (slot >> p.page_shift) * p.page_stride + (slot & (ps - 1)) * p.D;
    const int64_t cache_head = ps * p.D;

    if (busy) {
        PF cs, sn;
        if (pair && !bad) {
            cs = *reinterpret_cast<const PF *>(p.table + pos * p.rot + c * VEC);
            sn = *reinterpret_cast<const PF *>(p.table + pos * p.rot + half + c * VEC);
        }
        for (int h = h0;;) {
            const int next = h + HG;
            PT na, nb;
            if (next < heads) load(next, na, nb);
            if (bad) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    from_f(a.v[e], 0.f);
                    from_f(b.v[e], 0.f);
                }
            } else if (pair) {
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
                        PT &z = e < VEC / 2 ? a : b;
                        const int i = 2 * e % VEC;
                        const float x = to_f(z.v[i]), y = to_f(z.v[i + 1]);
                        from_f(z.v[i], x * cs.v[e] - y * sn.v[e]);
                        from_f(z.v[i + 1], y * cs.v[e] + x * sn.v[e]);
                    }
                }
            }
            T *dst;
            if (h < p.Hq) dst = reinterpret_cast<T *>(p.q_out) + (t * p.Hq + h) * p.D;
            else if (p.k_cache) dst = reinterpret_cast<T *>(p.k_cache) + cache_at + (h - p.Hq) * cache_head;
            else dst = reinterpret_cast<T *>(p.k_out) + (t * p.Hk + (h - p.Hq)) * p.D;
            if (h < p.Hq || !p.k_cache || slot >= 0) {
                *reinterpret_cast<PT *>(dst + e0) = a;
                if (pair) *reinterpret_cast<PT *>(dst + e1) = b;
            }
            if (next >= heads) break;
            h = next, a = na, b = nb;
        }
    }
    for (int i = threadIdx.x; i < v_all && slot >= 0; i += blockDim.x) {
        if (i != (int)threadIdx.x) w = load_v(i);
        const int h = i / v_per;
        *reinterpret_cast<PT *>(reinterpret_cast<T *>(p.v_cache) + cache_at + h * cache_head + (i - h * v_per) * VEC) = w;
    }
}

template <typename T>
static int launch(const Params &p, int64_t tokens, bool half, bool vec, cudaStream_t st) {
    const int VEC = vec ? 8 : 1;
    const int C = p.rot / 2 / VEC + (p.D - p.rot) / VEC;
    int nt = C * (p.Hq + p.Hk);
    if (nt > 128) nt = 128;
    if (nt < C) nt = C;
    nt = (nt + 31) / 32 * 32;
    const unsigned grid = (unsigned)tokens;
    auto kernel = vec ? (half ? rope_kernel<T, 8, true> : rope_kernel<T, 8, false>)
                      : (half ? rope_kernel<T, 1, true> : rope_kernel<T, 1, false>);
    QL_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(nt), 0, st, 1, p));
    return QL_OK;
}

}  // namespace ropek

int launch_rope(const ropek::Params &p, int dtype, int64_t tokens, bool half, bool vec, cudaStream_t st) {
    if (dtype == QL_F32) return ropek::launch<float>(p, tokens, half, vec, st);
    if (dtype == QL_BF16) return ropek::launch<__nv_bfloat16>(p, tokens, half, vec, st);
    return ropek::launch<__half>(p, tokens, half, vec, st);
}

}  // namespace ql
