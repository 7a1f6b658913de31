// attn_rows.cu -- paged attention for few rows per kv head: single tokens and short drafts
// (rows = new tokens x heads of a group, up to 16 at a time; more rows run as more CTAs).
//
// Bound: HBM -- every cached key and value is read once per kv head and 16 rows.  So the
// kernel is built around the loads: each of a CTA's four or eight warps walks its own blocks of 16
// positions with its own ring of cp.async stages, with no barrier between the warps until the
// end, and CTAs split a long axis (joined by join_kernel).  16 rows are one m16 tile of
// mma.sync, whose operand layouts let the scores become the second product's operand in
// registers; a 128-row tcgen05 tile would spend its softmax on rows that do not exist.
// Softmax: running maximum and sum per row in fp32, weights 2^(s - max) <= 1 (in f16 times 2^15:
// kWeightShift) rounded to the cache's type for the second product, the sum taken before that rounding.
//
// Measured (24 / 8 heads of 128, a graph's replay): 64 sequences of 311 - 8003 positions 178 us = 6.14
// TB/s (189 in calls back to back), 2 x 131k positions 181 us = 5.92 TB/s (a copy: 6.56 TB/s), one
// sequence of 777 positions 6.9 us.
//
// Positions that no row of the CTA sees are zero-filled in shared memory, whatever the cache
// holds there (a page's unused tail may hold anything); scores of positions that a row does
// not see are replaced by -inf.
#include "attn_common.cuh"

namespace ql {
namespace attn {

constexpr int RKV = 16;  // positions of one warp step

// ALONE: a CTA of eight warps that takes an SM's shared memory by itself (D = 256: four warps in
// both cases), for one wave of CTAs.  Of four warps, two that would fit one to an SM each share
// one while another SM idles (2 x 131k positions in 144 pieces: 221 us); kept apart by padding
// they take 177 us, and 198 where the power cap lowers the clock; of eight warps 180 in both.
template <int D, bool ALONE>
struct RowsCfg {
    static constexpr int RW = ALONE && D < 256 ? 8 : 4;  // warps
    static constexpr int ROW_BYTES = D * 2 + 16;  // padded: ldmatrix reads 8 rows free of bank conflicts
    static constexpr int TILE_BYTES = RKV * ROW_BYTES;
    // stages so that two CTAs of four warps (one for D = 256) fill an SM's shared memory
    static constexpr int STAGES = D == 64 ? 6 : D == 96 ? 4 : 3;
    static constexpr int WARP_BYTES = STAGES * 2 * TILE_BYTES;
    static constexpr int SMEM = RW * WARP_BYTES;
    static_assert((RW + 1) * ROWS_TILE * (D + 2) * 4 <= SMEM, "the warps' and the CTA's results fit in the ring");
};

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_t(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// One stretch of positions [lo, hi) for one row block of a (sequence, kv head).  Its result is
// partial result number `slot` of `slots`, or the output itself where slots is 1 (and not CLUSTER).
template <typename T, int D, bool CLUSTER, bool ALONE>
__device__ __forceinline__ void rows_stretch(const Params &p, const Seq &s, int b, int kvh, int rb, int lo, int hi, int slot,
                                             int slots, uint8_t *smem) {
    using C = RowsCfg<D, ALONE>;
    constexpr int RW = C::RW;
    constexpr float SHIFT = kWeightShift<T, 0>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = s.q_len * p.G, r0 = rb * ROWS_TILE, nrows = min(ROWS_TILE, rows - r0);

    // this thread's two rows, g and g + 8, and what they see
    const int g = lane >> 2, t4 = lane & 3;
    int rlo[2], rhi[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        if (r < nrows) visible(p, s, (r0 + r) / p.G, rlo[i], rhi[i]);
        else rlo[i] = rhi[i] = 0;
    }

    // q as the first product's A fragments
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        const bool in = r < nrows;
        const int tok = in ? (r0 + r) / p.G : 0, hd = in ? kvh * p.G + (r0 + r) % p.G : 0;
        const uint16_t *qp = reinterpret_cast<const uint16_t *>(p.q) + (s.q0 + (int64_t)tok) * p.q_token + hd * p.q_head;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qf[k][i] = in ? *reinterpret_cast<const uint32_t *>(qp + k * 16 + t4 * 2) : 0u;
            qf[k][i + 2] = in ? *reinterpret_cast<const uint32_t *>(qp + k * 16 + t4 * 2 + 8) : 0u;
        }
    }

    float o[D / 8][4], m[2] = {NEG_INF, NEG_INF}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;

    const int blk0 = lo / RKV, nblk = hi > lo ? (hi + RKV - 1) / RKV - blk0 : 0;
    const int mine = nblk > warp ? (nblk - warp + RW - 1) / RW : 0;  // blocks blk0 + warp + i * RW
    const uint32_t ring = smem_u32(smem) + warp * C::WARP_BYTES;
    const int64_t head_at = (int64_t)kvh * ((int64_t)D << p.page_shift);
    const int in_page = (1 << p.page_shift) - 1;

    auto issue = [&](int i, int page) {  // block i of this warp into its stage
        const int pos = (blk0 + warp + i * RW) * RKV;
        const uint32_t ks = ring + (i % C::STAGES) * 2 * C::TILE_BYTES, vs = ks + C::TILE_BYTES;
        const int64_t at = page * p.page_stride + head_at + (int64_t)(pos & in_page) * D;
        const uint16_t *kp = reinterpret_cast<const uint16_t *>(p.k_cache) + at;
        const uint16_t *vp = reinterpret_cast<const uint16_t *>(p.v_cache) + at;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            const int idx = j * 32 + lane, row = idx / (D / 8), col = idx % (D / 8);
            const bool in = pos + row >= lo && pos + row < hi;
            cp_async16(ks + row * C::ROW_BYTES + col * 16, kp + row * D + col * 8, in);
            cp_async16(vs + row * C::ROW_BYTES + col * 16, vp + row * D + col * 8, in);
        }
    };
    auto page_at = [&](int i) { return i < mine ? page_of(p, b, (blk0 + warp + i * RW) * RKV) : 0; };

    int pages[C::STAGES];
#pragma unroll
    for (int i = 0; i < C::STAGES; ++i) pages[i] = page_at(i);
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; ++i) {
        if (i < mine) issue(i, pages[i]);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int next_page = pages[C::STAGES - 1];

    for (int i = 0; i < mine; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
        __syncwarp();  // every lane's part of the block has landed; the oldest stage is free
        const int ahead = i + C::STAGES - 1;
        if (ahead < mine) issue(ahead, next_page);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next_page = page_at(ahead + 1);

        const uint32_t ks = ring + (i % C::STAGES) * 2 * C::TILE_BYTES, vs = ks + C::TILE_BYTES;
        float sc[2][4] = {};
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            uint32_t kb[4];
            ldmatrix_x4(kb, ks + ((lane & 7) + ((lane >> 4) & 1) * 8) * C::ROW_BYTES + k * 32 + ((lane >> 3) & 1) * 16);
            mma16816<T>(sc[0], qf[k], kb[0], kb[1]);
            mma16816<T>(sc[1], qf[k], kb[2], kb[3]);
        }
        const int pos = (blk0 + warp + i * RW) * RKV + t4 * 2;
        float mx[2] = {NEG_INF, NEG_INF};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = pos + n * 8 + (e & 1), r = e >> 1;
                const bool in = at >= max(rlo[r], lo) && at < min(rhi[r], hi);
                sc[n][e] = in ? sc[n][e] * p.scale_log2 : NEG_INF;
                mx[r] = fmaxf(mx[r], sc[n][e]);
            }
        float f[2], base[2];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            const float nm = fmaxf(m[r], mx[r]);
            moved |= nm != m[r];
            base[r] = nm == NEG_INF ? 0.f : nm;  // nothing seen yet: every weight is 2^-inf = 0
            f[r] = ex2(m[r] - base[r]);
            base[r] -= SHIFT;
            m[r] = nm;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
                o[n][0] *= f[0];
                o[n][1] *= f[0];
                o[n][2] *= f[1];
                o[n][3] *= f[1];
            }
            l[0] *= f[0];
            l[1] *= f[1];
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sc[n][e] = ex2(sc[n][e] - base[e >> 1]);
                l[e >> 1] += sc[n][e];
            }
        const uint32_t pf[4] = {pack2<T>(sc[0][0], sc[0][1]), pack2<T>(sc[0][2], sc[0][3]),
                                pack2<T>(sc[1][0], sc[1][1]), pack2<T>(sc[1][2], sc[1][3])};
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            uint32_t vb[4];
            ldmatrix_x4_t(vb, vs + ((lane & 7) + ((lane >> 3) & 1) * 8) * C::ROW_BYTES + n * 32 + ((lane >> 4) & 1) * 16);
            mma16816<T>(o[2 * n], pf, vb[0], vb[1]);
            mma16816<T>(o[2 * n + 1], pf, vb[2], vb[3]);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }

    // the warps' results meet in the ring's memory
    __syncthreads();
    float *so = reinterpret_cast<float *>(smem);        // [RW][16][D]
    float *sm = so + RW * ROWS_TILE * D, *sl = sm + RW * ROWS_TILE;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2 *>(so + (warp * ROWS_TILE + r) * D + n * 8 + t4 * 2) =
                make_float2(o[n][2 * i], o[n][2 * i + 1]);
        if (t4 == 0) {
            sm[warp * ROWS_TILE + r] = m[i];
            sl[warp * ROWS_TILE + r] = l[i];
        }
    }
    __syncthreads();
    const int64_t row0 = s.q0 * (int64_t)p.Hq + kvh * p.G;
    auto row_at = [&](int r) { return row0 + (int64_t)((r0 + r) / p.G) * p.Hq + (r0 + r) % p.G; };
    float *jo = sl + RW * ROWS_TILE, *jl = jo + ROWS_TILE * D;  // CLUSTER: this CTA's [16][D] and its lse
    for (int idx = threadIdx.x; idx < nrows * (D / 4); idx += RW * 32) {
        const int r = idx / (D / 4), e = idx % (D / 4) * 4;
        float mx = NEG_INF;
#pragma unroll
        for (int w = 0; w < RW; ++w) mx = fmaxf(mx, sm[w * ROWS_TILE + r]);
        // (a maximum leaves NaN out: a warp whose scores are all NaN has -inf and a NaN sum, and 0 * NaN
        // carries it on; one that saw nothing adds zeros)
        const float base = mx == NEG_INF ? 0.f : mx;
        float total = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            const float f = ex2(sm[w * ROWS_TILE + r] - base);
            const float4 v = *reinterpret_cast<const float4 *>(so + (w * ROWS_TILE + r) * D + e);
            total += f * sl[w * ROWS_TILE + r];
            a.x += f * v.x;
            a.y += f * v.y;
            a.z += f * v.z;
            a.w += f * v.w;
        }
        const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
        a = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
        const float lse = total > 0.f || total != total ? mx + (log2f(total) - SHIFT) : NEG_INF;
        if (CLUSTER) {
            if (e == 0) jl[r] = lse;
            *reinterpret_cast<float4 *>(jo + r * D + e) = a;
        } else if (slots > 1) {
            const int64_t row = row_at(r);
            if (e == 0) p.part_lse[row * p.nsplit + slot] = lse;
            if (lse != NEG_INF) *reinterpret_cast<float4 *>(p.part_o + (row * p.nsplit + slot) * D + e) = a;
        } else {
            *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p.out) + row_at(r) * D + e) =
                make_uint2(pack2<T>(a.x, a.y), pack2<T>(a.z, a.w));
        }
    }
    if constexpr (CLUSTER) {
        cluster_sync_all();
        // every CTA joins its share of the rows' elements, in the order of the splits
        for (int idx = slot * RW * 32 + threadIdx.x; idx < nrows * (D / 4); idx += slots * RW * 32) {
            const int r = idx / (D / 4), e = idx % (D / 4) * 4;
            float mx = NEG_INF, lse[MAX_CLUSTER];
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; ++c) {
                lse[c] = c < slots ? ld_cluster(mapa_shared(smem_u32(jl + r), c)) : NEG_INF;
                mx = fmaxf(mx, lse[c]);
            }
            float total = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
            const float base = mx == NEG_INF ? 0.f : mx;
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; ++c) {
                if (lse[c] == NEG_INF) continue;
                const float f = ex2(lse[c] - base);
                const float4 v = ld_cluster4(mapa_shared(smem_u32(jo + r * D + e), c));
                total += f;
                a.x += f * v.x;
                a.y += f * v.y;
                a.z += f * v.z;
                a.w += f * v.w;
            }
            const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
            *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p.out) + row_at(r) * D + e) =
                make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
        }
        cluster_sync_all();  // no CTA leaves while another reads its shared memory
    }
}

// The positions of one split when a few sequences (up to 32) are to fill the SMs, whatever their
// lengths: of the candidates n = 1 .. nsplit pieces for the longest, the one whose waves of CTAs
// (one per SM) take the least time, a piece costing its positions and about 500 more.  Lane by
// lane, two candidates each.  (2 x 131k positions: 9 pieces in one wave 180 us, 64 fixed 203.)
__device__ __forceinline__ int adapted_chunk(const Params &p, int B) {
    const int lane = threadIdx.x & 31;
    int len = 0;
    if (lane < B) {
        const Seq s = load_seq(p, lane);
        if (s.ok && s.q_len > 0) {
            int lo, hi;
            visible_rows(p, s, 0, s.q_len * p.G, lo, hi);
            len = hi - (lo & ~127);
        }
    }
    int most = len;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    float best = INFINITY;
    int chunk = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int n = k * 32 + lane + 1;
        const int c = ((most + n - 1) / n + 63) & ~63;
        int pieces = 0;
        for (int b = 0; b < B; ++b) pieces += (__shfl_sync(0xffffffffu, len, b) + c - 1) / max(c, 1);
        const float cost = (float)((pieces * p.Hkv + kSMs - 1) / kSMs) * (float)(c + 500);
        if (n <= p.nsplit && cost < best) best = cost, chunk = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oc = __shfl_xor_sync(0xffffffffu, chunk, o);
        if (ob < best || (ob == best && oc > chunk)) best = ob, chunk = oc;
    }
    return max(chunk, 64);
}

// CLUSTER: the splits of a (sequence, kv head, row block) are one thread-block cluster and join
// through distributed shared memory: no partial results in global memory, no second launch.
// grid: kv head * rowblocks + row block, sequence and split; the split runs fastest (x) with
// CLUSTER and slowest (z) without, so that pieces which hold something come before empty ones and
// the first of them go one to an SM.
template <typename T, int D, bool CLUSTER, bool ALONE>
__global__ void __launch_bounds__(RowsCfg<D, ALONE>::RW * 32) rows_kernel(const Params p, int rowblocks) {
    extern __shared__ __align__(16) uint8_t smem[];
    pdl_trigger();
    pdl_wait();
    const int b = CLUSTER ? blockIdx.z : blockIdx.y, split = CLUSTER ? blockIdx.x : blockIdx.z;
    const int item = CLUSTER ? blockIdx.y : blockIdx.x, kvh = item / rowblocks, rb = item % rowblocks;
    const Seq s = load_seq(p, b);
    if (!s.ok) {
        if (threadIdx.x == 0) raise_dev_error(DEV_ERR_BAD_INDEX);
        return;
    }
    const int rows = s.q_len * p.G, r0 = rb * ROWS_TILE;
    if (r0 >= rows || rows > p.rows_kernel_most) return;
    int lo, hi;
    visible_rows(p, s, r0, min(rows, r0 + ROWS_TILE), lo, hi);
    take_split(p, split, ALONE ? adapted_chunk(p, gridDim.y) : p.chunk, lo, hi);
    if (!CLUSTER && p.nsplit > 1 && lo >= hi) {  // nothing in this split
        const int r = threadIdx.x;
        if (r < min(ROWS_TILE, rows - r0))
            p.part_lse[((s.q0 + (int64_t)((r0 + r) / p.G)) * p.Hq + kvh * p.G + (r0 + r) % p.G) * p.nsplit + split] = NEG_INF;
        return;
    }
    rows_stretch<T, D, CLUSTER, ALONE>(p, s, b, kvh, rb, lo, hi, split, p.nsplit, smem);
}

template <typename T, int D, bool CLUSTER, bool ALONE>
static int launch_rows_c(const Params &p, int64_t B, int rowblocks, cudaStream_t st) {
    using C = RowsCfg<D, ALONE>;
    auto kernel = rows_kernel<T, D, CLUSTER, ALONE>;
    static PerDeviceFlag configured;
    const int dev = current_device();
    if (!configured.test(dev)) {
        QL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        configured.set(dev);
    }
    const dim3 grid = CLUSTER ? dim3(p.nsplit, p.Hkv * rowblocks, (unsigned)B) : dim3(p.Hkv * rowblocks, (unsigned)B, p.nsplit);
    QL_CUDA_TRY(launch_pdl(kernel, grid, dim3(C::RW * 32), C::SMEM, st, CLUSTER ? p.nsplit : 1, p, rowblocks));
    return QL_OK;
}

template <typename T, int D>
static int launch_rows_t(const Params &p, int64_t B, int rowblocks, cudaStream_t st) {
    if (p.cluster) return launch_rows_c<T, D, true, false>(p, B, rowblocks, st);
    return p.adapt ? launch_rows_c<T, D, false, true>(p, B, rowblocks, st)
                   : launch_rows_c<T, D, false, false>(p, B, rowblocks, st);
}

}  // namespace attn
}  // namespace ql
