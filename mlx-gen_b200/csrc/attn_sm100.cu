// attn_sm100.cu -- paged attention for chunks of new tokens on the tcgen05 tensor cores.
//
// One CTA takes 256 packed rows (tokens x heads of a group) of one kv head as two tiles of
// 128, and walks over the positions they see in steps of 128:
//     S_t = Q_t K^T      (A = Q from shared memory, B = K, fp32 into TMEM)
//     P_t = 2^(c S_t - c m),  l_t += rowsum(P_t)      (one thread per row)
//     O_t += P_t V       (A = P from TMEM, B = V as stored, fp32 in TMEM)
// Each tile of keys and values is read from L2 once for 256 rows, and while one tile's
// scores are in the softmax the other tile's products run on the tensor core.
//
// Roles (384 threads): warps 0-3 and 4-7 softmax and epilogue of tile 0 and 1 (a thread owns
// a row, so the running maximum and sum need no shuffles); warp 8 loads K and V page by page
// (a TMA box per page and 64-element half, its lanes issue the pages of a step) and clears the
// V rows of the first and last step that no row of the CTA sees (a page's unused tail may hold
// anything, and 0 * inf is not 0); warps 9 and 10 issue the MMAs of tile 0 and 1 (two issuers:
// a commit holds up only its own tile); warp 11 only fills the third warpgroup.
//
// TMEM (512 columns): S_0, S_1 at 0 and 128, then O_0, O_1.  P_t (16-bit) overlays S_t once its
// thread holds the scores in registers; with D = 64 there is room for it beside S_t, and the next
// step's scores are computed while this step's are in the softmax.  Shared memory: Q_0, Q_1 and a ring of
// K / V stages in 128-byte swizzled rows of 64 elements.
//
// The running maximum is lazy: O and l are rescaled only when a row's maximum rises by more
// than 2^8 over the one in use; until then the weights may exceed 1 (by up to 2^8, for which every
// format has room; f16 takes the rest of its range for small weights, kWeightShift), which the
// final division by l cancels.  O is rescaled by the softmax
// threads: S_t of step j is committed after O_t of step j - 1, so seeing it means O_t is at
// rest.  The same order lets S_t of step j + 1 overwrite P_t of step j: both products are
// issued by one thread and execute in order.
//
// Bound: the chain scores -> softmax -> product of a tile, about 3700 cycles a step of 128 positions
// for D = 128 (softmax 2050, of it 1024 at least in the special-function unit; products 1650), on
// which two tiles alternate; the tensor pipe and the special-function unit are each 52 % active.
// TMEM has no room for a third tile's S and O; the 64 columns of S_t that P_t leaves free are unused.
// Measured (24 / 8 heads of 128): 512 tokens over 16021 positions 101 us = 1013 TFLOP/s in a graph's
// replay and 115 us = 887 in calls back to back, where the power cap lowers the clock; 4096 tokens causal
// 114 us = 902 and 123 us = 836; cuBLAS reaches 1644 TFLOP/s in bf16.  With sinks: 1024 tokens over 30011 positions, window 4096
// and 64 sinks, 79 us; 4096 tokens, window 1024 and 4 sinks, 74 us; 17 chunks of heads of 64, window 256 and 16 sinks, 50 us.
#include "attn_common.cuh"

namespace ql {
namespace attn {

constexpr int TQ = 128, TKV = 128;
constexpr int PFIRST = 96;  // positions of P_t handed over first: O_t's product starts under the last weights
constexpr int SM100_THREADS = 384;
constexpr int SM100_ROWS = 2 * TQ;  // rows of a CTA

template <int D>
struct Sm100Cfg {
    static constexpr int HALVES = D / 64;
    static constexpr int HALF_BYTES = 128 * 128;           // 128 rows of 64 elements
    static constexpr int TILE_BYTES = HALVES * HALF_BYTES;  // of Q, K or V
    static constexpr int STAGES = D == 128 ? 5 : 8;
    // TMEM columns: S_t at 128 t, O_t next, and for D = 64 what is left is enough for P_t beside S_t
    static constexpr bool P_APART = D == 64;
    static constexpr int COL_O = 256, COL_P = P_APART ? 256 + 2 * D : 0, P_STEP = P_APART ? TKV / 2 : TKV;
    static constexpr int SMEM_Q = 0, SMEM_KV = 2 * TILE_BYTES;
    static constexpr int SMEM_BAR = SMEM_KV + STAGES * TILE_BYTES;
    static constexpr int NBAR = 2 * STAGES + 2 * 8 + 3;
    static constexpr int SMEM = SMEM_BAR + NBAR * 8 + 16 + 1024;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2,
                                            int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
        "[%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// the n lowest bits (none for n <= 0, all for n >= 32)
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

// Barrier 1: the loader and the issuers (and warp 11) wait until every role is done, so that none sets the
// abort flag any more; the softmax warps only arrive.
__device__ __forceinline__ void roles_done() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(SM100_THREADS) : "memory"); }
__device__ __forceinline__ void softmax_done() { asm volatile("barrier.cta.arrive 1, %0;" ::"n"(SM100_THREADS) : "memory"); }

// 32 bytes in one store: a whole DRAM sector of a thread's own row
__device__ __forceinline__ void st_global_32(void *dst, const uint32_t v[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// V as stored is [position][element]: for O = P V its N axis (elements) is the contiguous one.
// Swizzled MN-major operand: 64-element atoms along N are HALF_BYTES apart (leading offset),
// groups of 8 positions 1024 bytes apart (stride offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t n_atom_bytes) {
    return umma_desc_k_sw128(smem_addr) - ((uint64_t)1 << 16) + ((uint64_t)(n_atom_bytes >> 4) << 16);
}

template <typename T>
__host__ __device__ constexpr uint32_t attn_idesc(int N, bool b_mn_major) {
    // D f32; A and B both of T (bf16 = 1, f16 = 0); bit 16: B is MN-major
    return (1u << 4) | (sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? (1u << 7) | (1u << 10) : 0u) |
           (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(TQ >> 4) << 24);
}

template <typename T, int D, bool SINKS>
__global__ void __launch_bounds__(SM100_THREADS, 1)
    sm100_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
    using C = Sm100Cfg<D>;
    constexpr int STAGES = C::STAGES;
    // with P_t beside S_t the next scores are ready early and the tiles' softmaxes overlap freely
    // (with turns the same: 89 us on the mixed batch either way)
    constexpr bool TURNS = !C::P_APART;
    constexpr float SHIFT = kWeightShift<T, 8>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::SMEM_BAR);  // K / V stage landed
    uint64_t *empty = full + STAGES;   // stage read by every tile's MMAs
    uint64_t *qfull = empty + STAGES;  // [2] Q_t written
    uint64_t *sfull = qfull + 2;       // [2] S_t of the step computed (and O_t of the step before)
    uint64_t *pfull = sfull + 2;       // [2][2] P_t written: its first PFIRST positions, the rest
    uint64_t *ofull = pfull + 4;       // [2] O_t complete (P_APART: of the step)
    uint64_t *drain = ofull + 2;       // [2] an aborted tile's MMAs are done
    uint64_t *turn = drain + 2;        // [2] the other tile's exponentials of the step are done
    uint64_t *sread = turn + 2;        // [2] S_t of the step is in registers (P_APART)
    uint64_t *vfix = sread + 2;        // [3] V of the last step of the gap before the window / of the last / of the gap's other step cleared where no row sees it
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(vfix + 3);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const Seq s = load_seq(p, blockIdx.z);
    if (!s.ok) {
        if (threadIdx.x == 0) raise_dev_error(DEV_ERR_BAD_INDEX);
        return;
    }
    const int b = blockIdx.z, kvh = blockIdx.x % p.Hkv, split = blockIdx.x / p.Hkv;
    const int rows = s.q_len * p.G;
    // with `causal` the last tiles see most: they start first
    const int row0 = (p.causal ? gridDim.y - 1 - blockIdx.y : blockIdx.y) * SM100_ROWS;
    if (row0 >= rows || rows <= p.rows_kernel_most) return;
    const int nrows = min(SM100_ROWS, rows - row0), ntiles = nrows > TQ ? 2 : 1;

    int vlo, vhi, unused;
    visible(p, s, row0 / p.G, vlo, unused);
    visible(p, s, (row0 + nrows - 1) / p.G, unused, vhi);
    take_split(p, split, p.chunk, vlo, vhi);
    if (vhi <= vlo) {  // nothing to see: no partial result, or zeros
        for (int idx = threadIdx.x; idx < nrows; idx += SM100_THREADS) {
            const int r = row0 + idx;
            const int64_t row = (s.q0 + (int64_t)(r / p.G)) * p.Hq + kvh * p.G + r % p.G;
            if (p.nsplit > 1) p.part_lse[row * p.nsplit + split] = NEG_INF;
            else
                for (int e = 0; e < D / 8; ++e) reinterpret_cast<uint4 *>(p.out)[row * (D / 8) + e] = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    // The steps go over places.  Without sinks a place is its position; with SINKS, first come the sinks in whole
    // blocks of 16 (`lead` of them; by the first split, and only if the window begins behind them), then
    // the window's positions from its block of 16 on, each `shift` lower than its place.
    [[maybe_unused]] int lead = 0, shift = 0, sunk = 0, gap0 = 0, gap = 0;  // (places below `sunk` are sinks)
    [[maybe_unused]] bool fix_lead = false;
    if constexpr (SINKS) {
        int origin = vlo & ~15;
        if (split == 0) {
            if (p.sinks < origin) lead = (p.sinks + 15) & ~15;
            else origin = 0;
        }
        shift = lead - origin;
        sunk = lead ? p.sinks : p.sinks - origin;
        vlo += shift, vhi += shift;
        // the places up to the window that no row sees lie in one step or in two
        gap0 = max(sunk, 0) / TKV, gap = (vlo - 1) / TKV;
        fix_lead = sunk < vlo && gap0 < gap;
    }
    const int t0 = SINKS ? 0 : vlo / TKV, n = (vhi + TKV - 1) / TKV - t0;
    const bool fix_first = vlo > (SINKS ? max(sunk, 0) : t0 * TKV), fix_last = vhi < (t0 + n) * TKV;
    const int jf = SINKS && fix_first ? gap : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], ntiles);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&qfull[t], TQ);
            mbar_init(&sfull[t], 1);
            mbar_init(&pfull[2 * t], 4);
            mbar_init(&pfull[2 * t + 1], 4);
            mbar_init(&ofull[t], 1);
            mbar_init(&drain[t], 1);
            mbar_init(&turn[t], 4);
            mbar_init(&sread[t], 4);
            mbar_init(&vfix[t], 1);
        }
        if constexpr (SINKS) mbar_init(&vfix[2], 1);
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tm_k);
        prefetch_tmap(&tm_v);
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // only now: a dependent kernel that allocates tensor memory before its own wait must not take
    // it from a CTA of this one
    pdl_trigger();

    // registers: 3 warpgroups x 168 at launch = 2 x 216 + 72 (a softmax thread holds 128 scores)
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int t = warp >> 2;
        if (t < ntiles) {
            // ------------------------------------------------------------ softmax of tile t
            const int tid = threadIdx.x & 127;  // == row of the tile == TMEM lane
            {
                // Q_t by asynchronous copies of 16 bytes, rows past the end as zeros; a thread's rows
                // are 128 / CPR apart, so token and head advance without a division
                constexpr int CPR = D / 8, STEP = 128 / CPR;
                const uint32_t qs = smem_u32(smem + C::SMEM_Q + t * C::TILE_BYTES);
                const int c = tid % CPR, step_tok = STEP / p.G, step_g = STEP % p.G;
                int rr = tid / CPR, gr = row0 + t * TQ + rr, tok = gr / p.G, g = gr % p.G;
#pragma unroll
                for (int i = 0; i < CPR; ++i) {
                    const bool in = gr < rows;
                    const uint16_t *src = reinterpret_cast<const uint16_t *>(p.q) +
                                          (in ? (s.q0 + (int64_t)tok) * p.q_token + (kvh * p.G + g) * p.q_head + c * 8 : 0);
                    cp_async16(qs + (c >> 3) * C::HALF_BYTES + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), src, in);
                    rr += STEP, gr += STEP, tok += step_tok, g += step_g;
                    if (g >= p.G) g -= p.G, ++tok;
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&qfull[t]);
            }
            const int r = row0 + t * TQ + tid;
            int rlo = 0, rhi = 0, min_hi, max_lo;
            if (r < rows) visible(p, s, r / p.G, rlo, rhi);
            // a step inside [max_lo, min_hi) is seen whole by every row of the tile
            visible(p, s, (row0 + t * TQ) / p.G, unused, min_hi);
            visible(p, s, min(rows - 1, row0 + t * TQ + TQ - 1) / p.G, max_lo, unused);
            if constexpr (SINKS) min_hi += shift, max_lo += shift, rlo += shift, rhi += shift;
            min_hi = min(min_hi, vhi);
            max_lo = max(max_lo, vlo);
            rlo = max(rlo, vlo);
            rhi = min(rhi, vhi);

            const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            const uint32_t s_col = lane_base + t * TKV, o_col = lane_base + C::COL_O + t * D;
            const uint32_t p_col = lane_base + C::COL_P + t * C::P_STEP;
            const float c = p.scale_log2;
            float m = NEG_INF, l = 0.f;  // reference maximum (of unscaled scores) in use, sum
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                ok = __all_sync(0xffffffffu, mbar_wait(&sfull[t], j & 1, abort_flag, DEV_ERR_TIMEOUT_FULL));
                if (!ok) break;
                tc_fence_after();
                if (tid == 0) {  // K of this step and V of the step before have been read
                    mbar_arrive(&empty[(2 * j) % STAGES]);
                    if (!C::P_APART && j > 0) mbar_arrive(&empty[(2 * j - 1) % STAGES]);
                }
                __syncwarp();
                float sc[TKV];
#pragma unroll
                for (int i = 0; i < TKV / 32; ++i) tmem_ld32(s_col + i * 32, reinterpret_cast<uint32_t *>(sc) + i * 32);
                tmem_ld_wait();
                if constexpr (C::P_APART) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sread[t]);
                }
                const int kv0 = (t0 + j) * TKV;
                // a step that some row of the tile does not see whole (the same for all its threads)
                if (kv0 < max_lo || kv0 + TKV > min_hi) {
#pragma unroll
                    for (int w = 0; w < TKV / 32; ++w) {  // one bit per position: two instructions a score
                        uint32_t see = bits_below(rhi - kv0 - w * 32) & ~bits_below(rlo - kv0 - w * 32);
                        if constexpr (SINKS) see |= bits_below(min(rhi, sunk) - kv0 - w * 32);
#pragma unroll
                        for (int i = 0; i < 32; ++i) sc[w * 32 + i] = (see & (1u << i)) ? sc[w * 32 + i] : NEG_INF;
                    }
                }
                float mx[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
                for (int i = 4; i < 124; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], sc[i + 2 * k], sc[i + 2 * k + 1]);
#pragma unroll
                for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], sc[124 + k]);
                if (C::P_APART && j > 0) {  // O_t of the step before: P_t and its V stage are free, O_t is at rest
                    ok = __all_sync(0xffffffffu, mbar_wait(&ofull[t], (j - 1) & 1, abort_flag, DEV_ERR_TIMEOUT_ACC));
                    if (!ok) break;
                    tc_fence_after();
                    if (tid == 0) mbar_arrive(&empty[(2 * j - 1) % STAGES]);
                    __syncwarp();
                }
                const float nm = max3(max3(mx[0], mx[1], mx[2]), mx[3], m);
                const bool grow = (nm - m) * c > 8.f;  // also from -inf; false while nothing is seen (nan)
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? ex2((m - nm) * c) : 1.f;
                    if (grow) m = nm;
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int i = 0; i < D / 32; ++i) {
                            uint32_t o[32];
                            tmem_ld32(o_col + i * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st32(o_col + i * 32, o);
                        }
                    }
                }
                const float base = m == NEG_INF ? 0.f : m * c;
                // the tiles take turns: tile 1 follows tile 0's step, tile 0 tile 1's step before
                if (TURNS && ntiles == 2 && (t == 1 || j > 0)) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&turn[t], (t == 1 ? j : j - 1) & 1, abort_flag, DEV_ERR_TIMEOUT_ACC));
                    if (!ok) break;
                }
                const uint64_t c2 = f2_make(c, c), nb2 = f2_make(SHIFT - base, SHIFT - base);
                auto hand_over = [&](int h) {  // P_t's positions so far are in TMEM
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&pfull[2 * t + h]);
                };
                uint64_t sum[2] = {0ull, 0ull};
                // pairs of scores in flight: x2 of pair i + AHEAD is made while pair i is in the
                // special-function unit, so that unit, which bounds the loop, does not wait
                constexpr int AHEAD = 2;
                uint64_t x2[AHEAD];
                uint32_t pk[16];
                auto pair = [&](int i) { return f2_fma(f2_make(sc[2 * i], sc[2 * i + 1]), c2, nb2); };
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) x2[i] = pair(i);
                float px, py;
#pragma unroll
                for (int i = 0; i < TKV / 2; ++i) {
                    float x, y;
                    f2_split(x2[i % AHEAD], x, y);
                    x = ex2(x), y = ex2(y);
                    if (i + AHEAD < TKV / 2) x2[i % AHEAD] = pair(i + AHEAD);
                    if (i > 0) {
                        sum[i & 1] = f2_add(sum[i & 1], f2_make(px, py));
                        pk[(i - 1) & 15] = pack2<T>(px, py);
                        if (((i - 1) & 15) == 15) tmem_st16(p_col + (i - 16), pk);
                    }
                    if (i == PFIRST / 2) hand_over(0);
                    px = x, py = y;
                }
                sum[0] = f2_add(sum[0], f2_make(px, py));
                pk[15] = pack2<T>(px, py);
                tmem_st16(p_col + TKV / 2 - 16, pk);
                hand_over(1);
                if (TURNS && lane == 0 && ntiles == 2) mbar_arrive(&turn[t ^ 1]);
                float sx, sy;
                f2_split(f2_add(sum[0], sum[1]), sx, sy);
                l += sx + sy;
            }
            // ------------------------------------------------------------ epilogue of tile t
            if (ok && __all_sync(0xffffffffu, mbar_wait(&ofull[t], C::P_APART ? (n - 1) & 1 : 0, abort_flag, DEV_ERR_TIMEOUT_ACC))) {
                tc_fence_after();
                const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
                const int64_t row = (s.q0 + (int64_t)(r / p.G)) * p.Hq + kvh * p.G + r % p.G;
                const bool seen = m != NEG_INF || l != l;
                if (p.nsplit > 1 && r < rows)
                    p.part_lse[row * p.nsplit + split] = seen ? fmaf(m, c, log2f(l) - SHIFT) : NEG_INF;
#pragma unroll 1
                for (int i = 0; i < D / 32; ++i) {
                    uint32_t o[32];
                    tmem_ld32(o_col + i * 32, o);
                    tmem_ld_wait();
                    if (p.nsplit > 1) {
                        float *dst = p.part_o + (row * p.nsplit + split) * D + i * 32;
                        if (seen && r < rows) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
#pragma unroll
                            for (int e = 0; e < 32; e += 8) st_global_32(dst + e, o + e);
                        }
                    } else if (r < rows) {  // (a row that saw nothing has O = 0 and inv = 0)
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            w[e] = pack2<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
                        uint16_t *dst = reinterpret_cast<uint16_t *>(p.out) + row * D + i * 32;
                        st_global_32(dst, w);
                        st_global_32(dst + 16, w + 8);
                    }
                    __syncwarp();
                }
            }
            tmem_st_wait();  // (an aborted step's rescaling)
            tc_fence_before();
        }
        softmax_done();
    } else if (warp == 8) {
        // ---------------------------------------------------------------- K / V loads
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const unsigned inject = *reinterpret_cast<volatile unsigned *>(&g_debug_inject);
        if (!(inject & 2u)) {
            const int loads = inject & 4u ? n : 2 * n;  // of K and V, one each a step (n: the test hook's half)
            const int ps = 1 << p.page_shift, box = SINKS ? 16 : min(ps, TKV), nb = TKV / box;
            // clears what no row sees in V of step j, once it has landed; only this warp refills
            // the stage, so its barrier still stands at that load
            auto clear_v = [&](int j, uint64_t *done) {
                const int it = 2 * j + 1, st = it % STAGES, kv0 = (t0 + j) * TKV;
                if (!__all_sync(0xffffffffu, mbar_wait(&full[st], (it / STAGES) & 1, abort_flag, DEV_ERR_TIMEOUT_FULL))) return;
                uint8_t *vs = smem + C::SMEM_KV + st * C::TILE_BYTES;
                for (int idx = lane; idx < TKV * 8; idx += 32) {
                    const int row = idx >> 3;
                    if ((kv0 + row >= vlo || (SINKS && kv0 + row < sunk)) && kv0 + row < vhi) continue;
#pragma unroll
                    for (int h = 0; h < C::HALVES; ++h)
                        *reinterpret_cast<uint4 *>(vs + h * C::HALF_BYTES + row * 128 + (idx & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(done);
            };
            // this lane's page of step j, where there is something to see; indices are fetched four
            // steps ahead
            // places and their positions
            auto wanted = [&](int v) { return lane < nb && v < vhi && (v + box > vlo || (SINKS && v < sunk)); };
            auto position = [&](int v) { return SINKS && v >= lead ? v - shift : v; };
            auto page_index = [&](int j) {
                const int v = (t0 + j) * TKV + lane * box;
                return j < n && wanted(v) ? p.table[b * p.table_stride + (position(v) >> p.page_shift)] : 0;
            };
            int it = 0, page = 0, ahead[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) ahead[j] = page_index(j);
            for (; it < loads; ++it) {
                // V of step j is cleared before the load that waits for its products
                if (SINKS && fix_lead && it == min(2 * gap0 + STAGES, 2 * n - 1)) clear_v(gap0, &vfix[2]);
                if (it == min(2 * jf + STAGES, 2 * n - 1) && fix_first && jf < n - 1) clear_v(jf, &vfix[0]);
                const int st = it % STAGES, place = (t0 + (it >> 1)) * TKV + lane * box, pos = position(place);
                const bool in = wanted(place);
                if (!(it & 1)) {
                    page = ahead[0], ahead[0] = ahead[1], ahead[1] = ahead[2], ahead[2] = ahead[3];
                    ahead[3] = page_index((it >> 1) + 4);
                    if (in && (unsigned)page >= (unsigned)p.num_pages) {
                        raise_dev_error(DEV_ERR_BAD_INDEX);
                        page = 0;
                    }
                }
                if (it >= STAGES &&
                    !__all_sync(0xffffffffu, mbar_wait(&empty[st], ((it / STAGES) & 1) ^ 1, abort_flag, DEV_ERR_TIMEOUT_EMPTY)))
                    break;
                const int boxes = __popc(__ballot_sync(0xffffffffu, in));
                if (lane == 0) mbar_arrive_expect_tx(&full[st], boxes * box * D * 2);
                __syncwarp();
                if (in) {
                    const uint32_t dst = smem_u32(smem + C::SMEM_KV + st * C::TILE_BYTES) + lane * box * 128;
#pragma unroll
                    for (int h = 0; h < C::HALVES; ++h)
                        tma_load_4d(dst + h * C::HALF_BYTES, (it & 1) ? &tm_v : &tm_k, &full[st], h * 64, pos & (ps - 1), kvh,
                                    page);
                }
            }
            if (it == 2 * n) {
                if (jf == n - 1 && (fix_first || fix_last)) clear_v(jf, &vfix[0]);
                if (fix_last && jf < n - 1) clear_v(n - 1, &vfix[1]);
            }
            // after an abort, whichever wait ran out, the copies land before their memory is given up
            roles_done();
            if (*abort_flag) {
                const uint64_t from = globaltimer_ns();
                for (int i = max(0, it - STAGES); i < it; ++i)
                    while (!mbar_try_wait(&full[i % STAGES], (i / STAGES) & 1) && globaltimer_ns() - from < 100000000ull) {
                    }
            }
        } else {
            roles_done();
        }
    } else if (warp == 11) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        roles_done();
    } else {
        // ---------------------------------------------------------------- MMAs of tile t
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const int t = warp - 9;
        if (t < ntiles && lane == 0) {
            constexpr uint32_t qk = attn_idesc<T>(TKV, false), pv = attn_idesc<T>(D, true);
            const uint32_t s_col = tmem + t * TKV, o_col = tmem + C::COL_O + t * D, p_col = tmem + C::COL_P + t * C::P_STEP;
            const uint32_t qs = smem_u32(smem + C::SMEM_Q + t * C::TILE_BYTES), ring = smem_u32(smem + C::SMEM_KV);
            auto scores = [&](int j) {  // S_t = Q_t K^T of step j
                const int st = (2 * j) % STAGES;
                if (!mbar_wait(&full[st], (2 * j / STAGES) & 1, abort_flag, DEV_ERR_TIMEOUT_FULL)) return false;
                tc_fence_after();
                const uint32_t ks = ring + st * C::TILE_BYTES;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t at = (k >> 2) * C::HALF_BYTES + (k & 3) * 32;
                    tc_mma_ss(s_col, umma_desc_k_sw128(qs + at), umma_desc_k_sw128(ks + at), qk, k != 0);
                }
                return true;
            };
            bool ok = mbar_wait(&qfull[t], 0, abort_flag, DEV_ERR_TIMEOUT_FULL) && scores(0);
            if (ok) tc_commit(&sfull[t]);
            for (int j = 0; ok && j < n; ++j) {
                if (C::P_APART && j + 1 < n) {  // the next step's scores before this step's weights
                    ok = mbar_wait(&sread[t], j & 1, abort_flag, DEV_ERR_TIMEOUT_ACC) && scores(j + 1);
                    if (!ok) break;
                    tc_commit(&sfull[t]);
                }
                const int it = 2 * j + 1, st = it % STAGES;
                ok = mbar_wait(&full[st], (it / STAGES) & 1, abort_flag, DEV_ERR_TIMEOUT_FULL);
                if (SINKS && ok && fix_lead && j == gap0) ok = mbar_wait(&vfix[2], 0, abort_flag, DEV_ERR_TIMEOUT_FULL);
                if (ok && j == jf && (fix_first || (jf == n - 1 && fix_last))) ok = mbar_wait(&vfix[0], 0, abort_flag, DEV_ERR_TIMEOUT_FULL);
                if (ok && j > jf && j == n - 1 && fix_last) ok = mbar_wait(&vfix[1], 0, abort_flag, DEV_ERR_TIMEOUT_FULL);
                const uint32_t vs = ring + st * C::TILE_BYTES;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    ok = ok && mbar_wait(&pfull[2 * t + h], j & 1, abort_flag, DEV_ERR_TIMEOUT_ACC);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = h ? PFIRST / 16 : 0; k < (h ? TKV : PFIRST) / 16; ++k)
                        tc_mma_ts(o_col, p_col + k * 8, umma_desc_mn_sw128(vs + k * 2048, C::HALF_BYTES), pv, (j | k) != 0);
                }
                if (!ok) break;
                if (C::P_APART || j + 1 == n) {
                    tc_commit(&ofull[t]);
                } else {
                    ok = scores(j + 1);
                    if (ok) tc_commit(&sfull[t]);
                }
            }
        }
        __syncwarp();
        roles_done();
        if (*abort_flag && lane == 0) {  // the same for the products, before TMEM is freed
            tc_commit(&drain[t]);
            const uint64_t from = globaltimer_ns();
            while (!mbar_try_wait(&drain[t], 0) && globaltimer_ns() - from < 100000000ull) {
            }
        }
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

// keys or values of one layer as [pages][heads][page][D]; a box is the rows of one page that
// fall in a step (up to `rows`), 64 elements wide
template <typename T>
static int cache_map(CUtensorMap *map, const void *base, const Params &p, int D, int rows) {
    gemm::PFN_encodeTiled enc = gemm::get_encode();
    if (!enc) return fail(QL_ECUDA, "cuTensorMapEncodeTiled unavailable");
    const uint64_t ps = 1ull << p.page_shift;
    cuuint64_t dims[4] = {(cuuint64_t)D, ps, (cuuint64_t)p.Hkv, (cuuint64_t)p.num_pages};
    cuuint64_t strides[3] = {(cuuint64_t)D * 2, ps * D * 2, (cuuint64_t)p.page_stride * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)(ps < rows ? ps : rows), 1, 1}, es[4] = {1, 1, 1, 1};
    const CUresult r =
        enc(map, __is_same(T, __nv_bfloat16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? QL_OK : fail(QL_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

template <typename T, int D, bool SINKS>
static int launch_sm100_s(const Params &p, int64_t B, cudaStream_t st) {
    using C = Sm100Cfg<D>;
    static PerDeviceFlag configured;
    const int dev = current_device();
    if (!configured.test(dev)) {
        QL_CUDA_TRY(cudaFuncSetAttribute(sm100_kernel<T, D, SINKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        configured.set(dev);
    }
    CUtensorMap mk, mv;
    const int rows = SINKS ? 16 : TKV;  // the sinks and the window begin at any block of 16
    if (int rc = cache_map<T>(&mk, p.k_cache, p, D, rows)) return rc;
    if (int rc = cache_map<T>(&mv, p.v_cache, p, D, rows)) return rc;
    const int tiles = (int)(((int64_t)p.max_q * p.G + SM100_ROWS - 1) / SM100_ROWS);
    QL_CUDA_TRY(launch_pdl(sm100_kernel<T, D, SINKS>, dim3(p.Hkv * p.nsplit, tiles, (unsigned)B), dim3(SM100_THREADS), C::SMEM, st, 1,
                           mk, mv, p));
    return QL_OK;
}

template <typename T, int D>
static int launch_sm100_t(const Params &p, int64_t B, cudaStream_t st) {
    return p.sinks ? launch_sm100_s<T, D, true>(p, B, st) : launch_sm100_s<T, D, false>(p, B, st);
}

}  // namespace attn
}  // namespace ql
