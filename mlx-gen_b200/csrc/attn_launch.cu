// attn_launch.cu -- which kernel a paged-attention call runs and how its work is divided.
#include <math.h>

#include "attn_common.cuh"

namespace ql {
namespace attn {

struct Plan {
    int nsplit, chunk;
};

// Splits of the position axis.  The small-row kernel is bound by HBM, so what it needs is
// enough CTAs to keep every SM's loads in flight (two CTAs fill an SM) and pieces small
// enough to even out sequences of different lengths; a join costs one small launch.
static Plan plan_rows(int64_t items, int64_t max_kv) {
    const int64_t slots = 2 * kSMs;
    int64_t ns = 1;
    if (items < 4 * slots) ns = (4 * slots + items - 1) / items;
    const int64_t most = (max_kv + 127) / 128;  // pieces of at least 128 positions
    if (ns > most) ns = most;
    if (ns > 64) ns = 64;
    if (ns < 1) ns = 1;
    int64_t chunk = ((max_kv + ns - 1) / ns + 127) / 128 * 128;
    if (chunk < 128) chunk = 128;
    ns = (max_kv + chunk - 1) / chunk;
    return {(int)(ns < 1 ? 1 : ns), (int)chunk};
}

// The tensor-core kernel runs one CTA per SM, so its splits fill whole waves: of all counts, the
// one with the least estimated time in steps of 128 positions (about 1.2 us each); a CTA's
// start and end cost about 4 steps, the join 2 and the partial results' traffic.
static Plan plan_tiles(int64_t T, int Hq, int Hkv, int D, int64_t B, int64_t max_q, int64_t max_kv) {
    const int64_t G = Hq / Hkv;
    int64_t tiles = (T * G + SM100_ROWS - 1) / SM100_ROWS;  // of all sequences, if they fill their tiles
    if (tiles < B) tiles = B;
    const int64_t items = tiles * Hkv;
    const double seen = max_kv > max_q ? 1.0 - 0.5 * (double)max_q / (double)max_kv : 0.5;  // of max_kv, on average
    Plan best{1, 0};
    double best_cost = 0;
    for (int ns = 1; ns <= 32; ++ns) {
        const int64_t chunk = ((max_kv + ns - 1) / ns + TKV - 1) / TKV * TKV;
        if (ns > 1 && (max_kv + chunk - 1) / chunk != ns) continue;  // a last split would be empty
        const double work = (double)items * ns * (ns > 1 ? seen + (1 - seen) / ns : 1.0);
        double waves = work / kSMs;
        waves = waves < 6 ? ceil(waves) : waves + 0.5;
        double cost = waves * ((double)(chunk / TKV) * (ns > 1 ? 1.0 : seen + 0.15) + 4);
        if (ns > 1) cost += 2 + (double)T * Hq * ns * D * 8 / 5e6;
        if (ns == 1 || cost < best_cost) {
            best = {ns, (int)(chunk > 0 ? chunk : TKV)};
            best_cost = cost;
        }
    }
    return best;
}

// Sequences with up to 16 rows per kv head go to the small-row kernel, the others to the
// tensor-core kernel, which exists for D = 64 and 128.
struct Kernels {
    bool rows, tiles;
};
static Kernels kernels_of(int Hq, int Hkv, int D, int64_t T, int64_t B, int64_t max_q) {
    const int64_t most = max_q * (Hq / Hkv);
    if (most <= ROWS_TILE || (D != 64 && D != 128)) return {true, false};
    return {T < B * max_q, true};  // all chunks of the longest length: none is short
}

static Plan make_plan(int Hq, int Hkv, int D, int64_t T, int64_t B, int64_t max_q, int64_t max_kv) {
    if (kernels_of(Hq, Hkv, D, T, B, max_q).tiles) return plan_tiles(T, Hq, Hkv, D, B, max_q, max_kv);
    const int64_t rows = max_q * (Hq / Hkv);
    return plan_rows(B * Hkv * ((rows + ROWS_TILE - 1) / ROWS_TILE), max_kv);
}

static size_t lse_bytes(int64_t T, int Hq, int nsplit) { return ((size_t)T * Hq * nsplit * 4 + 255) / 256 * 256; }

template <typename T, int D>
static int launch_t(Params &p, int64_t B, cudaStream_t st) {
    const Kernels ks = kernels_of(p.Hq, p.Hkv, D, p.T, B, p.max_q);
    p.rows_kernel_most = ks.tiles ? (ks.rows ? ROWS_TILE : 0) : INT32_MAX;
    if constexpr (D == 64 || D == 128) {
        if (ks.tiles)
            if (int rc = launch_sm100_t<T, D>(p, B, st)) return rc;
    }
    if (ks.rows) {
        const int64_t most = (int64_t)p.max_q * p.G;
        if (int rc = launch_rows_t<T, D>(p, B, ks.tiles ? ROWS_TILE : most, st)) return rc;
    }
    return p.nsplit > 1 ? launch_join<T, D>(p, st) : QL_OK;
}

template <typename T>
static int launch_d(Params &p, int D, int64_t B, cudaStream_t st) {
    switch (D) {
        case 64: return launch_t<T, 64>(p, B, st);
        case 96: return launch_t<T, 96>(p, B, st);
        case 128: return launch_t<T, 128>(p, B, st);
        default: return launch_t<T, 256>(p, B, st);
    }
}

}  // namespace attn

size_t paged_attention_workspace(int64_t T, int Hq, int Hkv, int D, int64_t B, int64_t max_q, int64_t max_kv) {
    const attn::Plan pl = attn::make_plan(Hq, Hkv, D, T, B, max_q, max_kv);
    if (pl.nsplit <= 1) return 0;
    return attn::lse_bytes(T, Hq, pl.nsplit) + (size_t)T * Hq * pl.nsplit * D * 4;
}

int launch_paged_attention(attn::Params &p, int dtype, int D, int64_t B, void *workspace, cudaStream_t st) {
    const attn::Plan pl = attn::make_plan(p.Hq, p.Hkv, D, p.T, B, p.max_q, p.max_kv);
    p.nsplit = pl.nsplit;
    p.chunk = pl.chunk;
    p.part_lse = reinterpret_cast<float *>(workspace);
    p.part_o = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + attn::lse_bytes(p.T, p.Hq, pl.nsplit));
    return dtype == QL_BF16 ? attn::launch_d<__nv_bfloat16>(p, D, B, st) : attn::launch_d<__half>(p, D, B, st);
}

}  // namespace ql
