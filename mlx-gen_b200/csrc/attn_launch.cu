// attn_launch.cu -- which kernel a paged-attention call runs and how its work is divided.
#include <math.h>

#include "attn_common.cuh"

namespace ql {
namespace attn {

constexpr double kMostPartial = 128 << 20;  // bytes of partial results of the small-row kernel's pieces

struct Plan {
    int nsplit, chunk;
    bool adapt, cluster;
};

// The small-row kernel, for `items` (sequence, kv head, row block)s of up to `span` visible
// positions each; `split_bytes`: the partial results of one split of every row.
static Plan plan_rows(int64_t B, int64_t items, int64_t span, bool window, double split_bytes) {
    const int64_t pieces = (span + 127) / 128;  // at least 128 positions each
    if (pieces <= 1) return {1, 128, false, false};
    // Few items of moderate length: up to 8 splits in a cluster, one launch and no workspace.
    // One sequence of 8 kv heads: 777 positions 6.0 us (joined by a second launch 9.0), 4000
    // positions 11.1 us (12.5 in 16 joined splits), 16000 positions 31.5 us (24.3); one kv head, 6000
    // positions 14.2 us, 6001 by lengths 17.8.
    if (2 * items <= kSMs && span <= 6000) {
        int64_t ns = (kSMs + items - 1) / items;
        ns = ns < MAX_CLUSTER ? ns : MAX_CLUSTER;
        ns = ns < pieces ? ns : pieces;
        const int64_t most = window ? span + 127 : span;  // a window starts anywhere in its first 128
        return {(int)ns, (int)(((most + ns - 1) / ns + 63) / 64 * 64), false, true};
    }
    const int64_t most = span + 127;  // from the 128-boundary under a row's first position
    // A few sequences, at most a quarter of the SMs in items: adapted_chunk divides them.  It may
    // cut the longest into as many pieces as give each SM two if the lengths are equal, and into 8
    // of 4096 if they are not.
    if (4 * items <= kSMs && B <= 32) {
        int64_t ns = (2 * kSMs + items - 1) / items, uneven = (most + 4095) / 4096;
        uneven = uneven < 8 ? uneven : 8;
        ns = ns > uneven ? ns : uneven;
        ns = ns < 64 ? ns : 64;
        return {(int)(ns < pieces ? ns : pieces), 0, true, false};
    }
    // Many items: pieces of 2048 even out different lengths by their number (8 kv heads: 64
    // sequences of 311 - 8003 positions whole 218 us, in pieces of 4096 / 2048 / 1024 positions 189
    // / 180 / 189; 10 of 20000 159 / 141 / 152; 16 of 4000 62 / 52 / 54).  Up to 2048 positions there is
    // one piece, however few items: 10 sequences of 2000 33 us, where 9 are split in clusters and take 17.
    if (span <= 2048) return {1, 2048, false, false};
    // Chunks of heads of 96 and 256 run here too, with row blocks that fill the SMs by themselves and
    // gigabytes of partial results in such pieces: those are held to 128 MiB, by fewer, longer pieces
    // (16 / 8 heads of 256, 4096 tokens over 32768 positions: 17 pieces 17.2 ms and 1092 MB, 2 pieces
    // 13.8 ms; 512 over 131072: 64 pieces 9.0 ms, 16 pieces 7.7 ms; decode batches stay below it).
    int64_t ns = (most + 2047) / 2048, fit = (int64_t)(kMostPartial / split_bytes);
    fit = fit < 64 ? fit : 64;
    if (fit <= 1) return {1, 128, false, false};
    if (ns <= fit) return {(int)ns, 2048, false, false};
    return {(int)fit, (int)(((most + fit - 1) / fit + 127) / 128 * 128), false, false};
}

// The tensor-core kernel runs one CTA per SM, so its splits fill whole waves: of all counts, the
// one with the least estimated time in steps of 128 positions (about 1.2 us each); a CTA's
// start and end cost about 4 steps, the join 2 and the partial results' traffic.
static Plan plan_tiles(int64_t T, int Hq, int Hkv, int D, int64_t B, int64_t max_q, int64_t max_kv, int64_t window) {
    const int64_t G = Hq / Hkv;
    int64_t tiles = (T * G + SM100_ROWS - 1) / SM100_ROWS;  // of all sequences, if they fill their tiles
    if (tiles < B) tiles = B;
    const int64_t items = tiles * Hkv;
    // what one tile sees: at most `span` positions, on average a share `seen` of them
    const int64_t windowed = window ? window + SM100_ROWS / G + 1 : max_kv, span = windowed < max_kv ? windowed : max_kv;
    const double seen = span < max_kv || max_kv <= 0 ? 1.0 : 1.0 - 0.5 * (double)(max_q < max_kv ? max_q : max_kv) / (double)max_kv;
    Plan best{1, TKV, false, false};
    double best_cost = 0;
    for (int ns = 1; ns <= 32; ++ns) {
        // (the splits start at a row's own boundary: one step more than the span)
        const int64_t chunk = ns == 1 ? (span + TKV - 1) / TKV * TKV : (span / ns + TKV) / TKV * TKV;
        if (ns > 1 && (span + TKV - 1) / chunk + 1 != ns && (span + TKV - 1) / chunk != ns) continue;  // a last split would be empty
        const double work = (double)items * ns * (ns > 1 ? seen + (1 - seen) / ns : 1.0);
        double waves = work / kSMs;
        waves = waves < 6 ? ceil(waves) : waves + 0.5;
        double cost = waves * ((double)(chunk / TKV) * (ns > 1 ? 1.0 : seen + 0.15) + 4);
        if (ns > 1) cost += 2 + (double)T * Hq * ns * D * 8 / 5e6;
        if (ns == 1 || cost < best_cost) {
            best = {ns, (int)(chunk > 0 ? chunk : TKV), false, false};
            best_cost = cost;
        }
    }
    // every split of the longest row must be there: from its 128-boundary on
    while (best.nsplit > 1 && (int64_t)best.nsplit * best.chunk < span + TKV - 1) best.chunk += TKV;
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

// Row blocks of a sequence; one even where the bound is no rows, to report sequences that have some.
static int64_t row_blocks(int64_t rows) { return rows > 0 ? (rows + ROWS_TILE - 1) / ROWS_TILE : 1; }

static Plan make_plan(int Hq, int Hkv, int D, int64_t T, int64_t B, int64_t max_q, int64_t max_kv, int64_t window) {
    if (kernels_of(Hq, Hkv, D, T, B, max_q).tiles) return plan_tiles(T, Hq, Hkv, D, B, max_q, max_kv, window);
    const int64_t rowblocks = row_blocks(max_q * (Hq / Hkv)), windowed = window ? window + max_q : max_kv;
    return plan_rows(B, B * Hkv * rowblocks, windowed < max_kv ? windowed : max_kv, window != 0, 4.0 * T * Hq * D);
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
        const int blocks = ks.tiles ? 1 : (int)row_blocks((int64_t)p.max_q * p.G);
        if (int rc = launch_rows_t<T, D>(p, B, blocks, st)) return rc;
    }
    return p.nsplit > 1 && !p.cluster ? launch_join<T, D>(p, st) : QL_OK;
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

size_t paged_attention_workspace(int64_t T, int Hq, int Hkv, int D, int64_t B, int64_t max_q, int64_t max_kv,
                                 int64_t window) {
    const attn::Plan pl = attn::make_plan(Hq, Hkv, D, T, B, max_q, max_kv, window);
    if (pl.nsplit <= 1 || pl.cluster) return 0;
    return attn::lse_bytes(T, Hq, pl.nsplit) + (size_t)T * Hq * pl.nsplit * D * 4;
}

int launch_paged_attention(attn::Params &p, int dtype, int D, int64_t B, void *workspace, cudaStream_t st) {
    const attn::Plan pl = attn::make_plan(p.Hq, p.Hkv, D, p.T, B, p.max_q, p.max_kv, p.window);
    p.nsplit = pl.nsplit;
    p.chunk = pl.chunk;
    p.cluster = pl.cluster;
    p.adapt = pl.adapt;
    p.part_lse = reinterpret_cast<float *>(workspace);
    p.part_o = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(workspace) + attn::lse_bytes(p.T, p.Hq, pl.nsplit));
    return dtype == QL_BF16 ? attn::launch_d<__nv_bfloat16>(p, D, B, st) : attn::launch_d<__half>(p, D, B, st);
}

}  // namespace ql
