// plan.cu -- the index tensors of a forward pass over the paged cache, from the sequences' lengths:
//     kv_b = have_b + new_b,  q_starts = exclusive sum of new_b
//     held_b = ceil(have_b / page_size), fresh_b = ceil(kv_b / page_size) - held_b
//     table[b][held_b + i] = free[taken + (exclusive sum of fresh_b) + i],  i < fresh_b
//     token t of sequence b (t = q_starts_b + i): position have_b + i, slot table[b][position /
//     page_size] * page_size + position % page_size
// so that a decode step needs nothing from the host and can be captured in a graph and replayed.  All or nothing: too few
// pages, columns or rows, or a sequence past max_kv, and the step has no token.
//
// Bound: latency (a chain of dependent loads and barriers; 16 bytes a token written).  Split: every
// CTA sums the counts of all sequences by itself (a thread has B / threads neighbours), then takes
// tiles of one token a thread: each sequence marks its first token in the tile, and a token's
// sequence is the last mark at or before it.  A page is entered in its table by the token
// at its first position, which is always a new one.  Many tokens: a CTA for each tile.  Where lengths or the count
// of taken pages are updated in place, a cluster of 8 shares the tiles instead, so that all CTAs have read them (cluster
// barrier) before one writes them.
// Measured (a graph's replay): 64 sequences of one token 2.9 us, 203 of 62119 tokens 6.6 us (by the cluster of 8 18.7).
#include "pdl.cuh"

namespace ql {
namespace plank {

constexpr int MAX_THREADS = 1024, MAX_CTAS = 8;

struct Params {
    int32_t *table;
    int64_t table_stride, table_width;
    const int32_t *lengths, *new_tokens;
    int64_t B, max_tokens, max_kv;  // (max_kv: at most INT32_MAX)
    int page_shift;
    const int32_t *free_pages;  // NULL: the tables hold every page already
    int64_t num_free;
    const int32_t *taken;
    int64_t *positions, *slots;
    int32_t *q_starts, *kv_lens, *taken_out;
};

struct Shared {
    int64_t tokens[32], pages[32];  // sums of the warps
    int bad;
    int last[32];                   // last mark of each warp's tokens
    int seq[MAX_THREADS], start[MAX_THREADS];  // of the sequence that marks a token
    int64_t page[MAX_THREADS];      // its first entry of free_pages
};

template <bool CLUSTER>
__global__ void __launch_bounds__(MAX_THREADS) plan_kernel(const __grid_constant__ Params p) {
    __shared__ Shared sh;
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, nt = blockDim.x, warp = tid >> 5, lane = tid & 31, nw = nt >> 5;
    const int rank = blockIdx.x, ctas = gridDim.x;
    const int ps = 1 << p.page_shift;
    const int64_t per = (p.B + nt - 1) / nt, b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    if (tid == 0) sh.bad = 0;
    __syncthreads();

    // ---- sums over all sequences
    const int64_t taken = p.free_pages ? (int64_t)p.taken[0] : 0;
    auto pages_of = [&](int64_t n) { return (n + ps - 1) >> p.page_shift; };
    int64_t tokens = 0, pages = 0;
    bool bad = taken < 0;
    for (int64_t b = b0; b < b1; ++b) {
        const int64_t have = p.lengths[b], n = p.new_tokens[b];
        bad = bad || have < 0 || n < 0 || have + n > p.max_kv || pages_of(have + n) > p.table_width;
        tokens += n;
        if (p.free_pages) pages += pages_of(have + n) - pages_of(have);
    }
    int64_t tokens_upto = tokens, pages_upto = pages;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, tokens_upto, o), g = __shfl_up_sync(0xffffffffu, pages_upto, o);
        if (lane >= o) tokens_upto += t, pages_upto += g;
    }
    if (lane == 31) sh.tokens[warp] = tokens_upto, sh.pages[warp] = pages_upto;
    if (bad) sh.bad = 1;
    __syncthreads();
    int64_t total = 0, total_pages = 0;
    tokens_upto -= tokens, pages_upto -= pages;  // exclusive
    for (int w = 0; w < nw; ++w) {
        if (w == warp) tokens_upto += total, pages_upto += total_pages;
        total += sh.tokens[w], total_pages += sh.pages[w];
    }
    // all or nothing
    const bool ok = !sh.bad && total <= p.max_tokens && (!p.free_pages || taken + total_pages <= p.num_free);

    // ---- tiles of tokens
    for (int64_t base = (int64_t)rank * nt; base < p.max_tokens; base += (int64_t)ctas * nt) {
        const int64_t t = base + tid;
        if (ok && base < total) {
            sh.seq[tid] = -1;
            __syncthreads();
            int64_t at = tokens_upto, page = pages_upto;
            for (int64_t b = b0; b < b1 && at < base + nt; ++b) {
                const int64_t n = p.new_tokens[b];
                if (n > 0 && at + n > base) {
                    const int m = (int)max((int64_t)0, at - base);
                    sh.seq[m] = (int)b;
                    sh.start[m] = (int)at;
                    sh.page[m] = page;
                }
                at += n;
                if (p.free_pages) {
                    const int64_t have = p.lengths[b];
                    page += pages_of(have + n) - pages_of(have);
                }
            }
            __syncthreads();
            // the last mark at or before this token: within the warp, else of the warps before
            const unsigned marks = __ballot_sync(0xffffffffu, sh.seq[tid] >= 0);
            if (lane == 0) sh.last[warp] = marks ? warp * 32 + 31 - __clz(marks) : -1;
            __syncthreads();
            const unsigned mine = marks & (0xffffffffu >> (31 - lane));
            const unsigned before = __ballot_sync(0xffffffffu, lane < warp && sh.last[lane] >= 0);
            if (t < total) {
                const int m = mine ? warp * 32 + 31 - __clz(mine) : sh.last[31 - __clz(before)];
                const int64_t b = sh.seq[m];
                const int64_t have = p.lengths[b], pos = have + (t - sh.start[m]), at_page = pos >> p.page_shift;
                int32_t *entry = p.table + b * p.table_stride + at_page;
                int pg;
                if (p.free_pages && at_page >= pages_of(have)) {
                    pg = p.free_pages[taken + sh.page[m] + at_page - pages_of(have)];
                    if ((pos & (ps - 1)) == 0) *entry = pg;
                } else pg = *entry;
                if (pg < 0) raise_dev_error(DEV_ERR_BAD_INDEX);
                p.positions[t] = pos;
                p.slots[t] = pg < 0 ? -1 : ((int64_t)pg << p.page_shift) + (pos & (ps - 1));
            }
            __syncthreads();  // before the next tile's marks
        }
        if (t < p.max_tokens && (!ok || t >= total)) {  // padding: a token that is not cached
            p.positions[t] = 0;
            p.slots[t] = -1;
        }
    }

    // ---- offsets, lengths, the pages taken: from here on the inputs may change
    if (CLUSTER) cluster_sync_all();
    else __syncthreads();
    if (rank != 0) return;
    int64_t at = tokens_upto;
    for (int64_t b = b0; b < b1; ++b) {
        const int64_t have = p.lengths[b], n = ok ? p.new_tokens[b] : 0;
        p.q_starts[b] = ok ? (int)at : 0;
        p.kv_lens[b] = (int)(have + n);
        at += n;
    }
    if (tid == 0) {
        p.q_starts[p.B] = ok ? (int)total : 0;
        if (p.free_pages) p.taken_out[0] = (int)(taken + (ok ? total_pages : 0));
        if (!ok) raise_dev_error(DEV_ERR_NO_ROOM);
    }
}

}  // namespace plank

int launch_plan_step(const plank::Params &p, cudaStream_t st) {
    using namespace plank;
    const int64_t most = p.B > p.max_tokens ? p.B : p.max_tokens;
    const int threads = most >= MAX_THREADS ? MAX_THREADS : most < 32 ? 32 : (int)((most + 31) / 32 * 32);
    int64_t ctas = (p.max_tokens + threads - 1) / threads;
    auto overlap = [](const int32_t *a, const int32_t *b, int64_t n) { return a < b + n && b < a + n; };
    const bool in_place = overlap(p.kv_lens, p.lengths, p.B) || (p.free_pages && p.taken == p.taken_out);
    const int64_t most_ctas = in_place ? MAX_CTAS : 8 * 148;  // (more tiles than that: several each)
    ctas = ctas < 1 ? 1 : ctas < most_ctas ? ctas : most_ctas;
    if (ctas > 1 && in_place)
        QL_CUDA_TRY(launch_pdl(plan_kernel<true>, dim3((unsigned)ctas), dim3(threads), 0, st, (unsigned)ctas, p));
    else QL_CUDA_TRY(launch_pdl(plan_kernel<false>, dim3((unsigned)ctas), dim3(threads), 0, st, 1, p));
    return QL_OK;
}

}  // namespace ql
