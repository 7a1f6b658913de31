// sample.cu -- one token per row of logits, from a given random number:
//     w_i = exp((x_i - max x) / temperature)
//     order: x descending, equal ones by index;  kept, each a prefix of that order:
//         top-k   the first k
//         top-p   of those, the shortest prefix with a sum of at least p times their sum
//         min-p   of those, the ones with w_i >= min_p
//     token = the first kept i, by index, with (sum of the kept up to i) > u * (sum of the kept)
//
// Precision: the token is a whole number next to borders, and a border that is off by d moves one row
// in 1 / (d * kept tokens): with 128256 tokens, sums in fp32 (d = 1e-7) would give another token for one row in
// a hundred.  So each weight is computed in fp64 and held as the whole number
// W = round(w * 2^S), S = 46 for up to 2^17 tokens, and all sums are of whole numbers: exact, free of
// any order, so that a row's token does not depend on how the row was divided or on its batch.
// The exponential (method: table and short polynomial, P. T. P. Tang 1989): 256 y = k + r with whole
// k and |r| <= 1/2, 2^-y = 2^-(k >> 8) * table[k & 255] * exp(-r ln 2 / 256), whose series ends
// after the fourth power (the fifth is below 2^-54).
//
// Bound: fp64 instructions (10 of 64 lanes a clock and SM for each logit) for many rows, the chain of
// cluster barriers for few.  Split: a cluster of CTAs takes a row, each CTA keeps its slice in shared memory,
// so that the row is read once whatever filters it has.  A threshold is found without sorting: counts
// (or weights) of the keys in 1024 bins below the largest key, the bin that holds the border divided
// again, until it holds at most LIST elements, of which every one then counts what precedes it.
#include "pdl.cuh"

namespace ql {
namespace samplek {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 1024, GROUP = 32, GROUPS = BINS / GROUP;
constexpr int LIST = 512;         // elements that are compared one by one (one a thread)
constexpr int MAX_CTAS = 8;       // of a cluster
constexpr int MAX_SLICE = 160 << 10;  // bytes of a row in one CTA's shared memory
constexpr uint32_t NO_INDEX = 0xffffffffu;
static_assert(LIST <= THREADS && GROUPS == 32, "one element a thread; one group a lane");

struct Params {
    const void *logits;
    int64_t stride;  // elements between rows
    int V, slice;    // tokens; of one CTA
    int scale;       // S
    const float *u;
    const float *temperature, *top_p, *min_p;  // one for each row, or NULL: the value for all
    const int32_t *top_k;
    double temperature_all, top_p_all, min_p_all;
    int64_t top_k_all;
    int64_t *tokens;
    float *logprobs;  // or NULL
};

struct Hist {
    uint32_t count[BINS], lo[BINS], hi[BINS];  // elements; their weights' sum as lo + 2^32 hi
};
struct Cut {  // the kept: key > this, or equal and the index at most this
    uint32_t key, index;
};

// Shared memory besides the slice.  What other CTAs read after a barrier is not written again before
// another barrier has passed: hence one slot a phase, and two histograms in turn.
struct Shared {
    Hist hist[2];
    uint64_t group[2][GROUPS];
    uint32_t list_key[LIST], list_index[LIST];      // this CTA's
    uint32_t all_key[LIST], all_index[LIST];        // the cluster's
    uint64_t all_weight[LIST];
    double table[256];
    uint64_t warp_sum[WARPS];
    uint64_t cta_sum[2][2];                         // totals, by phase and select
    uint32_t warp_max[WARPS], cta_max, cta_first;
    uint32_t list_count[2], tie_count[2], tie_index[2];
    uint64_t found_before;                          // of the search: the sum before the bin
    uint32_t found_bin, found_count;
    Cut cut;
};

template <typename T>
struct Type;
template <>
struct Type<float> {
    static constexpr int N = 4, UNIT = 0;  // elements of 16 bytes; zero bits at the end of their fp32 form
    static __device__ __forceinline__ void load(const uint4 &v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    }
};
template <>
struct Type<__nv_bfloat16> {
    static constexpr int N = 8, UNIT = 16;
    static __device__ __forceinline__ void load(const uint4 &v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = bf16lo(w[i]), x[2 * i + 1] = bf16hi(w[i]);
    }
};
template <>
struct Type<__half> {
    static constexpr int N = 8, UNIT = 13;
    static __device__ __forceinline__ void load(const uint4 &v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __half2float(__ushort_as_half((unsigned short)(w[i] & 0xffffu)));
            x[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16)));
        }
    }
};

// Whole numbers in the order of the values; -0 is 0, NaN above everything.
template <int UNIT>
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0xffffffffu >> UNIT;
    const uint32_t b = __float_as_uint(x + 0.f);
    return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> UNIT;
}
template <int UNIT>
__device__ __forceinline__ float value_of(uint32_t key) {
    const uint32_t k = key << UNIT;
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~(k | ((1u << UNIT) - 1u)));
}

__device__ __forceinline__ uint32_t ld_cluster_u32(const void *p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t ld_cluster_u64(const void *p, uint32_t rank) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ uint64_t warp_scan(uint64_t v) {  // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// fp32 to fp64 without the conversion unit (a quarter of the fp64 rate); values below 2^-126 become 0, which
// changes a logit by less than anything that a weight can tell.  Not for infinities.
__device__ __forceinline__ double widen(float x) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t hi = ((b & 0x7fffffffu) >> 3) + 0x38000000u;
    return (b & 0x7f800000u) ? __hiloint2double((int)(hi | (b & 0x80000000u)), (int)(b << 29)) : 0.0;
}

struct Weigher {
    double max, rate;   // rate: 256 log2(e) / temperature
    double limit;       // 256 y from which on weights are 0
    int scale;
    bool infinite;      // the row holds +inf: those share everything
    const double *table;

    __device__ __forceinline__ double distance(float x) const {  // 256 y
        if (infinite) return x == INFINITY ? 0.0 : INFINITY;
        return x == -INFINITY ? (double)INFINITY : (max - widen(x)) * rate;
    }
    // w * 2^S, before its rounding
    __device__ __forceinline__ double scaled(double y) const {
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
        constexpr double C1 = 2.7076061740622863e-03, C2 = C1 * C1 / 2, C3 = C1 * C1 * C1 / 6, C4 = C1 * C1 * C1 * C1 / 24;
        if (!(y < limit)) return 0.0;
        const double t = y + MAGIC;
        const int k = __double2loint(t);
        const double r = (t - MAGIC) - y;
        const double e = fma(fma(fma(fma(C4, r, C3), r, C2), r, C1), r, 1.0) * table[k & 255];
        return e * __hiloint2double((1023 + scale - (k >> 8)) << 20, 0);
    }
    static __device__ __forceinline__ uint64_t whole(double s) {  // s < 2^51
        const double t = s + 4503599627370496.0;  // 2^52
        return (uint64_t)__double_as_longlong(t) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ uint64_t operator()(float x) const { return whole(scaled(distance(x))); }
};

template <bool CLUSTER>
__device__ __forceinline__ void sync_all() {
    if (CLUSTER) cluster_sync_all();
    else __syncthreads();
}

// One row's view: the slice in shared memory as 16-byte words, `words` of them, divided among the
// warps in order; places outside the slice hold -inf.
template <typename T, bool CLUSTER>
struct Row {
    using Ty = Type<T>;
    static constexpr int N = Ty::N, UNIT = Ty::UNIT;
    const uint4 *data;
    Shared *sh;
    int words, first, last;  // this warp's words
    int skew;                // places before the slice in the first word
    uint32_t base;           // index of the slice's first token
    uint32_t ctas, rank;

    __device__ __forceinline__ uint32_t index(int word, int e) const { return base + (uint32_t)(word * N + e - skew); }

    // f(x, word, e) of each of this warp's elements above -inf, 32 words at a time, in the order of indices
    // across calls
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int w = first + (threadIdx.x & 31); w < last; w += 32) {
            float x[N];
            Ty::load(data[w], x);
#pragma unroll
            for (int e = 0; e < N; ++e) f(x[e], w, e);
        }
    }

    // Sum over the cluster of a value of each thread; warp_sum[] and the sums before this CTA come with it.
    __device__ __forceinline__ uint64_t total(uint64_t v, uint64_t *slot, uint64_t &before) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh->warp_sum[warp] = v;
        __syncthreads();
        uint64_t cta = lane < WARPS ? sh->warp_sum[lane] : 0ull;
        cta = warp_sum(cta);
        if (!CLUSTER) {
            before = 0;
            return cta;
        }
        if (threadIdx.x == 0) *slot = cta;
        cluster_sync_all();
        const uint64_t mine = lane < ctas ? ld_cluster_u64(slot, lane) : 0ull;
        before = warp_sum(lane < rank ? mine : 0ull);
        return warp_sum(mine);
    }
};

// The cut after the shortest prefix, in the order of the values, whose measure (elements, or weights
// with WEIGHT) reaches `need` >= 1, among the elements within `cut` whose keys are from `low` up to `high`.
// Elements left out by `low` must not be needed.  `turn` counts histograms, over both calls.
template <bool WEIGHT, typename T, bool CLUSTER>
__device__ Cut select(const Row<T, CLUSTER> &row, const Weigher &weigh, Cut cut, uint32_t high, uint32_t low, uint64_t need,
                      int &turn) {
    constexpr int UNIT = Type<T>::UNIT;
    constexpr int SLOT = WEIGHT;
    Shared *sh = row.sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    low = max(low, cut.key);
    auto inside = [&](uint32_t key, int w, int e) {
        return key >= low && key <= high && (key != cut.key || row.index(w, e) <= cut.index);
    };
    for (;;) {
        const uint32_t range = high - low;
        const int bits = 32 - __clz((int)range), shift = bits > 10 ? bits - 10 : 0;
        Hist &h = sh->hist[turn & 1];
        uint64_t *group = sh->group[turn & 1];
        ++turn;
        for (int i = tid; i < BINS; i += THREADS) h.count[i] = h.lo[i] = h.hi[i] = 0;
        __syncthreads();
        row.each([&](float x, int w, int e) {
            const uint32_t key = key_of<UNIT>(x);
            if (!inside(key, w, e)) return;
            const uint32_t b = (high - key) >> shift;
            atomicAdd(&h.count[b], 1u);
            if (WEIGHT) {
                const uint64_t weight = weigh(x);
                const uint32_t lo = (uint32_t)weight, old = atomicAdd(&h.lo[b], lo);
                const uint32_t hi = (uint32_t)(weight >> 32) + (old + lo < old ? 1u : 0u);
                if (hi) atomicAdd(&h.hi[b], hi);
            }
        });
        __syncthreads();
        for (int g = warp; g < GROUPS; g += WARPS) {
            const int i = g * GROUP + lane;
            const uint64_t s = warp_sum(WEIGHT ? (uint64_t)h.hi[i] << 32 | 0u : (uint64_t)h.count[i]) +
                               (WEIGHT ? warp_sum((uint64_t)h.lo[i]) : 0ull);
            if (lane == 0) group[g] = s;
        }
        sync_all<CLUSTER>();
        if (warp == 0) {
            // the group, then the bin of it, that holds the border
            uint64_t s = 0;
            for (uint32_t c = 0; c < row.ctas; ++c) s += ld_cluster_u64(&group[lane], c);
            uint64_t upto = warp_scan(s);
            const unsigned past = __ballot_sync(0xffffffffu, upto >= need);
            const int g = past ? __ffs(past) - 1 : 0;
            uint64_t before = __shfl_sync(0xffffffffu, upto - s, g);
            s = 0;
            uint32_t n = 0;
            for (uint32_t c = 0; c < row.ctas; ++c) {
                const uint32_t k = ld_cluster_u32(&h.count[g * GROUP + lane], c);
                n += k;
                if (WEIGHT)
                    s += (uint64_t)ld_cluster_u32(&h.lo[g * GROUP + lane], c) +
                         ((uint64_t)ld_cluster_u32(&h.hi[g * GROUP + lane], c) << 32);
                else s += k;
            }
            upto = before + warp_scan(s);
            const unsigned here = __ballot_sync(0xffffffffu, upto >= need);
            const int b = here ? __ffs(here) - 1 : 0;
            if (lane == b) {
                sh->found_bin = past ? (uint32_t)(g * GROUP + b) : NO_INDEX;
                sh->found_count = n;
                sh->found_before = upto - s;
            }
        }
        __syncthreads();
        const uint32_t bin = sh->found_bin, count = sh->found_count;
        if (bin == NO_INDEX) return cut;  // all of them together do not reach it
        need -= sh->found_before;
        high -= bin << shift;
        low = max(low, high - min(high, (1u << shift) - 1u));
        __syncthreads();
        if (count <= LIST || shift == 0) {
            if (count <= LIST) {
                // every element against every other
                if (tid == 0) sh->list_count[SLOT] = 0;
                __syncthreads();
                row.each([&](float x, int w, int e) {
                    const uint32_t key = key_of<UNIT>(x);
                    if (!inside(key, w, e)) return;
                    const uint32_t at = atomicAdd(&sh->list_count[SLOT], 1u);
                    sh->list_key[at] = key;
                    sh->list_index[at] = row.index(w, e);
                });
                sync_all<CLUSTER>();
                uint32_t at = tid, from = 0;  // this thread's element: the at-th of CTA `from`
                while (from < row.ctas) {
                    const uint32_t n = ld_cluster_u32(&sh->list_count[SLOT], from);
                    if (at < n) break;
                    at -= n;
                    ++from;
                }
                uint32_t key = 0, index = 0;
                uint64_t own = 0;
                if (from < row.ctas) {
                    key = ld_cluster_u32(&sh->list_key[at], from);
                    index = ld_cluster_u32(&sh->list_index[at], from);
                    own = WEIGHT ? weigh(value_of<UNIT>(key)) : 1ull;
                    sh->all_key[tid] = key;
                    sh->all_index[tid] = index;
                    sh->all_weight[tid] = own;
                }
                __syncthreads();
                uint64_t upto = own;
                if (from < row.ctas)
                    for (uint32_t i = 0; i < count; ++i) {
                        const uint32_t k = sh->all_key[i];
                        if (k > key || (k == key && sh->all_index[i] < index)) upto += sh->all_weight[i];
                    }
                if (from < row.ctas && upto >= need && upto - own < need) sh->cut = {key, index};
                __syncthreads();
                // no CTA may refill its list before the others have read it: a second call of select uses
                // it only after the barrier of its own histogram
                return sh->cut;
            }
            // more equal elements than that: the last of them that is needed, by index
            const uint64_t each = WEIGHT ? weigh(value_of<UNIT>(high)) : 1ull;
            const uint64_t ties = (need + each - 1) / each;
            if (ties >= count) return {high, cut.key == high ? cut.index : NO_INDEX};
            uint64_t mine = 0, before;
            row.each([&](float x, int w, int e) { mine += inside(key_of<UNIT>(x), w, e) ? 1u : 0u; });
            row.total(mine, &sh->cta_sum[1][SLOT], before);
            // the warp whose elements hold it looks for it; its CTA tells the others
            if (tid == 0) sh->tie_index[SLOT] = NO_INDEX;
            __syncthreads();
            uint64_t at = before;
            for (int i = 0; i < warp; ++i) at += sh->warp_sum[i];
            if (at < ties && at + sh->warp_sum[warp] >= ties) {
                for (int w0 = row.first; w0 < row.last; w0 += 32) {
                    const int w = w0 + lane;
                    float x[Type<T>::N];
                    int n = 0;
                    if (w < row.last) {
                        Type<T>::load(row.data[w], x);
#pragma unroll
                        for (int e = 0; e < Type<T>::N; ++e) n += inside(key_of<UNIT>(x[e]), w, e) ? 1 : 0;
                    }
                    const uint64_t upto = at + warp_scan((uint64_t)n);
                    if (upto >= ties && upto - n < ties) {
                        uint64_t left = ties - (upto - n);
#pragma unroll
                        for (int e = 0; e < Type<T>::N; ++e)
                            if (inside(key_of<UNIT>(x[e]), w, e) && --left == 0) sh->tie_index[SLOT] = row.index(w, e);
                    }
                    at = __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            sync_all<CLUSTER>();
            uint32_t index = NO_INDEX;
            for (uint32_t c = 0; c < row.ctas; ++c) index = min(index, ld_cluster_u32(&sh->tie_index[SLOT], c));
            return {high, index};
        }
    }
}

template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(THREADS) sample_kernel(const Params p) {
    using Ty = Type<T>;
    constexpr int N = Ty::N, UNIT = Ty::UNIT;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared *sh = reinterpret_cast<Shared *>(smem);
    uint4 *data = reinterpret_cast<uint4 *>(smem + (sizeof(Shared) + 15) / 16 * 16);
    pdl_trigger();
    pdl_wait();
    Row<T, CLUSTER> row;
    row.ctas = CLUSTER ? gridDim.x : 1;
    row.rank = CLUSTER ? blockIdx.x : 0;
    const int64_t b = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- the slice: whole words by asynchronous copies, the ends one by one
    row.base = row.rank * (uint32_t)p.slice;
    const int n = max(0, min(p.slice, p.V - (int)min(row.base, (uint32_t)p.V)));
    const T *src = reinterpret_cast<const T *>(p.logits) + b * p.stride + row.base;
    row.skew = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
    row.words = n ? (n + row.skew + N - 1) / N : 0;
    for (int w = tid; w < row.words; w += THREADS) {
        const int at = w * N - row.skew;
        if (at >= 0 && at + N <= n) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(data + w)), "l"(src + at) : "memory");
        } else {
            T *dst = reinterpret_cast<T *>(data + w);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (at + e >= 0 && at + e < n) dst[e] = src[at + e];
                else dst[e] = T(-INFINITY);
            }
        }
    }
    const double temperature = p.temperature ? (double)p.temperature[b] : p.temperature_all;
    const double top_p = p.top_p ? (double)p.top_p[b] : p.top_p_all;
    const double min_p = p.min_p ? (double)p.min_p[b] : p.min_p_all;
    const int64_t top_k = p.top_k ? (int64_t)p.top_k[b] : p.top_k_all;
    const float u = p.u[b];
    if (tid < 256) sh->table[tid] = exp2(-tid / 256.0);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    row.data = data;
    row.sh = sh;
    const int per = (row.words + THREADS - 1) / THREADS * 32;
    row.first = min(row.words, warp * per);
    row.last = min(row.words, row.first + per);

    // ---- the largest logit
    uint32_t top = 0;
    row.each([&](float x, int, int) { top = max(top, key_of<UNIT>(x)); });
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) sh->warp_max[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < WARPS ? sh->warp_max[lane] : 0u);
    if (CLUSTER) {
        if (tid == 0) sh->cta_max = top;
        cluster_sync_all();
        top = __reduce_max_sync(0xffffffffu, lane < row.ctas ? ld_cluster_u32(&sh->cta_max, lane) : 0u);
    }
    const uint32_t none = key_of<UNIT>(-INFINITY);
    int64_t token = -1;
    float logprob = __uint_as_float(0x7fc00000u);
    bool writer = row.rank == 0 && tid == 0;
    // a NaN among the logits or the settings, nothing above -inf, a negative temperature: no token
    const bool bad = top > key_of<UNIT>(INFINITY) || top <= none || !(temperature >= 0.0) || top_p != top_p || min_p != min_p || u != u;
    if (bad) {
    } else if (temperature == 0.0) {
        // ---- greedy: the lowest index with the largest logit
        uint32_t at = NO_INDEX;
        row.each([&](float x, int w, int e) {
            if (key_of<UNIT>(x) == top) at = min(at, row.index(w, e));
        });
        at = __reduce_min_sync(0xffffffffu, at);
        if (tid == 0) sh->cta_first = NO_INDEX;
        __syncthreads();
        if (lane == 0) atomicMin(&sh->cta_first, at);
        sync_all<CLUSTER>();
        at = __reduce_min_sync(0xffffffffu, lane < row.ctas ? ld_cluster_u32(&sh->cta_first, lane) : NO_INDEX);
        token = at;
        logprob = 0.f;
    } else {
        Weigher weigh;
        const float largest = value_of<UNIT>(top);
        weigh.infinite = largest == INFINITY;
        weigh.max = weigh.infinite ? 0.0 : (double)largest;
        weigh.rate = fmin(369.3299304675746 / temperature, 1e300);  // 256 log2(e)
        weigh.scale = p.scale;
        weigh.limit = 256.0 * (p.scale + 2);
        weigh.table = sh->table;
        Cut cut{none + 1, NO_INDEX};
        int turn = 0;
        uint64_t before;
        if (top_k > 0 && top_k < p.V) cut = select<false>(row, weigh, cut, top, none + 1, (uint64_t)top_k, turn);
        auto kept = [&](uint32_t key, int w, int e) { return key > cut.key || (key == cut.key && row.index(w, e) <= cut.index); };
        if (top_p < 1.0) {
            uint64_t sum = 0;
            row.each([&](float x, int w, int e) {
                if (kept(key_of<UNIT>(x), w, e)) sum += weigh(x);
            });
            sum = row.total(sum, &sh->cta_sum[0][0], before);
            const double target = ceil((double)sum * top_p);
            const uint64_t need = target >= 1.0 ? min(sum, (uint64_t)target) : 1ull;
            // Weights below half of (1 - p) sum / V sum up to less than (1 - p) sum, so none of them is in
            // the prefix, and only keys above that (rounded down with a margin) are looked at.
            const double least = fmax(0.5, 0.5 * (1.0 - top_p) * (double)sum / p.V);
            const double reach = (p.scale - log2(least)) * 256.0 / weigh.rate * 1.000001;
            const float bound = (float)(weigh.max - reach - 1e-6 * fabs(weigh.max));
            uint32_t low = none + 1;
            if (!weigh.infinite && bound > -INFINITY) low = max(low, key_of<UNIT>(bound) - 1u);
            cut = select<true>(row, weigh, cut, top, min(low, top), need, turn);
        }
        // ---- the kept ones' sum, and the place of u in it
        const double least = fmin(fmax(min_p, 0.0), 1.0) * exp2((double)p.scale);
        auto weight_kept = [&](float x, int w, int e) -> uint64_t {
            if (!kept(key_of<UNIT>(x), w, e)) return 0ull;
            const double s = weigh.scaled(weigh.distance(x));
            return s >= least ? Weigher::whole(s) : 0ull;
        };
        uint64_t sum = 0;
        row.each([&](float x, int w, int e) { sum += weight_kept(x, w, e); });
        sum = row.total(sum, &sh->cta_sum[0][1], before);
        const double place = fmax((double)u, 0.0) * (double)sum;
        const uint64_t target = place < (double)sum ? min((uint64_t)place, sum - 1) : sum - 1;
        uint64_t at = before;
        for (int i = 0; i < warp; ++i) at += sh->warp_sum[i];
        writer = false;
        if (at <= target && target < at + sh->warp_sum[warp]) {
            for (int w0 = row.first; w0 < row.last; w0 += 32) {
                const int w = w0 + lane;
                float x[N];
                uint64_t mine = 0;
                if (w < row.last) {
                    Ty::load(data[w], x);
#pragma unroll
                    for (int e = 0; e < N; ++e) mine += weight_kept(x[e], w, e);
                }
                const uint64_t upto = at + warp_scan(mine);
                if (upto > target && upto - mine <= target) {
                    uint64_t run = upto - mine;
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const uint64_t own = weight_kept(x[e], w, e);
                        if (run <= target && target < run + own) {
                            token = row.index(w, e);
                            // ln(w / sum): w from its distance, the sum without its factor 2^S
                            logprob = (float)(weigh.distance(x[e]) * -2.7076061740622863e-03 -
                                              (log((double)sum) - p.scale * 0.6931471805599453));
                            writer = true;
                        }
                        run += own;
                    }
                }
                at = __shfl_sync(0xffffffffu, upto, 31);
                if (at > target) break;
            }
        }
    }
    if (writer) {
        p.tokens[b] = token;
        if (p.logprobs) p.logprobs[b] = logprob;
    }
    if (CLUSTER) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <typename T>
static int launch(const Params &q, int64_t B, cudaStream_t st) {
    Params p = q;
    const int64_t bytes = (int64_t)p.V * (int64_t)sizeof(T);
    int ctas = MAX_CTAS;
    while (ctas > 1 && B * ctas >= 8 * 148 && bytes * 2 / ctas <= (64 << 10)) ctas /= 2;
    while (ctas > 1 && bytes / ctas < 2048) ctas /= 2;
    p.slice = ((p.V + ctas - 1) / ctas + 15) / 16 * 16;
    const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (size_t)p.slice * sizeof(T) + 32;
    auto kernel = ctas > 1 ? sample_kernel<T, true> : sample_kernel<T, false>;
    static PerDeviceFlag configured;
    const int dev = current_device();
    if (!configured.test(dev)) {
        const int most = (int)((sizeof(Shared) + 15) / 16 * 16 + MAX_SLICE + 32);
        QL_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        QL_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        configured.set(dev);
    }
    const unsigned gy = (unsigned)(B < 32768 ? B : 32768);
    for (int64_t b0 = 0; b0 < B; b0 += (int64_t)gy) {
        const int64_t rows = B - b0 < gy ? B - b0 : gy;
        Params r = p;
        r.logits = reinterpret_cast<const T *>(p.logits) + b0 * p.stride;
        r.u = p.u + b0;
        r.temperature = p.temperature ? p.temperature + b0 : nullptr;
        r.top_p = p.top_p ? p.top_p + b0 : nullptr;
        r.min_p = p.min_p ? p.min_p + b0 : nullptr;
        r.top_k = p.top_k ? p.top_k + b0 : nullptr;
        r.tokens = p.tokens + b0;
        r.logprobs = p.logprobs ? p.logprobs + b0 : nullptr;
        QL_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)ctas, (unsigned)rows), dim3(THREADS), smem, st, (unsigned)ctas, r));
    }
    return QL_OK;
}

}  // namespace samplek

// bytes of one row's logits that a call can take
int64_t sample_row_limit() { return (int64_t)samplek::MAX_CTAS * samplek::MAX_SLICE - 16 * 4 * samplek::MAX_CTAS; }

int launch_sample(const samplek::Params &p, int dtype, int64_t B, cudaStream_t st) {
    using namespace samplek;
    if (dtype == QL_F32) return launch<float>(p, B, st);
    return dtype == QL_BF16 ? launch<__nv_bfloat16>(p, B, st) : launch<__half>(p, B, st);
}

}  // namespace ql
