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
constexpr int BINS = 2048, GROUPS = 32, GROUP = BINS / GROUPS;  // of a histogram
constexpr int LIST = 512;         // elements that are compared one by one (one a thread)
constexpr int MAX_CTAS = 8;       // of a cluster
constexpr int MAX_SLICE = 160 << 10;  // bytes of a row in one CTA's shared memory
constexpr uint32_t NO_INDEX = 0xffffffffu;
static_assert(LIST <= THREADS && GROUPS == 32 && GROUP == 64 && BINS == 4 * THREADS, "the divisions among threads and lanes below");

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

// Larger for what comes first: by the value, equal ones by the index.
__device__ __forceinline__ uint64_t place_of(uint32_t key, uint32_t index) { return (uint64_t)key << 32 | ~index; }

struct Cut {  // the kept: a logit above this, or equal and the index at most this
    float value;
    uint32_t index;
};

// Shared memory besides the slice.  What other CTAs read after a barrier is not written again before
// another barrier has passed: hence counts and sums in turn.
struct Shared {
    uint32_t count[2][BINS];
    union {
        struct {
            uint32_t lo[BINS / 2], hi[BINS / 2];    // sums of weights as lo + 2^32 hi
        };
        struct {                                    // the cluster's list
            ulonglong2 all[LIST];                   // place in the order (place_of), weight
        };
    };
    uint64_t group[2][GROUPS];                      // sums of a histogram's groups of bins
    uint32_t group_count[2][GROUPS];
    uint32_t list_key[LIST], list_index[LIST];      // this CTA's part of it
    double table[16];
    uint64_t warp_sum[WARPS];
    uint64_t cta_sum[2];
    uint32_t warp_max[WARPS], warp_min[WARPS], cta_max, cta_min, cta_first;
    uint32_t list_count[2], tie_index[2];
    // what warp 0 found in a histogram
    uint64_t found_before, found_estimate;
    uint32_t found_bin, found_count, found_first, found_last;
    int hit;
    Cut cut;
};

template <typename T>
struct Type;
template <>
struct Type<float> {
    static constexpr int N = 4, UNIT = 0;  // elements of 16 bytes; zero bits at the end of their fp32 form
    static constexpr uint32_t NONE = 0xff800000u;  // a word of -inf
    static __device__ __forceinline__ void load(const uint4 &v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    }
    // largest of the elements, NaN if one is
    static __device__ __forceinline__ float largest(const uint4 &v) {
        float m, n;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(__uint_as_float(v.x)), "f"(__uint_as_float(v.y)));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(n) : "f"(__uint_as_float(v.z)), "f"(__uint_as_float(v.w)));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(n));
        return m;
    }
};
template <>
struct Type<__nv_bfloat16> {
    static constexpr int N = 8, UNIT = 16;
    static constexpr uint32_t NONE = 0xff80ff80u;
    static __device__ __forceinline__ void load(const uint4 &v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = bf16lo(w[i]), x[2 * i + 1] = bf16hi(w[i]);
    }
    static __device__ __forceinline__ float largest(const uint4 &v) {
        uint32_t m, n;
        float r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(v.x), "r"(v.y));
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(n) : "r"(v.z), "r"(v.w));
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(n));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(bf16lo(m)), "f"(bf16hi(m)));
        return r;
    }
};
template <>
struct Type<__half> {
    static constexpr int N = 8, UNIT = 13;
    static constexpr uint32_t NONE = 0xfc00fc00u;
    static __device__ __forceinline__ float lower(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
    static __device__ __forceinline__ float upper(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
    static __device__ __forceinline__ void load(const uint4 &v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = lower(w[i]), x[2 * i + 1] = upper(w[i]);
    }
    static __device__ __forceinline__ float largest(const uint4 &v) {
        uint32_t m, n;
        float r;
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(v.x), "r"(v.y));
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(n) : "r"(v.z), "r"(v.w));
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(n));
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(lower(m)), "f"(upper(m)));
        return r;
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
// f(CTA) of each of the cluster's, its loads in flight together; 0 past the last
template <typename V, typename F>
__device__ __forceinline__ void of_all(V (&v)[MAX_CTAS], uint32_t ctas, F f) {
#pragma unroll
    for (uint32_t c = 0; c < MAX_CTAS; ++c) v[c] = c < ctas ? f(c) : V(0);
}
__device__ __forceinline__ uint32_t sum_u32(const void *p, uint32_t ctas) {
    uint32_t v[MAX_CTAS], s = 0;
    of_all(v, ctas, [&](uint32_t c) { return ld_cluster_u32(p, c); });
#pragma unroll
    for (int c = 0; c < MAX_CTAS; ++c) s += v[c];
    return s;
}
__device__ __forceinline__ uint64_t sum_u64(const void *p, uint32_t ctas) {
    uint64_t v[MAX_CTAS], s = 0;
    of_all(v, ctas, [&](uint32_t c) { return ld_cluster_u64(p, c); });
#pragma unroll
    for (int c = 0; c < MAX_CTAS; ++c) s += v[c];
    return s;
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

// fp32 to fp64 in integer instructions (the conversion has a quarter of the fp64 rate).  Values below 2^-126 keep their
// sign and some magnitude below 2^-125, infinities become 2^128: neither makes a difference to a weight
// at the temperatures in use (Weigher).
__device__ __forceinline__ double widen(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);  // (-0 as 0)
    return __hiloint2double((int)((((b & 0x7fffffffu) >> 3) + 0x38000000u) | (b & 0x80000000u)), (int)(b << 29));
}

struct Weigher {
    static constexpr uint64_t BIAS = 0x4330000000000000ull;  // bits of 2^52
    static constexpr double C = 0.04332169878499658;          // ln 2 / 16
    double max, rate;  // of the row; 16 log2(e) / temperature
    int far;           // upper word of the distance from which on weights are 0
    int scale;         // S
    const double *table;

    __device__ __forceinline__ Weigher(float largest, double temperature, int scale_, const double *table_)
        : max(widen(largest)), scale(scale_), table(table_) {
        // The temperature is held between 2e-29 and 4e28: beyond, only logits below 1e-26 or above 1e26 could
        // tell the difference.
        const double limit = 16.0 * (scale + 2);
        rate = fmin(fmax(23.083120654223414 / temperature, limit * 7.888609052210118e-31), 1.2676506002282294e30);
        far = __double2hiint(limit / rate);
    }
    // w and its factor 2^S in one number; 0 with `keep` false and where w is below 2^-(S + 1)
    __device__ __forceinline__ void parts(float x, bool keep, double &t, double &e) const {
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
        double d = max - widen(x);
        const int hi = __double2hiint(d);
        d = __hiloint2double(keep && hi < far ? hi : far, __double2loint(d));
        const double s = fma(d, rate, MAGIC);
        const int k = __double2loint(s);
        const double r = fma(-d, rate, s - MAGIC);
        e = fma(fma(fma(fma(fma(C * C * C * C * C / 120, r, C * C * C * C / 24), r, C * C * C / 6), r, C * C / 2), r, C), r, 1.0);
        t = table[k & 15];
        t = __hiloint2double(__double2hiint(t) + (scale << 20) - ((k & ~15) << 16), __double2loint(t));
    }
    // W + BIAS: sums of n of them are n * BIAS too large (modulo 2^64)
    __device__ __forceinline__ uint64_t biased(float x, bool keep) const {
        double t, e;
        parts(x, keep, t, e);
        return (uint64_t)__double_as_longlong(fma(t, e, 4503599627370496.0));
    }
    __device__ __forceinline__ uint64_t operator()(float x, bool keep = true) const { return biased(x, keep) - BIAS; }
    // ln(w / sum): w from its distance, the sum without its factor 2^S
    __device__ __forceinline__ float logprob(float x, uint64_t sum) const {
        return (float)((widen(x) - max) * (rate * C) - log((double)sum * exp2(-(double)scale)));
    }
    // the same, 0 where w 2^S is below `least`
    __device__ __forceinline__ uint64_t at_least(float x, bool keep, double least) const {
        double t, e;
        parts(x, keep, t, e);
        return t * e >= least ? (uint64_t)__double_as_longlong(fma(t, e, 4503599627370496.0)) - BIAS : 0ull;
    }
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
    uint4 *data;
    Shared *sh;
    int first, last;         // this warp's words
    int skew;                // places before the slice in the first word
    uint32_t base;           // index of the slice's first token
    uint32_t ctas, rank;
    uint64_t *slot;          // of the next sum
    int turn;                // of the next histogram

    __device__ __forceinline__ uint32_t index(int word, int e) const { return base + (uint32_t)(word * N + e - skew); }

    // f(v, w) of this warp's words in order, 32 at a time, a lane each; -inf past the last
    template <typename F>
    __device__ __forceinline__ void words(F f) const {
        const int lane = threadIdx.x & 31;
        for (int w0 = first; w0 < last; w0 += 32) {
            uint4 v = make_uint4(Ty::NONE, Ty::NONE, Ty::NONE, Ty::NONE);
            if (w0 + lane < last) v = data[w0 + lane];
            f(v, w0 + lane);
        }
    }
    // the same without words of which no lane has an element of at least `low`
    template <typename F>
    __device__ __forceinline__ void words_from(float low, F f) const {
        words([&](const uint4 &v, int w) {
            if (__any_sync(0xffffffffu, Ty::largest(v) >= low)) f(v, w);
        });
    }
    // f(x, w, e) of their elements
    template <typename F>
    __device__ __forceinline__ void each_from(float low, F f) const {
        words_from(low, [&](const uint4 &v, int w) {
            float x[N];
            Ty::load(v, x);
#pragma unroll
            for (int e = 0; e < N; ++e) f(x[e], w, e);
        });
    }
    __device__ __forceinline__ bool kept(const Cut &cut, float x, int w, int e) const {
        return x > cut.value || (x == cut.value && index(w, e) <= cut.index);
    }

    // Sum over the cluster of a value of each thread; `before` is that of the CTAs before this one, and
    // warp_sum[] holds the warps'.
    __device__ __forceinline__ uint64_t total(uint64_t v, uint64_t &before) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh->warp_sum[warp] = v;
        __syncthreads();
        const uint64_t cta = warp_sum(lane < WARPS ? sh->warp_sum[lane] : 0ull);
        if (!CLUSTER) {
            before = 0;
            return cta;
        }
        if (threadIdx.x == 0) *slot = cta;
        cluster_sync_all();
        const uint64_t mine = lane < ctas ? ld_cluster_u64(slot, lane) : 0ull;
        slot = slot == &sh->cta_sum[0] ? &sh->cta_sum[1] : &sh->cta_sum[0];
        before = warp_sum(lane < rank ? mine : 0ull);
        return warp_sum(mine);
    }

    // This CTA's elements for which f(x, w, e) holds, as its part of the list; the number of the cluster's.
    // All CTAs may read it after the barrier inside.
    template <typename F>
    __device__ __forceinline__ uint32_t collect(int which, float low, F f) {
        if (threadIdx.x == 0) sh->list_count[which] = 0;
        __syncthreads();
        each_from(low, [&](float x, int w, int e) {
            if (f(x, w, e)) append(which, x, w, e);
        });
        sync_all<CLUSTER>();
        return sum_u32(&sh->list_count[which], ctas);
    }
    __device__ __forceinline__ void append(int which, float x, int w, int e) const {
        const uint32_t at = atomicAdd(&sh->list_count[which], 1u);
        if (at < LIST) {
            sh->list_key[at] = key_of<UNIT>(x);
            sh->list_index[at] = index(w, e);
        }
    }
    // Brings the cluster's list (at most LIST) together in all[]; true where this thread has an element of it.
    // No CTA may refill its part before the others have read it: a barrier of the cluster stands
    // before every collect.
    template <typename M>
    __device__ __forceinline__ bool gather(int which, uint64_t &place, uint64_t &own, M measure) const {
        uint32_t n[MAX_CTAS], at = threadIdx.x, from = MAX_CTAS;
        of_all(n, ctas, [&](uint32_t c) { return ld_cluster_u32(&sh->list_count[which], c); });
#pragma unroll
        for (uint32_t c = 0; c < MAX_CTAS; ++c) {  // this thread's element: the at-th of CTA `from`
            if (from == MAX_CTAS && at < n[c]) from = c;
            if (from == MAX_CTAS) at -= n[c];
        }
        const bool has = from < MAX_CTAS;
        place = own = 0;
        if (has) {
            const uint32_t key = ld_cluster_u32(&sh->list_key[at], from);
            place = place_of(key, ld_cluster_u32(&sh->list_index[at], from));
            own = measure(value_of<UNIT>(key));
            sh->all[threadIdx.x] = make_ulonglong2(place, own);
        }
        __syncthreads();
        return has;
    }
    // Of the list's `count` elements in their order, the one at which the sum of the measure reaches
    // `need`: sh->cut, and true; false if it does not.
    template <typename M>
    __device__ __forceinline__ bool resolve(int which, uint32_t count, uint64_t need, M measure) const {
        uint64_t place, own;
        if (threadIdx.x == 0) sh->hit = 0;
        if (gather(which, place, own, measure)) {
            uint64_t before = 0;
#pragma unroll 4
            for (uint32_t i = 0; i < count; ++i) {
                const ulonglong2 a = sh->all[i];
                before += a.x > place ? a.y : 0ull;
            }
            if (before + own >= need && before < need) {
                sh->cut = {value_of<UNIT>((uint32_t)(place >> 32)), ~(uint32_t)place};
                sh->hit = 1;
            }
        }
        __syncthreads();
        const bool hit = sh->hit != 0;
        __syncthreads();
        return hit;
    }
};

// The token from a list that holds all that may be drawn (at most LIST, in all CTAs' parts): top-k (none where k
// is 0), top-p by p of the first k's sum -- or by `need`, where that is not 0 --, min-p by `least`, the draw.
// By one CTA.
template <typename T, bool CLUSTER>
__device__ __forceinline__ void finish(const Row<T, CLUSTER> &row, const Weigher &weigh, int which, uint32_t count, uint64_t k, double p,
                                       uint64_t need, double least, double u, int64_t *token, float *logprob) {
    constexpr int UNIT = Type<T>::UNIT;
    Shared *sh = row.sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto block_sum = [&](uint64_t v) {
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh->warp_sum[warp] = v;
        __syncthreads();
        return warp_sum(lane < WARPS ? sh->warp_sum[lane] : 0ull);
    };
    uint64_t place, own;
    bool stays = row.gather(which, place, own, [&](float x) { return weigh(x); });
    const float x = value_of<UNIT>((uint32_t)(place >> 32));
    uint64_t before = 0;
    uint32_t rank = 0;
    if (stays)
#pragma unroll 4
        for (uint32_t i = 0; i < count; ++i) {
            const ulonglong2 a = sh->all[i];
            before += a.x > place ? a.y : 0ull;
            rank += a.x > place ? 1u : 0u;
        }
    if (k) {
        stays = stays && rank < k;
        if (p < 1.0) {
            const uint64_t sum = block_sum(stays ? own : 0ull);
            const double target = ceil((double)sum * p);
            need = target >= 1.0 ? min(sum, (uint64_t)target) : 1ull;
        }
    }
    if (need) stays = stays && before < need;
    if (stays && least > 0.0) own = weigh.at_least(x, true, least);
    if (!stays) own = 0;
    const uint64_t sum = block_sum(own);  // (all[] has been read)
    sh->all[tid] = make_ulonglong2(~(uint32_t)place, own);
    __syncthreads();
    if (!own) return;
    const double at = fmax(u, 0.0) * (double)sum;
    const uint64_t target = at < (double)sum ? min((uint64_t)at, sum - 1) : sum - 1;
    const uint32_t index = ~(uint32_t)place;
    uint64_t upto = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < count; ++i) {
        const ulonglong2 a = sh->all[i];
        upto += (uint32_t)a.x < index ? a.y : 0ull;
    }
    if (upto <= target && target < upto + own) {
        *token = index;
        if (logprob) *logprob = weigh.logprob(x, sum);
    }
}

// A value below which nothing is among the k largest: of the 16-byte words' largest elements, from `least` up to
// `top`, k are at least that large.  -inf if they are not that many.
template <typename T, bool CLUSTER>
__device__ __forceinline__ float bound_of_largest(Row<T, CLUSTER> &row, float top, float least, uint64_t k) {
    Shared *sh = row.sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float c = top > least ? (BINS - 1) / (top - least) : 0.f;
    uint32_t *count = sh->count[row.turn & 1], *group = sh->group_count[row.turn & 1];
    ++row.turn;
    *reinterpret_cast<uint4 *>(count + 4 * tid) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    row.words([&](const uint4 &v, int) {
        const float x = Type<T>::largest(v);
        if (x >= least) atomicAdd(&count[min((int)((top - x) * c), BINS - 1)], 1u);
    });
    __syncthreads();
    for (int g = warp; g < GROUPS; g += WARPS) {
        const uint2 n = *reinterpret_cast<const uint2 *>(count + g * GROUP + 2 * lane);
        const uint32_t s = __reduce_add_sync(0xffffffffu, n.x + n.y);
        if (lane == 0) group[g] = s;
    }
    sync_all<CLUSTER>();
    if (warp == 0) {
        const uint64_t s = sum_u32(&group[lane], row.ctas);
        uint64_t upto = warp_scan(s);
        const unsigned past = __ballot_sync(0xffffffffu, upto >= k);
        const int g = past ? __ffs(past) - 1 : 0;
        const uint64_t before = __shfl_sync(0xffffffffu, upto - s, g);
        const uint64_t a = sum_u32(&count[g * GROUP + 2 * lane], row.ctas), b = sum_u32(&count[g * GROUP + 2 * lane + 1], row.ctas);
        upto = before + warp_scan(a + b);
        const unsigned here = __ballot_sync(0xffffffffu, upto >= k);
        if (here && lane == __ffs(here) - 1) sh->found_bin = g * GROUP + 2 * lane + (upto - b >= k ? 0 : 1);
        if (!past && lane == 0) sh->found_bin = NO_INDEX;
    }
    __syncthreads();
    const uint32_t bin = sh->found_bin;
    __syncthreads();
    if (bin == NO_INDEX || c == 0.f) return -INFINITY;
    // the bin's lower edge, less what the roundings of the bin's number may amount to
    const float range = top - least, edge = top - (float)(bin + 1) / c - 1e-5f * range - 1e-6f * fabsf(top);
    return edge > -INFINITY ? edge : -INFINITY;
}

// The cut after the shortest prefix, in the order of the values, whose measure (elements, or weights
// with WEIGHT) reaches `need` >= 1, among the elements within `cut` whose keys are from `low` up to `high`.
// Elements left out by `low` must not be needed.  By histograms of keys, each dividing the bin that
// holds the border, until it holds at most LIST elements or one value.
template <bool WEIGHT, typename T, bool CLUSTER>
__device__ __noinline__ Cut select(Row<T, CLUSTER> &row, const Weigher &weigh, Cut cut, uint32_t high, uint32_t low, uint64_t need) {
    constexpr int UNIT = Type<T>::UNIT, LOG = WEIGHT ? 10 : 11, PER = (1 << LOG) / GROUPS / 32;  // bins of a group's lane
    Shared *sh = row.sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t cut_key = key_of<UNIT>(cut.value);
    low = max(low, cut_key);
    auto inside = [&](uint32_t key, int w, int e) {
        return key >= low && key <= high && (key != cut_key || row.index(w, e) <= cut.index);
    };
    auto measure = [&](float x) { return WEIGHT ? weigh(x) : 1ull; };
    for (;;) {
        const float from = value_of<UNIT>(low);
        const uint32_t range = high - low;
        const int bits = 32 - __clz((int)range), shift = bits > LOG ? bits - LOG : 0;
        uint32_t *count = sh->count[row.turn & 1];
        uint64_t *group = sh->group[row.turn & 1];
        ++row.turn;
        if (WEIGHT) sync_all<CLUSTER>();  // (one set of sums: the others have read those of the round before)
        *reinterpret_cast<uint4 *>(count + 4 * tid) = make_uint4(0, 0, 0, 0);
        if (WEIGHT) sh->lo[2 * tid] = sh->lo[2 * tid + 1] = sh->hi[2 * tid] = sh->hi[2 * tid + 1] = 0;
        __syncthreads();
        row.each_from(from, [&](float x, int w, int e) {
            const uint32_t key = key_of<UNIT>(x);
            const bool in = inside(key, w, e);
            const unsigned active = __ballot_sync(0xffffffffu, in);
            if (!active) return;
            uint64_t weight = WEIGHT ? weigh(x, in) : 0ull;
            // equal elements of a warp (a row of few values) count as one
            uint32_t n = 1;
            const uint32_t one = __shfl_sync(0xffffffffu, key, __ffs(active) - 1);
            if (__all_sync(0xffffffffu, !in || key == one)) {
                if (lane != __ffs(active) - 1) return;
                n = __popc(active);
                weight *= n;
            }
            if (!in) return;
            const uint32_t b = (high - key) >> shift;
            atomicAdd(&count[b], n);
            if (WEIGHT) {
                const uint32_t lo = (uint32_t)weight, old = atomicAdd(&sh->lo[b], lo);
                const uint32_t hi = (uint32_t)(weight >> 32) + (old + lo < old ? 1u : 0u);
                if (hi) atomicAdd(&sh->hi[b], hi);
            }
        });
        __syncthreads();
        for (int g = warp; g < GROUPS; g += WARPS) {
            uint64_t s = 0;
            for (int k = 0; k < PER; ++k) {
                const int i = (g * PER + k) * 32 + lane;
                s += WEIGHT ? ((uint64_t)sh->hi[i] << 32) + sh->lo[i] : (uint64_t)count[i];
            }
            s = warp_sum(s);
            if (lane == 0) group[g] = s;
        }
        sync_all<CLUSTER>();
        if (warp == 0) {
            // the group, then the bin of it, that holds the border
            uint64_t s = 0;
            s = sum_u64(&group[lane], row.ctas);
            uint64_t upto = warp_scan(s);
            const unsigned past = __ballot_sync(0xffffffffu, upto >= need);
            const int g = past ? __ffs(past) - 1 : 0;
            uint64_t before = __shfl_sync(0xffffffffu, upto - s, g);
            bool found = false;
            for (int k = 0; k < PER && !found; ++k) {
                const int i = (g * PER + k) * 32 + lane;
                const uint32_t n = sum_u32(&count[i], row.ctas);
                s = n;
                if (WEIGHT) {
                    s = 0;
                    for (uint32_t c = 0; c < row.ctas; ++c)
                        s += (uint64_t)ld_cluster_u32(&sh->lo[i], c) + ((uint64_t)ld_cluster_u32(&sh->hi[i], c) << 32);
                }
                upto = before + warp_scan(s);
                const unsigned here = __ballot_sync(0xffffffffu, upto >= need);
                found = here != 0;
                if (found && lane == __ffs(here) - 1) {
                    sh->found_bin = i;
                    sh->found_count = n;
                    sh->found_before = upto - s;
                }
                before = __shfl_sync(0xffffffffu, upto, 31);
            }
            if (!past && lane == 0) sh->found_bin = NO_INDEX;
        }
        __syncthreads();
        const uint32_t bin = sh->found_bin, n = sh->found_count;
        if (bin == NO_INDEX) return cut;  // all of them together do not reach it
        need -= sh->found_before;
        high -= bin << shift;
        low = max(low, high - min(high, (1u << shift) - 1u));
        __syncthreads();
        if (n <= LIST) {
            row.collect(WEIGHT, value_of<UNIT>(low), [&](float x, int w, int e) { return inside(key_of<UNIT>(x), w, e); });
            return row.resolve(WEIGHT, n, need, measure) ? sh->cut : cut;
        }
        if (shift == 0) {
            // more equal elements than that: the last of them that is needed, by index
            const float value = value_of<UNIT>(high);
            const uint64_t ties = (need + measure(value) - 1) / measure(value);
            if (ties >= n) return {value, cut_key == high ? cut.index : NO_INDEX};
            uint64_t mine = 0, before;
            row.each_from(value, [&](float x, int w, int e) { mine += inside(key_of<UNIT>(x), w, e) ? 1u : 0u; });
            row.total(mine, before);
            // the warp whose elements hold it looks for it; its CTA tells the others
            if (tid == 0) sh->tie_index[WEIGHT] = NO_INDEX;
            __syncthreads();
            uint64_t at = before;
            for (int i = 0; i < warp; ++i) at += sh->warp_sum[i];
            if (at < ties && at + sh->warp_sum[warp] >= ties) {
                row.words([&](const uint4 &v, int w) {
                    float x[Type<T>::N];
                    Type<T>::load(v, x);
                    int m = 0;
#pragma unroll
                    for (int e = 0; e < Type<T>::N; ++e) m += inside(key_of<UNIT>(x[e]), w, e) ? 1 : 0;
                    const uint64_t upto = at + warp_scan((uint64_t)m);
                    if (upto >= ties && upto - m < ties) {
                        uint64_t left = ties - (upto - m);
#pragma unroll
                        for (int e = 0; e < Type<T>::N; ++e)
                            if (inside(key_of<UNIT>(x[e]), w, e) && --left == 0) sh->tie_index[WEIGHT] = row.index(w, e);
                    }
                    at = __shfl_sync(0xffffffffu, upto, 31);
                });
            }
            sync_all<CLUSTER>();
            uint32_t ix = NO_INDEX;
            for (uint32_t c = 0; c < row.ctas; ++c) ix = min(ix, ld_cluster_u32(&sh->tie_index[WEIGHT], c));
            return {value, ix};
        }
    }
}

// Top-p among the elements within `cut`: their weights' sum `total`, of which the prefix has to reach `need` = p times that.  One
// pass sums the weights and counts the elements in bins of equal width; each counted as an element at its bin's
// middle, they say about where the border is.  (Sums of weights in each bin would cost three atomic additions
// for every element.)  Where all elements down to the border fit the list, the list is all that is needed: true, its
// length in `listed`.  Else a pass over the elements above a few bins around the border sums them exactly and lists
// those in the bins; where the border is not among these after all, the sum tells by how much the
// estimate is off.  `cut` is then the one after the prefix.
template <typename T, bool CLUSTER>
__device__ __forceinline__ bool nucleus(Row<T, CLUSTER> &row, const Weigher &weigh, Cut &cut, float top, double p, int V, uint64_t &need,
                                        uint32_t &listed) {
    constexpr int UNIT = Type<T>::UNIT, N = Type<T>::N;
    Shared *sh = row.sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Weights below (1 - p) / (2 V) of the largest (1, so of the sum) sum up to less than (1 - p), so none of them is in
    // the prefix, and only logits above that (with a margin for roundings) are counted.
    const double smallest = fmax(0.5, 0.5 * (1.0 - p) / V * exp2((double)weigh.scale));
    const double reach = (weigh.scale - log2(smallest)) * 16.0 / weigh.rate * 1.000001;
    const float low = fmaxf(fminf(top, fmaxf((float)((double)top - reach - 1e-6 * fabs((double)top)), -3.4028234e38f)), cut.value);
    const float c = top > low ? (BINS - 1) / (top - low) : 0.f, width = top > low ? (top - low) / (BINS - 1) : 0.f;
    // (not decreasing as x falls: every step is a rounded operation of that kind)
    auto bin_of = [&](float x) { return min((int)((top - x) * c), BINS - 1); };
    auto middle = [&](int b) { return weigh(fmaf(-(float)b - 0.5f, width, top)); };
    uint32_t *count = sh->count[row.turn & 1], *group_count = sh->group_count[row.turn & 1];
    uint64_t *group = sh->group[row.turn & 1];
    ++row.turn;
    *reinterpret_cast<uint4 *>(count + 4 * tid) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint64_t mine = 0, before;
    const bool whole = cut.value == -INFINITY;
    row.words_from(cut.value, [&](const uint4 &v, int w) {
        float x[N];
        Type<T>::load(v, x);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const bool in = whole || row.kept(cut, x[e], w, e);
            mine += weigh.biased(x[e], in);
            if (in && x[e] >= low) atomicAdd(&count[bin_of(x[e])], 1u);
        }
        mine -= N * Weigher::BIAS;
    });
    __syncthreads();
    {
        const uint4 n = *reinterpret_cast<const uint4 *>(count + 4 * tid);
        uint64_t s = 0;
        if (n.x | n.y | n.z | n.w)
            s = n.x * middle(4 * tid) + n.y * middle(4 * tid + 1) + n.z * middle(4 * tid + 2) + n.w * middle(4 * tid + 3);
        uint32_t k = n.x + n.y + n.z + n.w;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), k += __shfl_xor_sync(0xffffffffu, k, o);
        if ((tid & 15) == 0) group[tid >> 4] = s, group_count[tid >> 4] = k;
    }
    const uint64_t sum = row.total(mine, before);
    const double target = ceil((double)sum * p);
    need = target >= 1.0 ? min(sum, (uint64_t)target) : 1ull;
    // the border is in bin `first` or after it, and before bin `end`
    int first = 0, end = BINS;
    uint64_t seek = need;  // in sums of the estimate
    for (;;) {
        if (warp == 0) {
            const uint64_t s = sum_u64(&group[lane], row.ctas);
            const uint32_t k = sum_u32(&group_count[lane], row.ctas);
            uint64_t upto = warp_scan(s);
            const uint32_t elements = (uint32_t)warp_scan((uint64_t)k);
            // up to which group the weights reach `need` for certain: none is less than the middle's by more than half a bin
            const double sure = exp2(-0.51 * width * weigh.rate / 16.0) * (1.0 - 1e-6);
            const unsigned reached = __ballot_sync(0xffffffffu, (double)upto * sure >= (double)need);
            const int last = reached ? __ffs(reached) - 1 : 0;
            const uint32_t all = __shfl_sync(0xffffffffu, elements, last);
            if (first == 0 && end == BINS && reached && all <= LIST) {
                if (lane == 0) sh->found_bin = last * GROUP + GROUP - 1, sh->found_count = all;
            } else {
                const unsigned past = __ballot_sync(0xffffffffu, upto >= seek);
                const int g = past ? __ffs(past) - 1 : GROUPS - 1;
                const uint64_t start = __shfl_sync(0xffffffffu, upto - s, g);  // before the group
                const int i = g * GROUP + 2 * lane;
                const uint32_t a = sum_u32(&count[i], row.ctas), b = sum_u32(&count[i + 1], row.ctas);
                const uint64_t wa = a ? a * middle(i) : 0ull, wb = b ? b * middle(i + 1) : 0ull;
                upto = start + warp_scan(wa + wb);
                const unsigned here = __ballot_sync(0xffffffffu, upto >= seek);
                int bin = BINS - 1;
                if (here) {
                    const int l = __ffs(here) - 1;
                    bin = g * GROUP + 2 * l + (__shfl_sync(0xffffffffu, upto - wb >= seek ? 1 : 0, l) ? 0 : 1);
                }
                if (bin < first || bin >= end) bin = (first + end) / 2;  // (the estimate has not come closer)
                // the bins around it that fit the list: 2^n to either side
                const int at = bin - 16 + lane;
                const uint32_t n = at >= first && at < end ? sum_u32(&count[at], row.ctas) : 0u;
                uint32_t m = __reduce_add_sync(0xffffffffu, n);
                int side = 16;
                while (m > LIST && side > 0) {
                    side >>= 1;
                    m = __reduce_add_sync(0xffffffffu, lane >= 16 - side && lane <= 16 + side ? n : 0u);
                }
                const int b0 = max(bin - side, first), b1 = min(bin + min(side, 15), end - 1);
                // the estimate of what is before the first of them, from the start of the group
                uint64_t est = start + warp_sum((i < b0 ? wa : 0ull) + (i + 1 < b0 ? wb : 0ull));
                if (b0 < g * GROUP) est = start - warp_sum(at >= b0 && at < g * GROUP && n ? n * middle(at) : 0ull);
                if (lane == 0) {
                    sh->found_bin = NO_INDEX;
                    sh->found_count = m;
                    sh->found_first = b0;
                    sh->found_last = b1;
                    sh->found_estimate = est;
                }
            }
        }
        __syncthreads();
        const uint32_t through = sh->found_bin, n = sh->found_count;
        const int b0 = sh->found_first, b1 = sh->found_last;
        const uint64_t est = sh->found_estimate;
        __syncthreads();
        if (through != NO_INDEX) {
            listed = row.collect(1, low, [&](float x, int w, int e) { return x >= low && bin_of(x) <= (int)through && row.kept(cut, x, w, e); });
            return true;
        }
        if (n > LIST) {  // a bin of many elements, likely equal ones
            Row<T, CLUSTER> other = row;
            cut = select<true>(other, weigh, cut, key_of<UNIT>(top), key_of<UNIT>(low), need);
            row.turn = other.turn;
            return false;
        }
        mine = 0;
        if (tid == 0) sh->list_count[1] = 0;
        __syncthreads();
        row.each_from(low, [&](float x, int w, int e) {
            const int b = bin_of(x);
            const bool in = x >= low && b <= b1 && (whole || row.kept(cut, x, w, e));
            mine += weigh(x, in && b < b0);
            if (in && b >= b0) row.append(1, x, w, e);
        });
        const uint64_t above = row.total(mine, before);
        if (above >= need) end = b0;
        else if (row.resolve(1, n, need - above, [&](float x) { return weigh(x); })) {
            cut = sh->cut;
            return false;
        } else first = b1 + 1;
        if (first >= end) return false;  // all of them together do not reach it
        seek = need + est - above;
        sync_all<CLUSTER>();  // the lists are filled again
    }
}

template <typename T, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const Params p) {
    using Ty = Type<T>;
    constexpr int N = Ty::N, UNIT = Ty::UNIT;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared *sh = reinterpret_cast<Shared *>(smem);
    pdl_trigger();
    pdl_wait();
    Row<T, CLUSTER> row;
    row.sh = sh;
    row.data = reinterpret_cast<uint4 *>(smem + (sizeof(Shared) + 15) / 16 * 16);
    row.ctas = CLUSTER ? gridDim.x : 1;
    row.rank = CLUSTER ? blockIdx.x : 0;
    row.slot = &sh->cta_sum[0];
    row.turn = 0;
    const int64_t b = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- the slice: whole words by asynchronous copies, the ends one by one
    row.base = row.rank * (uint32_t)p.slice;
    const int n = max(0, min(p.slice, p.V - (int)min(row.base, (uint32_t)p.V)));
    const T *src = reinterpret_cast<const T *>(p.logits) + b * p.stride + row.base;
    row.skew = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
    const int words = n ? (n + row.skew + N - 1) / N : 0;
    for (int w = tid; w < words; w += THREADS) {
        const int at = w * N - row.skew;
        if (at >= 0 && at + N <= n) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(row.data + w)), "l"(src + at) : "memory");
        } else {
            T *dst = reinterpret_cast<T *>(row.data + w);
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
    if (tid < 16) sh->table[tid] = exp2(-tid / 16.0);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const int per = (words + THREADS - 1) / THREADS * 32;
    row.first = min(words, warp * per);
    row.last = min(words, row.first + per);

    // ---- the largest logit
    float largest = -INFINITY, smallest = INFINITY;  // of the words' largest; of those above -inf
    row.words([&](const uint4 &v, int) {
        const float x = Ty::largest(v);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(largest) : "f"(x));
        if (x > -INFINITY) smallest = fminf(smallest, x);
    });
    uint32_t top = __reduce_max_sync(0xffffffffu, key_of<UNIT>(largest)), bottom = __reduce_min_sync(0xffffffffu, key_of<UNIT>(smallest));
    if (lane == 0) sh->warp_max[warp] = top, sh->warp_min[warp] = bottom;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < WARPS ? sh->warp_max[lane] : 0u);
    bottom = __reduce_min_sync(0xffffffffu, lane < WARPS ? sh->warp_min[lane] : NO_INDEX);
    if (CLUSTER) {
        if (tid == 0) sh->cta_max = top, sh->cta_min = bottom;
        cluster_sync_all();
        top = __reduce_max_sync(0xffffffffu, lane < row.ctas ? ld_cluster_u32(&sh->cta_max, lane) : 0u);
        bottom = __reduce_min_sync(0xffffffffu, lane < row.ctas ? ld_cluster_u32(&sh->cta_min, lane) : NO_INDEX);
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
        const float value = value_of<UNIT>(top);
        uint32_t at = NO_INDEX;
        row.each_from(value, [&](float x, int w, int e) {
            if (x == value) at = min(at, row.index(w, e));
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
        if (top == key_of<UNIT>(INFINITY)) {
            // infinite logits share everything: they are 0 in the slice from here on, the others -inf
            for (int w = row.first + lane; w < row.last; w += 32) {
                T *x = reinterpret_cast<T *>(row.data + w);
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = (float)x[e] == INFINITY ? T(0.f) : T(-INFINITY);
            }
            __syncwarp();
            top = bottom = key_of<UNIT>(0.f);
        }
        const float peak = value_of<UNIT>(top);
        const Weigher weigh(peak, temperature, p.scale, sh->table);
        const double least = fmin(fmax(min_p, 0.0), 1.0) * exp2((double)p.scale);
        Cut cut{-INFINITY, NO_INDEX};
        // whether all that may be drawn is in the list, its length, which counter, and what is left to do with it
        bool in_list = false;
        uint32_t listed = 0;
        uint64_t k = 0, need = 0, before;
        if (top_k > 0 && top_k < p.V) {
            const float low = top_k <= p.V / N ? bound_of_largest(row, peak, value_of<UNIT>(bottom), (uint64_t)top_k) : -INFINITY;
            if (top_k <= LIST && low > -INFINITY) {
                listed = row.collect(0, low, [&](float x, int, int) { return x >= low; });
                in_list = listed <= LIST;
                k = (uint64_t)top_k;
            }
            if (!in_list) {
                Row<T, CLUSTER> other = row;
                cut = select<false>(other, weigh, cut, top, low > -INFINITY ? max(none + 1, key_of<UNIT>(low)) : none + 1, (uint64_t)top_k);
                row.turn = other.turn;
                k = 0;
            }
        }
        if (!in_list && top_p < 1.0) in_list = nucleus(row, weigh, cut, peak, top_p, p.V, need, listed);
        writer = false;
        if (in_list) {
            if (row.rank == 0)
                finish(row, weigh, k ? 0 : 1, listed, k, top_p, need, least, (double)u, p.tokens + b, p.logprobs ? p.logprobs + b : nullptr);
        } else {
            // ---- the kept ones' sum, and the place of u in it
            auto weight_kept = [&](float x, int w, int e) { return weigh.at_least(x, row.kept(cut, x, w, e), least); };
            uint64_t mine = 0;
            const bool plain = cut.value == -INFINITY && least == 0.0;
            row.words_from(cut.value, [&](const uint4 &v, int w) {
                float x[N];
                Ty::load(v, x);
                if (plain) {
#pragma unroll
                    for (int e = 0; e < N; ++e) mine += weigh.biased(x[e], true);
                    mine -= N * Weigher::BIAS;
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) mine += weight_kept(x[e], w, e);
                }
            });
            const uint64_t sum = row.total(mine, before);
            const double place = fmax((double)u, 0.0) * (double)sum;
            const uint64_t target = place < (double)sum ? min((uint64_t)place, sum - 1) : sum - 1;
            uint64_t at = before;
            for (int i = 0; i < warp; ++i) at += sh->warp_sum[i];
            if (at <= target && target < at + sh->warp_sum[warp]) {
                row.words_from(cut.value, [&](const uint4 &v, int w) {
                    float x[N];
                    Ty::load(v, x);
                    uint64_t own[N], mine = 0;
#pragma unroll
                    for (int e = 0; e < N; ++e) mine += own[e] = weight_kept(x[e], w, e);
                    const uint64_t upto = at + warp_scan(mine);
                    if (upto > target && upto - mine <= target) {
                        uint64_t run = upto - mine;
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            if (run <= target && target < run + own[e]) {
                                token = row.index(w, e);
                                logprob = weigh.logprob(x[e], sum);
                                writer = true;
                            }
                            run += own[e];
                        }
                    }
                    at = __shfl_sync(0xffffffffu, upto, 31);
                });
            }
        }
    }
    if (writer) {
        p.tokens[b] = token;
        if (p.logprobs) p.logprobs[b] = logprob;
    }
    __syncwarp();
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
