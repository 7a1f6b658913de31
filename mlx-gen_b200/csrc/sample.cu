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
// The exponential (method: table and short polynomial, P. T. P. Tang 1989): 16 y = k + r with whole
// k and |r| <= 1/2, 2^-y = 2^-(k >> 4) * table[k & 15] * exp(-r ln 2 / 16), whose series ends after the
// fifth power (the sixth is below 2^-42: borders move by less than a 10^-12th of the sum).
//
// Bound: for many rows fp64 and integer instructions (9 and about 20 for each logit and pass; 64 and 128 lanes a
// clock and SM) and the two to four passes that top-p takes; for few rows the chain of passes and cluster barriers, about
// 1200 cycles each with what is exchanged.  Split: a cluster of up to 16 CTAs takes a row.  Slices that fit stay in shared
// memory, so that the row is read once whatever filters it has; longer ones are read again by each pass.
// Nothing is sorted but short lists: top-k takes a bound from the words' largest elements and lists what is above it;
// top-p counts in 2048 bins and lists a few bins around the border, or all above it where these are few.
// Scalars travel by stores into the other CTAs' shared memory before a barrier; what every warp would compute for itself is
// computed by one.
// Measured (bf16, 128256 logits from N(0, 2) with 24 likely ones among them, a graph's replay of the same rows): one row greedy
// 4.3 us, without filter 8.4, top-k 50 11.5, top-p 0.95 at temperature 0.8 16.2 (18.7 with log-probabilities and other rows
// each time); 64 rows 7.8, 22, 16, 62; 256 rows with top-p 0.98 at temperature 1.5 (half the vocabulary stays) 250, without
// the likely ones 301.
#include <string.h>

#include "pdl.cuh"

namespace ql {
namespace samplek {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 2048, GROUPS = 32, GROUP = BINS / GROUPS;  // of a histogram
constexpr int LIST = 512;         // elements that are put in order one by one (one a thread)
constexpr int WINDOW = 128;       // .. that top-p's border is looked for among
constexpr int FEW = 128;          // .. up to which each is compared with every other
constexpr int NEAR = 128;         // bins around a group that are looked at together
constexpr int MAX_CTAS = 16;      // of a cluster
constexpr int MAX_SLICE = 66 << 10;  // bytes of a row in one CTA's shared memory
constexpr int MAX_ROW = 1310208;     // bytes of a row: the longest that is tested
constexpr uint32_t NO_INDEX = 0xffffffffu;
static_assert(LIST <= THREADS && THREADS == 512 && MAX_CTAS <= WARPS && NEAR == 4 * 32 && GROUPS == 32 && GROUP == 64 && BINS == 4 * THREADS, "the divisions among threads and lanes below");

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
// another barrier has passed: hence counts and sums in turn.  (45 KB: two CTAs an SM beside slices of 66 KB.)
struct Shared {
    uint32_t count[2][BINS];
    union {
        struct {
            uint32_t lo[BINS / 2], hi[BINS / 2];    // sums of weights as lo + 2^32 hi
        };
        uint64_t near_group[MAX_CTAS][GROUPS];      // what the warps read of the CTAs' histograms
        uint32_t near_bins[MAX_CTAS / 2][2 * NEAR];
    };
    uint32_t offset[BINS];                          // sums of the elements' places in their bins, in 256ths
    uint64_t group[2][GROUPS];                      // sums of a histogram's groups of bins
    uint32_t group_count[2][GROUPS], elements[GROUPS];
    uint64_t list[LIST];                            // this CTA's part of it: places
    uint64_t other[THREADS];                        // a value of each thread
    ulonglong2 all[FEW];                            // of few elements: places and weights
    double table[16];
    uint64_t warp_sum[WARPS], scratch[3][WARPS];
    uint32_t warp_max[WARPS], warp_min[WARPS], first, tie;
    uint32_t list_count[2];
    // written by each CTA of the cluster, for itself and the others, before a barrier
    uint64_t sum_of[2][MAX_CTAS];
    uint32_t max_of[MAX_CTAS], min_of[MAX_CTAS], first_of[MAX_CTAS], tie_of[2][MAX_CTAS], listed_of[2][MAX_CTAS];
    // what warp 0 found
    uint64_t sum, before;
    uint32_t listed;
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
__device__ __forceinline__ void st_cluster_u32(void *p, uint32_t rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u64(void *p, uint32_t rank, uint64_t v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapa_shared(smem_u32(p), rank)), "l"(v) : "memory");
}
// *p += n where `in`, without a branch: a warp's elements stay one block of instructions
__device__ __forceinline__ void add_if(uint32_t *p, uint32_t n, bool in) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p red.shared::cta.add.u32 [%0], %1;\n\t}" ::"r"(smem_u32(p)), "r"(n), "r"((uint32_t)in)
                 : "memory");
}
// Sum of a word of all CTAs.  Eight loads are in flight together, without a branch between them: they take as long as
// one (5000 cycles for three such sums of 16 CTAs one after the other).  ctas: a power of two.
template <typename V, typename L>
__device__ __forceinline__ V sum_of_ctas(uint32_t ctas, L load) {
    V s = 0;
    for (uint32_t c0 = 0; c0 < ctas; c0 += 8) {
        V v[8];
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) v[c] = load((c0 + c) & (ctas - 1));
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) s += c0 + c < ctas ? v[c] : V(0);
    }
    return s;
}
__device__ __noinline__ uint32_t sum_u32(const uint32_t *p, uint32_t ctas) {
    return sum_of_ctas<uint32_t>(ctas, [&](uint32_t c) { return ld_cluster_u32(p, c); });
}
__device__ __noinline__ uint64_t sum_u64(const uint64_t *p, uint32_t ctas) {
    return sum_of_ctas<uint64_t>(ctas, [&](uint32_t c) { return ld_cluster_u64(p, c); });
}
// (modulo 2^64, in three parts whose sums fit 32 bits: a third of the time of five rounds of shuffles)
__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
    const uint32_t a = __reduce_add_sync(0xffffffffu, (uint32_t)v & 0x3fffffu);
    const uint32_t b = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 22) & 0x1fffffu);
    const uint32_t c = __reduce_add_sync(0xffffffffu, (uint32_t)(v >> 43));
    return a + ((uint64_t)b << 22) + ((uint64_t)c << 43);
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

// The block's values in falling order, thread t the t-th; only the first 2^log threads hold any (else 0).  A bitonic
// network: distances within a warp by shuffles, the others through `buf`.
__device__ __noinline__ uint64_t sort_down(uint64_t v, int log, uint64_t *buf) {
    const int tid = threadIdx.x;
    for (int k = 1; k <= log; ++k)
        for (int j = k - 1; j >= 0; --j) {
            uint64_t o;
            if (j >= 5) {
                __syncthreads();
                buf[tid] = v;
                __syncthreads();
                o = buf[tid ^ (1 << j)];
            } else o = __shfl_xor_sync(0xffffffffu, v, 1 << j);
            const bool larger = ((tid >> j) & 1) == ((tid >> k) & 1);
            v = (v > o) == larger ? v : o;
        }
    __syncthreads();
    return v;
}
__device__ __forceinline__ int log_of(uint32_t n) { return n > 1 ? 32 - __clz((int)(n - 1)) : 0; }  // 2^log >= n
// Inclusive sum over the block's threads up to this one; `total` of all.  scratch: WARPS words, free after the next barrier.
__device__ __noinline__ uint64_t block_scan(uint64_t v, uint64_t *scratch, uint64_t &total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    v = warp_scan(v);
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const uint64_t x = scratch[w];
        before += w < warp ? x : 0ull;
        all += x;
    }
    total = all;
    return v + before;
}

// Of `count` <= FEW elements, thread t's the t-th: how many have a larger place, and the sum of their weights.
__device__ __noinline__ ulonglong2 sum_over_few(Shared *sh, uint32_t count, uint64_t place, uint64_t weight) {
    const uint32_t tid = threadIdx.x;
    __syncthreads();
    if (tid < FEW) sh->all[tid] = make_ulonglong2(place, weight);
    __syncthreads();
    uint64_t s = 0;
    uint32_t n = 0;
    if (tid < count)
#pragma unroll 8
        for (uint32_t k = 0; k < count; ++k) {
            const ulonglong2 a = sh->all[k];
            s += a.x > place ? a.y : 0ull;
            n += a.x > place ? 1u : 0u;
        }
    return make_ulonglong2(n, s);
}

// fp32 to fp64 in integer instructions (the conversion has a quarter of the fp64 rate).  Values below 2^-126, zeros among
// them, keep their sign and some magnitude below 2^-125, infinities become 2^128: neither makes a difference to a
// weight at the temperatures in use (Weigher).  UNIT: zero bits at the end.
template <int UNIT>
__device__ __forceinline__ double widen(float x) {
    const uint32_t b = __float_as_uint(x);
    return __hiloint2double((int)((((b & 0x7fffffffu) >> 3) + 0x38000000u) | (b & 0x80000000u)), UNIT >= 3 ? 0 : (int)(b << 29));
}

template <int UNIT>
struct Weigher {
    static constexpr uint64_t BIAS = 0x4330000000000000ull;  // bits of 2^52
    static constexpr double C = 0.04332169878499658;          // ln 2 / 16
    double max, rate;  // of the row; 16 log2(e) / temperature
    int far;           // upper word of the distance from which on weights are 0
    int scale;         // S
    const double *table;

    // all but the row's largest logit, which comes later
    __device__ __forceinline__ Weigher(double temperature, int scale_, const double *table_) : max(0.0), scale(scale_), table(table_) {
        // The temperature is held between 2e-17 and 4e28: beyond, only logits that differ by less than 1e-14, or above
        // 1e26, could tell the difference (and -0 and 0, whose distance is 2^-126 here, weigh the same).
        const double limit = 16.0 * (scale + 2);
        rate = fmin(fmax(23.083120654223414 / temperature, limit * 7.888609052210118e-31), 1.152921504606847e18);
        far = __double2hiint(limit / rate);
    }
    // w and its factor 2^S in one number, of an element d below the largest; 0 with `keep` false and where w is below
    // 2^-(S + 1)
    __device__ __forceinline__ void parts(double d, bool keep, double &t, double &e) const {
        constexpr double MAGIC = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the nearest whole number
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
        return biased_below(max - widen<UNIT>(x), keep);
    }
    __device__ __forceinline__ uint64_t biased_below(double d, bool keep) const {
        double t, e;
        parts(d, keep, t, e);
        return (uint64_t)__double_as_longlong(fma(t, e, 4503599627370496.0));
    }
    __device__ __forceinline__ uint64_t operator()(float x, bool keep = true) const { return biased(x, keep) - BIAS; }
    // ln(w / sum): w from its distance, the sum without its factor 2^S
    __device__ __noinline__ float logprob(float x, uint64_t sum) const {
        return (float)((widen<UNIT>(x) - max) * (rate * C) - log((double)sum * exp2(-(double)scale)));
    }
    // the same, 0 where w 2^S is below `least`
    __device__ __forceinline__ uint64_t at_least(float x, bool keep, double least) const {
        double t, e;
        parts(max - widen<UNIT>(x), keep, t, e);
        return t * e >= least ? (uint64_t)__double_as_longlong(fma(t, e, 4503599627370496.0)) - BIAS : 0ull;
    }
};

// One weight, where no loop needs it inlined (most of the kernel's time with few rows is instruction fetches).
template <int UNIT>
__device__ __noinline__ uint64_t weight_of(const Weigher<UNIT> w, float x, double least) { return w.at_least(x, true, least); }

template <bool CLUSTER>
__device__ __forceinline__ void sync_all() {
    if (CLUSTER) cluster_sync_all();
    else __syncthreads();
}

// Infinite logits become 0, the others -inf.
template <typename T>
__device__ __noinline__ uint4 only_infinite(uint4 v) {
    uint32_t *w = reinterpret_cast<uint32_t *>(&v);
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 4) w[i] = w[i] == 0x7f800000u ? 0u : Type<T>::NONE;
        else {
            const uint32_t inf = Type<T>::NONE & 0x7fffu;
            w[i] = ((w[i] & 0xffffu) == inf ? 0u : Type<T>::NONE & 0xffffu) | ((w[i] >> 16) == inf ? 0u : Type<T>::NONE & 0xffff0000u);
        }
    }
    return v;
}

// One row's view: the slice as 16-byte words in shared memory or, GLOBAL, where the caller has it (two words of a lane on their
// way while one is worked on), divided among the warps in order; places outside the slice hold -inf.
template <typename T, bool CLUSTER, bool GLOBAL>
struct Row {
    using Ty = Type<T>;
    static constexpr int N = Ty::N, UNIT = Ty::UNIT;
    uint4 *data;             // in shared memory
    const T *src;            // the slice's first token
    bool infinite;           // GLOBAL: the row holds +inf
    Shared *sh;
    int first, last;         // this warp's words, `per` of them
    int per, tokens;         // .. and the slice's tokens
    int all_words;           // of the slice
    int skew;                // places before the slice in the first word
    uint32_t base;           // index of the slice's first token
    uint32_t ctas, rank;
    int sums;                // so far
    int turn;                // of the next histogram

    __device__ __forceinline__ uint32_t index(int word, int e) const { return base + (uint32_t)(word * N + e - skew); }

    __device__ __forceinline__ uint4 word(int w) const {
        uint4 v = make_uint4(Ty::NONE, Ty::NONE, Ty::NONE, Ty::NONE);
        if (w >= last) return v;
        if (!GLOBAL) return data[w];
        const int at = w * N - skew;
        if (at >= 0 && at + N <= tokens) v = __ldg(reinterpret_cast<const uint4 *>(src + at));
        else
#pragma unroll 1
            for (int e = 0; e < N; ++e)
                if (at + e >= 0 && at + e < tokens) v = with(v, e, src[at + e]);
        return infinite ? only_infinite<T>(v) : v;
    }
    static __device__ __forceinline__ uint4 with(uint4 v, int e, T x) {
        uint32_t bits = 0, mask = sizeof(T) == 4 ? 0xffffffffu : 0xffffu;
        memcpy(&bits, &x, sizeof(T));
        const int i = e * (int)sizeof(T) / 4, shift = sizeof(T) == 4 ? 0 : (e & 1) * 16;
        const uint32_t old = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w, now = (old & ~(mask << shift)) | bits << shift;
        if (i == 0) v.x = now;
        if (i == 1) v.y = now;
        if (i == 2) v.z = now;
        if (i == 3) v.w = now;
        return v;
    }
    // f(v, w) of this warp's words in order, 32 at a time, a lane each; -inf past the last
    template <typename F>
    __device__ __forceinline__ void words(F f) const {
        const int lane = threadIdx.x & 31;
        if (GLOBAL) {
            uint4 next = word(first + lane), after = word(first + 32 + lane);
            for (int w0 = first; w0 < last; w0 += 32) {
                const uint4 v = next;
                next = after;
                after = word(w0 + 64 + lane);
                f(v, w0 + lane);
            }
        } else {
            for (int w0 = first; w0 < last; w0 += 32) f(word(w0 + lane), w0 + lane);
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

    // A value of this CTA to all CTAs (lanes of one warp); read after a barrier.
    __device__ __forceinline__ void tell(uint32_t *of, uint32_t v) const {
        const uint32_t lane = threadIdx.x & 31;
        if (CLUSTER ? lane < ctas : lane == 0) {
            if (CLUSTER) st_cluster_u32(&of[rank], lane, v);
            else of[0] = v;
        }
    }
    // Sum over the block (every thread has it); scratch[i] is free again after the next barrier.
    __device__ __forceinline__ uint64_t block_sum(uint64_t v, int i) const {
        v = warp_sum(v);
        if ((threadIdx.x & 31) == 0) sh->scratch[i][threadIdx.x >> 5] = v;
        __syncthreads();
        return warp_sum((threadIdx.x & 31) < WARPS ? sh->scratch[i][threadIdx.x & 31] : 0ull);
    }
    // Sum over the cluster of a value of each thread; `before` is that of the CTAs before this one, and
    // warp_sum[] holds the warps'.
    __device__ __forceinline__ uint64_t total(uint64_t v, uint64_t &before) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh->warp_sum[warp] = v;
        __syncthreads();
        if (!CLUSTER) {
            before = 0;
            return warp_sum(lane < WARPS ? sh->warp_sum[lane] : 0ull);
        }
        uint64_t *of = sh->sum_of[sums++ & 1];
        if (warp == 0) {
            const uint64_t cta = warp_sum(lane < WARPS ? sh->warp_sum[lane] : 0ull);
            if (lane < ctas) st_cluster_u64(&of[rank], lane, cta);
        }
        cluster_sync_all();
        // (one warp for all: what every warp does for itself takes sixteen times the issue slots)
        if (warp == 0) {
            const uint64_t x = lane < ctas ? of[lane] : 0ull;
            const uint64_t sum = warp_sum(x), first = warp_sum(lane < rank ? x : 0ull);
            if (lane == 0) sh->sum = sum, sh->before = first;
        }
        __syncthreads();
        before = sh->before;
        return sh->sum;
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
        return share_list(which);
    }
    __device__ __forceinline__ void append(int which, float x, int w, int e) const {
        const uint32_t at = atomicAdd(&sh->list_count[which], 1u);
        if (at < LIST) sh->list[at] = place_of(key_of<UNIT>(x), index(w, e));
    }
    __device__ __forceinline__ uint32_t share_list(int which) const {
        __syncthreads();
        if (threadIdx.x < 32) tell(sh->listed_of[which], sh->list_count[which]);
        sync_all<CLUSTER>();
        if (threadIdx.x < 32) {
            const uint32_t n = __reduce_add_sync(0xffffffffu, threadIdx.x < ctas ? sh->listed_of[which][threadIdx.x] : 0u);
            if (threadIdx.x == 0) sh->listed = n;
        }
        __syncthreads();
        return sh->listed;
    }
    // The cluster's list (`count`, at most LIST), an element a thread: its place, 0 past the last.  More than FEW come in
    // their order.  No CTA may refill its part before the others have read it: a barrier of the cluster
    // stands before every collect.
    __device__ __forceinline__ uint64_t listed(int which, uint32_t count) const {
        uint64_t place = 0;
        if (threadIdx.x < count) {
            uint32_t at = threadIdx.x, from = 0;  // the at-th of CTA `from`
            for (uint32_t n; from < ctas && at >= (n = sh->listed_of[which][from]); ++from) at -= n;
            if (from < ctas) place = CLUSTER ? ld_cluster_u64(&sh->list[at], from) : sh->list[at];
        }
        return count > FEW ? sort_down(place, log_of(count), sh->other) : place;
    }
    // Of the list's `count` elements in their order, the one at which the sum of the measure reaches
    // `need`: sh->cut, and true; false if it does not.  place, own: this thread's element.
    template <typename M>
    __device__ __forceinline__ bool resolve(int which, uint32_t count, uint64_t need, M measure, uint64_t &place, uint64_t &own) const {
        if (threadIdx.x == 0) sh->hit = 0;
        place = listed(which, count);
        own = place ? measure(value_of<UNIT>((uint32_t)(place >> 32))) : 0ull;
        uint64_t before;
        if (count > FEW) before = block_scan(own, sh->scratch[2], before) - own;
        else before = sum_over_few(sh, count, place, own).y;
        if (before + own >= need && before < need) {
            sh->cut = {value_of<UNIT>((uint32_t)(place >> 32)), ~(uint32_t)place};
            sh->hit = 1;
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
template <typename T, bool CLUSTER, bool GLOBAL>
__device__ __forceinline__ void finish(const Row<T, CLUSTER, GLOBAL> &row, const Weigher<Type<T>::UNIT> &weigh, int which, uint32_t count, uint64_t k, double p,
                                       uint64_t need, double least, double u, int64_t *token, float *logprob) {
    constexpr int UNIT = Type<T>::UNIT;
    Shared *sh = row.sh;
    const uint32_t tid = threadIdx.x;
    const uint64_t place = row.listed(which, count);
    const float x = value_of<UNIT>((uint32_t)(place >> 32));
    uint64_t own = place ? weight_of(weigh, x, 0.0) : 0ull, before, sum;
    uint32_t rank = tid;
    if (count > FEW) {
        if (k && tid >= k) own = 0;
        before = block_scan(own, sh->scratch[0], sum) - own;
    } else {
        const ulonglong2 r = sum_over_few(sh, count, place, own);
        rank = (uint32_t)r.x, before = r.y;
        if (k && rank >= k) own = 0;
        if (k && p < 1.0) sum = row.block_sum(own, 0);
    }
    if (k && p < 1.0) {
        const double target = ceil((double)sum * p);
        need = target >= 1.0 ? min(sum, (uint64_t)target) : 1ull;
    }
    if (need && before >= need) own = 0;
    if (own && least > 0.0) own = weight_of(weigh, x, least);
    // those that stay, by their indices (the lower half of a place falls as the index rises)
    const uint32_t low = own ? (uint32_t)place : 0u;
    uint64_t drawn = own;
    uint32_t holder = tid;
    if (count > FEW) {
        // (sorted, so the first threads': a weight is never above the one before it)
        const int stay = __syncthreads_count(own != 0);
        const uint64_t by_index = sort_down(own ? (uint64_t)low << 32 | tid : 0ull, log_of(stay), sh->other);
        sh->other[tid] = own;
        __syncthreads();
        holder = (uint32_t)by_index;
        drawn = by_index ? sh->other[holder] : 0ull;
        before = block_scan(drawn, sh->scratch[1], sum) - drawn;
    } else {
        sum = row.block_sum(own, 1);
        before = sum_over_few(sh, count, low, own).y;
    }
    const double at = fmax(u, 0.0) * (double)sum;
    const uint64_t target = at < (double)sum ? min((uint64_t)at, sum - 1) : sum - 1;
    if (before <= target && target < before + drawn) sh->found_bin = holder;  // the thread that has its logit
    __syncthreads();
    if (tid == sh->found_bin) {
        *token = ~(uint32_t)place;
        if (logprob) *logprob = weigh.logprob(x, sum);
    }
}

// A value below which nothing is among the k largest: of the 16-byte words' largest elements, from `least` up to
// `top`, k are at least that large.  -inf if they are not that many.
template <typename T, bool CLUSTER, bool GLOBAL>
__device__ __forceinline__ float bound_of_largest(Row<T, CLUSTER, GLOBAL> &row, float top, float least, uint64_t k) {
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
        const uint32_t s = __reduce_add_sync(0xffffffffu, count[g * GROUP + lane] + count[g * GROUP + 32 + lane]);
        if (lane == 0) group[g] = s;
    }
    sync_all<CLUSTER>();
    if (warp == 0) {
        const uint64_t s = sum_u32(&group[lane], row.ctas);
        uint64_t upto = warp_scan(s);
        const unsigned past = __ballot_sync(0xffffffffu, upto >= k);
        const int g = past ? __ffs(past) - 1 : 0;
        const uint64_t before = __shfl_sync(0xffffffffu, upto - s, g);
        // (to two bins: the bound may be lower than it could be, not higher)
        upto = before + warp_scan((uint64_t)(sum_u32(&count[g * GROUP + 2 * lane], row.ctas) + sum_u32(&count[g * GROUP + 2 * lane + 1], row.ctas)));
        const unsigned here = __ballot_sync(0xffffffffu, upto >= k);
        if (here && lane == 0) sh->found_bin = g * GROUP + 2 * __ffs(here) - 1;
        if (!past && lane == 0) sh->found_bin = NO_INDEX;
    }
    __syncthreads();
    const uint32_t bin = sh->found_bin;
    __syncthreads();
    // (a range below 6e-36 or one that overflows has no bins: the search by keys takes such a row)
    if (bin == NO_INDEX || c == 0.f || c == INFINITY) return -INFINITY;
    // the bin's lower edge, less what the roundings of the bin's number may amount to
    const float range = top - least, edge = top - (float)(bin + 1) / c - 1e-5f * range - 1e-6f * fabsf(top);
    return edge > -INFINITY ? edge : -INFINITY;
}

// The cut after the shortest prefix, in the order of the values, whose measure (elements, or weights
// with WEIGHT) reaches `need` >= 1, among the elements within `cut` whose keys are from `low` up to `high`.
// Elements left out by `low` must not be needed.  By histograms of keys, each dividing the bin that
// holds the border, until it holds at most LIST elements or one value.
template <bool WEIGHT, typename T, bool CLUSTER, bool GLOBAL>
__device__ __noinline__ Cut select(Row<T, CLUSTER, GLOBAL> &row, const Weigher<Type<T>::UNIT> &weigh, Cut cut, uint32_t high, uint32_t low, uint64_t need) {
    constexpr int UNIT = Type<T>::UNIT, LOG = 10;
    constexpr int BINS = 1 << LOG, GROUP = BINS / GROUPS;  // (half of the others': two more words a bin)
    static_assert(GROUP == 32, "one bin a lane");
    Shared *sh = row.sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t cut_key = key_of<UNIT>(cut.value);
    low = max(low, cut_key);
    auto inside = [&](uint32_t key, int w, int e) {
        return key >= low && key <= high && (key != cut_key || row.index(w, e) <= cut.index);
    };
    auto measure = [&](float x) { return WEIGHT ? weight_of(weigh, x, 0.0) : 1ull; };
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
            const uint32_t b = in ? (high - key) >> shift : 0u;
            add_if(&count[b], 1u, in);
            if (WEIGHT && in) {
                const uint64_t weight = weigh(x);
                const uint32_t lo = (uint32_t)weight, old = atomicAdd(&sh->lo[b], lo);
                const uint32_t hi = (uint32_t)(weight >> 32) + (old + lo < old ? 1u : 0u);
                if (hi) atomicAdd(&sh->hi[b], hi);
            }
        });
        __syncthreads();
        for (int g = warp; g < GROUPS; g += WARPS) {
            const int i = g * GROUP + lane;
            const uint64_t s = warp_sum(WEIGHT ? ((uint64_t)sh->hi[i] << 32) + sh->lo[i] : (uint64_t)count[i]);
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
            const uint64_t before = __shfl_sync(0xffffffffu, upto - s, g);
            const int i = g * GROUP + lane;
            const uint32_t n = sum_u32(&count[i], row.ctas);
            s = n;
            if (WEIGHT) {
                s = 0;
                for (uint32_t c = 0; c < row.ctas; ++c)
                    s += (uint64_t)ld_cluster_u32(&sh->lo[i], c) + ((uint64_t)ld_cluster_u32(&sh->hi[i], c) << 32);
            }
            upto = before + warp_scan(s);
            const unsigned here = __ballot_sync(0xffffffffu, upto >= need);
            if (here && lane == __ffs(here) - 1) {
                sh->found_bin = i;
                sh->found_count = n;
                sh->found_before = upto - s;
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
            uint64_t place, own;
            return row.resolve(WEIGHT, n, need, measure, place, own) ? sh->cut : cut;
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
            if (tid == 0) sh->tie = NO_INDEX;
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
                            if (inside(key_of<UNIT>(x[e]), w, e) && --left == 0) sh->tie = row.index(w, e);
                    }
                    at = __shfl_sync(0xffffffffu, upto, 31);
                });
            }
            __syncthreads();
            if (warp == 0) row.tell(sh->tie_of[WEIGHT], sh->tie);
            sync_all<CLUSTER>();
            uint32_t ix = NO_INDEX;
            for (uint32_t c = 0; c < row.ctas; ++c) ix = min(ix, sh->tie_of[WEIGHT][c]);
            return {value, ix};
        }
    }
}

// Weights below (1 - p) / (2 V) of the largest (1, so of the sum) sum up to less than (1 - p), so none of them is in
// top-p's prefix: how far below the largest logit the others may be (with a margin for roundings).
template <int UNIT>
__device__ __forceinline__ double reach_of(const Weigher<UNIT> &weigh, double p, int V) {
    const double smallest = fmax(0.5, 0.5 * (1.0 - p) / V * exp2((double)weigh.scale));
    return (weigh.scale - log2(smallest)) * 16.0 / weigh.rate * 1.000001;
}

// Where in the bins of width 1 / c below the largest logit an element is, and its bin, the nearest whole number, as 1.5 * 2^23
// more (without a conversion, which has a quarter of the rate); x falling, neither falls.  Every step is rounded by
// itself: passes that count and passes that list must agree on an element's bin, and a product and a sum that are
// fused in one of them only would part them.
constexpr float BIN0 = 12582912.f;
__device__ __forceinline__ float bins_below(float top, float x, float c) { return __fmul_rn(__fsub_rn(top, x), c); }
__device__ __forceinline__ float bin_at(float at) { return fminf(__fadd_rn(at, BIN0), BIN0 + (BINS - 1)); }

// The passes over the logits, each a function of its own: inlined into one kernel they share its registers, and spilled
// values in their loops tripled their time.
// Sum of the weights within the cut; elements of at least `low` counted in bins of the width 1 / c below `top`.
template <bool WHOLE, typename T, bool CLUSTER, bool GLOBAL>
__device__ __noinline__ uint64_t sum_and_count(const Row<T, CLUSTER, GLOBAL> row, const Weigher<Type<T>::UNIT> weigh, const Cut cut, float top, float low, float c,
                                               uint32_t *count) {
    constexpr int N = Type<T>::N;
    uint32_t *offset = row.sh->offset;
    uint64_t mine = 0;
    auto add = [&](const uint4 &v, int w) {
        float x[N];
        Type<T>::load(v, x);
#pragma unroll
        for (int e = 0; e < N; ++e) mine += weigh.biased(x[e], WHOLE || row.kept(cut, x[e], w, e));
        mine -= N * weigh.BIAS;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const bool in = x[e] >= low && (WHOLE || row.kept(cut, x[e], w, e));
            const float at = in ? bins_below(top, x[e], c) : 0.f, bin = bin_at(at);
            const uint32_t b = __float_as_uint(bin) - __float_as_uint(BIN0);
            add_if(&count[b], 1u, in);
            // (where in it, from its lower edge on: 0 to 256)
            add_if(&offset[b], __float_as_uint(fmaf(at - (bin - BIN0), 256.f, BIN0 + 128.f)) - __float_as_uint(BIN0), in);
        }
    };
    if (WHOLE) row.words(add);
    else row.words_from(cut.value, add);
    return mine;
}
// Sum of the weights within the cut, of at least `low` and before bin `first`; those in bins from that to `last` to the list.
template <bool WHOLE, typename T, bool CLUSTER, bool GLOBAL>
__device__ __noinline__ uint64_t sum_and_list(const Row<T, CLUSTER, GLOBAL> row, const Weigher<Type<T>::UNIT> weigh, const Cut cut, float top, float low, float c,
                                              float first, float last) {
    constexpr int N = Type<T>::N;
    uint64_t mine = 0;
    row.words_from(low, [&](const uint4 &v, int w) {
        float x[N];
        Type<T>::load(v, x);
        uint32_t listed = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float bin = bin_at(bins_below(top, x[e], c));
            const bool in = x[e] >= low && (WHOLE || row.kept(cut, x[e], w, e));
            mine += weigh.biased(x[e], in && bin < first);
            listed |= in && bin >= first && bin <= last ? 1u << e : 0u;
        }
        mine -= N * weigh.BIAS;
        if (listed)
#pragma unroll 1
            for (int e = 0; e < N; ++e)
                // (as `words` gives them: an infinite logit is 0)
                if (listed & (1u << e))
                    row.append(1, row.infinite ? 0.f : (float)(GLOBAL ? row.src[w * N - row.skew + e] : reinterpret_cast<const T *>(row.data + w)[e]), w, e);
    });
    return mine;
}
// Sum of the weights within the cut, of at least `least`.
template <bool PLAIN, typename T, bool CLUSTER, bool GLOBAL>
__device__ __noinline__ uint64_t sum_kept(const Row<T, CLUSTER, GLOBAL> row, const Weigher<Type<T>::UNIT> weigh, const Cut cut, double least) {
    constexpr int N = Type<T>::N;
    uint64_t mine = 0;
    auto add = [&](const uint4 &v, int w) {
        float x[N];
        Type<T>::load(v, x);
#pragma unroll
        for (int e = 0; e < N; ++e) mine += PLAIN ? weigh.biased(x[e], true) : weigh.at_least(x[e], row.kept(cut, x[e], w, e), least);
        if (PLAIN) mine -= N * weigh.BIAS;
    };
    if (PLAIN) row.words(add);
    else row.words_from(cut.value, add);
    return mine;
}
// One warp's elements within the cut and of at least `least`, `at` the sum of those before: the one at which it passes
// `target` is the token.
template <typename T, bool CLUSTER, bool GLOBAL>
__device__ __noinline__ void draw(const Row<T, CLUSTER, GLOBAL> row, const Weigher<Type<T>::UNIT> weigh, const Cut cut, double least, uint64_t at, uint64_t target,
                                  uint64_t sum, int64_t *token, float *logprob) {
    constexpr int N = Type<T>::N;
    row.words_from(cut.value, [&](const uint4 &v, int w) {
        if (at > target) return;
        float x[N];
        Type<T>::load(v, x);
        uint64_t own[N], mine = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) mine += own[e] = weigh.at_least(x[e], row.kept(cut, x[e], w, e), least);
        const uint64_t upto = at + warp_scan(mine);
        if (upto > target && upto - mine <= target) {
            uint64_t run = upto - mine;
            float found = 0.f;
            uint32_t index = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (run <= target && target < run + own[e]) index = row.index(w, e), found = x[e];
                run += own[e];
            }
            *token = index;
            if (logprob) *logprob = weigh.logprob(found, sum);
        }
        at = __shfl_sync(0xffffffffu, upto, 31);
    });
}

enum Outcome { LISTED, CUT, CUT_AND_SUM };
// Top-p among the elements within `cut`: their weights' sum `total`, of which the prefix has to reach `need` = p times that.  One
// pass sums the weights and counts the elements in bins of equal width; each counted as an element in the
// middle of those of its bin, they say about where the border is.  (Sums of weights in each bin would cost three atomic additions
// for every element.)  Where all elements down to the border fit the list, the list is all that is needed: true, its
// length in `listed`.  Else a pass over the elements above a few bins around the border sums them exactly and lists
// those in the bins; where the border is not among these after all, the sum tells by how much the
// estimate is off.  `cut` is then the one after the prefix.
template <typename T, bool CLUSTER, bool GLOBAL>
__device__ __forceinline__ Outcome nucleus(Row<T, CLUSTER, GLOBAL> &row, const Weigher<Type<T>::UNIT> &weigh, Cut &cut, float top, double p, double reach, uint64_t &need,
                                           uint32_t &listed, uint64_t &sum, uint64_t &before) {
    constexpr int UNIT = Type<T>::UNIT, N = Type<T>::N;
    Shared *sh = row.sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const float low = fmaxf(fminf(top, fmaxf((float)((double)top - reach - 1e-6 * fabs((double)top)), -3.4028234e38f)), cut.value);
    const float c = top > low ? (BINS - 1) / (top - low) : 0.f, width = top > low ? (top - low) / (BINS - 1) : 0.f;
    // four bins' elements, each counted as one in the middle of its bin's
    auto estimate = [&](const uint32_t (&n)[4], const uint32_t (&offset)[4], int b, uint64_t (&w)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float middle = (float)offset[q] / (256.f * (float)n[q]) - 0.5f;
            // (by the distance: next to a logit of 10^4 the bins may be narrower than fp32 can tell)
            w[q] = n[q] * (weigh.biased_below(fmax((double)((float)(b + q) + middle) * (double)width, 0.0), n[q] != 0) - weigh.BIAS);
        }
    };
    uint32_t *count = sh->count[row.turn & 1], *group_count = sh->group_count[row.turn & 1];
    uint64_t *group = sh->group[row.turn & 1];
    ++row.turn;
    *reinterpret_cast<uint4 *>(count + 4 * tid) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4 *>(sh->offset + 4 * tid) = make_uint4(0, 0, 0, 0);
    if (tid < GROUPS) sh->elements[tid] = 0;
    __syncthreads();
    const bool whole = cut.value == -INFINITY;
    uint64_t mine = whole ? sum_and_count<true>(row, weigh, cut, top, low, c, count) : sum_and_count<false>(row, weigh, cut, top, low, c, count);
    __syncthreads();
    {
        const uint4 n4 = *reinterpret_cast<const uint4 *>(count + 4 * tid), o4 = *reinterpret_cast<const uint4 *>(sh->offset + 4 * tid);
        const uint32_t n[4] = {n4.x, n4.y, n4.z, n4.w}, o[4] = {o4.x, o4.y, o4.z, o4.w};
        uint64_t w[4];
        estimate(n, o, 4 * tid, w);
        uint64_t s = w[0] + w[1] + w[2] + w[3];
        uint32_t k = n[0] + n[1] + n[2] + n[3];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), k += __shfl_xor_sync(0xffffffffu, k, o);
        if ((tid & 15) == 0) group[tid >> 4] = s, group_count[tid >> 4] = k;
    }
    sum = row.total(mine, before);
    const double target = ceil((double)sum * p);
    need = target >= 1.0 ? min(sum, (uint64_t)target) : 1ull;
    // the border is in bin `first` or after it, and before bin `end`
    int first = 0, end = BINS;
    uint64_t seek = need;  // in sums of the estimate
    const double sure = exp2(-1.01 * width * weigh.rate / 16.0) * (1.0 - 1e-6);
    for (;;) {
        // a warp for each CTA reads its groups, then its bins around the group of the border
        const uint32_t of = (uint32_t)warp < row.ctas ? warp : 0;
        sh->near_group[warp][lane] = ld_cluster_u64(&group[lane], of);
        const uint32_t counted = ld_cluster_u32(&group_count[lane], of);
        if ((uint32_t)warp < row.ctas) atomicAdd(&sh->elements[lane], counted);
        __syncthreads();
        if (warp == 0) {
            uint64_t s = 0;
            for (uint32_t k = 0; k < row.ctas; ++k) s += sh->near_group[k][lane];
            const uint64_t upto = warp_scan(s);
            const unsigned past = __ballot_sync(0xffffffffu, upto >= seek);
            const int g = past ? __ffs(past) - 1 : GROUPS - 1;
            // up to which group the weights reach `need` for certain: a bin's elements are no wider apart than it
            const unsigned reached = __ballot_sync(0xffffffffu, (double)upto * sure >= (double)need);
            const int last = reached ? __ffs(reached) - 1 : 0;
            const uint32_t all = __reduce_add_sync(0xffffffffu, lane <= last ? sh->elements[lane] : 0u);
            if (lane == g) sh->found_before = upto - s, sh->found_first = g;
            if (lane == 0) sh->found_count = first == 0 && end == BINS && reached && all <= LIST ? all : NO_INDEX, sh->found_last = last;
        }
        __syncthreads();
        const uint64_t start = sh->found_before;  // before the border's group
        const int g = sh->found_first, last = sh->found_last, near0 = min(max(g * GROUP - NEAR / 4, 0), BINS - NEAR);
        const bool listable = sh->found_count != NO_INDEX;
        const uint32_t all = sh->found_count;
        __syncthreads();
        if (warp == 0) sh->elements[lane] = 0;  // (for another round)
        if (!listable) {
            // (16 CTAs: two to a row)
            uint32_t v[2 * NEAR / 32];
#pragma unroll
            for (int q = 0; q < NEAR / 32; ++q) {
                v[q] = ld_cluster_u32(count + near0 + q * 32 + lane, of);
                v[NEAR / 32 + q] = ld_cluster_u32(sh->offset + near0 + q * 32 + lane, of);
            }
            uint32_t *row_of = sh->near_bins[warp & 7];
            if (warp < 8)
#pragma unroll
                for (int q = 0; q < 2 * NEAR / 32; ++q) row_of[q * 32 + lane] = v[q];
            __syncthreads();
            if (warp >= 8 && (uint32_t)warp < row.ctas)
#pragma unroll
                for (int q = 0; q < 2 * NEAR / 32; ++q) row_of[q * 32 + lane] += v[q];
        }
        __syncthreads();
        if (warp == 0) {
            if (listable) {
                if (lane == 0) sh->found_bin = last * GROUP + GROUP - 1, sh->found_count = all;
            } else {
                // four bins a lane
                uint32_t n[4], o[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) n[q] = o[q] = 0;
                for (uint32_t k = 0; k < min(row.ctas, 8u); ++k)
#pragma unroll
                    for (int q = 0; q < 4; ++q) n[q] += sh->near_bins[k][4 * lane + q], o[q] += sh->near_bins[k][NEAR + 4 * lane + q];
                uint64_t w[4];
                estimate(n, o, near0 + 4 * lane, w);
                const uint64_t mine4 = w[0] + w[1] + w[2] + w[3];
                // sums from near0 on; what lies before the group's start among them
                const uint64_t scan = warp_scan(mine4);
                const int lane_of_group = (g * GROUP - near0) / 4;
                const uint64_t head = lane_of_group ? __shfl_sync(0xffffffffu, scan, lane_of_group - 1) : 0ull;
                const uint64_t base = start - head;  // the estimate before near0
                uint64_t run = base + scan - mine4;
                int my_bin = BINS;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    run += w[q];
                    if (run >= seek && my_bin == BINS) my_bin = near0 + 4 * lane + q;
                }
                int bin = (int)__reduce_min_sync(0xffffffffu, (unsigned)my_bin);
                if (bin == BINS) bin = BINS - 1;
                const bool lost = bin < first || bin >= end || bin < near0 || bin >= near0 + NEAR;  // (the estimate has not come closer)
                if (bin < first || bin >= end) bin = (first + end) / 2;
                // the lanes (of four bins) around it that fit the window, else its bin alone
                int b0 = bin, b1 = bin;
                uint32_t m = 0;
                uint64_t est = 0;
                if (lost) m = sum_u32(&count[bin], row.ctas);
                else {
                    const int l = (bin - near0) / 4;
                    const uint32_t four = n[0] + n[1] + n[2] + n[3];
                    int side = 16;
                    for (;;) {
                        m = __reduce_add_sync(0xffffffffu, lane >= l - side && lane <= l + side ? four : 0u);
                        if (m <= WINDOW || side == 0) break;
                        side >>= 1;
                    }
                    if (m <= WINDOW) {
                        b0 = max(near0 + 4 * max(l - side, 0), first);
                        b1 = min(near0 + 4 * min(l + side, 31) + 3, end - 1);
                    }
                    m = 0;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int at = near0 + 4 * lane + q;
                        m += at >= b0 && at <= b1 ? n[q] : 0u;
                        est += at < b0 ? w[q] : 0ull;
                    }
                    m = __reduce_add_sync(0xffffffffu, m);
                    est = base + warp_sum(est);
                }
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
            listed = row.collect(1, low, [&](float x, int w, int e) { return x >= low && bin_at(bins_below(top, x, c)) <= BIN0 + (float)through && row.kept(cut, x, w, e); });
            return LISTED;
        }
        if (n > LIST) {  // a bin of many elements, likely equal ones
            Row<T, CLUSTER, GLOBAL> other = row;
            cut = select<true>(other, weigh, cut, key_of<UNIT>(top), key_of<UNIT>(low), need);
            row.turn = other.turn, row.sums = other.sums;
            return CUT;
        }
        if (tid == 0) sh->list_count[1] = 0;
        __syncthreads();
        mine = whole ? sum_and_list<true>(row, weigh, cut, top, low, c, BIN0 + b0, BIN0 + b1) : sum_and_list<false>(row, weigh, cut, top, low, c, BIN0 + b0, BIN0 + b1);
        __syncthreads();
        if (warp == 0) row.tell(sh->listed_of[1], sh->list_count[1]);
        const uint64_t above = row.total(mine, before);
        uint64_t place, own;
        if (above >= need) end = b0;
        else if (row.resolve(1, n, need - above, [&](float x) { return weight_of(weigh, x, 0.0); }, place, own)) {
            cut = sh->cut;
            // what the list adds to the sums before this CTA, of its warps, of all
            const uint32_t ix = ~(uint32_t)place;
            if (place < place_of(key_of<UNIT>(cut.value), cut.index)) own = 0;
            sum = above + row.block_sum(own, 0);
            before += row.block_sum(ix < row.base ? own : 0ull, 1);
            if (own && ix >= row.base && ix - row.base < (uint32_t)row.tokens)
                atomicAdd(reinterpret_cast<unsigned long long *>(&sh->warp_sum[(ix - row.base + row.skew) / N / row.per]), own);
            __syncthreads();
            return CUT_AND_SUM;
        } else first = b1 + 1;
        if (first >= end) return CUT;  // all of them together do not reach it
        seek = need + est - above;
        sync_all<CLUSTER>();  // the lists are filled again
    }
}

template <typename T, bool CLUSTER, bool GLOBAL>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const Params p) {
    using Ty = Type<T>;
    constexpr int N = Ty::N, UNIT = Ty::UNIT;
    extern __shared__ __align__(16) uint8_t smem[];
    Shared *sh = reinterpret_cast<Shared *>(smem);
    pdl_trigger();
    if (CLUSTER) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    pdl_wait();
    Row<T, CLUSTER, GLOBAL> row;
    row.sh = sh;
    row.data = reinterpret_cast<uint4 *>(smem + (sizeof(Shared) + 15) / 16 * 16);
    row.ctas = CLUSTER ? gridDim.x : 1;
    row.rank = CLUSTER ? blockIdx.x : 0;
    row.sums = 0;
    row.turn = 0;
    const int64_t b = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- the slice: to shared memory, whole words by asynchronous copies, the ends one by one
    row.base = row.rank * (uint32_t)p.slice;
    const int n = max(0, min(p.slice, p.V - (int)min(row.base, (uint32_t)p.V)));
    const T *src = reinterpret_cast<const T *>(p.logits) + b * p.stride + row.base;
    row.skew = (int)((reinterpret_cast<uintptr_t>(src) & 15u) / sizeof(T));
    const int words = n ? (n + row.skew + N - 1) / N : 0;
    row.src = src;
    row.infinite = false;
    for (int w = tid; !GLOBAL && w < words; w += THREADS) {
        const int at = w * N - row.skew;
        if (at >= 0 && at + N <= n) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(row.data + w)), "l"(src + at) : "memory");
        } else {
            T *dst = reinterpret_cast<T *>(row.data + w);
#pragma unroll 1
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
    // (what takes divisions and functions of fp64, under the copies)
    Weigher<UNIT> weigh(temperature, p.scale, sh->table);
    const double least = fmin(fmax(min_p, 0.0), 1.0) * exp2((double)p.scale);
    const double reach = top_p < 1.0 ? reach_of(weigh, top_p, p.V) : 0.0;
    if (tid < 16) sh->table[tid] = exp2(-tid / 16.0);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    row.tokens = n;
    row.all_words = words;
    row.per = (words + THREADS - 1) / THREADS * 32;
    row.first = min(words, warp * row.per);
    row.last = min(words, row.first + row.per);

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
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA has started
        if (warp == 0) row.tell(sh->max_of, top), row.tell(sh->min_of, bottom);
        cluster_sync_all();
        top = __reduce_max_sync(0xffffffffu, lane < row.ctas ? sh->max_of[lane] : 0u);
        bottom = __reduce_min_sync(0xffffffffu, lane < row.ctas ? sh->min_of[lane] : NO_INDEX);
    }
    // no token, until one is drawn: whichever thread does that has this write behind it by a barrier below
    if (row.rank == 0 && tid == 0) {
        p.tokens[b] = -1;
        if (p.logprobs) p.logprobs[b] = __uint_as_float(0x7fc00000u);
    }
    const uint32_t none = key_of<UNIT>(-INFINITY);
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
        if (tid == 0) sh->first = NO_INDEX;
        __syncthreads();
        if (lane == 0) atomicMin(&sh->first, at);
        __syncthreads();
        if (warp == 0) row.tell(sh->first_of, sh->first);
        sync_all<CLUSTER>();
        at = __reduce_min_sync(0xffffffffu, lane < row.ctas ? sh->first_of[lane] : NO_INDEX);
        if (row.rank == 0 && tid == 0) {
            p.tokens[b] = at;
            if (p.logprobs) p.logprobs[b] = 0.f;
        }
    } else {
        if (top == key_of<UNIT>(INFINITY)) {
            // infinite logits share everything: they are 0 from here on, the others -inf
            row.infinite = true;
            for (int w = row.first + lane; !GLOBAL && w < row.last; w += 32) row.data[w] = only_infinite<T>(row.data[w]);
            __syncwarp();
            top = bottom = key_of<UNIT>(0.f);
        }
        const float peak = value_of<UNIT>(top);
        weigh.max = widen<UNIT>(peak);
        Cut cut{-INFINITY, NO_INDEX};
        // whether all that may be drawn is in the list, its length, which counter, and what is left to do with it
        bool in_list = false;
        uint32_t listed = 0;
        uint64_t k = 0, need = 0, before = 0, sum = 0;
        bool summed = false;  // whether sum, before and warp_sum[] are those of the kept
        if (top_k > 0 && top_k < p.V) {
            const float low = top_k <= p.V / N ? bound_of_largest(row, peak, value_of<UNIT>(bottom), (uint64_t)top_k) : -INFINITY;
            if (top_k <= LIST && low > -INFINITY) {
                listed = row.collect(0, low, [&](float x, int, int) { return x >= low; });
                in_list = listed <= LIST;
                k = (uint64_t)top_k;
            }
            if (!in_list) {
                Row<T, CLUSTER, GLOBAL> other = row;
                cut = select<false>(other, weigh, cut, top, low > -INFINITY ? max(none + 1, key_of<UNIT>(low)) : none + 1, (uint64_t)top_k);
                row.turn = other.turn, row.sums = other.sums;
                k = 0;
            }
        }
        if (!in_list && top_p < 1.0) {
            const Outcome o = nucleus(row, weigh, cut, peak, top_p, reach, need, listed, sum, before);
            in_list = o == LISTED;
            summed = o == CUT_AND_SUM && least == 0.0;
        }
        if (in_list) {
            if (row.rank == 0)
                finish(row, weigh, k ? 0 : 1, listed, k, top_p, need, least, (double)u, p.tokens + b, p.logprobs ? p.logprobs + b : nullptr);
        } else {
            // ---- the kept ones' sum, and the place of u in it
            if (!summed) {
                const uint64_t mine = cut.value == -INFINITY && least == 0.0 ? sum_kept<true>(row, weigh, cut, 0.0) : sum_kept<false>(row, weigh, cut, least);
                sum = row.total(mine, before);
            }
            const double place = fmax((double)u, 0.0) * (double)sum;
            const uint64_t target = place < (double)sum ? min((uint64_t)place, sum - 1) : sum - 1;
            // the warp in whose words it is, here or in another CTA; then all warps look through these
            uint64_t at = before;
            int owner = 0;
            for (; owner < WARPS && target >= at + sh->warp_sum[owner]; ++owner) at += sh->warp_sum[owner];
            if (target >= at && owner < WARPS) {
                Row<T, CLUSTER, GLOBAL> part = row;
                const int from = min(row.all_words, owner * row.per), words = min(row.per, row.all_words - from);
                const int each = (words + THREADS - 1) / THREADS * 32;
                part.first = from + min(words, warp * each);
                part.last = min(from + words, part.first + each);
                const uint64_t mine = warp_sum(sum_kept<false>(part, weigh, cut, least));
                if (lane == 0) sh->scratch[0][warp] = mine;
                __syncthreads();
                for (int i = 0; i < warp; ++i) at += sh->scratch[0][i];
                if (at <= target && target < at + mine)
                    draw(part, weigh, cut, least, at, target, sum, p.tokens + b, p.logprobs ? p.logprobs + b : nullptr);
            }
        }
    }
    __syncwarp();
    if (CLUSTER) cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

template <typename T>
static int launch(const Params &q, int64_t B, cudaStream_t st) {
    Params p = q;
    const int64_t bytes = (int64_t)p.V * (int64_t)sizeof(T);
    // CTAs of a row: up to 16 while all rows together have at most 400 (296 are resident at a time), slices of 4 KB at least.
    // 128256 bf16 logits, us without filter / with top-p 0.95 / with settings of each row's own:
    //      64 rows  4 CTAs 22 / 76 / 79    2 CTAs 38 / 121 / 124  8 CTAs 31 / 100 / 67
    //      96       4 CTAs 33 / 114 / 87   2 CTAs 40 / 125 / 140  8 CTAs 44 / 149 / 87
    //     200       2 CTAs 61 / 193 / 158  1 CTA  71 / 221 / 244  4 CTAs 63 / 211 / 120
    //     256       1 CTA  74 / 246 / 257  2 CTAs 79 / 246 / 173
    // (96 of 151643 in f32: 4 CTAs 51 / 136 / 100, 2 CTAs 56 / 163 / 149).  The rule knows the number of rows, not the settings, and gives
    // away most next to where it steps, and for settings of the rows' own, whose CTAs run unequally long:
    //      24 rows 16 CTAs 22 / 72 / 40    8 CTAs 15 / 51 / 45
    //     110       2 CTAs 40 / 158 / 135  4 CTAs 43 / 141 / 94
    //     160       2 CTAs 59 / 186 / 142  4 CTAs 51 / 178 / 102
    int ctas = MAX_CTAS;
    while (ctas > 1 && (B * ctas > 400 || bytes / ctas < 4096)) ctas /= 2;
    p.slice = ((p.V + ctas - 1) / ctas + 15) / 16 * 16;
    // Slices of which two fit an SM stay in shared memory for all passes (64 rows of 256 KB, top-k 50: 16 us, 19 read again by
    // each pass); longer ones are read again, from L2 mostly (256 rows: 41 us, 60 in slices of 64 KB).
    const bool global = (int64_t)p.slice * (int64_t)sizeof(T) > MAX_SLICE;
    const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + (global ? 0 : (size_t)p.slice * sizeof(T) + 32);
    auto kernel = ctas > 1 ? (global ? sample_kernel<T, true, true> : sample_kernel<T, true, false>)
                           : (global ? sample_kernel<T, false, true> : sample_kernel<T, false, false>);
    static PerDeviceFlag configured;
    const int dev = current_device();
    if (!configured.test(dev)) {
        const int most = (int)((sizeof(Shared) + 15) / 16 * 16 + MAX_SLICE + 32);
        for (auto k : {sample_kernel<T, true, true>, sample_kernel<T, true, false>, sample_kernel<T, false, true>, sample_kernel<T, false, false>}) {
            QL_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
            QL_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        }
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

int launch_sample(const samplek::Params &p, int dtype, int64_t B, cudaStream_t st) {
    using namespace samplek;
    if (dtype == QL_F32) return launch<float>(p, B, st);
    return dtype == QL_BF16 ? launch<__nv_bfloat16>(p, B, st) : launch<__half>(p, B, st);
}

}  // namespace ql
