// The next token of every row from a random number that the caller gives, with a temperature, top-k, top-p and min-p for each row (ns_sample_tokens).
// ns_f32_sample_rows (ns_sampler.cu) is the reference's sampler, pass for pass: one setting for all rows, numbers drawn inside, ties kept
// together, k + 30 passes by one CTA; this one serves a batch of requests.
//
// For a row x with temperature T: w_j = e^((x_j - max x) / T).  Kept are the first k tokens by (x descending, index ascending); of those the shortest beginning whose
// weights add up to p times all of theirs; of those the ones with w >= min_p.  The drawn token is the first in the order of the vocabulary at which the
// running sum of kept weights exceeds u times their sum.
//
// A draw is decided by whether a sum of up to 10^5 weights lies left or right of a border, so the weights are computed to 2^-33 of themselves and summed as
// integers of 2^-42: exact, whatever the order, the number of CTAs or the atomics.  (With 32-bit weights one row in a few thousand draws another token than the
// definition's.)
//
// A cluster of 1 to 8 CTAs holds a row in shared memory; it is read from global memory once.  What remains costs passes over shared memory:
//   - A top-k of up to ST_WIDE_K: a histogram of every 8th token (of every one, in vocabularies up to 16384) over (max - x) / T, 45 bins to each halving of the weight, names
//     a cutoff that hardly ever fails to leave k candidates and leaves few more; they are gathered into one CTA.  Few are sorted (value, then index), cut by all three rules, sorted by index and drawn from; of more, the three places (of the
//     k-th token, of p of the weight, of u of what is left) are found by a histogram and the tokens of one bin each.  (64 rows of 32 000 in turn 34.9 us with cutoffs of the whole cluster, so 27.7.)
//   - Else cutoffs are found one after the other: a histogram, by number (from such a cutoff on) or by weight, names the bin in which a cutoff lies, and that bin's tokens
//     alone are gathered and sorted (or, where they are too many, counted by the bits of x, 11 at a time).  The draw is then one more pass over the row, or, after a
//     cutoff by weight, the sums of the pass that gathered.
#include <cooperative_groups.h>
#include <math.h>

#include "ns_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int ST_THREADS = 512;
constexpr int ST_BINS = 2048;
constexpr int ST_MAX_CLUSTER = 8;
constexpr int ST_FIX = 42;                 // weights are multiples of 2^-42: 2^20 of them fit 64 bits
constexpr int ST_FAR = 45;                 // 2^-45 and less is no weight
constexpr int ST_OCTAVE = 45;              // bins of the first histogram that halve the weight
constexpr int ST_GUESS = ST_BINS / ST_THREADS;
constexpr float ST_MAGIC = 12582912.0f;    // 1.5 * 2^23: the low bits of a sum with it are the rounded value
constexpr int ST_TABLE = 1024;             // 2^(-i / 1024)
constexpr int ST_LIST = ST_THREADS;         // candidates that are sorted: one a thread
constexpr int ST_SORT_K = 128;             // a top-k whose candidates are looked for in a short vocabulary too
constexpr int ST_WIDE = 4 * ST_LIST;       // candidates that one CTA cuts with histograms of its own: four a thread
constexpr int ST_WIDE_K = 1024;            // the largest top-k whose candidates one CTA takes
constexpr int ST_SAMPLE = 8;               // its cutoff is guessed from every 8th token

struct SampleArgs {
    const void* x;
    int64_t row_stride;
    int rows, vocab, each;                 // each: tokens a CTA holds, of its row
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* ids;
    float* probs;
};

struct SampleTable {
    uint64_t twice[ST_TABLE];              // in units of 2^-43
    float value[ST_TABLE];                 // in units of 2^-42
};

// 2^42 * 2^(-i / 1024), rounded, made by the compiler from the series of e^x (64-bit exponentials would take every CTA microseconds).
struct SamplePowers {
    uint64_t v[ST_TABLE];
    constexpr SamplePowers() : v()
    {
        for (int i = 0; i < ST_TABLE; i++) {
            const double x = -0.69314718055994531 * i / ST_TABLE;
            double sum = 0.0;
            for (int k = 24; k > 0; k--) sum = (sum + 1.0) * x / k;
            v[i] = (uint64_t)((sum + 1.0) * (double)(1ull << ST_FIX) + 0.5);
        }
    }
};
__device__ constexpr SamplePowers st_powers;

struct SampleFound {
    int bin;
    uint64_t before;                       // number or weight of the bins before it
};
// Kept are the tokens whose (key, index) is not above `last`.
struct SampleCut {
    uint64_t last;
    int bin;                               // its bin, where the run sums of gather() are to be used; -1: they are not
};

struct alignas(16) SampleShared {
    union {
        struct {
            uint32_t word[2][ST_BINS];     // numbers, or weights: the low word, the high word
        };
        struct {
            __align__(16) uint64_t list[ST_LIST];        // candidates: key, index
            uint64_t sorted[ST_LIST], weights[ST_LIST];
            int ranks[ST_THREADS];
        };
        struct {
            uint64_t wide[ST_WIDE];
        };
    };
    int listed[ST_MAX_CLUSTER], mine;
    SampleTable table;
    uint64_t part[ST_MAX_CLUSTER], draw[ST_MAX_CLUSTER];       // of every CTA of the cluster, written between its barriers
    union {
        uint64_t extra[ST_THREADS];        // of each thread's run
        uint32_t guess[ST_THREADS];        // a histogram of a sample: of ST_GUESS bins of the first one
    };
    int guessed;
    uint64_t scan[ST_THREADS / 32], scan2[ST_THREADS / 32];
    float max[ST_MAX_CLUSTER], red[ST_THREADS / 32];
    SampleFound found;
    uint64_t cut;
    int run_first, run_end;
    uint64_t run_before;
};

__device__ __forceinline__ float st_value(float x) { return x; }
__device__ __forceinline__ float st_bits(float x, const float*) { return x; }
__device__ __forceinline__ uint16_t st_bits(float x, const uint16_t*) { return (uint16_t)(__float_as_uint(x) >> 16); }       // (of zero and infinity)
__device__ __forceinline__ float st_value(uint16_t x) { return ns_bf16_bits_to_f32(x); }
// As a token is kept: what is no number counts as -infinity (a maximum leaves NaN out), and both zeros are one value (adding 0 gives the positive one).
__device__ __forceinline__ float st_clean(float x) { return fmaxf(x + 0.0f, -INFINITY); }
__device__ __forceinline__ uint32_t st_clean2(uint32_t x)
{
    uint32_t y;
    asm("{\n\t.reg .b32 t;\n\tadd.bf16x2 t, %1, %2;\n\tmax.bf16x2 %0, t, %3;\n\t}" : "=r"(y) : "r"(x), "r"(0u), "r"(0xFF80FF80u));
    return y;
}
__device__ __forceinline__ uint16_t st_clean(uint16_t x) { return (uint16_t)st_clean2(x); }
__device__ __forceinline__ uint32_t st_max2(uint32_t a, uint32_t b)
{
    uint32_t y;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
    return y;
}
// a vector of tokens as they are kept; best: the largest so far
__device__ __forceinline__ void st_take(uint4& v, float& best, const float*)
{
    float* e = reinterpret_cast<float*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        e[i] = st_clean(e[i]);
        best = fmaxf(best, e[i]);
    }
}
__device__ __forceinline__ void st_take(uint4& v, float& best, const uint16_t*)
{
    uint32_t* e = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) e[i] = st_clean2(e[i]);
    const uint32_t m = st_max2(st_max2(e[0], e[1]), st_max2(e[2], e[3]));
    best = fmaxf(best, fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u)));
}
// what is below `value` becomes -infinity; ties: something equals it
__device__ __forceinline__ void st_erase(uint4& v, float value, bool& ties, const float*)
{
    float* e = reinterpret_cast<float*>(&v);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        ties = ties || e[i] == value;
        e[i] = e[i] < value ? -INFINITY : e[i];
    }
}
__device__ __forceinline__ void st_erase(uint4& v, float value, bool& ties, const uint16_t*)
{
    uint32_t* e = reinterpret_cast<uint32_t*>(&v);
    const uint32_t both = __byte_perm(__float_as_uint(value), 0, 0x3232);
    uint32_t equal = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t less, same;
        asm("set.lt.u32.bf16x2 %0, %1, %2;" : "=r"(less) : "r"(e[i]), "r"(both));
        asm("set.eq.u32.bf16x2 %0, %1, %2;" : "=r"(same) : "r"(e[i]), "r"(both));
        equal |= same;
        e[i] = (e[i] & ~less) | (0xFF80FF80u & less);
    }
    ties = equal != 0;
}
// Which of a vector's tokens reach `floor` (a bf16): of 4, a bit each; of 8, the even ones in the low half and the odd ones in the high half, two bits each.
__device__ __forceinline__ uint32_t st_reach(const uint4& v, float floor, const float*)
{
    const float* e = reinterpret_cast<const float*>(&v);
    return (e[0] >= floor ? 1 : 0) | (e[1] >= floor ? 2 : 0) | (e[2] >= floor ? 4 : 0) | (e[3] >= floor ? 8 : 0);
}
__device__ __forceinline__ uint32_t st_reach(const uint4& v, float floor, const uint16_t*)
{
    const uint32_t* e = reinterpret_cast<const uint32_t*>(&v);
    const uint32_t both = __byte_perm(__float_as_uint(floor), 0, 0x3232);
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t m;
        asm("set.ge.u32.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(e[i]), "r"(both));
        mask |= m & (0x00010001u << (2 * i));
    }
    return mask;
}
__device__ __forceinline__ int st_reached(int bit, const float*) { return bit; }
__device__ __forceinline__ int st_reached(int bit, const uint16_t*) { return (bit & 15) + (bit >> 4); }
// ascending where the value descends
__device__ __forceinline__ uint32_t st_key(float x)
{
    const uint32_t b = __float_as_uint(x);
    return (b >> 31) ? b : ~b ^ 0x80000000u;
}

__device__ __forceinline__ float st_unkey(uint32_t key) { return __uint_as_float((key >> 31) ? key : ~key ^ 0x80000000u); }

// the sum that a top-p asks for: the fewest units that are at least p times all of them, one at least
__device__ __forceinline__ uint64_t st_goal(float p, uint64_t all)
{
    const uint64_t goal = p > 0.0f ? (uint64_t)ceil((double)p * (double)all) : 1;
    return goal == 0 ? 1 : goal;
}
// A running sum exceeds u * total where it exceeds that number's floor.
__device__ __forceinline__ uint64_t st_aim(float u, uint64_t total)
{
    const uint64_t aim = u < 1.0f ? (u > 0.0f ? (uint64_t)((double)u * (double)total) : 0) : total - 1;
    return aim >= total ? total - 1 : aim;
}

// e^(-d / T) in units of 2^-42, d = max - x >= 0, within 2^-33 of itself (64-bit floats would take five times as long here: a warp's instruction 16 cycles).
// d is a float and the rest of it, exactly; t = d / (T ln 2) the same to 2^-46 of itself; t = n + i / 1024 + r with |r| <= 2^-11;
// 2^(-i / 1024) from a table, 2^(-r) = 1 + q with q a polynomial of degree 3 and below 2^-11.5 (0.7 * 2^-11), so that each rounding of its float counts 2^-35.5; its product with
// the table's 2^42, below 2^31 therefore, is rounded to an integer of 32 bits once, added to the table's and shifted by n.
__device__ __forceinline__ uint64_t st_pair(float lo, float hi)
{
    uint64_t y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(lo), "f"(hi));
    return y;
}
__device__ __forceinline__ void st_split(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
// two sums, products, fused multiply-adds: each rounded as the single ones are
__device__ __forceinline__ uint64_t st_add2(uint64_t a, uint64_t b)
{
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ uint64_t st_mul2(uint64_t a, uint64_t b)
{
    uint64_t y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ uint64_t st_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}

// a * b + c
__device__ __forceinline__ uint64_t st_mad(int a, int b, uint64_t c)
{
    uint64_t y;
    asm("mad.wide.s32 %0, %1, %2, %3;" : "=l"(y) : "r"(a), "r"(b), "l"(c));
    return y;
}

struct SampleWeight {
    float max, rate, rate_lo;              // 1 / (T ln 2): the float and the rest of it
    const SampleTable* table;
    __device__ __forceinline__ SampleWeight(float m, float temperature, const SampleTable* t) : max(m), table(t)
    {
        const double r = 1.4426950408889634 / (double)temperature;
        rate = (float)fmin(r, 3e38);
        rate_lo = (float)(fmin(r, 3e38) - (double)rate);
    }
    // 2^-p in units of 2^-42, for p's steps of 1/1024 as the low bits of ni and q = 2^-rest - 1: the products add in 64 bits on the multipliers' pipe, the others are
    // this kernel's bound
    __device__ __forceinline__ uint64_t finish(float ni, float q) const
    {
        const int steps = __float_as_int(ni), i = steps & (ST_TABLE - 1), n = (steps >> 10) & 63;       // n * 1024 + i
        const uint64_t w = st_mad(__float2int_rn(table->value[i] * q), 2, table->twice[i]);
        return st_mad(1, 1, w >> n) >> 1;
    }
    // steps of 2^-1/1024 from the maximum down, as the low bits of ni: no more than for the largest p that leaves no weight (infinity and 0 * infinity become that too)
    __device__ __forceinline__ float limit(float p) const { return fminf(p, (float)ST_FAR); }
    // The weights of two tokens, and their bins.
    __device__ __forceinline__ void two(float x0, float x1, uint64_t& w0, uint64_t& w1, int& b0, int& b1) const
    {
        const uint64_t x = st_pair(x0, x1), m = st_pair(max, max), r2 = st_pair(rate, rate), magic = st_pair(ST_MAGIC, ST_MAGIC);
        // (differences as products with -1: the sign of a pair would be two more integer operations)
        const uint64_t minus = st_pair(-1.0f, -1.0f), minus_m = st_pair(-max, -max), d = st_fma2(x, minus, m);
        float p0, p1;
        st_split(st_mul2(d, r2), p0, p1);
        const uint64_t p = st_pair(limit(p0), limit(p1));
        const uint64_t ni = st_fma2(p, st_pair(1024.0f, 1024.0f), magic);
        float n0, n1;
        st_split(ni, n0, n1);
        b0 = bin(n0);
        b1 = bin(n1);
        w0 = w1 = 0;
        if (fminf(p0, p1) >= (float)ST_FAR) return;
        // d + d_lo = max - x; p + p_lo = its product with the rate
        const uint64_t back = st_add2(d, minus_m), minus_d_lo = st_fma2(st_fma2(st_fma2(back, minus, d), minus, m), minus, st_add2(x, back));
        const uint64_t e = st_add2(x, minus_m), minus_p_lo = st_fma2(minus_d_lo, r2, st_fma2(e, st_pair(rate_lo, rate_lo), st_fma2(e, r2, p)));
        const uint64_t r = st_fma2(minus_p_lo, minus, st_fma2(st_add2(ni, st_pair(-ST_MAGIC, -ST_MAGIC)), st_pair(-0.0009765625f, -0.0009765625f), p));      // (the product and its sum are exact)
        const uint64_t q = st_mul2(r, st_fma2(r, st_fma2(r, st_pair(-0.055504109f, -0.055504109f), st_pair(0.24022651f, 0.24022651f)), st_pair(-0.69314718f, -0.69314718f)));
        float q0, q1;
        st_split(q, q0, q1);
        w0 = finish(n0, q0);           // (where p was limited, whatever q is leaves less than half a unit: the conversion saturates)
        w1 = finish(n1, q1);
    }
    __device__ __forceinline__ void two(float x0, float x1, uint64_t& w0, uint64_t& w1) const
    {
        int b0, b1;
        two(x0, x1, w0, w1, b0, b1);
    }
    // The first histogram's bin, never less for a smaller token: ST_OCTAVE of them halve the weight.
    __device__ __forceinline__ int bin(float ni) const { return (__float_as_int(ni) - 0x4B400000) * ST_OCTAVE >> 10; }
    __device__ __forceinline__ int coarse(float x) const { return bin(fmaf(limit((max - x) * rate), 1024.0f, ST_MAGIC)); }
    __device__ __forceinline__ uint64_t operator()(float x) const
    {
        uint64_t w0, w1;
        two(x, -INFINITY, w0, w1);
        return w0;
    }
};

// exclusive sums over the CTA of one 64-bit value a thread; total = their sum.  (A barrier before the next use of `warps`.)
__device__ __forceinline__ uint64_t st_scan(uint64_t v, uint64_t* warps, uint64_t& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    if (lane == 31) warps[warp] = inc;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < ST_THREADS / 32; w++) {
        const uint64_t t = warps[w];
        if (w < warp) before += t;
        total += t;
    }
    return before + inc - v;
}

// Puts `count` different values of `from` into `to` in order.  Every value is compared with all others, by as many threads as there are for each.
__device__ void st_sort(const uint64_t* from, uint64_t* to, int* ranks, int count)
{
    const int tid = threadIdx.x, shares = count <= ST_THREADS / 4 ? 4 : count <= ST_THREADS / 2 ? 2 : 1, width = ST_THREADS / shares;
    const int i = tid & (width - 1), share = tid / width, per = ((count + shares - 1) / shares + 1) & ~1, first = min(share * per, count), end = min(first + per, count);
    ranks[tid] = 0;
    __syncthreads();
    const uint64_t v = i < count ? from[i] : 0;
    if (i < count) {
        int r = 0, j = first;
        const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(from);
#pragma unroll 4
        for (; j + 1 < end; j += 2) {
            const ulonglong2 w = pairs[j >> 1];
            r += (w.x < v ? 1 : 0) + (w.y < v ? 1 : 0);
        }
        if (j < end) r += from[j] < v ? 1 : 0;
        if (r != 0) atomicAdd(&ranks[i], r);
    }
    __syncthreads();
    if (tid < count) to[ranks[tid]] = v;
    __syncthreads();
}

struct SampleCuts {
    int k;
    float top_p, u;
    uint64_t least;                        // smallest weight
};

// Draws from `count` candidates in s.list (key above, index below): by one CTA, the others have left.
__device__ void st_draw(SampleShared& s, int count, const SampleCuts& cuts, const SampleWeight& weight, int row, const SampleArgs& p)
{
    const int tid = threadIdx.x;
    st_sort(s.list, s.sorted, s.ranks, count);
    const uint64_t v = tid < count ? s.sorted[tid] : 0;
    uint64_t w = tid < count && tid < cuts.k ? weight(st_unkey((uint32_t)(v >> 32))) : 0, total;
    uint64_t before = st_scan(w, s.scan, total);
    const uint64_t goal = cuts.top_p < 1.0f ? st_goal(cuts.top_p, total) : ~0ull;
    // kept is the beginning; then by index
    const int kept = __syncthreads_count(tid < count && tid < cuts.k && before < goal && w >= cuts.least);
    if (tid < kept) s.list[tid] = v << 32 | (uint32_t)tid;
    s.weights[tid] = w;
    __syncthreads();
    st_sort(s.list, s.sorted, s.ranks, kept);
    w = tid < kept ? s.weights[(uint32_t)s.sorted[tid]] : 0;
    before = st_scan(w, s.scan2, total);
    const uint64_t aim = st_aim(cuts.u, total);
    if (before <= aim && aim < before + w) {
        p.ids[row] = (int)(s.sorted[tid] >> 32);
        if (p.probs != nullptr) p.probs[row] = (float)((double)w / (double)total);
    }
}

// What one CTA needs to cut up to ST_WIDE candidates; it lies over the CTA's tokens.
struct SampleNarrow {
    uint32_t lo[ST_THREADS], hi[ST_THREADS];           // a histogram of amounts
    uint64_t list[ST_LIST], sorted[ST_LIST];           // a bin's candidates
    int ranks[ST_THREADS];
    uint64_t before, key;
    int found, count;
};

// st_draw for the candidates in s.wide, in no order, four a thread.  Three places are looked for in the same way: the key at which, in the keys' order, sums of amounts reach a
// goal -- the k-th token, the one at which p of their weight is reached, and, with what is left in the order of the vocabulary, the drawn one.
__device__ void st_draw_wide(SampleShared& s, SampleNarrow& m, int count, const SampleCuts& cuts, const SampleWeight& weight, int row, const SampleArgs& p)
{
    const int tid = threadIdx.x, shift = max(0, 32 - __clz(p.vocab) - 9);
    uint64_t key[4], v[4], total = 0, last = ~0ull;
    uint32_t live = 0;                                 // of the four, those that are left
    int bin[4];                                        // a monotone function of the key
    auto weigh = [&](uint64_t k) { return weight(st_unkey((uint32_t)(k >> 32))); };
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int at = tid + i * ST_THREADS;
        key[i] = at < count ? s.wide[at] : ~0ull;
        live |= at < count ? 1u << i : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        weight.two(st_unkey((uint32_t)(key[i] >> 32)), st_unkey((uint32_t)(key[i + 1] >> 32)), v[i], v[i + 1], bin[i], bin[i + 1]);
        bin[i] /= ST_BINS / ST_THREADS;
        bin[i + 1] /= ST_BINS / ST_THREADS;
    }
#pragma unroll 1
    for (int step = 0; step < 3; step++) {
        if (step == 1 && !(cuts.top_p < 1.0f)) continue;
        uint64_t goal = (uint64_t)cuts.k;
        auto amount = [&](int i) -> uint64_t { return (live >> i & 1) == 0 ? 0 : step == 0 ? 1 : v[i]; };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (key[i] > last || (step == 2 && v[i] < cuts.least)) live &= ~(1u << i);
            if (step == 2) {
                bin[i] = min((int)((uint32_t)key[i] >> shift), ST_THREADS - 1);
                key[i] = key[i] << 32 | (uint32_t)(tid + i * ST_THREADS);
            }
        }
        if (step > 0) {
            st_scan(amount(0) + amount(1) + amount(2) + amount(3), s.scan2, total);
            goal = step == 1 ? st_goal(cuts.top_p, total) : st_aim(cuts.u, total) + 1;
        }
        m.lo[tid] = m.hi[tid] = 0;
        if (tid == 0) m.count = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (amount(i) != 0) {
                const uint32_t lo = (uint32_t)amount(i), hi = (uint32_t)(amount(i) >> 32) + (atomicAdd(&m.lo[bin[i]], lo) + lo < lo ? 1 : 0);
                if (hi != 0) atomicAdd(&m.hi[bin[i]], hi);
            }
        __syncthreads();
        const uint64_t mine = (uint64_t)m.hi[tid] << 32 | m.lo[tid];
        uint64_t all;
        const uint64_t before = st_scan(mine, s.scan, all);
        if (before < goal && goal <= before + mine) {
            m.found = tid;
            m.before = before;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (amount(i) != 0 && bin[i] == m.found) {
                const int at = atomicAdd(&m.count, 1);
                if (at < ST_LIST) m.list[at] = key[i];
            }
        __syncthreads();
        const int listed = m.count;
        if (listed <= ST_LIST) {
            st_sort(m.list, m.sorted, m.ranks, listed);
            const uint64_t k = tid < listed ? m.sorted[tid] : 0, of = tid >= listed ? 0 : step == 0 ? 1 : weigh(step == 1 ? k : s.wide[(uint32_t)k]);
            const uint64_t ahead = m.before + st_scan(of, s.scan2, all);
            if (ahead < goal && goal <= ahead + of) m.key = k;
        } else {
            // more than can be sorted: by halves
            uint64_t least = 0, most = ~0ull;
            while (least < most) {
                const uint64_t middle = least + (most - least) / 2;
                uint64_t sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) sum += key[i] <= middle ? amount(i) : 0;
                __syncthreads();
                st_scan(sum, s.scan2, all);
                if (all >= goal) most = middle;
                else least = middle + 1;
            }
            if (tid == 0) m.key = least;
        }
        __syncthreads();
        last = m.key;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (key[i] == last && (live >> i & 1) != 0) {
            p.ids[row] = (int)(last >> 32);
            if (p.probs != nullptr) p.probs[row] = (float)((double)v[i] / (double)total);
        }
}

template <typename T>
struct SampleRow {
    static constexpr int VEC = 16 / sizeof(T);
    SampleShared& s;
    T* vals;                               // this CTA's tokens; they begin `skew` after a vector
    int n, first, skew;                    // how many, the first's index
    cg::cluster_group cl;
    int rank, ranks;
    const SampleWeight& weight;

    // f(number in the CTA, value) for its tokens: vectors first, first + step .. below end
    template <typename F>
    __device__ __forceinline__ void each(int at, int step, int end, F f) const
    {
        const uint4* vecs = reinterpret_cast<const uint4*>(vals - skew);
        for (int v = at; v < end; v += step) {
            const uint4 raw = vecs[v];
            const T* e = reinterpret_cast<const T*>(&raw);
            const int i0 = v * VEC - skew;
            if (i0 >= 0 && i0 + VEC <= n) {
#pragma unroll
                for (int i = 0; i < VEC; i++) f(i0 + i, st_value(e[i]));
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    if (i0 + i >= 0 && i0 + i < n) f(i0 + i, st_value(e[i]));
            }
        }
    }
    // f(number in the CTA of the first, value, value) for pairs of neighbouring tokens, -infinity where there is none
    template <typename F>
    __device__ __forceinline__ void pairs(int at, int step, int end, F f) const
    {
        const uint4* vecs = reinterpret_cast<const uint4*>(vals - skew);
        for (int v = at; v < end; v += step) {
            const uint4 raw = vecs[v];
            const T* e = reinterpret_cast<const T*>(&raw);
            const int i0 = v * VEC - skew;
            if (i0 >= 0 && i0 + VEC <= n) {
#pragma unroll
                for (int i = 0; i < VEC; i += 2) f(i0 + i, st_value(e[i]), st_value(e[i + 1]));
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i += 2)
                    f(i0 + i, i0 + i >= 0 && i0 + i < n ? st_value(e[i]) : -INFINITY, i0 + i + 1 >= 0 && i0 + i + 1 < n ? st_value(e[i + 1]) : -INFINITY);
            }
        }
    }
    // f(number in the CTA, value) for the tokens that reach `floor`, where they are few
    template <typename F>
    __device__ __forceinline__ void above(int at, int step, int end, float floor, F f) const
    {
        const uint4* vecs = reinterpret_cast<const uint4*>(vals - skew);
        for (int v = at; v < end; v += step)
            for (uint32_t mask = st_reach(vecs[v], floor, vals); mask != 0; mask &= mask - 1) {
                const int i = v * VEC - skew + st_reached(__ffs((int)mask) - 1, vals);
                if (i >= 0 && i < n) f(i, st_value(vals[i]));
            }
    }
    __device__ __forceinline__ int vectors() const { return n > 0 ? (n + skew + VEC - 1) / VEC : 0; }
    // a thread's run of neighbouring vectors: an odd number, so that neighbouring threads read from different banks
    __device__ __forceinline__ int run_length() const { return (vectors() + ST_THREADS - 1) / ST_THREADS | 1; }
    __device__ __forceinline__ int run_begin(int thread) const { return min(thread * run_length(), vectors()); }
    template <typename F>
    __device__ __forceinline__ void run(F f) const { each(run_begin(threadIdx.x), 1, run_begin(threadIdx.x + 1), f); }
    __device__ __forceinline__ uint64_t place(int i, float x) const { return ((uint64_t)st_key(x) << 32) | (uint32_t)(first + i); }
    template <typename F>
    __device__ __forceinline__ void all(F f) const { each(threadIdx.x, ST_THREADS, vectors(), f); }

    __device__ void clear(bool mass)
    {
        uint32_t* w = s.word[0];
        for (int i = threadIdx.x; i < (mass ? 2 : 1) * ST_BINS; i += ST_THREADS) w[i] = 0;
        __syncthreads();
    }
    // adds a token to a histogram
    __device__ __forceinline__ void put(bool mass, int bin, uint64_t weight)
    {
        if (!mass) {
            atomicAdd(&s.word[0][bin], 1u);
            return;
        }
        // (one addition for most: a 64-bit one took several times as long)
        const uint32_t lo = (uint32_t)weight;
        if (weight == 0) return;
        const uint32_t hi = (uint32_t)(weight >> 32) + (atomicAdd(&s.word[0][bin], lo) + lo < lo ? 1 : 0);
        if (hi != 0) atomicAdd(&s.word[1][bin], hi);
    }
    // The bin in which the sums over the cluster's histograms reach goal(whole sum) (1 to the whole sum), the same in every CTA.
    template <typename G>
    __device__ SampleFound find(bool mass, G goal)
    {
        cl.sync();
        const int bins = ST_BINS / ranks, per = bins < ST_THREADS ? 1 : bins / ST_THREADS, at = rank * bins + threadIdx.x * per;
        const bool active = (int)threadIdx.x * per < bins;
        uint64_t mine[4] = {0, 0, 0, 0}, sum = 0;
        if (active) {
            // (all loads ahead of their sums: they come from other SMs)
            if (per == 1) {
                uint32_t lo[ST_MAX_CLUSTER], hi[ST_MAX_CLUSTER];
#pragma unroll
                for (int r = 0; r < ST_MAX_CLUSTER; r++) {
                    const SampleShared* o = cl.map_shared_rank(&s, min(r, ranks - 1));
                    lo[r] = o->word[0][at];
                    hi[r] = mass ? o->word[1][at] : 0;
                }
#pragma unroll
                for (int r = 0; r < ST_MAX_CLUSTER; r++)
                    if (r < ranks) mine[0] += (uint64_t)hi[r] << 32 | lo[r];
            } else {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const SampleShared* o = cl.map_shared_rank(&s, min(r, ranks - 1));
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (i < per && r < ranks) mine[i] += (uint64_t)(mass ? o->word[1][at + i] : 0) << 32 | o->word[0][at + i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) sum += mine[i];
        uint64_t total;
        uint64_t before = st_scan(sum, s.scan, total);
        if ((int)threadIdx.x < ranks) cl.map_shared_rank(&s, threadIdx.x)->part[rank] = total;
        cl.sync();
        total = 0;
        for (int r = 0; r < ranks; r++) {
            if (r < rank) before += s.part[r];
            total += s.part[r];
        }
        const uint64_t target = goal(total);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (active && i < per && before < target && target <= before + mine[i])
                for (int r = 0; r < ranks; r++) cl.map_shared_rank(&s, r)->found = SampleFound{at + i, before};
            before += mine[i];
        }
        cl.sync();
        return s.found;
    }
    // pass(list) goes over the CTA's tokens; those that it gives to list(number, value) are listed, in no order.  Then the cluster's lists are gathered into the first CTA's;
    // their tokens' number, or -1 where they are too many.  The lists lie over the histograms.  (A barrier of the cluster before the others' lists change.)
    template <int MOST = ST_LIST, typename F>
    __device__ int gather(F pass)
    {
        if (threadIdx.x == 0) s.mine = 0;
        __syncthreads();
        pass([&](int i, float x) {
            const int at = atomicAdd(&s.mine, 1);
            if (at < MOST) s.wide[at] = place(i, x);
        });
        __syncthreads();
        if ((int)threadIdx.x < ranks) cl.map_shared_rank(&s, threadIdx.x)->listed[rank] = s.mine;
        cl.sync();
        int sum = 0;
        bool fits = true;
        for (int r = 0; r < ranks; r++) {
            fits = fits && s.listed[r] <= MOST;
            sum += s.listed[r];
        }
        if (!fits || sum > MOST) return -1;
        if (rank == 0) {
            for (int i = threadIdx.x; i < sum; i += ST_THREADS) {
                int r = 0, at = i;
                while (at >= s.listed[r]) at -= s.listed[r++];
                if (r > 0) s.wide[i] = cl.map_shared_rank(&s, r)->wide[at];
            }
            __syncthreads();
        }
        return sum;
    }
    __device__ void tell(uint64_t last)
    {
        for (int r = 0; r < ranks; r++) cl.map_shared_rank(&s, r)->cut = last;
    }
    // Among `count` listed tokens, in order: the one at which sums reach `rest`, told to the cluster.
    __device__ void cut_list(bool mass, int count, uint64_t rest)
    {
        const int tid = threadIdx.x;
        st_sort(s.list, s.sorted, s.ranks, count);
        const uint64_t v = tid < count ? s.sorted[tid] : 0;
        const uint64_t w = tid >= count ? 0 : mass ? weight(st_unkey((uint32_t)(v >> 32))) : 1;
        uint64_t total;
        const uint64_t before = st_scan(w, s.scan, total);
        if (before < rest && rest <= before + w) tell(v);
    }
    // Finds the token at which, in order, sums reach goal(their whole sum), by weight or by number.  few: of the tokens that reach `floor`, which are few.  sum, by weight: the
    // thread's run's weights from `least` on of the bins before the token's, for the draw.
    template <typename G>
    __device__ SampleCut select(bool mass, bool few, float floor, uint64_t least, uint64_t& sum, G goal)
    {
        const int tid = threadIdx.x;
        clear(mass);
        if (few) {
            above(tid, ST_THREADS, vectors(), floor, [&](int, float x) { put(mass, weight.coarse(x), mass ? weight(x) : 0); });
        } else {
            pairs(tid, ST_THREADS, vectors(), [&](int, float x0, float x1) {
                uint64_t w0 = 0, w1 = 0;
                int b0, b1;
                if (mass) {
                    weight.two(x0, x1, w0, w1, b0, b1);
                } else {
                    b0 = weight.coarse(x0);
                    b1 = weight.coarse(x1);
                }
                put(mass, b0, w0);
                put(mass, b1, w1);
            });
        }
        uint64_t target = 0, whole = 0;
        SampleFound f = find(mass, [&](uint64_t all) {
            whole = all;
            return target = goal(all);
        });
        if (target > whole) return SampleCut{~0ull, -2};
        const int bin = f.bin;
        if (bin > (ST_FIX + 1) * ST_OCTAVE) return SampleCut{~0ull, -1};      // it and all after it have no weight
        uint64_t rest = target - f.before;
        sum = 0;
        int count = 0;
        const int begin = run_begin(tid), end = run_begin(tid + 1);
        count = gather([&](auto list) {
            if (few) {
                above(begin, 1, end, floor, [&](int i, float x) {
                    const int b = weight.coarse(x);
                    if (b == bin) list(i, x);
                    if (!mass || b >= bin) return;
                    const uint64_t w = weight(x);
                    if (w >= least) sum += w;
                });
            } else if (!mass) {
                pairs(begin, 1, end, [&](int i, float x0, float x1) {
                    if (weight.coarse(x0) == bin) list(i, x0);
                    if (weight.coarse(x1) == bin) list(i + 1, x1);
                });
            } else {
                auto body = [&](auto kept) {
                    pairs(begin, 1, end, [&](int i, float x0, float x1) {
                        uint64_t w0, w1;
                        int b0, b1;
                        weight.two(x0, x1, w0, w1, b0, b1);
                        if (b0 == bin) list(i, x0);
                        if (b1 == bin) list(i + 1, x1);
                        sum += (b0 < bin ? kept(w0) : 0) + (b1 < bin ? kept(w1) : 0);
                    });
                };
                if (least == 0) body([](uint64_t w) { return w; });
                else body([least](uint64_t w) { return w >= least ? w : 0; });
            }
        });
        if (count >= 0) {
            if (rank == 0) cut_list(mass, count, rest);
            cl.sync();
            return SampleCut{s.cut, bin};
        }
        // too many: the key by its bits, then the token by its number among the key's
        constexpr int LEVELS = sizeof(T) == 2 ? 2 : 3, LOW = sizeof(T) == 2 ? 16 : 0;
        uint32_t prefix = 0;
#pragma unroll 1
        for (int level = 0; level < LEVELS; level++) {
            const int shift = level == 0 ? 21 : level == LEVELS - 1 ? LOW : 10, bits = level == 0 ? 11 : level == 1 ? 21 - shift : 10;
            cl.sync();
            clear(mass);
            all([&](int i, float x) {
                const uint32_t k = st_key(x);
                if (weight.coarse(x) == bin && (level == 0 || (k >> (shift + bits)) == prefix))
                    put(mass, (int)((k >> shift) & ((1u << bits) - 1)), mass ? weight(x) : 0);
            });
            f = find(mass, [&](uint64_t) { return rest; });
            rest -= f.before;
            prefix = (prefix << bits) | (uint32_t)f.bin;
        }
        if (LOW != 0) prefix = prefix << LOW | ((prefix >> 15) != 0 ? 0u : 0xFFFFu);        // (the lower half of a bf16's key)
        if (mass) {
            const uint64_t w = weight(st_unkey(prefix));
            rest = (rest + w - 1) / w;
        }
        uint64_t ties = 0, total;
        run([&](int, float x) { ties += st_key(x) == prefix ? 1 : 0; });
        uint64_t before = st_scan(ties, s.scan, total);
        if ((int)threadIdx.x < ranks) cl.map_shared_rank(&s, threadIdx.x)->part[rank] = total;
        cl.sync();
        for (int r = 0; r < rank; r++) before += s.part[r];
        if (before < rest && rest <= before + ties)
            run([&](int i, float x) {
                if (st_key(x) == prefix && ++before == rest) tell(place(i, x));
            });
        cl.sync();
        return SampleCut{s.cut, -1};
    }
    // What lies after `last` becomes -infinity.
    __device__ void erase(uint64_t last)
    {
        const float value = st_unkey((uint32_t)(last >> 32));
        uint4* vecs = reinterpret_cast<uint4*>(vals - skew);
        for (int v = threadIdx.x; v < vectors(); v += ST_THREADS) {
            uint4 raw = vecs[v];
            bool ties = false;
            st_erase(raw, value, ties, vals);
            if (ties) {
                T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
                for (int i = 0; i < VEC; i++)
                    if (st_value(e[i]) == value && first + v * VEC - skew + i > (int)(uint32_t)last) e[i] = st_bits(-INFINITY, vals);
            }
            vecs[v] = raw;
        }
        __syncthreads();
    }
};

template <typename T>
__global__ void __launch_bounds__(ST_THREADS) ns_sample_tokens_kernel(const SampleArgs p)
{
    extern __shared__ __align__(16) uint8_t st_smem[];
    SampleShared& s = *reinterpret_cast<SampleShared*>(st_smem);
    ns_pdl_wait();
    ns_pdl_trigger();
    cg::cluster_group cl = cg::this_cluster();
    // (answered before the first write to another CTA's shared memory, which exists only from that CTA's start on; the row is read in between)
    auto begun = cl.barrier_arrive();
    const int rank = (int)cl.block_rank(), ranks = (int)cl.num_blocks();
    const int row = blockIdx.x / ranks, tid = threadIdx.x;
    const int first = min(rank * p.each, p.vocab), n = min(p.each, p.vocab - first);
    const T* src = reinterpret_cast<const T*>(p.x) + row * p.row_stride + first;
    // the row lies in shared memory as it lies in global memory, modulo 16 bytes
    constexpr int VEC = 16 / sizeof(T);
    const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    T* vals = reinterpret_cast<T*>(st_smem + sizeof(SampleShared)) + skew;

    // asked for ahead of the row
    const float temperature = p.temperature != nullptr ? p.temperature[row] : 1.0f;
    int k = p.top_k != nullptr ? p.top_k[row] : 0;
    const float top_p = p.top_p != nullptr ? p.top_p[row] : 1.0f, min_p = p.min_p != nullptr ? p.min_p[row] : 0.0f;
    uint64_t power[ST_TABLE / ST_THREADS];
#pragma unroll
    for (int i = 0; i < ST_TABLE / ST_THREADS; i++) power[i] = st_powers.v[tid + i * ST_THREADS];
    float best = -INFINITY;
    const int head = min(n, skew == 0 ? 0 : VEC - skew), vecs = (n - head) / VEC, tail = head + vecs * VEC;
    auto take_one = [&](int i) {
        vals[i] = st_clean(src[i]);
        best = fmaxf(best, st_value(vals[i]));
    };
    if (tid < head) take_one(tid);
    {
        constexpr int U = 4;
        const uint4* from = reinterpret_cast<const uint4*>(src + head);
        uint4* to = reinterpret_cast<uint4*>(vals + head);
        for (int at = tid; at < vecs; at += U * ST_THREADS) {
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (at + u * ST_THREADS < vecs) v[u] = from[at + u * ST_THREADS];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (at + u * ST_THREADS < vecs) {
                    st_take(v[u], best, src);
                    to[at + u * ST_THREADS] = v[u];
                }
        }
    }
    if (tail + tid < n) take_one(tail + tid);
#pragma unroll
    for (int i = 0; i < ST_TABLE / ST_THREADS; i++) {
        s.table.twice[tid + i * ST_THREADS] = 2 * power[i];
        s.table.value[tid + i * ST_THREADS] = (float)power[i];
    }
    s.guess[tid] = 0;
    // ---- the maximum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((tid & 31) == 0) s.red[tid >> 5] = best;
    __syncthreads();
    cl.barrier_wait(static_cast<decltype(begun)&&>(begun));      // every CTA of the cluster runs
    if (tid < ranks) {
        for (int w = 0; w < ST_THREADS / 32; w++) best = fmaxf(best, s.red[w]);
        cl.map_shared_rank(&s, tid)->max[rank] = best;
    }
    cl.sync();
    float max = s.max[0];
    for (int r = 1; r < ranks; r++) max = fmaxf(max, s.max[r]);

    if (k <= 0 || k > p.vocab) k = p.vocab;
    // Greedily, or nothing to choose from: every CTA sees the same and leaves, the first that has the maximum once it has found where.
    if (max == -INFINITY || !(temperature > 0.0f) || k == 1) {
        int owner = 0;
        while (s.max[owner] != max) owner++;
        if (rank == owner) {
            if (tid == 0) s.mine = n;
            __syncthreads();
            int at = n;
            for (int i = tid; i < n && at == n; i += ST_THREADS)
                if (st_value(vals[i]) == max) at = i;
            if (at < n) atomicMin(&s.mine, at);
            __syncthreads();
            if (tid == 0) {
                p.ids[row] = max == -INFINITY ? -1 : first + s.mine;
                if (p.probs != nullptr) p.probs[row] = max == -INFINITY ? 0.0f : 1.0f;
            }
        }
        return;
    }
    if (max == INFINITY) {
        // infinite tokens share everything: as zeros among tokens of -infinity
        for (int i = tid; i < n; i += ST_THREADS) vals[i] = st_value(vals[i]) == INFINITY ? st_bits(0.0f, vals) : st_bits(-INFINITY, vals);
        max = 0.0f;
        __syncthreads();
    }
    const SampleWeight weight(max, temperature, &s.table);
    SampleRow<T> me{s, vals, n, first, skew, cl, rank, ranks, weight};
    uint64_t least = 0;
    if (min_p > 0.0f) least = (uint64_t)ceil((double)fminf(min_p, 1.0f) * (double)(1ull << ST_FIX));

    // ---- the first k
    SampleCut cut{~0ull, -1};
    uint64_t sum = 0;
    float floor = -INFINITY;
    bool few = false;                      // few tokens reach `floor`, and all that are left do
    if (k < p.vocab) {
        if (k <= ST_SORT_K || (p.vocab > 2048 * ST_SAMPLE && k <= p.vocab / 16)) {
            // A value that about k tokens or some more reach, from a sample: so much of it that k hardly ever fail to be among those it stands for.
            int every = 1;
            uint64_t need = k;
            if (p.vocab > 2048 * ST_SAMPLE) {
                every = ST_SAMPLE;
                const float share = (float)k / ST_SAMPLE;
                need = (uint64_t)(1.25f * share + 3.0f * sqrtf(share) + 4.0f);
            }
            for (int i = (every - first % every) % every + tid * every; i < n; i += ST_THREADS * every) atomicAdd(&s.guess[weight.coarse(st_value(vals[i])) / ST_GUESS], 1u);
            cl.sync();
            uint64_t in_bin = 0, sample;   // every CTA sums them all: that takes one barrier instead of three
            uint32_t of[ST_MAX_CLUSTER];
#pragma unroll
            for (int r = 0; r < ST_MAX_CLUSTER; r++) of[r] = cl.map_shared_rank(&s, min(r, ranks - 1))->guess[tid];
#pragma unroll
            for (int r = 0; r < ST_MAX_CLUSTER; r++) in_bin += r < ranks ? of[r] : 0;
            const uint64_t ahead = st_scan(in_bin, s.scan, sample), wanted = need < sample ? need : sample;
            if (ahead < wanted && wanted <= ahead + in_bin) s.guessed = tid * ST_GUESS + ST_GUESS - 1;
            __syncthreads();
            floor = fmaxf(max - ((float)s.guessed + 1.0f) * (temperature * (0.69314718f / ST_OCTAVE)), -3e38f);
            floor = __uint_as_float(__float_as_uint(floor) & 0xFFFF0000u);
            few = true;
        }
        if (few && k <= ST_WIDE_K) {
            int count = 0;
            count = me.template gather<ST_WIDE>([&](auto list) { me.above(me.run_begin(tid), 1, me.run_begin(tid + 1), floor, list); });
            const bool room = p.each * sizeof(T) >= sizeof(SampleNarrow), wide = count > (room ? ST_LIST / 2 : ST_LIST);
            if (count >= k && (room || !wide)) {
                const SampleCuts cuts{k, top_p, p.u[row], least};
                auto listed = cl.barrier_arrive();         // the first CTA has the others' lists
                if (rank == 0) {
                    if (wide) st_draw_wide(s, *reinterpret_cast<SampleNarrow*>(st_smem + sizeof(SampleShared)), count, cuts, weight, row, p);
                    else st_draw(s, count, cuts, weight, row, p);
                }
                cl.barrier_wait(static_cast<decltype(listed)&&>(listed));
                return;
            }
            cl.sync();
            few = count < 0 || count >= k;                 // too many, or not enough
        }
        auto number = [&](uint64_t) { return (uint64_t)k; };
        cut = me.select(false, few, floor, least, sum, number);
        if (cut.bin == -2) {               // the guess was too high
            cl.sync();
            few = false;
            cut = me.select(false, few, floor, least, sum, number);
        }
        if (cut.last != ~0ull) {
            if (few && cut.bin >= 0) {
                // what reaches the value of the last token and lies after it is among the CTA's part of the lists
                if (tid < s.mine && s.list[tid] > cut.last) vals[(int)(uint32_t)s.list[tid] - first] = st_bits(-INFINITY, vals);
                __syncthreads();
            } else {
                me.erase(cut.last);
                few = k <= p.vocab / 16;
            }
            floor = st_unkey((uint32_t)(cut.last >> 32));
            cut = SampleCut{~0ull, -1};
        } else {
            few = false;
        }
    }
    // ---- of those, the first that have p of the weight
    if (top_p < 1.0f) {
        cl.sync();
        cut = me.select(true, few, floor, least, sum, [&](uint64_t whole) { return st_goal(top_p, whole); });
        if (cut.bin < 0 && cut.last != ~0ull) {
            me.erase(cut.last);
            cut = SampleCut{~0ull, -1};
        }
    }

    // ---- the draw: the weights of each thread's run
    if (cut.bin < 0) {
        sum = 0;
        const int begin = me.run_begin(tid), end = me.run_begin(tid + 1);
        auto sums = [&](auto kept) {
            me.pairs(begin, 1, end, [&](int, float x0, float x1) {
                uint64_t w0, w1;
                weight.two(x0, x1, w0, w1);
                sum += kept(w0) + kept(w1);
            });
        };
        if (few)
            me.above(begin, 1, end, floor, [&](int, float x) {
                const uint64_t w = weight(x);
                if (w >= least) sum += w;
            });
        else if (least == 0) sums([](uint64_t w) { return w; });
        else sums([least](uint64_t w) { return w >= least ? w : 0; });
    } else {
        // all but the cutoff's bin are in the sums: its tokens are this CTA's part of the lists
        s.extra[tid] = 0;
        __syncthreads();
        if (tid < s.mine) {
            const uint64_t v = s.list[tid];
            if (v <= cut.last) {
                const uint64_t w = weight(st_unkey((uint32_t)(v >> 32)));
                const int thread = ((int)(uint32_t)v - first + skew) / me.VEC / me.run_length();
                if (w >= least) atomicAdd(reinterpret_cast<unsigned long long*>(&s.extra[thread]), (unsigned long long)w);
            }
        }
        __syncthreads();
        sum += s.extra[tid];
    }
    uint64_t total;
    uint64_t before = st_scan(sum, s.scan, total);
    if (tid < ranks) cl.map_shared_rank(&s, tid)->draw[rank] = total;
    cl.sync();
    total = 0;
    for (int r = 0; r < ranks; r++) {
        if (r < rank) before += s.draw[r];
        total += s.draw[r];
    }
    const uint64_t aim = st_aim(p.u[row], total);
    const bool mine = before <= aim && aim < before + sum;
    // One run of the cluster's holds the token: its CTA goes over it a token a thread.
    if (mine) {
        s.run_first = me.run_begin(tid);
        s.run_end = me.run_begin(tid + 1);
        s.run_before = before;
    }
    if (__syncthreads_or(mine)) {
        const int i = s.run_first * me.VEC - skew + tid;
        uint64_t w = 0, unused;
        if (i >= 0 && i < n && i < s.run_end * me.VEC - skew) {
            const float x = st_value(vals[i]);
            w = weight(x);
            if (w < least || (few && x < floor) || me.place(i, x) > cut.last) w = 0;
        }
        const uint64_t at = s.run_before + st_scan(w, s.scan2, unused);
        if (at <= aim && aim < at + w) {
            p.ids[row] = first + i;
            if (p.probs != nullptr) p.probs[row] = (float)((double)w / (double)total);
        }
    }
    cl.sync();      // a CTA's shared memory stays until the others have written to it
}

// Shared memory for `each` tokens and what goes before them.
size_t st_bytes(int each, int size) { return sizeof(SampleShared) + (size_t)each * size + 16; }

}  // namespace

extern "C" int ns_sample_tokens(ns_device_t h, uint64_t logits, int dtype, int64_t row_stride, int rows, int vocab, uint64_t temperature, uint64_t top_k, uint64_t top_p,
                                uint64_t min_p, uint64_t u, uint64_t ids, uint64_t probs)
{
    NS_REQUIRE(logits && u && ids, NS_ERR_ARGUMENT, "ns_sample_tokens: null argument");
    NS_REQUIRE(dtype == NS_F32 || dtype == NS_BF16, NS_ERR_ARGUMENT, "ns_sample_tokens: dtype must be NS_F32 or NS_BF16");
    NS_REQUIRE(rows >= 0 && vocab > 0 && row_stride >= 0, NS_ERR_ARGUMENT, "ns_sample_tokens: bad shape");
    const int size = dtype == NS_F32 ? 4 : 2;
    NS_REQUIRE((logits & (uint64_t)(size - 1)) == 0 && ((temperature | top_k | top_p | min_p | u | ids | probs) & 3) == 0, NS_ERR_ARGUMENT,
               "ns_sample_tokens: misaligned argument");
    constexpr int most = 227 * 1024;
    const int most_each = (most - (int)sizeof(SampleShared) - 16) / size / 8 * 8;
    NS_REQUIRE((int64_t)vocab <= (int64_t)ST_MAX_CLUSTER * most_each, NS_ERR_ARGUMENT, "ns_sample_tokens: at most %d tokens of this type",
               ST_MAX_CLUSTER * most_each);
    NS_REQUIRE(rows <= (1 << 27), NS_ERR_ARGUMENT, "ns_sample_tokens: too many rows");
    NsDevice* d = ns_dev(h);
    int rc = ns_device_make_current(d);
    if (rc != NS_OK) return rc;
    if (rows == 0) return NS_OK;
    SampleArgs p;
    p.x = reinterpret_cast<const void*>(logits);
    p.row_stride = row_stride; p.rows = rows; p.vocab = vocab;
    p.temperature = reinterpret_cast<const float*>(temperature);
    p.top_k = reinterpret_cast<const int32_t*>(top_k);
    p.top_p = reinterpret_cast<const float*>(top_p);
    p.min_p = reinterpret_cast<const float*>(min_p);
    p.u = reinterpret_cast<const float*>(u);
    p.ids = reinterpret_cast<int32_t*>(ids);
    p.probs = reinterpret_cast<float*>(probs);
    // CTAs a row: as many as leave room for two of them an SM (one has too few warps for the latency of its passes: 256 rows of 131 001 bf16 182 us with two a row,
    // 150 with four, 186 with eight), and until the SMs are full or a thread has few tokens left.
    int ranks = 1;
    auto each = [&](int r) { return ((vocab + r - 1) / r + 7) / 8 * 8; };
    while (ranks < ST_MAX_CLUSTER && (2 * st_bytes(each(ranks), size) > (size_t)most || ((int64_t)rows * ranks < d->sm_count && each(ranks) > 8 * ST_THREADS))) ranks *= 2;
    p.each = each(ranks);
    const size_t smem = st_bytes(p.each, size);
    auto kernel = dtype == NS_F32 ? ns_sample_tokens_kernel<float> : ns_sample_tokens_kernel<uint16_t>;
    NS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ranks));
    cfg.blockDim = dim3(ST_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = d->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    NS_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return NS_OK;
}
