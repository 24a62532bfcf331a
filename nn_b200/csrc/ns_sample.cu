// The next token of every row from a random number that the caller gives, with a temperature, top-k, top-p and min-p for each row (ns_sample_tokens).
// ns_f32_sample_rows (ns_sampler.cu) is the reference's sampler, pass for pass: one setting for all rows, numbers drawn inside, ties kept
// together, k + 30 passes by one CTA; this one serves a batch of requests.
//
// For a row x with temperature T: w_j = e^((x_j - max x) / T).  Kept are the first k tokens by (x descending, index ascending); of those the shortest beginning whose
// weights add up to p times all of theirs; of those the ones with w >= min_p.  The drawn token is the first in the order of the vocabulary at which the
// running sum of kept weights exceeds u times their sum.
//
// A draw is decided by whether a sum of up to 10^5 weights lies left or right of a border, so the weights are computed in 64 bits and summed as integers
// of 2^-44: exact, whatever the order, the number of CTAs or the atomics.  (With 32-bit weights one row in a few thousand draws another token than the
// definition's.)
//
// A cluster of 1 to 8 CTAs holds a row in shared memory; it is read from global memory once.  The cutoffs are found by histograms: first over
// (max - x) / T in steps of 1/64, where weights down to 2^-44 spread over 2048 bins, then inside the bin over the bits of x, 11 at a time.
#include <cooperative_groups.h>
#include <math.h>

#include "ns_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int ST_THREADS = 512;
constexpr int ST_BINS = 2048;
constexpr int ST_MAX_CLUSTER = 8;
constexpr int ST_FIX = 44;                 // weights are multiples of 2^-44: 2^20 of them fit 64 bits
constexpr int ST_TABLE = 128;              // 2^(-i / 128)
constexpr uint32_t ST_NO_CUT = 0xFFFFFFFFu;

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

struct SampleFound {
    int bin;
    uint32_t count;                        // tokens of that bin
    uint64_t before;                       // count or mass of the bins before it
};

struct alignas(16) SampleShared {
    uint32_t count[ST_BINS], lo[ST_BINS], hi[ST_BINS];
    double table[ST_TABLE];
    uint64_t part[ST_MAX_CLUSTER], mass[ST_MAX_CLUSTER], ties[ST_MAX_CLUSTER];       // of every CTA of the cluster; each written once or between barriers
    uint64_t scan[ST_THREADS / 32], scan2[ST_THREADS / 32];
    float max[ST_MAX_CLUSTER];
    int max_at[ST_MAX_CLUSTER];
    float red[ST_THREADS / 32];
    int red_at[ST_THREADS / 32];
    SampleFound found;
};

// not a number counts as -infinity, and both zeros are one value
__device__ __forceinline__ float st_clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ float st_value(float x) { return st_clean(x); }
__device__ __forceinline__ float st_value(uint16_t x) { return st_clean(ns_bf16_bits_to_f32(x)); }
// ascending where the value descends
__device__ __forceinline__ uint32_t st_key(float x)
{
    const uint32_t b = __float_as_uint(x);
    return (b >> 31) ? b : ~b ^ 0x80000000u;
}

// e^(-d / T) in units of 2^-44, d = max - x >= 0.  z = 128 d / (T ln 2) = n + r; 2^(-z / 128) = 2^(-n / 128) times a polynomial of degree 4 in r (its next term is
// below 2^-49); rounded to an integer once.  64-bit floats: d in 32 loses x's last bits, and z's fraction needs 44 of them.
struct SampleWeight {
    float max;
    double rate;                           // 128 / (T ln 2)
    const double* table;
    __device__ __forceinline__ uint64_t operator()(float x) const
    {
        if (x == max) return 1ull << ST_FIX;           // infinities among them
        const double z = ((double)max - (double)x) * rate;
        if (!(z < 128.0 * (ST_FIX + 2))) return 0;
        const double n = rint(z), r = (z - n) * -0.0054152123481245726;        // -ln 2 / 128
        const double e = fma(fma(fma(fma(r, 1.0 / 24, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0);
        const int i = (int)n;
        const double w = e * table[i & (ST_TABLE - 1)];        // (1/2, 1], or an ulp above
        return (uint64_t)__double2ll_rn(__longlong_as_double(__double_as_longlong(w) + ((long long)(ST_FIX - (i >> 7)) << 52)));
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

__device__ __forceinline__ bool st_better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

template <typename T>
struct SampleRow {
    const SampleArgs& p;
    SampleShared& s;
    const T* vals;                         // this CTA's tokens
    int n, first;                          // how many, and the first's index
    cg::cluster_group cl;
    int rank, ranks;

    // Clears the histogram, lets f(x) name each token's bin (negative: none) and adds it up, by weight too where `mass`.
    template <typename F>
    __device__ void histogram(bool mass, const SampleWeight& weight, F f)
    {
        for (int i = threadIdx.x; i < ST_BINS; i += ST_THREADS) { s.count[i] = 0; s.lo[i] = 0; s.hi[i] = 0; }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += ST_THREADS) {
            const float x = st_value(vals[i]);
            const int bin = f(x);
            if (bin < 0) continue;
            atomicAdd(&s.count[bin], 1u);
            if (mass) {
                // a 64-bit sum in two words: the lower word's carry goes to the upper
                const uint64_t w = weight(x);
                const uint32_t lo = (uint32_t)w;
                uint32_t hi = (uint32_t)(w >> 32);
                if (lo != 0 && atomicAdd(&s.lo[bin], lo) + lo < lo) hi++;
                if (hi != 0) atomicAdd(&s.hi[bin], hi);
            }
        }
        cl.sync();
    }
    // The bin in which the sums over the cluster's histograms reach `target` (1 to the whole sum), the same in every CTA.
    __device__ SampleFound find(bool mass, uint64_t target)
    {
        const int bins = ST_BINS / ranks, per = bins < ST_THREADS ? 1 : bins / ST_THREADS, at = rank * bins + threadIdx.x * per;
        const bool active = (int)threadIdx.x * per < bins;
        uint64_t mine[4], sum = 0;
        uint32_t counts[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            mine[i] = 0;
            counts[i] = 0;
            if (active && i < per) {
                for (int r = 0; r < ranks; r++) {
                    const SampleShared* o = cl.map_shared_rank(&s, r);
                    counts[i] += o->count[at + i];
                    if (mass) mine[i] += o->lo[at + i] + ((uint64_t)o->hi[at + i] << 32);
                }
                if (!mass) mine[i] = counts[i];
                sum += mine[i];
            }
        }
        uint64_t total;
        uint64_t before = st_scan(sum, s.scan, total);
        if ((int)threadIdx.x < ranks) cl.map_shared_rank(&s, threadIdx.x)->part[rank] = total;
        cl.sync();
        for (int r = 0; r < rank; r++) before += s.part[r];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (active && i < per && before < target && target <= before + mine[i])
                for (int r = 0; r < ranks; r++) cl.map_shared_rank(&s, r)->found = SampleFound{at + i, counts[i], before};
            before += mine[i];
        }
        cl.sync();
        return s.found;
    }
    // The key at which the tokens before it and `target` of its own (by count or by mass) make up `target`, among keys below `limit`; before: their sum.
    __device__ uint32_t select(bool mass, uint64_t target, uint32_t limit, const SampleWeight& weight, float scale, uint64_t& before)
    {
        const float max = weight.max;
        auto coarse = [&](float x) {
            const float d = x == max ? 0.0f : max - x;
            return (int)fminf(d * scale, (float)(ST_BINS - 1));
        };
        histogram(mass, weight, [&](float x) { return st_key(x) < limit ? coarse(x) : -1; });
        SampleFound f = find(mass, target);
        before = f.before;
        const int bin = f.bin;
        if (!mass && bin == ST_BINS - 1) return ST_NO_CUT;      // weights of 2^-44 and less
        uint32_t prefix = 0;
#pragma unroll 1
        for (int level = 0; level < 3; level++) {
            const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
            histogram(mass, weight, [&](float x) {
                const uint32_t k = st_key(x);
                if (k >= limit || coarse(x) != bin || (level > 0 && (k >> (shift + bits)) != prefix)) return -1;
                return (int)((k >> shift) & ((1u << bits) - 1));
            });
            f = find(mass, target - before);
            before += f.before;
            prefix = (prefix << bits) | (uint32_t)f.bin;
        }
        return prefix;
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
    const int rank = (int)cl.block_rank(), ranks = (int)cl.num_blocks();
    const int row = blockIdx.x / ranks, tid = threadIdx.x;
    const int first = min(rank * p.each, p.vocab), n = min(p.each, p.vocab - first);
    const T* src = reinterpret_cast<const T*>(p.x) + row * p.row_stride + first;
    // the row lies in shared memory as it lies in global memory, modulo 16 bytes
    constexpr int VEC = 16 / sizeof(T);
    const int skew = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    T* vals = reinterpret_cast<T*>(st_smem + sizeof(SampleShared)) + skew;
    for (int i = tid; i < ST_TABLE; i += ST_THREADS) s.table[i] = exp2(-(double)i / ST_TABLE);

    float best = -INFINITY;
    int best_at = p.vocab;
    auto take = [&](T raw, int i) {
        const float v = st_value(raw);
        if (v > best) { best = v; best_at = first + i; }
    };
    const int head = min(n, skew == 0 ? 0 : VEC - skew), vecs = (n - head) / VEC, tail = head + vecs * VEC;
    if (tid < head) { vals[tid] = src[tid]; take(src[tid], tid); }
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
                    to[at + u * ST_THREADS] = v[u];
                    const T* e = reinterpret_cast<const T*>(&v[u]);
#pragma unroll
                    for (int i = 0; i < VEC; i++) take(e[i], head + (at + u * ST_THREADS) * VEC + i);
                }
        }
    }
    if (tail + tid < n) { vals[tail + tid] = src[tail + tid]; take(src[tail + tid], tail + tid); }

    // ---- the first maximum
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, best, o);
        const int i = __shfl_xor_sync(0xffffffffu, best_at, o);
        if (st_better(v, i, best, best_at)) { best = v; best_at = i; }
    }
    if ((tid & 31) == 0) { s.red[tid >> 5] = best; s.red_at[tid >> 5] = best_at; }
    __syncthreads();
    if (tid < ranks) {
        for (int w = 0; w < ST_THREADS / 32; w++)
            if (w == 0 || st_better(s.red[w], s.red_at[w], best, best_at)) { best = s.red[w]; best_at = s.red_at[w]; }
        SampleShared* o = cl.map_shared_rank(&s, tid);
        o->max[rank] = best;
        o->max_at[rank] = best_at;
    }
    cl.sync();
    float max = s.max[0];
    int max_at = s.max_at[0];
    for (int r = 1; r < ranks; r++)
        if (st_better(s.max[r], s.max_at[r], max, max_at)) { max = s.max[r]; max_at = s.max_at[r]; }

    const float temperature = p.temperature != nullptr ? p.temperature[row] : 1.0f;
    int k = p.top_k != nullptr ? p.top_k[row] : 0;
    const float top_p = p.top_p != nullptr ? p.top_p[row] : 1.0f, min_p = p.min_p != nullptr ? p.min_p[row] : 0.0f;
    if (k <= 0 || k > p.vocab) k = p.vocab;
    // greedily, or nothing to choose from: every CTA sees the same and leaves
    if (max == -INFINITY || !(temperature > 0.0f) || k == 1) {
        if (rank == 0 && tid == 0) {
            p.ids[row] = max == -INFINITY ? -1 : max_at;
            if (p.probs != nullptr) p.probs[row] = max == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }
    const SampleWeight weight{max, 184.6649652337873 / (double)temperature, s.table};       // 128 / ln 2
    const float scale = fminf(64.0f / temperature, 1e30f);
    SampleRow<T> me{p, s, vals, n, first, cl, rank, ranks};

    // ---- cutoffs: kept are keys below `cut`, and the first `ties` tokens of key `cut`
    uint32_t cut = ST_NO_CUT, ties = 0;
    uint64_t tie_weight = 0;
    auto mass_below = [&](uint32_t limit) {
        uint64_t sum = 0, total;
        for (int i = tid; i < n; i += ST_THREADS) {
            const float x = st_value(vals[i]);
            if (st_key(x) < limit) sum += weight(x);
        }
        st_scan(sum, s.scan2, total);
        if (tid < ranks) cl.map_shared_rank(&s, tid)->mass[rank] = total;
        cl.sync();
        total = 0;
        for (int r = 0; r < ranks; r++) total += s.mass[r];
        return total;
    };
    auto key_weight = [&](uint32_t key) { return weight(__uint_as_float((key >> 31) ? key : ~key ^ 0x80000000u)); };
    if (k < p.vocab) {
        uint64_t before;
        cut = me.select(false, (uint64_t)k, ST_NO_CUT, weight, scale, before);
        if (cut != ST_NO_CUT) {
            ties = (uint32_t)(k - before);
            tie_weight = key_weight(cut);
        }
    }
    if (top_p < 1.0f) {
        const uint64_t above = mass_below(cut), all = above + ties * tie_weight;
        uint64_t target = top_p > 0.0f ? (uint64_t)ceil((double)top_p * (double)all) : 1;
        if (target == 0) target = 1;
        uint64_t before = above;
        if (target <= above) {
            cut = me.select(true, target, cut, weight, scale, before);
            tie_weight = key_weight(cut);
            ties = 0xFFFFFFFFu;
        }
        // the fewest tokens of the cutoff's weight that reach the target
        if (tie_weight != 0) ties = (uint32_t)min((uint64_t)ties, (target - before + tie_weight - 1) / tie_weight);
    }
    uint64_t least = 0;
    if (min_p > 0.0f) least = (uint64_t)ceil((double)fminf(min_p, 1.0f) * (double)(1ull << ST_FIX));
    if (tie_weight < least) ties = 0;

    // ---- the draw: runs of neighbouring tokens, one a thread, in the vocabulary's order
    const int seg = (p.each + ST_THREADS - 1) / ST_THREADS | 1, j0 = min(tid * seg, n), j1 = min(j0 + seg, n);
    uint64_t sum = 0, tie_count = 0;
    for (int j = j0; j < j1; j++) {
        const float x = st_value(vals[j]);
        const uint32_t key = st_key(x);
        if (key < cut) {
            const uint64_t w = weight(x);
            if (w >= least) sum += w;
        } else if (key == cut) {
            tie_count++;
        }
    }
    uint64_t all_sum, all_ties;
    __syncthreads();
    uint64_t before = st_scan(sum, s.scan, all_sum), ties_before = st_scan(tie_count, s.scan2, all_ties);
    if (tid < ranks) {
        SampleShared* o = cl.map_shared_rank(&s, tid);
        o->part[rank] = all_sum;
        o->ties[rank] = all_ties;
    }
    cl.sync();
    all_sum = 0;
    all_ties = 0;
    for (int r = 0; r < ranks; r++) {
        if (r < rank) { before += s.part[r]; ties_before += s.ties[r]; }
        all_sum += s.part[r];
        all_ties += s.ties[r];
    }
    const uint64_t kept_ties = ties;
    const uint64_t total = all_sum + min(all_ties, kept_ties) * tie_weight;
    const float u = p.u[row];
    // a running sum exceeds u * total where it exceeds that number's floor
    uint64_t target = u < 1.0f ? (u > 0.0f ? (uint64_t)((double)u * (double)total) : 0) : total - 1;
    if (target >= total) target = total - 1;
    uint64_t run = before + min(ties_before, kept_ties) * tie_weight;
    const uint64_t after = run + sum + (min(ties_before + tie_count, kept_ties) - min(ties_before, kept_ties)) * tie_weight;
    if (run <= target && target < after) {
        uint64_t tie = ties_before;
        for (int j = j0; j < j1; j++) {
            const float x = st_value(vals[j]);
            const uint32_t key = st_key(x);
            uint64_t w = 0;
            if (key < cut) {
                w = weight(x);
                if (w < least) w = 0;
            } else if (key == cut) {
                if (tie < kept_ties) w = tie_weight;
                tie++;
            }
            run += w;
            if (run > target) {
                p.ids[row] = first + j;
                if (p.probs != nullptr) p.probs[row] = (float)((double)w / (double)total);
                break;
            }
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
    // CTAs a row: until the SMs are full or a thread has few tokens left, and as many as its shared memory takes
    int ranks = 1;
    auto each = [&](int r) { return ((vocab + r - 1) / r + 7) / 8 * 8; };
    while (ranks < ST_MAX_CLUSTER && (each(ranks) > most_each || ((int64_t)rows * ranks < d->sm_count && each(ranks) > 8 * ST_THREADS))) ranks *= 2;
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
