// Rotary positions: the leading columns of every query and key head are turned, pair by pair, by an angle that grows with the token's
// position -- as rows of a matrix (ns_rotary), and on the way from the fused projection into the pages of a key/value cache
// (ns_kv_append_rotary).  No counterpart in the reference, whose positions are a table added to the embedding (Layers/Attention.cs:236-269).
//
//   (a, b) <- amplitude (a cos t - b sin t, a sin t + b cos t),  t = position * freq[pair]
//
// The pairs are neighbouring columns or column p of the first half and column p of the second.  t is formed and reduced in 64 bits: a float
// product of a position of 500 000 is off by up to 0.02 radians.  What a row's heads share, the cosines and sines of its position, is computed once
// for each row into shared memory, while the row's first columns are on their way.  Both kernels move each byte once and are bound by
// that (8192 rows of 40 heads x 128 bf16, 168 MB: see the launch).
#include <type_traits>

#include "ns_cache.cuh"
#include "ns_mma.cuh"
#include "ns_seq.cuh"

namespace {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_DIM = 4096;
constexpr int ROT_MAX_COLUMNS = 1 << 19;

// amplitude * (cos, sin) of position * freq.  The angle in turns, reduced to half a turn either way, in 64 bits; its doubled value as a float and the
// rest of it, which moves the result along its derivative: within an ulp or two of the exact value.
__device__ __forceinline__ float2 rot_cos_sin(double position, float freq, float amplitude, float sign = 1.0f)
{
    double turns = position * (double)freq * 0.15915494309189535;
    turns -= rint(turns);
    const double twice = turns + turns;
    const float hi = (float)twice, lo = (float)(twice - (double)hi) * 3.14159274f;
    float s, c;
    sincospif(hi, &s, &c);
    return make_float2(amplitude * fmaf(-lo, s, c), sign * amplitude * fmaf(lo, c, s));
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
    T v[VEC];
};

template <int VEC>
__device__ __forceinline__ void rot_unpack(const RotVec<float, VEC>& x, float (&f)[VEC])
{
#pragma unroll
    for (int i = 0; i < VEC; i++) f[i] = x.v[i];
}
template <int VEC>
__device__ __forceinline__ void rot_unpack(const RotVec<uint16_t, VEC>& x, float (&f)[VEC])
{
    if constexpr (VEC == 1) {
        f[0] = ns_bf16_bits_to_f32(x.v[0]);
    } else {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
}
template <int VEC>
__device__ __forceinline__ void rot_pack(RotVec<float, VEC>& x, const float (&f)[VEC])
{
#pragma unroll
    for (int i = 0; i < VEC; i++) x.v[i] = f[i];
}
template <int VEC>
__device__ __forceinline__ void rot_pack(RotVec<uint16_t, VEC>& x, const float (&f)[VEC])
{
    if constexpr (VEC == 1) {
        x.v[0] = ns_f32_to_bf16_bits(f[0]);
    } else {
        uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) w[i] = ns_pack_bf16x2(f[2 * i], f[2 * i + 1]);
    }
}

// How a head's columns are dealt out.  A task turns PAIRS neighbouring pairs: VEC neighbouring columns of each half, VEC neighbouring columns that hold VEC / 2
// pairs (the last task may hold columns behind the turned ones), or, column by column, one pair.  The columns from `rest` on are copied.
template <bool HALVES, int VEC>
struct RotTasks {
    static constexpr int PAIRS = HALVES || VEC == 1 ? VEC : VEC / 2;
    static constexpr bool TWO = HALVES || VEC == 1;                       // two vectors a task
    int half, turned, rest;
    __host__ __device__ RotTasks(int dim, int rot) : half(rot / 2), turned((rot / 2 + PAIRS - 1) / PAIRS), rest(TWO ? rot : turned * VEC) {}
    __device__ __forceinline__ int first(int t) const { return HALVES ? t * VEC : t * (VEC == 1 ? 2 : VEC); }
    __device__ __forceinline__ int second() const { return HALVES ? half : 1; }      // from the first vector's column to the second's
    // Where a row's cosine and sine of pair p lie: neighbouring tasks' side by side, so that neighbouring threads read them without conflicts.
    __host__ __device__ int table() const { return PAIRS * turned; }
    __device__ __forceinline__ int slot(int p) const { return p % PAIRS * turned + p / PAIRS; }
    __device__ __forceinline__ void angles(const float2* row, int t, float2 (&w)[PAIRS]) const
    {
#pragma unroll
        for (int i = 0; i < PAIRS; i++) w[i] = row[i * turned + t];
    }
    // the columns of task t in 32 bits
    __device__ __forceinline__ void turn(int t, const float2 (&w)[PAIRS], float (&a)[VEC], float (&b)[VEC]) const
    {
        const int live = half - t * PAIRS;
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            float& x = TWO ? a[i] : a[(2 * i) % VEC];
            float& y = TWO ? b[i] : a[(2 * i + 1) % VEC];
            const float u = x, v = y;
            if (TWO || i < live) {
                x = fmaf(u, w[i].x, -(v * w[i].y));
                y = fmaf(u, w[i].y, v * w[i].x);
            }
        }
    }
};

// How a CTA's threads are dealt out: `tasks` threads a head, `heads` of them at a time, `rows` of those; a thread keeps its pairs' cosines and sines in registers
// and walks heads.
struct RotLanes {
    int tasks, heads, rows;
};
RotLanes rot_lanes(const NsDevice* d, int64_t rows, int heads, int turned, int table, int columns)
{
    RotLanes best{turned < ROT_THREADS ? turned : ROT_THREADS, 1, 1};
    const int slots = ROT_THREADS / best.tasks;
    // few rows: all heads at once.  Else the fewest idle threads, with four to eight heads a thread where that is level.
    if (rows < 2 * d->sm_count) {
        best.heads = heads < slots ? heads : slots;
        return best;
    }
    double most = 0.0;
    for (int h = 1; h <= slots && h <= heads; h++) {
        int r = slots / h;
        if ((int64_t)r * table > 2048) r = 2048 / table > 1 ? 2048 / table : 1;
        if (r > (1 << 16) / columns) r = (1 << 16) / columns > 1 ? (1 << 16) / columns : 1;       // (RotDiv)
        if (r > rows / (4 * d->sm_count)) r = (int)(rows / (4 * d->sm_count));
        if (r < 1) r = 1;
        const int walk = (heads + h - 1) / h;
        const double busy = (double)r * heads * best.tasks / ((double)walk * ROT_THREADS) * (walk < 4 ? 0.8 + 0.05 * walk : walk > 8 ? 0.9 : 1.0);
        if (busy > most) { most = busy; best.heads = h; best.rows = r; }
    }
    return best;
}

// n / d, exact while n * d < 2^32 (m d - 2^32 < d)
struct RotDiv {
    uint32_t d, m;
    explicit RotDiv(int divisor = 0) : d((uint32_t)divisor), m(divisor > 1 ? (uint32_t)(((1ull << 32) + divisor - 1) / divisor) : 0u) {}
    __device__ __forceinline__ int of(int n) const { return d == 1 ? n : (int)__umulhi((uint32_t)n, m); }
};

// ---------------------------------------------------------------------------------------------
// rows of a matrix
// ---------------------------------------------------------------------------------------------
struct RotaryArgs {
    const void* x;
    void* y;
    int x_ld, x_head, y_ld, y_head;
    const int32_t* pos;
    const float* freq;
    float amplitude, sign;
    int64_t rows;
    int dim, rot;
    int copies;            // y is another matrix: the columns that are not turned are copied
    int heads, heads_each; // heads a CTA takes of its rows (blockIdx.y)
    RotLanes lanes;
    RotDiv half, rest, rest_row;         // pairs of a row, vectors of a head and of a row that are copied
};

// A CTA takes a few rows: their first columns are asked for, the cosines and sines of all the rows computed meanwhile, one or two a thread, and then
// the rows' heads stream through.
template <typename T, bool HALVES, int VEC>
__global__ void __launch_bounds__(ROT_THREADS, 4) ns_rotary_kernel(const RotaryArgs p)
{
    using V = RotVec<T, VEC>;
    using N = RotTasks<HALVES, VEC>;
    constexpr int U = N::TWO ? 2 : 4;          // heads a thread has on their way
    extern __shared__ float2 rot_table[];
    ns_pdl_wait();
    ns_pdl_trigger();
    const N n(p.dim, p.rot);
    const int half = p.rot / 2, h0 = blockIdx.y * p.heads_each, heads = min(p.heads_each, p.heads - h0);
    const int slot = threadIdx.x / p.lanes.tasks, t0 = threadIdx.x - slot * p.lanes.tasks, my_row = slot / p.lanes.heads, my_head = slot - my_row * p.lanes.heads;
    for (int64_t r0 = (int64_t)blockIdx.x * p.lanes.rows; r0 < p.rows; r0 += (int64_t)gridDim.x * p.lanes.rows) {
        const int rows = (int)min((int64_t)p.lanes.rows, p.rows - r0);
        const int32_t* pos = p.pos + r0;
        const T* x0 = reinterpret_cast<const T*>(p.x) + r0 * p.x_ld + (int64_t)h0 * p.x_head;
        T* y0 = reinterpret_cast<T*>(p.y) + r0 * p.y_ld + (int64_t)h0 * p.y_head;
        const T* x = x0 + (int64_t)my_row * p.x_ld;
        T* y = y0 + (int64_t)my_row * p.y_ld;
        const bool mine = my_row < rows;
        V a[U], b[U];
        auto load = [&](int t, int h) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int head = h + u * p.lanes.heads;
                if (head < heads) {
                    const T* src = x + (int64_t)head * p.x_head + n.first(t);
                    a[u] = *reinterpret_cast<const V*>(src);
                    if (N::TWO) b[u] = *reinterpret_cast<const V*>(src + n.second());
                }
            }
        };
        if (mine) load(t0, my_head);
        if (p.copies != 0 && n.rest < p.dim) {
            const int per_head = (p.dim - n.rest) / VEC, per_row = heads * per_head;
            constexpr int C = 4;
            for (int e = threadIdx.x; e < rows * per_row; e += C * ROT_THREADS) {
                V v[C];
                T* to[C];
#pragma unroll
                for (int u = 0; u < C; u++) {
                    const int i = e + u * ROT_THREADS, r = rows == 1 ? 0 : p.rest_row.of(i), in = i - r * per_row, head = p.rest.of(in);
                    const int c = n.rest + (in - head * per_head) * VEC;
                    to[u] = nullptr;
                    if (i < rows * per_row && pos[r] >= 0) {
                        v[u] = *reinterpret_cast<const V*>(x0 + (int64_t)r * p.x_ld + (int64_t)head * p.x_head + c);
                        to[u] = y0 + (int64_t)r * p.y_ld + (int64_t)head * p.y_head + c;
                    }
                }
#pragma unroll
                for (int u = 0; u < C; u++)
                    if (to[u] != nullptr) *reinterpret_cast<V*>(to[u]) = v[u];
            }
        }
        __syncthreads();                       // the rows before have been turned
        for (int i = threadIdx.x; i < rows * half; i += ROT_THREADS) {
            const int r = p.half.of(i), pair = i - r * half;
            rot_table[r * n.table() + n.slot(pair)] = rot_cos_sin((double)pos[r], p.freq[pair], p.amplitude, p.sign);
        }
        __syncthreads();
        if (mine && pos[my_row] >= 0) {
            for (int t = t0; t < n.turned; t += p.lanes.tasks) {
                float2 w[N::PAIRS];
                n.angles(rot_table + my_row * n.table(), t, w);
                if (t != t0) load(t, my_head);
                for (int h = my_head; h < heads; h += U * p.lanes.heads) {
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const int head = h + u * p.lanes.heads;
                        if (head < heads) {
                            float fa[VEC], fb[VEC];
                            rot_unpack(a[u], fa);
                            if (N::TWO) rot_unpack(b[u], fb);
                            n.turn(t, w, fa, fb);
                            V o;
                            T* dst = y + (int64_t)head * p.y_head + n.first(t);
                            rot_pack(o, fa);
                            *reinterpret_cast<V*>(dst) = o;
                            if (N::TWO) {
                                rot_pack(o, fb);
                                *reinterpret_cast<V*>(dst + n.second()) = o;
                            }
                        }
                    }
                    load(t, h + U * p.lanes.heads);
                }
            }
        }
    }
}

// The widest vector that divides the half (or, for neighbours, the head) and that every row starts on.
int rot_vector(int most, bool halves, int dim, int rot, uint64_t addresses, int64_t strides)
{
    int v = most;
    const int width = halves ? (rot / 2) | (dim - rot) : dim;
    const int size = 16 / most;
    while (v > 1 && ((width | strides) % v != 0 || (addresses & (uint64_t)(v * size - 1)) != 0)) v >>= 1;
    return v;
}

template <typename F>
int rot_pick(bool halves, int vec, F f)
{
    auto by = [&](auto h) {
        switch (vec) {
            case 8: return f(h, std::integral_constant<int, 8>());
            case 4: return f(h, std::integral_constant<int, 4>());
            case 2: return f(h, std::integral_constant<int, 2>());
            default: return f(h, std::integral_constant<int, 1>());
        }
    };
    return halves ? by(std::true_type()) : by(std::false_type());
}

// ---------------------------------------------------------------------------------------------
// into the cache
// ---------------------------------------------------------------------------------------------
struct AppendArgs {
    NsSource src;
    int q_col, k_col, v_col, heads, kv_heads, dim, rot;
    const float* freq;
    float amplitude;
    const int32_t* offset;      // one word, or null
    const int32_t* pos;         // [batch]
    const int32_t* lens;        // [batch], or null
    const int32_t* page_table;
    int max_pages, page_shift, num_pages;
    int batch, steps;
    uint16_t* q;
    int64_t q_ld;
    uint16_t* k_pool;
    uint16_t* v_pool;
    int lane_tasks;                        // lanes a head, at most 32
    int parts, heads_each;                 // warps a row, and heads of each
    int stage_at;                          // bytes: where the warps' source heads lie in shared memory, behind their angles
    RotDiv rest, value;                    // vectors of a head that are not turned, and of a value head
    int* status;
};

// VEC neighbouring values of the source as they are held until they are used: bf16 as it lies there, float slabs as their sum.
constexpr int ROT_BF16 = -1;               // in place of a number of slabs
template <int VEC, int SLABS>
using RotHeld = typename std::conditional<SLABS == ROT_BF16, RotVec<uint16_t, VEC>, RotVec<float, VEC>>::type;
template <int VEC, int SLABS>
__device__ __forceinline__ void rot_source(const NsSource& s, int64_t idx, RotHeld<VEC, SLABS>& v)
{
    if constexpr (SLABS == ROT_BF16) {
        v = *reinterpret_cast<const RotVec<uint16_t, VEC>*>(reinterpret_cast<const uint16_t*>(s.ptr) + idx);
    } else if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 f = ns_source_at4<SLABS>(s, idx + i);
            v.v[i] = f.x; v.v[i + 1] = f.y; v.v[i + 2] = f.z; v.v[i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v.v[i] = ns_source_at<SLABS>(s, idx + i);
    }
}
template <int VEC>
__device__ __forceinline__ void rot_store(uint16_t* dst, const RotVec<uint16_t, VEC>& v) { *reinterpret_cast<RotVec<uint16_t, VEC>*>(dst) = v; }
template <int VEC>
__device__ __forceinline__ void rot_store(uint16_t* dst, const RotVec<float, VEC>& v)
{
    RotVec<uint16_t, VEC> o;
    rot_pack(o, v.v);
    rot_store<VEC>(dst, o);
}

// A warp a row, or several, each with a range of its heads (queries, keys, values); no barrier joins them.  What a token's place and angles come from is a chain of
// three loads (position, page, data), so what counts is that many bytes are on their way: a bf16 source's heads all at once, through shared memory.  (Through registers,
// four vectors a lane at a time, 13 x 777 tokens of 48 heads x 128 took 42 us, with two warps a row 34; so they take 26, 4.7 TB/s.)
template <bool HALVES, int VEC, int SLABS>
__global__ void __launch_bounds__(ROT_THREADS, SLABS == NS_TOGETHER ? 1 : SLABS == ROT_BF16 ? 4 : 3) ns_kv_append_rotary_kernel(const AppendArgs p)
{
    using N = RotTasks<HALVES, VEC>;
    using H = RotHeld<VEC, SLABS>;
    constexpr bool STAGED = SLABS == ROT_BF16 && VEC == 8;
    constexpr int U = SLABS == NS_TOGETHER ? 1 : SLABS == ROT_BF16 && !N::TWO ? 4 : 2;      // heads a lane has on their way
    constexpr int K = SLABS == NS_TOGETHER ? 1 : SLABS == ROT_BF16 ? 4 : 2;                 // vectors to copy
    extern __shared__ __align__(16) uint8_t rot_smem[];
    ns_pdl_wait();
    ns_pdl_trigger();
    const N n(p.dim, p.rot);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = p.rot / 2;
    const int item = blockIdx.x * (ROT_THREADS / 32) + warp, r = item / p.parts, part = item - r * p.parts;
    if (r >= p.batch * p.steps) return;
    const int b = r / p.steps, i = r - b * p.steps;
    const int first_pos = p.pos[b], offset = p.offset != nullptr ? p.offset[0] : 0;
    if (p.lens != nullptr && i >= p.lens[b]) return;
    // this warp's heads: turned ones below `all_heads`, values behind
    const int all_heads = p.heads + p.kv_heads, head0 = part * p.heads_each, head1 = min(head0 + p.heads_each, all_heads + p.kv_heads);
    const int64_t src0 = (int64_t)r * p.src.ld, head_step = (int64_t)p.dim << p.page_shift;
    auto column = [&](int head) {
        return head < p.heads ? p.q_col + head * p.dim : head < all_heads ? p.k_col + (head - p.heads) * p.dim : p.v_col + (head - all_heads) * p.dim;
    };
    float2* table = reinterpret_cast<float2*>(rot_smem) + warp * n.table();
    const uint16_t* staged = reinterpret_cast<const uint16_t*>(rot_smem + p.stage_at) + warp * p.heads_each * p.dim;
    if constexpr (STAGED) {
        const int per = p.dim / 8, total = (head1 - head0) * per;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(p.src.ptr) + src0;
        for (int e = lane; e < total; e += 32) {
            const int head = p.value.of(e), c = (e - head * per) * 8;
            ns_cp_async16(ns_smem_u32(staged + head * p.dim + c), src + column(head0 + head) + c);
        }
        ns_cp_commit();
    }
    // positions in 64 bits: nothing wraps around
    const int64_t at = (int64_t)first_pos + i;
    int page = -1;
    if (at >= 0 && (at >> p.page_shift) < p.max_pages) page = p.page_table[(int64_t)b * p.max_pages + (at >> p.page_shift)];
    auto read = [&](int head, int c, H& v) {
        if constexpr (STAGED) v = *reinterpret_cast<const H*>(staged + (head - head0) * p.dim + c);
        else rot_source<VEC, SLABS>(p.src, src0 + column(head) + c, v);
    };

    // ---- turned heads: lanes of a head, heads side by side
    const int across = 32 / p.lane_tasks, t0 = lane % p.lane_tasks, sub = lane / p.lane_tasks;
    H x[U], y[U];
    auto load = [&](int t, int h) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (h + u * across < min(head1, all_heads)) {
                read(h + u * across, n.first(t), x[u]);
                if (N::TWO) read(h + u * across, n.first(t) + n.second(), y[u]);
            }
    };
    const bool mine = sub < across;
    const int h0 = head0 + sub;
    if (!STAGED && mine) load(t0, h0);
    if (head0 < all_heads)
        for (int e = lane; e < half; e += 32) table[n.slot(e)] = rot_cos_sin((double)(at + offset), p.freq[e], p.amplitude);
    if constexpr (STAGED) ns_cp_wait<0>();
    __syncwarp();
    const bool stored = page >= 0 && page < p.num_pages;
    if (!stored && lane == 0) *reinterpret_cast<volatile int*>(p.status) = 500;
    const int64_t slab = (((int64_t)page * p.kv_heads << p.page_shift) + (at & ((1 << p.page_shift) - 1))) * p.dim;      // head 0's row in the page
    auto target = [&](int head) {
        return head < p.heads ? p.q + (int64_t)r * p.q_ld + (int64_t)head * p.dim
                              : (head < all_heads ? p.k_pool + (int64_t)(head - p.heads) * head_step : p.v_pool + (int64_t)(head - all_heads) * head_step) + slab;
    };
    const int end = min(head1, stored ? all_heads : p.heads);
    if (mine) {
        for (int t = t0; t < n.turned; t += p.lane_tasks) {
            float2 w[N::PAIRS];
            n.angles(table, t, w);
            if (STAGED || t != t0) load(t, h0);
            for (int h = h0; h < end; h += U * across) {
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (h + u * across < end) {
                        uint16_t* dst = target(h + u * across) + n.first(t);
                        float fa[VEC], fb[VEC];
                        rot_unpack(x[u], fa);
                        if (N::TWO) rot_unpack(y[u], fb);
                        n.turn(t, w, fa, fb);
                        RotVec<uint16_t, VEC> o;
                        rot_pack(o, fa);
                        rot_store<VEC>(dst, o);
                        if (N::TWO) {
                            rot_pack(o, fb);
                            rot_store<VEC>(dst + n.second(), o);
                        }
                    }
                load(t, h + U * across);
            }
        }
    }
    // ---- what is not turned of those heads, and the values
    H v[K];
    auto copy = [&](int count, auto where) {
        for (int e = lane; e < count; e += K * 32) {
            uint16_t* to[K];
#pragma unroll
            for (int u = 0; u < K; u++)
                if (e + u * 32 < count) {
                    int c;
                    const int head = where(e + u * 32, c);
                    read(head, c, v[u]);
                    to[u] = target(head) + c;
                }
#pragma unroll
            for (int u = 0; u < K; u++)
                if (e + u * 32 < count) rot_store<VEC>(to[u], v[u]);
        }
    };
    const int rest = (p.dim - n.rest) / VEC;
    copy(max(end - head0, 0) * rest, [&](int e, int& c) {
        const int head = p.rest.of(e);
        c = n.rest + (e - head * rest) * VEC;
        return head0 + head;
    });
    const int per = p.dim / VEC, value0 = max(head0, all_heads);
    copy(stored ? max(head1 - value0, 0) * per : 0, [&](int e, int& c) {
        const int head = p.value.of(e);
        c = (e - head * per) * VEC;
        return value0 + head;
    });
}

bool rot_layout(int layout) { return layout == NS_ROTARY_PAIRS || layout == NS_ROTARY_HALVES; }

}  // namespace

extern "C" int ns_rotary(ns_device_t h, uint64_t x, int dtype, int64_t x_ld, int64_t x_head, uint64_t pos, uint64_t freq, float amplitude, int layout, int inverse,
                         int64_t rows, int heads, int dim, int rot_dims, uint64_t y, int64_t y_ld, int64_t y_head)
{
    NS_REQUIRE(x && y && pos && freq, NS_ERR_ARGUMENT, "ns_rotary: null argument");
    NS_REQUIRE(dtype == NS_F32 || dtype == NS_BF16, NS_ERR_ARGUMENT, "ns_rotary: dtype must be NS_F32 or NS_BF16");
    NS_REQUIRE(rot_layout(layout), NS_ERR_ARGUMENT, "ns_rotary: unknown layout %d", layout);
    NS_REQUIRE(rows >= 0 && heads > 0 && dim > 0 && dim <= ROT_MAX_DIM, NS_ERR_ARGUMENT, "ns_rotary: bad shape (heads of 1 to %d columns)", ROT_MAX_DIM);
    NS_REQUIRE(rot_dims >= 2 && rot_dims <= dim && rot_dims % 2 == 0, NS_ERR_ARGUMENT, "ns_rotary: rot_dims must be even, 2 to %d (got %d)", dim, rot_dims);
    NS_REQUIRE(((pos | freq) & 3) == 0, NS_ERR_ARGUMENT, "ns_rotary: pos and freq must be 4-byte aligned");
    const int size = dtype == NS_F32 ? 4 : 2;
    NS_REQUIRE(((x | y) & (uint64_t)(size - 1)) == 0, NS_ERR_ARGUMENT, "ns_rotary: rows must be aligned to their type");
    NS_REQUIRE((int64_t)heads * dim <= ROT_MAX_COLUMNS, NS_ERR_ARGUMENT, "ns_rotary: at most 2^19 columns a row");
    // no two (row, head) of the output share a column: heads inside rows, or rows inside heads
    auto apart = [&](int64_t inner, int64_t n_inner, int64_t outer, int64_t n_outer) {
        const bool in = n_inner == 1 || inner >= dim;
        return in && (n_outer == 1 || (outer >= dim && (n_inner == 1 || (outer - dim) / inner >= n_inner - 1)));
    };
    NS_REQUIRE(x_ld >= 0 && x_head >= 0 && y_ld >= 0 && y_head >= 0, NS_ERR_ARGUMENT, "ns_rotary: negative pitch");
    NS_REQUIRE(x_ld < (1LL << 31) && x_head < (1LL << 31) && y_ld < (1LL << 31) && y_head < (1LL << 31), NS_ERR_ARGUMENT, "ns_rotary: a pitch of 2^31 elements or more");
    NS_REQUIRE(apart(y_head, heads, y_ld, rows) || apart(y_ld, rows, y_head, heads), NS_ERR_ARGUMENT, "ns_rotary: rows or heads of the output overlap");
    NS_REQUIRE(x != y || (x_ld == y_ld && x_head == y_head), NS_ERR_ARGUMENT, "ns_rotary: in place, both pitches have to be the input's");
    NsDevice* d = ns_dev(h);
    int rc = ns_device_make_current(d);
    if (rc != NS_OK) return rc;
    if (rows == 0) return NS_OK;
    RotaryArgs p;
    p.x = reinterpret_cast<const void*>(x); p.y = reinterpret_cast<void*>(y);
    p.x_ld = (int)x_ld; p.x_head = (int)x_head; p.y_ld = (int)y_ld; p.y_head = (int)y_head;
    p.pos = reinterpret_cast<const int32_t*>(pos);
    p.freq = reinterpret_cast<const float*>(freq);
    p.amplitude = amplitude; p.sign = inverse ? -1.0f : 1.0f;
    p.rows = rows; p.heads = heads; p.dim = dim; p.rot = rot_dims;
    p.copies = x != y ? 1 : 0;
    const bool halves = layout == NS_ROTARY_HALVES;
    const int vec = rot_vector(16 / size, halves, dim, rot_dims, x | y, x_ld | x_head | y_ld | y_head);
    return rot_pick(halves, vec, [&](auto hv, auto vc) {
        constexpr bool HALVES = decltype(hv)::value;
        constexpr int VEC = decltype(vc)::value;
        const RotTasks<HALVES, VEC> n(dim, rot_dims);
        // few rows: their heads are spread over CTAs, a task a thread at least
        int parts = 1;
        while (parts < heads && rows * parts < d->sm_count && (int64_t)heads * n.turned > (int64_t)parts * ROT_THREADS) parts *= 2;
        p.heads_each = (heads + parts - 1) / parts;
        parts = (heads + p.heads_each - 1) / p.heads_each;
        p.lanes = rot_lanes(d, rows, p.heads_each, n.turned, n.table(), p.heads_each * dim);
        p.half = RotDiv(rot_dims / 2);
        p.rest = RotDiv((dim - n.rest) / VEC);
        p.rest_row = RotDiv(heads * ((dim - n.rest) / VEC));       // (several rows a CTA: parts is 1)
        int64_t ctas = (rows + p.lanes.rows - 1) / p.lanes.rows;
        if (ctas > (1 << 30)) ctas = 1 << 30;
        const size_t smem = (size_t)p.lanes.rows * n.table() * sizeof(float2);
        const dim3 grid((unsigned)ctas, (unsigned)parts);
        if constexpr (VEC <= 4) {
            if (size == 4) {
                NS_CUDA(ns_launch_plain(ns_rotary_kernel<float, HALVES, VEC>, grid, dim3(ROT_THREADS), smem, d->stream, p));
                return (int)NS_OK;
            }
        }
        NS_CUDA(ns_launch_plain(ns_rotary_kernel<uint16_t, HALVES, VEC>, grid, dim3(ROT_THREADS), smem, d->stream, p));
        return (int)NS_OK;
    });
}

extern "C" int ns_kv_append_rotary(ns_device_t h, ns_kv_cache_t cache, uint64_t src, int splits, int src_dtype, int src_ld, int q_col, int k_col, int v_col, int heads,
                                   uint64_t freq, float amplitude, int layout, int rot_dims, uint64_t offset, uint64_t pos, uint64_t lens, uint64_t page_table,
                                   int max_pages, int batch, int steps, uint64_t q, int64_t q_ld)
{
    NsKvCacheView c;
    int rc = ns_kv_cache_view(cache, &c);
    if (rc != NS_OK) return rc;
    NS_REQUIRE(src && freq && pos && page_table, NS_ERR_ARGUMENT, "ns_kv_append_rotary: null argument");
    NS_REQUIRE(ns_source_ok(src, splits, src_dtype), NS_ERR_ARGUMENT, "ns_kv_append_rotary: bad source");
    NS_REQUIRE(rot_layout(layout), NS_ERR_ARGUMENT, "ns_kv_append_rotary: unknown layout %d", layout);
    NS_REQUIRE(batch >= 0 && steps >= 0 && max_pages > 0 && heads >= 0 && (int64_t)batch * steps < (1LL << 30), NS_ERR_ARGUMENT, "ns_kv_append_rotary: bad shape");
    NS_REQUIRE(q == 0 || heads > 0, NS_ERR_ARGUMENT, "ns_kv_append_rotary: queries of no heads");
    const int dim = c.head_dim;
    NS_REQUIRE(rot_dims >= 2 && rot_dims <= dim && rot_dims % 2 == 0, NS_ERR_ARGUMENT, "ns_kv_append_rotary: rot_dims must be even, 2 to %d (got %d)", dim, rot_dims);
    if (q == 0) heads = 0;
    NS_REQUIRE((int64_t)(heads + 2LL * c.heads) * dim <= ROT_MAX_COLUMNS, NS_ERR_ARGUMENT, "ns_kv_append_rotary: at most 2^19 columns a row");
    NS_REQUIRE(k_col >= 0 && v_col >= 0 && (q == 0 || q_col >= 0) && (int64_t)k_col + c.heads * dim <= src_ld && (int64_t)v_col + c.heads * dim <= src_ld &&
                   (q == 0 || (int64_t)q_col + heads * dim <= src_ld),
               NS_ERR_ARGUMENT, "ns_kv_append_rotary: columns outside the source's rows");
    NS_REQUIRE(q == 0 || (q_ld >= (int64_t)heads * dim && (q & 1) == 0), NS_ERR_ARGUMENT, "ns_kv_append_rotary: query rows are shorter than their heads");
    NS_REQUIRE((src & (src_dtype == NS_F32 ? 3 : 1)) == 0 && ((freq | offset | pos | lens | page_table) & 3) == 0, NS_ERR_ARGUMENT,
               "ns_kv_append_rotary: misaligned argument");
    NsDevice* d = ns_dev(h);
    rc = ns_device_make_current(d);
    if (rc != NS_OK) return rc;
    NS_REQUIRE(c.ordinal == d->ordinal, NS_ERR_ARGUMENT, "ns_kv_append_rotary: the cache is another device's");
    const int rows = batch * steps;
    if (rows == 0) return NS_OK;
    AppendArgs p;
    p.src = ns_source(src, splits, src_dtype, rows, src_ld);
    p.q_col = q == 0 ? 0 : q_col; p.k_col = k_col; p.v_col = v_col;
    p.heads = heads; p.kv_heads = c.heads; p.dim = dim; p.rot = rot_dims;
    p.freq = reinterpret_cast<const float*>(freq);
    p.amplitude = amplitude;
    p.offset = reinterpret_cast<const int32_t*>(offset);
    p.pos = reinterpret_cast<const int32_t*>(pos);
    p.lens = reinterpret_cast<const int32_t*>(lens);
    p.page_table = reinterpret_cast<const int32_t*>(page_table);
    p.max_pages = max_pages; p.num_pages = c.num_pages;
    p.page_shift = 0;
    while ((1 << p.page_shift) < c.page_size) p.page_shift++;
    p.batch = batch; p.steps = steps;
    p.q = reinterpret_cast<uint16_t*>(q); p.q_ld = q_ld;
    p.k_pool = c.k_pool; p.v_pool = c.v_pool;
    p.status = d->status_dev;
    const bool halves = layout == NS_ROTARY_HALVES;
    // source vectors of four values are one load: the source's addresses in bf16 terms where it is float, too
    const uint64_t at = (src_dtype == NS_F32 ? src >> 1 | (src & 1) : src) | q;
    const int vec = rot_vector(8, halves, dim, rot_dims, at, (int64_t)src_ld | p.q_col | k_col | v_col | (q == 0 ? 0 : q_ld));
    return rot_pick(halves, vec, [&](auto hv, auto vc) {
        constexpr bool HALVES = decltype(hv)::value;
        constexpr int VEC = decltype(vc)::value;
        const RotTasks<HALVES, VEC> n(dim, rot_dims);
        p.lane_tasks = n.turned < 32 ? n.turned : 32;
        // Warps a row: two where rows are many (one: 41 us for 13 x 777, four: 37), more for few rows, until there are eight warps an SM or each has one turn, and
        // for rows that the staging memory of a warp does not hold.
        const int row_heads = heads + 2 * c.heads, across = 32 / p.lane_tasks;
        const bool staged = src_dtype == NS_BF16 && VEC == 8;
        constexpr int stage_bytes = 6144;
        p.parts = 2;
        while (p.parts < row_heads && ((int64_t)rows * p.parts < 8 * d->sm_count ? row_heads > p.parts * across
                                                                                 : staged && (row_heads + p.parts - 1) / p.parts * dim * 2 > stage_bytes))
            p.parts *= 2;
        p.heads_each = (row_heads + p.parts - 1) / p.parts;
        p.parts = (row_heads + p.heads_each - 1) / p.heads_each;
        p.rest = RotDiv((dim - n.rest) / VEC);
        p.value = RotDiv(dim / VEC);
        const int64_t items = (int64_t)rows * p.parts;
        p.stage_at = (ROT_THREADS / 32 * n.table() * (int)sizeof(float2) + 15) / 16 * 16;
        const size_t smem = p.stage_at + (staged ? (size_t)(ROT_THREADS / 32) * p.heads_each * dim * 2 : 0);
        const dim3 grid((unsigned)((items + ROT_THREADS / 32 - 1) / (ROT_THREADS / 32)));
        auto launch = [&](auto kernel) {
            NS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
            NS_CUDA(ns_launch_plain(kernel, grid, dim3(ROT_THREADS), smem, d->stream, p));
            return (int)NS_OK;
        };
        if (src_dtype == NS_BF16) return launch(ns_kv_append_rotary_kernel<HALVES, VEC, ROT_BF16>);
        return ns_pick_slabs<NS_IN_TURN>(splits > 2 && rows <= 128, [&](auto sl) { return launch(ns_kv_append_rotary_kernel<HALVES, VEC, decltype(sl)::value>); });
    });
}
