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
#include "ns_seq.cuh"

namespace {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_DIM = 4096;

// amplitude * (cos, sin) of position * freq.  The angle in turns, reduced to half a turn either way, in 64 bits; its doubled value as a float and the
// rest of it, which moves the result along its derivative: within an ulp or two of the exact value.
__device__ __forceinline__ float2 rot_cos_sin(double position, float freq, float amplitude)
{
    double turns = position * (double)freq * 0.15915494309189535;
    turns -= rint(turns);
    const double twice = turns + turns;
    const float hi = (float)twice, lo = (float)(twice - (double)hi) * 3.14159274f;
    float s, c;
    sincospif(hi, &s, &c);
    return make_float2(amplitude * fmaf(-lo, s, c), amplitude * fmaf(lo, c, s));
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) RotVec {
    T v[VEC];
};

__device__ __forceinline__ float rot_float(float v) { return v; }
__device__ __forceinline__ float rot_float(uint16_t v) { return ns_bf16_bits_to_f32(v); }
__device__ __forceinline__ void rot_put(float& d, float v) { d = v; }
__device__ __forceinline__ void rot_put(uint16_t& d, float v) { d = ns_f32_to_bf16_bits(v); }

// How a head's columns are dealt out.  A task is VEC neighbouring pairs of halves, or VEC neighbouring columns (pairs of neighbours lie inside; columns
// behind the turned ones are copied).
template <bool HALVES, int VEC>
struct RotTasks {
    int half, dim, turned, per_head;      // turned: tasks that turn something
    __host__ __device__ RotTasks(int dim_, int rot, bool copies) : half(rot / 2), dim(dim_)
    {
        if (HALVES) {
            turned = half / VEC;
            per_head = turned + (copies ? (dim - rot) / VEC : 0);
        } else {
            // (scalar: a task is a pair, then single columns)
            const int columns = VEC > 1 ? VEC : 2;
            turned = (rot + columns - 1) / columns;
            per_head = copies ? (VEC > 1 ? dim / VEC : half + dim - rot) : turned;
        }
    }
    // first column of a task, and of its second vector
    __device__ __forceinline__ int first(int t) const
    {
        if (HALVES) return t < turned ? t * VEC : 2 * half + (t - turned) * VEC;
        if (VEC == 1) return t < turned ? 2 * t : 2 * half + (t - turned);
        return t * VEC;
    }
};

// the columns of one task in 32 bits: a, and for halves or scalar pairs b
template <bool HALVES, int VEC>
__device__ __forceinline__ void rot_turn(const RotTasks<HALVES, VEC>& n, int t, const float2* cs, float sign, float (&a)[VEC], float (&b)[VEC])
{
    if (t >= n.turned) return;
    if (HALVES || VEC == 1) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float2 w = cs[t * VEC + i];
            const float x = a[i], y = b[i], s = sign * w.y;
            a[i] = fmaf(x, w.x, -(y * s));
            b[i] = fmaf(x, s, y * w.x);
        }
    } else {
#pragma unroll
        for (int i = 0; i + 1 < VEC; i += 2) {
            const int p = (t * VEC + i) >> 1;
            if (p < n.half) {
                const float2 w = cs[p];
                const float x = a[i], y = a[i + 1], s = sign * w.y;
                a[i] = fmaf(x, w.x, -(y * s));
                a[i + 1] = fmaf(x, s, y * w.x);
            }
        }
    }
}

// whether a task has a second vector, and where it is
template <bool HALVES, int VEC>
__device__ __forceinline__ bool rot_second(const RotTasks<HALVES, VEC>& n, int t) { return (HALVES || VEC == 1) && t < n.turned; }
template <bool HALVES, int VEC>
__device__ __forceinline__ int rot_second_at(const RotTasks<HALVES, VEC>& n, int c) { return HALVES ? c + n.half : c + 1; }

// ---------------------------------------------------------------------------------------------
// rows of a matrix
// ---------------------------------------------------------------------------------------------
struct RotaryArgs {
    const void* x;
    void* y;
    int64_t x_ld, x_head, y_ld, y_head;
    const int32_t* pos;
    const float* freq;
    float amplitude, sign;
    int64_t rows;
    int heads, dim, rot;
    int copies;            // y is another matrix: the columns that are not turned are copied
    int group;             // threads a row
    int heads_each;        // heads a CTA takes of its rows (blockIdx.y)
};

template <typename T, bool HALVES, int VEC>
__global__ void __launch_bounds__(ROT_THREADS) ns_rotary_kernel(const RotaryArgs p)
{
    constexpr int U = VEC >= 4 ? 2 : 4;      // tasks in flight
    using V = RotVec<T, VEC>;
    extern __shared__ float2 rot_table[];
    ns_pdl_wait();
    ns_pdl_trigger();
    const RotTasks<HALVES, VEC> n(p.dim, p.rot, p.copies != 0);
    const int per_cta = ROT_THREADS / p.group, slot = threadIdx.x / p.group, lane = threadIdx.x % p.group;
    const int half = p.rot / 2;
    float2* cs = rot_table + slot * half;
    const int h0 = blockIdx.y * p.heads_each, heads = min(p.heads_each, p.heads - h0);
    const int tasks = heads * n.per_head;
    for (int64_t r0 = (int64_t)blockIdx.x * per_cta; r0 < p.rows; r0 += (int64_t)gridDim.x * per_cta) {
        const int64_t r = r0 + slot;
        const int pos = r < p.rows ? p.pos[r] : -1;
        const T* x = reinterpret_cast<const T*>(p.x) + r * p.x_ld + h0 * p.x_head;
        T* y = reinterpret_cast<T*>(p.y) + r * p.y_ld + h0 * p.y_head;
        bool table = false;
        // (the loop runs once at least in every thread: the barrier stands in it)
        for (int at = lane; at < tasks || !table; at += U * p.group) {
            V a[U], b[U];
            int head[U], task[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int e = at + u * p.group;
                head[u] = e / n.per_head;
                task[u] = e - head[u] * n.per_head;
                if (e < tasks && pos >= 0) {
                    const T* src = x + head[u] * p.x_head;
                    const int c = n.first(task[u]);
                    a[u] = *reinterpret_cast<const V*>(src + c);
                    if (rot_second(n, task[u])) b[u] = *reinterpret_cast<const V*>(src + rot_second_at(n, c));
                }
            }
            if (!table) {
                __syncthreads();       // the row before has been turned
                if (pos >= 0)
                    for (int i = lane; i < half; i += p.group) cs[i] = rot_cos_sin((double)pos, p.freq[i], p.amplitude);
                __syncthreads();
                table = true;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (at + u * p.group < tasks && pos >= 0) {
                    float fa[VEC], fb[VEC];
                    const bool second = rot_second(n, task[u]);
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        fa[i] = rot_float(a[u].v[i]);
                        fb[i] = second ? rot_float(b[u].v[i]) : 0.0f;
                    }
                    rot_turn(n, task[u], cs, p.sign, fa, fb);
                    V oa, ob;
#pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        rot_put(oa.v[i], fa[i]);
                        rot_put(ob.v[i], fb[i]);
                    }
                    T* dst = y + head[u] * p.y_head;
                    const int c = n.first(task[u]);
                    // columns that are not turned keep their bits
                    *reinterpret_cast<V*>(dst + c) = task[u] < n.turned ? oa : a[u];
                    if (second) *reinterpret_cast<V*>(dst + rot_second_at(n, c)) = ob;
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

// threads a row: as many as it has tasks, a warp at least and a CTA at most
int rot_group(int64_t tasks)
{
    int g = 32;
    while (g < ROT_THREADS && g < tasks) g *= 2;
    return g;
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
    int group, tasks_each;
    int* status;
};

// VEC values of the source from element idx on, in 32 bits
template <int VEC, int SLABS>
__device__ __forceinline__ void rot_source(const NsSource& s, int64_t idx, float (&v)[VEC])
{
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 f = ns_source_at4<SLABS>(s, idx + i);
            v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = ns_source_at<SLABS>(s, idx + i);
    }
}
template <int VEC>
__device__ __forceinline__ void rot_store(uint16_t* dst, const float (&v)[VEC])
{
    RotVec<uint16_t, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; i++) o.v[i] = ns_f32_to_bf16_bits(v[i]);
    *reinterpret_cast<RotVec<uint16_t, VEC>*>(dst) = o;
}

template <bool HALVES, int VEC, int SLABS>
__global__ void __launch_bounds__(ROT_THREADS) ns_kv_append_rotary_kernel(const AppendArgs p)
{
    extern __shared__ float2 rot_table[];
    ns_pdl_wait();
    ns_pdl_trigger();
    const RotTasks<HALVES, VEC> n(p.dim, p.rot, true);
    const int per_cta = ROT_THREADS / p.group, slot = threadIdx.x / p.group, lane = threadIdx.x % p.group;
    const int half = p.rot / 2;
    float2* cs = rot_table + slot * half;
    const int rows = p.batch * p.steps;
    // tasks of a row: the query heads', the key heads', then the values' columns
    const int turned = (p.heads + p.kv_heads) * n.per_head, tasks = turned + p.kv_heads * (p.dim / VEC);
    const int first = blockIdx.y * p.tasks_each, end = min(first + p.tasks_each, tasks);
    const int page_size = 1 << p.page_shift;
    const int offset = p.offset != nullptr ? p.offset[0] : 0;
    for (int r0 = blockIdx.x * per_cta; r0 < rows; r0 += gridDim.x * per_cta) {
        const int r = r0 + slot;
        const int b = r / p.steps, i = r - b * p.steps;
        const bool live = r < rows && (p.lens == nullptr || i < p.lens[b]);
        // positions in 64 bits: nothing a caller leaves in a padded row wraps around
        const int64_t at = live ? (int64_t)p.pos[b] + i : 0;
        __syncthreads();
        if (live)
            for (int e = lane; e < half; e += p.group) cs[e] = rot_cos_sin((double)(at + offset), p.freq[e], p.amplitude);
        __syncthreads();
        if (!live) continue;
        int page = -1;
        if (at >= 0 && (at >> p.page_shift) < p.max_pages) page = p.page_table[(int64_t)b * p.max_pages + (at >> p.page_shift)];
        const bool stored = page >= 0 && page < p.num_pages;
        if (!stored && lane == 0) *reinterpret_cast<volatile int*>(p.status) = 500;
        const int64_t row = (int64_t)r * p.src.ld;
        const int64_t slab = ((int64_t)page * p.kv_heads * page_size + (at & (page_size - 1))) * p.dim;      // head 0's row in the page
        const int64_t head_step = (int64_t)page_size * p.dim;
        for (int e = first + lane; e < end; e += p.group) {
            float a[VEC], c[VEC];
            if (e < turned) {
                const int head = e / n.per_head, t = e - head * n.per_head, col = n.first(t);
                const bool key = head >= p.heads;
                if (key && !stored) continue;
                const int64_t src = row + (key ? p.k_col + (head - p.heads) * p.dim : p.q_col + head * p.dim) + col;
                uint16_t* dst = key ? p.k_pool + slab + (head - p.heads) * head_step + col : p.q + (int64_t)r * p.q_ld + (int64_t)head * p.dim + col;
                rot_source<VEC, SLABS>(p.src, src, a);
                const bool second = rot_second(n, t);
                const int step = rot_second_at(n, col) - col;
                if (second) rot_source<VEC, SLABS>(p.src, src + step, c);
                rot_turn(n, t, cs, 1.0f, a, c);
                rot_store<VEC>(dst, a);
                if (second) rot_store<VEC>(dst + step, c);
            } else if (stored) {
                const int per = p.dim / VEC, head = (e - turned) / per, col = (e - turned - head * per) * VEC;
                rot_source<VEC, SLABS>(p.src, row + p.v_col + head * p.dim + col, a);
                rot_store<VEC>(p.v_pool + slab + head * head_step + col, a);
            }
        }
    }
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
    NS_REQUIRE((int64_t)heads * dim <= (1 << 24), NS_ERR_ARGUMENT, "ns_rotary: at most 2^24 columns a row");
    // no two (row, head) of the output share a column: heads inside rows, or rows inside heads
    auto apart = [&](int64_t inner, int64_t n_inner, int64_t outer, int64_t n_outer) {
        const bool in = n_inner == 1 || inner >= dim;
        return in && (n_outer == 1 || (outer >= dim && (n_inner == 1 || (outer - dim) / inner >= n_inner - 1)));
    };
    NS_REQUIRE(x_ld >= 0 && x_head >= 0 && y_ld >= 0 && y_head >= 0, NS_ERR_ARGUMENT, "ns_rotary: negative pitch");
    NS_REQUIRE(apart(y_head, heads, y_ld, rows) || apart(y_ld, rows, y_head, heads), NS_ERR_ARGUMENT, "ns_rotary: rows or heads of the output overlap");
    NS_REQUIRE(x != y || (x_ld == y_ld && x_head == y_head), NS_ERR_ARGUMENT, "ns_rotary: in place, both pitches have to be the input's");
    NsDevice* d = ns_dev(h);
    int rc = ns_device_make_current(d);
    if (rc != NS_OK) return rc;
    if (rows == 0) return NS_OK;
    RotaryArgs p;
    p.x = reinterpret_cast<const void*>(x); p.y = reinterpret_cast<void*>(y);
    p.x_ld = x_ld; p.x_head = x_head; p.y_ld = y_ld; p.y_head = y_head;
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
        const RotTasks<HALVES, VEC> n(dim, rot_dims, p.copies != 0);
        p.group = rot_group((int64_t)heads * n.per_head);
        const int per_cta = ROT_THREADS / p.group;
        // few rows: their heads are spread over CTAs, a task a thread at least
        int64_t ctas = (rows + per_cta - 1) / per_cta;
        int parts = 1;
        while (parts < heads && ctas * parts < d->sm_count && (int64_t)heads * n.per_head > (int64_t)parts * ROT_THREADS) parts *= 2;
        p.heads_each = (heads + parts - 1) / parts;
        parts = (heads + p.heads_each - 1) / p.heads_each;
        if (ctas > (1 << 30)) ctas = 1 << 30;
        const size_t smem = (size_t)per_cta * (rot_dims / 2) * sizeof(float2);
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
    NS_REQUIRE((int64_t)(heads + 2LL * c.heads) * dim <= (1 << 24), NS_ERR_ARGUMENT, "ns_kv_append_rotary: at most 2^24 columns a row");
    NS_REQUIRE(k_col >= 0 && v_col >= 0 && (q == 0 || q_col >= 0) && (int64_t)k_col + c.heads * dim <= src_ld && (int64_t)v_col + c.heads * dim <= src_ld &&
                   (q == 0 || (int64_t)q_col + heads * dim <= src_ld),
               NS_ERR_ARGUMENT, "ns_kv_append_rotary: columns outside the source's rows");
    NS_REQUIRE(q == 0 || (q_ld >= (int64_t)heads * dim && (q & 1) == 0), NS_ERR_ARGUMENT, "ns_kv_append_rotary: query rows are shorter than their heads");
    NS_REQUIRE((src & (src_dtype == NS_F32 ? 3 : 1)) == 0 && ((freq | offset | pos | lens | page_table) & 3) == 0, NS_ERR_ARGUMENT,
               "ns_kv_append_rotary: misaligned argument");
    NsDevice* d = ns_dev(h);
    rc = ns_device_make_current(d);
    if (rc != NS_OK) return rc;
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
        const RotTasks<HALVES, VEC> n(dim, rot_dims, true);
        const int tasks = (heads + c.heads) * n.per_head + c.heads * (dim / VEC);
        p.group = rot_group(tasks);
        const int per_cta = ROT_THREADS / p.group;
        const int ctas = (rows + per_cta - 1) / per_cta;
        int parts = 1;
        while (ctas * parts < 2 * d->sm_count && tasks > parts * ROT_THREADS) parts *= 2;
        p.tasks_each = (tasks + parts - 1) / parts;
        parts = (tasks + p.tasks_each - 1) / p.tasks_each;
        const size_t smem = (size_t)per_cta * (rot_dims / 2) * sizeof(float2);
        const dim3 grid((unsigned)ctas, (unsigned)parts);
        return ns_pick_slabs<NS_IN_TURN>(splits > 2 && rows <= 128, [&](auto sl) {
            NS_CUDA(ns_launch_plain(ns_kv_append_rotary_kernel<HALVES, VEC, decltype(sl)::value>, grid, dim3(ROT_THREADS), smem, d->stream, p));
            return (int)NS_OK;
        });
    });
}
