// Attention of a batch's new positions over a prefix that all its sequences share and over pages of their own (ns_attention_shared).
//
//   o = softmax over the shared positions [0, prefix_len) and the sequence's own positions [0, pos + i] of scale q.k, times v
//
// Softmax over a union of key sets is a fold: every part gives (maximum m, sum l of e^(s - m), weighted values o relative to m), and parts fold as
//   M = max m,  L = sum l e^(m - M),  O = sum o e^(m - M);  the result is O / L.
// So the prefix is one part (or several, by position) for the rows of ALL sequences together, whose keys and values are then read once and not once for each
// sequence, and each sequence's own pages are another.  Every part is computed from its keys alone, and parts fold in a fixed order.
//
// Rows: the query heads of a key/value head share its cached rows; row r of a key/value head is token r / group (sequence * steps + i), query head
// r % group of its group.
#include <math.h>

#include "ns_attention_shared.cuh"
#include "ns_mma.cuh"

namespace {

constexpr int SH_WARPS = 4;
constexpr int SH_THREADS = 32 * SH_WARPS;
constexpr int SH_KEYS = 16;                // keys a warp takes at a time
constexpr int SH_ROWS = 16;                // query rows of a CTA
constexpr int SH_STAGES = 2;

// 16 bytes to shared memory, zeros where there is nothing
__device__ __forceinline__ void sh_copy16(uint32_t dst, const void* src, bool there)
{
    const int n = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// A CTA: 16 rows of one key/value head against a range of keys.  Each warp walks 16 keys at a time on its own, through a ring of its own in shared memory, with
// its own running maximum and sum; the four warps' results fold at the end.  P.V takes the weights as two bf16 halves: the rounding of
// the output is then the only one that shows.
template <int DH>
__global__ void __launch_bounds__(SH_THREADS, 3) ns_attention_shared_walk_kernel(const SharedParams p)
{
    constexpr int LD = DH + 8;                         // elements a row in shared memory: ldmatrix without conflicts
    constexpr int TILE = SH_KEYS * LD * 2;             // bytes
    constexpr int CHUNKS = DH / 8;                     // 16-byte pieces of a row
    constexpr int PASS = 32 / CHUNKS;                  // rows a warp copies at once
    extern __shared__ __align__(16) uint8_t sh_smem[];
    __shared__ uint32_t masks[SH_WARPS][SH_STAGES];
    __shared__ float2 fold[SH_WARPS][SH_ROWS];
    ns_pdl_wait();
    ns_pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- which rows and which keys
    int item = blockIdx.x;
    const int n_prefix = p.kv_heads * p.prefix_tiles * p.prefix_parts;
    const bool prefix = item < n_prefix;
    if (!prefix) item -= n_prefix;
    const int splits = prefix ? p.prefix_parts : p.own_parts, tiles = prefix ? p.prefix_tiles : p.own_tiles;
    const int split = item % splits; item /= splits;
    const int tile = item % tiles; item /= tiles;
    const int kvh = item % p.kv_heads, b = item / p.kv_heads;       // b: 0 for the prefix
    const int rows_all = p.batch * p.steps * p.group;
    const int seq_rows = p.steps * p.group;
    const int row0 = (prefix ? 0 : b * seq_rows) + tile * SH_ROWS;
    const int row_end = prefix ? rows_all : (b + 1) * seq_rows;
    const int part = prefix ? split : p.prefix_parts + split;
    const int32_t* table = prefix ? p.prefix_table : p.page_table + (int64_t)b * p.max_pages;
    const int table_pages = prefix ? p.prefix_pages : p.max_pages;
    // own positions: how many the token of row r sees
    const int64_t own_pos = prefix ? 0 : (int64_t)p.pos[b] + 1;
    const int own_len = prefix || p.lens == nullptr ? p.steps : p.lens[b];
    auto seen = [&](int r) {
        if (r >= row_end) return 0;
        const int i = (r - b * seq_rows) / p.group;
        return i < own_len ? sh_clamp(own_pos + i, table_pages, p.page_shift) : 0;
    };
    int n_keys;
    if (prefix) {
        n_keys = sh_clamp(p.prefix_len[0], table_pages, p.page_shift);
    } else {
        n_keys = 0;
        for (int r = row0; r < min(row0 + SH_ROWS, row_end); r += p.group) n_keys = max(n_keys, seen(r));
        n_keys = max(n_keys, seen(min(row0 + SH_ROWS, row_end) - 1));
    }
    const int tiles_all = (n_keys + SH_KEYS - 1) / SH_KEYS, per = (tiles_all + splits - 1) / splits;
    const int t0 = min(split * per, tiles_all), t1 = min(t0 + per, tiles_all);

    // ---- queries: A fragments of 16 rows
    const int fr = lane >> 2, fc = (lane & 3) * 2;
    uint32_t qf[DH / 16][4];
    {
        const uint16_t* qr[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = row0 + fr + 8 * h;
            qr[h] = r < row_end ? p.q + (int64_t)(r / p.group) * p.q_stride + (int64_t)(kvh * p.group + r % p.group) * DH : nullptr;
        }
#pragma unroll
        for (int kk = 0; kk < DH / 16; kk++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                qf[kk][e] = qr[e & 1] != nullptr ? *reinterpret_cast<const uint32_t*>(qr[e & 1] + kk * 16 + fc + (e >> 1) * 8) : 0u;
    }
    int limit[2] = {n_keys, n_keys};
    if (!prefix) {
        limit[0] = seen(row0 + fr);
        limit[1] = seen(row0 + fr + 8);
    }

    // ---- keys and values
    const uint32_t ring = ns_smem_u32(sh_smem) + warp * SH_STAGES * 2 * TILE;
    const int64_t head_off = (int64_t)kvh << p.page_shift;
    const int page_mask = (1 << p.page_shift) - 1;
    auto load = [&](int t, int stage) {
        if (t < t1) {
            // the cached row of key t * 16 + lane % 16, or -1
            const int j = t * SH_KEYS + (lane & 15);
            int64_t at = -1;
            if (j < n_keys) {
                const int page = table[j >> p.page_shift];
                if (page >= 0 && page < p.num_pages) at = ((((int64_t)page * p.kv_heads) << p.page_shift) + head_off + (j & page_mask)) * DH;
                else *reinterpret_cast<volatile int*>(p.status) = SH_BAD_PAGE;
            }
            const uint32_t there = __ballot_sync(0xffffffffu, at >= 0) & 0xFFFFu;
            if (lane == 0) masks[warp][stage] = there;
            const uint32_t kd = ring + stage * 2 * TILE, vd = kd + TILE;
            const int c = lane % CHUNKS;
#pragma unroll
            for (int r0 = 0; r0 < SH_KEYS; r0 += PASS) {
                const int r = r0 + lane / CHUNKS;
                const int64_t row = __shfl_sync(0xffffffffu, at, r);
                const int64_t off = row < 0 ? 0 : row + c * 8;
                sh_copy16(kd + (r * LD + c * 8) * 2, p.k_pool + off, row >= 0);
                sh_copy16(vd + (r * LD + c * 8) * 2, p.v_pool + off, row >= 0);
            }
        }
        ns_cp_commit();
    };
    float acc[DH / 8][4];
#pragma unroll
    for (int n = 0; n < DH / 8; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[n][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < SH_STAGES - 1; s++) load(t0 + warp + s * SH_WARPS, s);
    int stage = 0;
    for (int t = t0 + warp; t < t1; t += SH_WARPS) {
        ns_cp_wait<SH_STAGES - 2>();
        __syncwarp();
        const uint32_t kt = ring + stage * 2 * TILE, vt = kt + TILE;
        const uint32_t there = masks[warp][stage];
        load(t + (SH_STAGES - 1) * SH_WARPS, stage == 0 ? SH_STAGES - 1 : stage - 1);
        float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int kk = 0; kk < DH / 16; kk++) {
            uint32_t kb[4];
            ns_ldsm4(kb, ns_addr_b(kt, LD, 0, kk * 16, lane));
            ns_mma_bf16(s[0], qf[kk], kb[0], kb[1]);
            ns_mma_bf16(s[1], qf[kk], kb[2], kb[3]);
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int c = n * 8 + fc + (e & 1);
                const bool live = ((there >> c) & 1u) != 0 && t * SH_KEYS + c < limit[e >> 1];
                s[n][e] = live ? s[n][e] * p.scale_log2 : -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
            }
        bool grew = false;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            grew |= mx[h] > m[h];
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const float up = fmaxf(m[h], mx[h]), f = m[h] == up ? 1.0f : ns_exp2(m[h] - up);
                m[h] = up;
                l[h] *= f;
#pragma unroll
                for (int n = 0; n < DH / 8; n++) {
                    acc[n][2 * h] *= f;
                    acc[n][2 * h + 1] *= f;
                }
            }
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                // (nothing seen yet: the scores are -infinity, their weights 0)
                const float base = m[h] == -INFINITY ? 0.0f : m[h];
                const float e0 = ns_exp2(s[n][2 * h] - base), e1 = ns_exp2(s[n][2 * h + 1] - base);
                l[h] += e0 + e1;
                const uint32_t w = ns_pack_bf16x2(e0, e1);
                hi[2 * n + h] = w;
                lo[2 * n + h] = ns_pack_bf16x2(e0 - __uint_as_float(w << 16), e1 - __uint_as_float(w & 0xFFFF0000u));
            }
#pragma unroll
        for (int n = 0; n < DH / 16; n++) {
            uint32_t vb[4];
            ns_ldsm4_t(vb, ns_addr_bt(vt, LD, 0, n * 16, lane));
            ns_mma_bf16(acc[2 * n], hi, vb[0], vb[1]);
            ns_mma_bf16(acc[2 * n + 1], hi, vb[2], vb[3]);
            ns_mma_bf16(acc[2 * n], lo, vb[0], vb[1]);
            ns_mma_bf16(acc[2 * n + 1], lo, vb[2], vb[3]);
        }
        __syncwarp();
        stage = stage == SH_STAGES - 1 ? 0 : stage + 1;
    }
    ns_cp_wait<0>();

    // ---- the warps' results fold, in warp order
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if ((lane & 3) == 0) fold[warp][fr + 8 * h] = make_float2(m[h], l[h]);
    }
    __syncthreads();                      // every ring is free
    float* out = reinterpret_cast<float*>(sh_smem) + warp * SH_ROWS * (DH + 4);
#pragma unroll
    for (int n = 0; n < DH / 8; n++)
#pragma unroll
        for (int h = 0; h < 2; h++)
            *reinterpret_cast<float2*>(out + (fr + 8 * h) * (DH + 4) + n * 8 + fc) = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
    __syncthreads();
    const bool alone = p.part_o == nullptr;
    for (int e = threadIdx.x; e < SH_ROWS * DH; e += SH_THREADS) {
        const int rr = e / DH, c = e % DH, r = row0 + rr;
        if (r >= row_end) break;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < SH_WARPS; w++) M = fmaxf(M, fold[w][rr].x);
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < SH_WARPS; w++) {
            // (a warp that saw nothing has a sum of 0)
            const float f = fold[w][rr].x == -INFINITY ? (fold[w][rr].y == 0.0f ? 0.0f : 1.0f) : ns_exp2(fold[w][rr].x - M);
            L = fmaf(fold[w][rr].y, f, L);
            O = fmaf(reinterpret_cast<float*>(sh_smem)[(w * SH_ROWS + rr) * (DH + 4) + c], f, O);
        }
        if (alone) {
            const int token = r / p.group, i = token % p.steps;
            if (p.lens != nullptr && i >= p.lens[token / p.steps]) continue;
            p.o[(int64_t)token * p.o_stride + (int64_t)(kvh * p.group + r % p.group) * DH + c] = ns_f32_to_bf16_bits(L == 0.0f ? 0.0f : O / L);
        } else {
            const int64_t at = ((int64_t)part * p.kv_heads + kvh) * rows_all + r;
            p.part_o[at * DH + c] = O;
            if (c == 0) p.part_ml[at] = make_float2(M, L);
        }
    }
}

template <int N>
struct alignas(4 * N) ShColumns {
    float v[N];
};

// The parts of every row fold, in order: a warp a row.  A lane weighs a part, 32 of them at a time; then every lane adds up its columns, whose loads do not wait for the
// weights.
template <int DH>
__global__ void __launch_bounds__(256) ns_attention_shared_fold_kernel(const SharedParams p)
{
    constexpr int N = DH / 32;
    ns_pdl_wait();
    ns_pdl_trigger();
    const int rows_all = p.batch * p.steps * p.group, parts = p.prefix_parts + p.own_parts;
    const int64_t idx = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (idx >= (int64_t)p.kv_heads * rows_all) return;
    const int kvh = (int)(idx / rows_all), r = (int)(idx % rows_all);
    const int token = r / p.group, i = token % p.steps;
    if (p.lens != nullptr && i >= p.lens[token / p.steps]) return;
    const int64_t step = (int64_t)p.kv_heads * rows_all;
    const float* src = p.part_o + idx * DH + lane * N;
    float M = -INFINITY, L = 0.0f, O[N];
#pragma unroll
    for (int n = 0; n < N; n++) O[n] = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
        const int count = min(32, parts - k0);
        const float2 ml = lane < count ? p.part_ml[idx + (k0 + lane) * step] : make_float2(-INFINITY, 0.0f);
        float m = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        // (fmaxf leaves a maximum of NaN out; the part's sum is NaN then, and so is the row)
        const float up = fmaxf(M, m), old = M == up ? 1.0f : ns_exp2(M - up);
        const bool none = ml.x == -INFINITY && ml.y == 0.0f;         // (its values were not written)
        const float f = none ? 0.0f : ml.x == -INFINITY ? 1.0f : ns_exp2(ml.x - up);
        float l = none ? 0.0f : ml.y * f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        L = fmaf(L, old, l);
#pragma unroll
        for (int n = 0; n < N; n++) O[n] *= old;
        M = up;
        const uint32_t there = __ballot_sync(0xffffffffu, !none);
        for (int k = 0; k < count; k += 8) {
            ShColumns<N> v[8];
#pragma unroll
            for (int u = 0; u < 8; u++)
                if ((there >> (k + u)) & 1u) v[u] = *reinterpret_cast<const ShColumns<N>*>(src + (k0 + k + u) * step * DH);
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float w = __shfl_sync(0xffffffffu, f, (k + u) & 31);
                if ((there >> (k + u)) & 1u) {
#pragma unroll
                    for (int n = 0; n < N; n++) O[n] = fmaf(v[u].v[n], w, O[n]);
                }
            }
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint16_t* dst = p.o + (int64_t)token * p.o_stride + (int64_t)(kvh * p.group + r % p.group) * DH + lane * N;
#pragma unroll
    for (int n = 0; n < N; n++) dst[n] = ns_f32_to_bf16_bits(L == 0.0f ? 0.0f : O[n] * inv);
}

template <int DH>
int launch_shared(NsDevice* d, const SharedParams& p)
{
    constexpr int smem = SH_WARPS * SH_STAGES * 2 * SH_KEYS * (DH + 8) * 2;
    static_assert(smem >= SH_WARPS * SH_ROWS * (DH + 4) * 4, "the fold's rows");
    const int64_t ctas = (int64_t)p.kv_heads * ((int64_t)p.prefix_tiles * p.prefix_parts + (int64_t)p.batch * p.own_tiles * p.own_parts);
    NS_REQUIRE(ctas < (1LL << 31), NS_ERR_ARGUMENT, "ns_attention_shared: too many rows");
    if (ctas > 0) {
        auto walk = ns_attention_shared_walk_kernel<DH>;
        NS_CUDA(cudaFuncSetAttribute(walk, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        NS_CUDA(ns_launch_plain(walk, dim3((unsigned)ctas), dim3(SH_THREADS), smem, d->stream, p));
    }
    if (p.part_o != nullptr) {
        const int64_t rows = (int64_t)p.batch * p.steps * p.heads;
        NS_CUDA(ns_launch_plain(ns_attention_shared_fold_kernel<DH>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, d->stream, p));
    }
    return NS_OK;
}

}  // namespace

extern "C" int ns_attention_shared(ns_device_t h, ns_kv_cache_t cache, uint64_t q, int64_t q_stride, uint64_t o, int64_t o_stride, int heads, uint64_t prefix_table,
                                   int prefix_pages, uint64_t prefix_len, uint64_t page_table, int max_pages, uint64_t pos, uint64_t lens, int batch, int steps,
                                   float scale)
{
    NsKvCacheView c;
    int rc = ns_kv_cache_view(cache, &c);
    if (rc != NS_OK) return rc;
    NS_REQUIRE(q && o, NS_ERR_ARGUMENT, "ns_attention_shared: null argument");
    NS_REQUIRE(batch >= 0 && steps >= 0 && prefix_pages >= 0 && max_pages >= 0, NS_ERR_ARGUMENT, "ns_attention_shared: bad shape");
    NS_REQUIRE(heads > 0 && heads % c.heads == 0, NS_ERR_ARGUMENT, "ns_attention_shared: %d query heads over %d key/value heads", heads, c.heads);
    NS_REQUIRE(prefix_pages == 0 || (prefix_table && prefix_len), NS_ERR_ARGUMENT, "ns_attention_shared: a prefix without its table or length");
    NS_REQUIRE(max_pages == 0 || (page_table && pos), NS_ERR_ARGUMENT, "ns_attention_shared: pages without their table or positions");
    NS_REQUIRE(prefix_pages > 0 || max_pages > 0, NS_ERR_ARGUMENT, "ns_attention_shared: neither a prefix nor pages of their own");
    NS_REQUIRE((int64_t)prefix_pages * c.page_size < (1LL << 31) && (int64_t)max_pages * c.page_size < (1LL << 31), NS_ERR_ARGUMENT,
               "ns_attention_shared: tables of 2^31 positions and more");
    NS_REQUIRE((int64_t)batch * steps * heads < (1LL << 30), NS_ERR_ARGUMENT, "ns_attention_shared: too many rows");
    NS_REQUIRE(q_stride % 8 == 0 && (q & 15) == 0, NS_ERR_ARGUMENT, "ns_attention_shared: query rows must be 16-byte aligned");
    NS_REQUIRE((o & 1) == 0 && ((prefix_table | prefix_len | page_table | pos | lens) & 3) == 0, NS_ERR_ARGUMENT, "ns_attention_shared: misaligned argument");
    NS_REQUIRE(q_stride >= (int64_t)heads * c.head_dim && o_stride >= (int64_t)heads * c.head_dim, NS_ERR_ARGUMENT,
               "ns_attention_shared: rows are shorter than their heads");
    NsDevice* d = ns_dev(h);
    rc = ns_device_make_current(d);
    if (rc != NS_OK) return rc;
    if (batch == 0 || steps == 0) return NS_OK;
    SharedParams p;
    p.q = reinterpret_cast<const uint16_t*>(q); p.q_stride = q_stride;
    p.o = reinterpret_cast<uint16_t*>(o); p.o_stride = o_stride;
    p.k_pool = c.k_pool; p.v_pool = c.v_pool;
    p.prefix_table = reinterpret_cast<const int32_t*>(prefix_table);
    p.prefix_len = reinterpret_cast<const int32_t*>(prefix_len);
    p.page_table = reinterpret_cast<const int32_t*>(page_table);
    p.pos = reinterpret_cast<const int32_t*>(pos);
    p.lens = reinterpret_cast<const int32_t*>(lens);
    p.prefix_pages = prefix_pages; p.max_pages = max_pages; p.num_pages = c.num_pages;
    p.page_shift = 0;
    while ((1 << p.page_shift) < c.page_size) p.page_shift++;
    p.batch = batch; p.steps = steps; p.heads = heads; p.kv_heads = c.heads; p.group = heads / c.heads;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.status = d->status_dev;
    const int64_t rows = (int64_t)batch * steps * p.group;
    // parts by position: until there are about four CTAs an SM, 64 keys a part at least
    auto parts = [&](int64_t ctas, int64_t positions) {
        int64_t n = (4LL * d->sm_count + ctas - 1) / ctas;
        if (n > (positions + 63) / 64) n = (positions + 63) / 64;
        return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
    };
    p.prefix_tiles = 0;
    const bool tiles = ns_attention_shared_tiles_fit(d, p, c.head_dim, scale, &p.prefix_parts);
    if (!tiles) {
        p.prefix_tiles = (int)((rows + SH_ROWS - 1) / SH_ROWS);
        p.prefix_parts = prefix_pages == 0 ? 0 : parts((int64_t)p.prefix_tiles * c.heads, (int64_t)prefix_pages * c.page_size);
    }
    p.own_tiles = (steps * p.group + SH_ROWS - 1) / SH_ROWS;
    p.own_parts = max_pages == 0 ? 0 : parts((int64_t)batch * p.own_tiles * c.heads, (int64_t)max_pages * c.page_size);
    const int n_parts = p.prefix_parts + p.own_parts;
    p.part_o = nullptr;
    p.part_ml = nullptr;
    if (tiles || n_parts > 1) {
        const size_t sums = (size_t)n_parts * c.heads * rows;
        void* s = nullptr;
        rc = ns_scratch_reserve(d, sums * (c.head_dim * 4 + 8), &s);
        if (rc != NS_OK) return rc;
        p.part_o = reinterpret_cast<float*>(s);
        p.part_ml = reinterpret_cast<float2*>(p.part_o + sums * c.head_dim);
    }
    if (tiles) {
        rc = ns_attention_shared_tiles(d, p, c.head_dim);
        if (rc != NS_OK) return rc;
    }
    switch (c.head_dim) {
        case 32: return launch_shared<32>(d, p);
        case 64: return launch_shared<64>(d, p);
        default: return launch_shared<128>(d, p);
    }
}
