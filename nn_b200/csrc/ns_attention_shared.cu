// Attention of a batch's new positions over a prefix that all its sequences share and over pages of their own (ns_attention_shared).
//
//   o = softmax over the shared positions [0, prefix_len) and the sequence's own positions [0, pos + i] of scale q.k, times v
//
// Softmax over a union of key sets is a fold: every part gives (maximum m, sum l of e^(s - m), weighted values o relative to m), and parts fold as
//   M = max m,  L = sum l e^(m - M),  O = sum o e^(m - M);  the result is O / L.
// So the prefix is one part (or several, by position) for the rows of ALL sequences together, whose keys and values are then read once for every tile of rows (256 of the
// tensor-core kernel, 8 or 16 here) and not once for each sequence, and each sequence's own pages are another.  Every part is computed from its keys alone, and parts fold in a fixed order.
//
// Rows: the query heads of a key/value head share its cached rows; row r of a key/value head is token r / group (sequence * steps + i), query head
// r % group of its group.
#include <limits.h>
#include <math.h>

#include "ns_attention_shared.cuh"
#include "ns_mma.cuh"

namespace {

constexpr int SH_WARPS = 4;
constexpr int SH_THREADS = 32 * SH_WARPS;
constexpr int SH_KEYS = 16;                // keys a warp takes at a time
constexpr int SH_STAGES = 2;

// 16 bytes to shared memory, zeros where there is nothing
__device__ __forceinline__ void sh_copy16(uint32_t dst, const void* src, bool there)
{
    const int n = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// (8 x 8 of 16-bit values, a register a lane: rows become columns)
__device__ __forceinline__ uint32_t sh_transpose(uint32_t v)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// A CTA: 8 NT rows of one key/value head against a range of keys.  Each warp walks 16 keys at a time on its own, through a ring of its own in shared memory, with
// its own running maximum and sum; the four warps' results fold at the end.  The keys are the M of the products, S' = K Q' and O' = V' P', so that a group of up
// to 8 query heads fills the N of 8: with the queries as M, 16 rows of which 4 are used, the MMAs took twice as long and bounded the kernel (34 GB/s an SM).
// P.V takes the weights as two bf16 halves: the rounding of the output is then the only one that shows.
template <int DH, int NT>
__global__ void __launch_bounds__(SH_THREADS, 3) ns_attention_shared_walk_kernel(const SharedParams p)
{
    constexpr int ROWS = 8 * NT;
    constexpr int LD = DH + 8;                         // elements a row in shared memory: ldmatrix without conflicts
    constexpr int TILE = SH_KEYS * LD * 2;             // bytes
    constexpr int CHUNKS = DH / 8;                     // 16-byte pieces of a row
    constexpr int PASS = 32 / CHUNKS;                  // rows a warp copies at once
    extern __shared__ __align__(16) uint8_t sh_smem[];
    __shared__ uint32_t masks[SH_WARPS][SH_STAGES];
    __shared__ float2 fold[SH_WARPS][ROWS];
    // (beside the tensor-core kernel, which needs the whole of the SMs it has: what came before that has completed, and nothing here needs its results)
    if (p.beside == nullptr) {
        ns_pdl_wait();
        ns_pdl_trigger();
    }
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
    const int row0 = (prefix ? 0 : b * seq_rows) + tile * ROWS;
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
    // lane (g, t) = (lane / 4, lane % 4): keys g and g + 8 of a tile, rows 2 t and 2 t + 1 of each 8
    const int fg = lane >> 2, ft = lane & 3;
    int limit[2 * NT], n_keys, all_see;                // all_see: keys that every row sees which sees any
    if (prefix) {
        n_keys = all_see = sh_clamp(p.prefix_len[0], table_pages, p.page_shift);
#pragma unroll
        for (int e = 0; e < 2 * NT; e++) limit[e] = n_keys;
    } else {
        n_keys = 0;
        all_see = INT_MAX;
#pragma unroll
        for (int e = 0; e < 2 * NT; e++) {
            limit[e] = seen(row0 + (e >> 1) * 8 + ft * 2 + (e & 1));
            n_keys = max(n_keys, limit[e]);
            all_see = min(all_see, limit[e] > 0 ? limit[e] : INT_MAX);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            n_keys = max(n_keys, __shfl_xor_sync(0xffffffffu, n_keys, o));
            all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, o));
        }
    }
    const int tiles_all = (n_keys + SH_KEYS - 1) / SH_KEYS, per = (tiles_all + splits - 1) / splits;
    const int t0 = min(split * per, tiles_all), t1 = min(t0 + per, tiles_all);

    // ---- keys and values
    const uint32_t ring = ns_smem_u32(sh_smem) + warp * SH_STAGES * 2 * TILE;
    const int64_t head_off = (int64_t)kvh << p.page_shift;
    const int page_mask = (1 << p.page_shift) - 1;
    // the page of key lane % 16 of tile t, -1 behind the last; and its cached row as an element of the pools, or -1
    auto page_of = [&](int t) {
        const int j = t * SH_KEYS + (lane & 15);
        return t < t1 && j < n_keys ? table[j >> p.page_shift] : -1;
    };
    auto locate = [&](int t, int page) {
        const int j = t * SH_KEYS + (lane & 15);
        if (t >= t1 || j >= n_keys) return (int64_t)-1;
        if (page < 0 || page >= p.num_pages) {
            *reinterpret_cast<volatile int*>(p.status) = SH_BAD_PAGE;
            return (int64_t)-1;
        }
        return ((((int64_t)page * p.kv_heads) << p.page_shift) + head_off + (j & page_mask)) * DH;
    };
    auto load = [&](int t, uint32_t dst, const uint16_t* pool, int64_t at) {
        if (t < t1) {
            const int c = lane % CHUNKS;
#pragma unroll
            for (int r0 = 0; r0 < SH_KEYS; r0 += PASS) {
                const int r = r0 + lane / CHUNKS;
                const int64_t row = __shfl_sync(0xffffffffu, at, r);
                sh_copy16(dst + (r * LD + c * 8) * 2, pool + (row < 0 ? 0 : row + c * 8), row >= 0);
            }
        }
        ns_cp_commit();
    };
    auto note = [&](int stage, int64_t at) {
        const uint32_t there = __ballot_sync(0xffffffffu, at >= 0) & 0xFFFFu;
        if (lane == 0) masks[warp][stage] = there;
    };
    int64_t ahead = -1;                                // of the tile after next: its keys' rows
    int page = -1;                                     // and of the one behind that: its pages, which nothing waits for yet
    int pages[SH_STAGES];
#pragma unroll
    for (int s = 0; s < SH_STAGES; s++) pages[s] = page_of(t0 + warp + s * SH_WARPS);
    page = page_of(t0 + warp + SH_STAGES * SH_WARPS);
#pragma unroll
    for (int s = 0; s < SH_STAGES; s++) {
        const int t = t0 + warp + s * SH_WARPS;
        ahead = locate(t, pages[s]);
        note(s, ahead);
        load(t, ring + s * 2 * TILE, p.k_pool, ahead);
        load(t, ring + s * 2 * TILE + TILE, p.v_pool, ahead);
    }

    // ---- queries: B fragments
    uint32_t qf[DH / 16][2 * NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = row0 + n * 8 + fg, token = r / p.group;
        const uint16_t* q = p.q + (int64_t)token * p.q_stride + (int64_t)(kvh * p.group + r - token * p.group) * DH + ft * 2;
#pragma unroll
        for (int kk = 0; kk < DH / 16; kk++)
#pragma unroll
            for (int e = 0; e < 2; e++) qf[kk][2 * n + e] = r < row_end ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + e * 8) : 0u;
    }
    float acc[DH / 16][4 * NT];
#pragma unroll
    for (int n = 0; n < DH / 16; n++)
#pragma unroll
        for (int e = 0; e < 4 * NT; e++) acc[n][e] = 0.0f;
    float m[2 * NT], l[2 * NT];                        // of rows 2 t and 2 t + 1 of each 8
#pragma unroll
    for (int e = 0; e < 2 * NT; e++) {
        m[e] = -INFINITY;
        l[e] = 0.0f;
    }
    int stage = 0;
    for (int t = t0 + warp; t < t1; t += SH_WARPS) {
        const uint32_t kt = ring + stage * 2 * TILE, vt = kt + TILE;
        // in order: K and V of this tile, K and V of the next
        ns_cp_wait<2 * SH_STAGES - 1>();
        __syncwarp();
        const uint32_t there = masks[warp][stage];
        float s[4 * NT];
#pragma unroll
        for (int e = 0; e < 4 * NT; e++) s[e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DH / 16; kk++) {
            uint32_t ka[4];
            ns_ldsm4(ka, ns_addr_a(kt, LD, 0, kk * 16, lane));
#pragma unroll
            for (int n = 0; n < NT; n++) ns_mma_bf16(*reinterpret_cast<float(*)[4]>(&s[4 * n]), ka, qf[kk][2 * n], qf[kk][2 * n + 1]);
        }
        __syncwarp();
        const int next = t + SH_STAGES * SH_WARPS;
        ahead = locate(next, page);
        page = page_of(next + SH_WARPS);
        note(stage, ahead);
        load(next, kt, p.k_pool, ahead);
        // s[4 n + 2 h + e]: key g + 8 h, row 2 t + e of the n-th 8
        float mx[2 * NT];
        bool grew = false;
#pragma unroll
        for (int i = 0; i < 2 * NT; i++) {
            const int n = i >> 1, e = i & 1;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int c = fg + 8 * h;
                const bool live = ((there >> c) & 1u) != 0 && t * SH_KEYS + c < limit[i];
                s[4 * n + 2 * h + e] = live ? s[4 * n + 2 * h + e] * p.scale_log2 : -INFINITY;
            }
            mx[i] = fmaxf(s[4 * n + e], s[4 * n + 2 + e]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
            grew |= mx[i] > m[i];
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int i = 0; i < 2 * NT; i++) {
                const float up = fmaxf(m[i], mx[i]), f = m[i] == up ? 1.0f : ns_exp2(m[i] - up);
                m[i] = up;
                l[i] *= f;
#pragma unroll
                for (int d = 0; d < DH / 16; d++) {
                    acc[d][4 * (i >> 1) + (i & 1)] *= f;
                    acc[d][4 * (i >> 1) + 2 + (i & 1)] *= f;
                }
            }
        }
        uint32_t hi[2 * NT], lo[2 * NT];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                // (nothing seen yet: the scores are -infinity, their weights 0)
                const float b0 = m[2 * n] == -INFINITY ? 0.0f : m[2 * n], b1 = m[2 * n + 1] == -INFINITY ? 0.0f : m[2 * n + 1];
                const float e0 = ns_exp2(s[4 * n + 2 * h] - b0), e1 = ns_exp2(s[4 * n + 2 * h + 1] - b1);
                l[2 * n] += e0;
                l[2 * n + 1] += e1;
                const uint32_t w = ns_pack_bf16x2(e0, e1);
                hi[2 * n + h] = sh_transpose(w);
                lo[2 * n + h] = sh_transpose(ns_pack_bf16x2(e0 - __uint_as_float(w << 16), e1 - __uint_as_float(w & 0xFFFF0000u)));
            }
        ns_cp_wait<2 * SH_STAGES - 1>();
        __syncwarp();
        // Where some rows do not see all of the tile's keys, a value that is no number must not reach them: 0 times NaN is NaN.  (0.3 us at most of 20 with five tokens a sequence.)
        bool odd = false;
        if (all_see < n_keys && all_see < (t + 1) * SH_KEYS) {
#pragma unroll
            for (int d = 0; d < DH / 16; d++) {
                uint32_t va[4];
                ns_ldsm4_t(va, ns_addr_at(vt, LD, d * 16, 0, lane));
#pragma unroll
                for (int e = 0; e < 4; e++) odd |= (va[e] & 0x7F80u) == 0x7F80u || (va[e] & 0x7F800000u) == 0x7F800000u;
            }
            odd = __any_sync(0xffffffffu, odd);
        }
        if (__builtin_expect(odd, 0)) {
            // key by key, where it has a weight
            const uint16_t* values = reinterpret_cast<const uint16_t*>(sh_smem) + ((warp * SH_STAGES + stage) * 2 + 1) * (TILE / 2) + fg;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float b0 = m[2 * n] == -INFINITY ? 0.0f : m[2 * n], b1 = m[2 * n + 1] == -INFINITY ? 0.0f : m[2 * n + 1];
                    const float e0 = ns_exp2(s[4 * n + 2 * h] - b0), e1 = ns_exp2(s[4 * n + 2 * h + 1] - b1);
#pragma unroll 1
                    for (int g = 0; g < 8; g++) {
                        const float w0 = __shfl_sync(0xffffffffu, e0, g * 4 + ft), w1 = __shfl_sync(0xffffffffu, e1, g * 4 + ft);
#pragma unroll
                        for (int d = 0; d < DH / 8; d++) {
                            const float v = ns_bf16_bits_to_f32(values[(8 * h + g) * LD + d * 8]);
                            float* a = &acc[d >> 1][4 * n + 2 * (d & 1)];
                            if (w0 != 0.0f) a[0] = fmaf(w0, v, a[0]);
                            if (w1 != 0.0f) a[1] = fmaf(w1, v, a[1]);
                        }
                    }
                }
        } else {
#pragma unroll
            for (int d = 0; d < DH / 16; d++) {
                uint32_t va[4];
                ns_ldsm4_t(va, ns_addr_at(vt, LD, d * 16, 0, lane));
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float(&a)[4] = *reinterpret_cast<float(*)[4]>(&acc[d][4 * n]);
                    ns_mma_bf16(a, va, hi[2 * n], hi[2 * n + 1]);
                    ns_mma_bf16(a, va, lo[2 * n], lo[2 * n + 1]);
                }
            }
        }
        __syncwarp();
        load(next, vt, p.v_pool, ahead);
        stage = stage == SH_STAGES - 1 ? 0 : stage + 1;
    }
    ns_cp_wait<0>();

    // ---- the warps' results fold, in warp order
#pragma unroll
    for (int i = 0; i < 2 * NT; i++) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
        if (fg == 0) fold[warp][(i >> 1) * 8 + ft * 2 + (i & 1)] = make_float2(m[i], l[i]);
    }
    __syncthreads();                      // every ring is free
    // acc[d][4 n + 2 h + e]: dimension 16 d + g + 8 h, row 2 t + e of the n-th 8
    float* out = reinterpret_cast<float*>(sh_smem) + warp * ROWS * (DH + 4);
#pragma unroll
    for (int d = 0; d < DH / 16; d++)
#pragma unroll
        for (int e = 0; e < 4 * NT; e++) out[((e >> 2) * 8 + ft * 2 + (e & 1)) * (DH + 4) + d * 16 + fg + ((e >> 1) & 1) * 8] = acc[d][e];
    __syncthreads();
    const bool alone = p.part_o == nullptr;
    for (int e = threadIdx.x; e < ROWS * DH; e += SH_THREADS) {
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
            O = fmaf(reinterpret_cast<float*>(sh_smem)[(w * ROWS + rr) * (DH + 4) + c], f, O);
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
    // The kernel that folds follows this one alone: the last CTA to get here waits for the other kernel.  (Were each to wait, those to come would find no room.)
    if (p.beside != nullptr) {
        __shared__ int last;
        if (threadIdx.x == 0) last = atomicAdd(p.beside, 1u) == gridDim.x - 1 ? 1 : 0;
        __syncthreads();
        if (last != 0) {
            if (threadIdx.x == 0) *p.beside = 0;
            ns_pdl_wait();
        }
    }
}

template <int N>
struct alignas(4 * N) ShColumns {
    float v[N];
};

// The parts of every row fold, in order: a warp a row, or W warps with a range of the parts each.  A lane weighs a part, 32 of them at a time; then every lane adds up its
// columns, whose loads do not wait for the weights.
template <int DH, int W>
__global__ void __launch_bounds__(256) ns_attention_shared_fold_kernel(const SharedParams p)
{
    constexpr int N = DH / 32;
    __shared__ ShColumns<N> held[8][32];
    __shared__ float2 held_ml[8];
    ns_pdl_wait();
    ns_pdl_trigger();
    const int rows_all = p.batch * p.steps * p.group, parts = p.prefix_parts + p.own_parts;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t idx = (int64_t)blockIdx.x * (8 / W) + warp / W;
    const bool there_is = idx < (int64_t)p.kv_heads * rows_all;
    const int kvh = (int)(idx / rows_all), r = (int)(idx % rows_all);
    const int token = r / p.group, i = token % p.steps;
    const bool live = there_is && (p.lens == nullptr || i < p.lens[token / p.steps]);
    const int64_t step = (int64_t)p.kv_heads * rows_all;
    const float* src = p.part_o + idx * DH + lane * N;
    float M = -INFINITY, L = 0.0f, O[N];
#pragma unroll
    for (int n = 0; n < N; n++) O[n] = 0.0f;
    const int per = (parts + W - 1) / W, first = warp % W * per, end = min(first + per, parts);
    for (int k0 = first; live && k0 < end; k0 += 32) {
        const int count = min(32, end - k0);
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
    if constexpr (W > 1) {
        ShColumns<N> mine;
#pragma unroll
        for (int n = 0; n < N; n++) mine.v[n] = O[n];
        held[warp][lane] = mine;
        if (lane == 0) held_ml[warp] = make_float2(M, L);
        __syncthreads();
        if (warp % W != 0) return;
#pragma unroll
        for (int w = 1; w < W; w++) M = fmaxf(M, held_ml[warp + w].x);
        L = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++) O[n] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float2 ml = held_ml[warp + w];
            const float f = ml.x == -INFINITY ? 1.0f : ns_exp2(ml.x - M);       // (a range without anything has sums of 0)
            L = fmaf(ml.y, f, L);
            const ShColumns<N> v = held[warp + w][lane];
#pragma unroll
            for (int n = 0; n < N; n++) O[n] = fmaf(v.v[n], f, O[n]);
        }
    }
    if (!live) return;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    uint16_t* dst = p.o + (int64_t)token * p.o_stride + (int64_t)(kvh * p.group + r % p.group) * DH + lane * N;
#pragma unroll
    for (int n = 0; n < N; n++) dst[n] = ns_f32_to_bf16_bits(L == 0.0f ? 0.0f : O[n] * inv);
}

template <int DH, int NT>
int launch_walk(NsDevice* d, const SharedParams& p, int64_t ctas)
{
    constexpr int smem = SH_WARPS * SH_STAGES * 2 * SH_KEYS * (DH + 8) * 2;
    static_assert(smem >= SH_WARPS * 8 * NT * (DH + 4) * 4, "the fold's rows");
    auto walk = ns_attention_shared_walk_kernel<DH, NT>;
    NS_CUDA(cudaFuncSetAttribute(walk, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (p.beside != nullptr) NS_CUDA(ns_launch_pdl(walk, dim3((unsigned)ctas), dim3(SH_THREADS), smem, d->stream, p));
    else NS_CUDA(ns_launch_plain(walk, dim3((unsigned)ctas), dim3(SH_THREADS), smem, d->stream, p));
    return NS_OK;
}

template <int DH>
int launch_shared(NsDevice* d, const SharedParams& p, int row_tile)
{
    const int64_t ctas = (int64_t)p.kv_heads * ((int64_t)p.prefix_tiles * p.prefix_parts + (int64_t)p.batch * p.own_tiles * p.own_parts);
    NS_REQUIRE(ctas < (1LL << 31), NS_ERR_ARGUMENT, "ns_attention_shared: too many rows");
    if (ctas > 0) {
        const int rc = row_tile == 8 ? launch_walk<DH, 1>(d, p, ctas) : launch_walk<DH, 2>(d, p, ctas);
        if (rc != NS_OK) return rc;
    }
    if (p.part_o != nullptr) {
        // (eight warps a row for more parts than a warp has on their way at once, where rows are few: 8 rows of 66 parts, the whole call 18.4 -> 8.9 us; 2048 of 18 37.3 -> 43.7)
        const int64_t rows = (int64_t)p.batch * p.steps * p.heads;
        const bool many = p.prefix_parts + p.own_parts > 16 && rows <= 1024;
        auto fold = many ? ns_attention_shared_fold_kernel<DH, 8> : ns_attention_shared_fold_kernel<DH, 1>;
        const dim3 grid((unsigned)(many ? rows : (rows + 7) / 8));
        // (early behind the walking kernel alone: 0.3 us of 6.5; where that runs beside the other one, its CTAs are in the way: 37.1 us became 38.1)
        if (p.beside == nullptr) NS_CUDA(ns_launch_pdl(fold, grid, dim3(256), 0, d->stream, p));
        else NS_CUDA(ns_launch_plain(fold, grid, dim3(256), 0, d->stream, p));
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
    NS_REQUIRE(c.ordinal == d->ordinal, NS_ERR_ARGUMENT, "ns_attention_shared: the cache is another device's");
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
    p.beside = nullptr;
    const int64_t rows = (int64_t)batch * steps * p.group;
    // rows of a CTA of the walking kernel: those of one token, or of all, where they fit into 8
    const int row_tile = steps * p.group <= 8 ? 8 : 16;
    p.prefix_tiles = 0;
    const bool tiles = ns_attention_shared_tiles_fit(d, p, c.head_dim, scale, &p.prefix_parts);
    if (!tiles && prefix_pages > 0) p.prefix_tiles = (int)((rows + row_tile - 1) / row_tile);
    p.own_tiles = (steps * p.group + row_tile - 1) / row_tile;
    // Parts by position, of 64 keys at least and 64 of them at most, alike for prefix and own pages: as short as leaves all CTAs of the walking kernel on the SMs at once (three an SM with
    // 128 columns, four with fewer, one less with 16 rows).  Parts for four CTAs an SM from the prefix and as many from the own pages: 16 sequences of 500 positions, 4 query heads for each of 8, over 500
    // 19.3 us, so 13.0; 8 of 2000 over 2000 24.3, 18.1; 8 x 5 x 16 heads of 64 columns, 300 over 2500, 18.4, 14.8; 4 of 500 over 4000 16.6, 12.5.  But no longer than a quarter more than
    // the keys of all divided by so many CTAs: where the own pages' alone are more than that, a prefix in one part would end long after them.
    const int64_t prefix_keys = tiles ? 0 : (int64_t)prefix_pages * c.page_size, own_keys = (int64_t)max_pages * c.page_size, most = prefix_keys > own_keys ? prefix_keys : own_keys;
    const int64_t prefix_ctas = (int64_t)p.prefix_tiles * c.heads, own_ctas = max_pages > 0 ? (int64_t)batch * p.own_tiles * c.heads : 0;
    const int64_t wave = (int64_t)d->sm_count * ((c.head_dim == 128 ? 3 : 4) - (row_tile == 16 ? 1 : 0));
    auto parts = [&](int64_t keys, int64_t length) { return keys == 0 ? 0 : (keys + length - 1) / length; };
    const int64_t enough = (prefix_ctas * prefix_keys + own_ctas * own_keys) / (wave * 4 / 5);
    int64_t length = most <= 64 * 64 ? 64 : (most + 4095) / 4096 * 64;
    while (length < most && length < enough && prefix_ctas * parts(prefix_keys, length) + own_ctas * parts(own_keys, length) > wave) length += length / 512 * 64 + 64;
    // (beside the tensor-core kernel, on what SMs it leaves, until there are four an SM in all: sequences are of many lengths, and the longest part is the last to end.  64 of up to 512 positions
    // over 4096, 512 CTAs 43.4 us, 1024 41.4.)
    if (tiles && own_ctas > 0) {
        const int64_t n = (4 * (int64_t)d->sm_count + own_ctas - 1) / own_ctas;
        length = (own_keys + n - 1) / n > 64 ? (own_keys + n - 1) / n : 64;
        if (length * 64 < own_keys) length = (own_keys + 63) / 64;
    }
    if (!tiles) p.prefix_parts = (int)parts(prefix_keys, length);
    p.own_parts = (int)parts(own_keys, length);
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
        if (ns_pdl_enabled() && max_pages > 0) p.beside = d->sync_words + NS_SYNC_BESIDE;
        rc = ns_attention_shared_tiles(d, p, c.head_dim);
        if (rc != NS_OK) return rc;
    }
    switch (c.head_dim) {
        case 32: return launch_shared<32>(d, p, row_tile);
        case 64: return launch_shared<64>(d, p, row_tile);
        default: return launch_shared<128>(d, p, row_tile);
    }
}
