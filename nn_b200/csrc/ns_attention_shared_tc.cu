// The shared prefix of ns_attention_shared on the sm_100a tensor cores: the query rows of all sequences against each key/value head's pages, S = Q.K^T and
// O += P.V as tcgen05.mma with accumulators in tensor memory, an online softmax between them.
//
// A tile is 256 query rows of one key/value head, its units the key blocks of 128; the units of all tiles, one after the other, are dealt out to the CTAs in equal
// shares, one persistent CTA of 384 threads per SM.  What a CTA has of a tile is a part of its rows' results.
//   warp 0       reads the page table and loads K and V blocks (a TMA box a page, or part of one) into rings of slots, for both groups
//   warp 1       issues the MMAs, in turn for group 0 and group 1: O += P.V of a block, then S = Q.K^T of the next
//   warps 4..11  two groups of four warps; thread r of a group owns one query row (tensor-memory lane r): it copies its query to shared memory, and for each
//                block reads 128 scores, takes maximum and sum, and writes P as bf16 over the scores in tensor memory, from where P.V takes it
// Group g owns rows [128 g, 128 g + 128) of the tile and both groups read every block; with 128 rows or fewer they own the same rows and take turns
// with the blocks, each a part of its own.
// One warp issues for both groups so that their MMAs run in that order.  With a warp for each the tensor pipe took them alternately, both groups' scores
// arrived together, both computed exponentials together (3 300 cycles a block for 1 700 alone) and both then waited 1 200 cycles for MMAs.
//
// A block's positions behind the prefix's end are masked, and their values, which may be anything, are zeroed in shared memory before the MMA reads them (0 times NaN
// is NaN); pages outside the pool read as zeros and are masked.  Parts leave as 32-bit sums; ns_attention_shared_fold_kernel joins them.
// Every mbarrier wait is bounded; a wait that runs out reports a status code (330 + role) and the CTA leaves.
#include <math.h>

#include "ns_attention_shared.cuh"

namespace {

constexpr int ST_THREADS = 384;
constexpr int ST_KB = 128;                             // keys a block
constexpr int ST_OWN = 300;                            // own positions of a key/value head that are as much work as a unit
constexpr int ST_EARLY = 4;                            // blocks in which every growth of the maximum is followed
constexpr uint32_t ST_STAGE_BYTES = 32 * 128;          // a softmax warp's 32 rows x 32 floats on their way out
constexpr uint32_t ST_S_COL = 128;                     // tensor memory of group g: O at columns 256 g, S 128 further on, P over the first half of S

// Rows of 128 bytes, 64 columns.  Heads of 32 columns lie two keys a row, key 2 i before key 2 i + 1 as they lie in the page: the first 64 scores are those of the even keys, the
// products' operands the first 32 columns, and the other 64 those of the odd ones.
template <int DH>
struct Layout {
    static constexpr bool TWO = DH == 32;                      // keys a row
    static constexpr int HALVES = DH == 128 ? 2 : 1;           // column blocks of 64
    static constexpr int SLOTS = DH == 128 ? 2 : 4;
    static constexpr int KEYS = TWO ? 2 : 1;
    static constexpr uint32_t HALF = ST_KB / KEYS * 128;
    static constexpr uint32_t KV = HALVES * HALF;
    static constexpr uint32_t Q = HALVES * 128 * 128;
    // the key of a block's score c
    static __device__ __forceinline__ constexpr int key(int c) { return TWO ? c % 64 * 2 + c / 64 : c; }
    static constexpr uint32_t K_AT = 2 * Q, V_AT = K_AT + SLOTS * KV, STAGE_AT = V_AT + SLOTS * KV, BAR_AT = STAGE_AT + 8 * ST_STAGE_BYTES;
    static constexpr uint32_t SMEM = 1024 + BAR_AT + 512;
    // barriers
    static constexpr int Q_FULL = 0, K_FULL = 2, K_EMPTY = K_FULL + SLOTS, V_FULL = K_EMPTY + SLOTS, V_EMPTY = V_FULL + SLOTS, S_FULL = V_EMPTY + SLOTS, P_FULL = S_FULL + 2,
                         O_DONE = P_FULL + 4, V_TAIL = O_DONE + 2, COUNT = V_TAIL + 1;
    static_assert(SMEM <= 232448 && COUNT * 8 + 16 <= 512, "shared memory of an SM");
};

// n / d for n < 2^30: the multiplier is rounded up, which is exact there for every d (32 + log2 d bits of it)
struct Divide {
    uint32_t m, shift;
    void by(int d)
    {
        shift = 0;
        while ((1 << shift) < d) shift++;
        m = (uint32_t)((((uint64_t)1 << (31 + shift)) + d - 1) / d);
    }
    __device__ __forceinline__ int of(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> (31 + shift)); }
};
struct TileParams {
    SharedParams s;
    Divide group;
    int rows;            // query rows of a key/value head
    int tiles;           // row tiles of a key/value head
    int turns;           // the groups own the same rows and take turns with the blocks
    int box;             // rows of a TMA box: a page, or 128 of it
    int parts;           // of a tile, at most (each two where the groups take turns)
    int sms;
};
struct TileMaps {
    CUtensorMap k, v;    // [64 columns, box rows] of (columns, page rows, heads, pages)
    CUtensorMap o;       // [32 columns, 32 rows] of (columns, rows, parts * heads), float
};

// What a CTA has of a tile: key blocks [b0, b1), and which part of the tile that is.
struct Item {
    int kvh, tile, part, b0, b1;
};
// The CTAs' shares: units [first, end) of all, walked item by item.
struct Share {
    int blocks;          // of a tile
    int64_t at, end, total;
    int ctas;
    // own: positions that the walking kernel has to read beside this one.  The SMs are divided between the two in proportion to their work, a unit being as much as 300
    // positions of a key/value head: the CTAs behind `most` leave, and the other kernel's take their place.  (256 sequences of 300 positions over 16384, 148 CTAs 141 us,
    // 88 129; 64 of 257 over 4096, 128 CTAs 42.6, 57 35.6.)
    __device__ __forceinline__ Share(const TileParams& p, int n_keys, float own)
    {
        blocks = (n_keys + ST_KB - 1) / ST_KB;
        total = (int64_t)blocks * p.tiles * p.s.kv_heads;
        const float units = (float)total * (p.turns ? 0.6f : 1.0f), beside = p.s.beside != nullptr ? own * (float)p.s.kv_heads * (1.0f / ST_OWN) : 0.0f;
        const int most = min((int)gridDim.x, max(1, (int)((float)p.sms * units / (units + beside) + 0.5f)));
        ctas = (int)(total < most ? total : most);                 // no share is empty but behind these
        at = end = 0;
        if ((int)blockIdx.x < ctas) {
            at = total * blockIdx.x / ctas;
            end = total * (blockIdx.x + 1) / ctas;
        }
    }
    __device__ __forceinline__ bool next(const TileParams& p, Item& t)
    {
        if (at >= end) return false;
        const int tile = (int)(at / blocks);
        const int64_t first = (int64_t)tile * blocks;
        t.kvh = tile / p.tiles;
        t.tile = tile - t.kvh * p.tiles;
        t.b0 = (int)(at - first);
        t.b1 = (int)(end - first < blocks ? end - first : blocks);
        // the CTA that has a unit x is the last one whose share begins at or before it
        t.part = (int)blockIdx.x - (int)(((first + 1) * ctas - 1) / total);
        at = first + t.b1;
        return true;
    }
};

__device__ __forceinline__ float st_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// maxima of which a NaN is one
__device__ __forceinline__ float st_max3(float a, float b, float c)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float st_row_max(const float (&s)[ST_KB])
{
    float m[8];
#pragma unroll
    for (int q = 0; q < 8; q++) m[q] = s[q];
#pragma unroll
    for (int c = 8; c + 16 <= ST_KB; c += 16)
#pragma unroll
        for (int q = 0; q < 8; q++) m[q] = st_max3(m[q], s[c + 2 * q], s[c + 2 * q + 1]);
#pragma unroll
    for (int q = 0; q < 8; q++) m[q] = st_max3(m[q], s[ST_KB - 8 + q], m[q]);
    return st_max3(st_max3(m[0], m[1], m[2]), st_max3(m[3], m[4], m[5]), st_max3(m[6], m[7], m[7]));
}
__device__ __forceinline__ uint64_t st_pair(float lo, float hi)
{
    uint64_t y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(lo), "f"(hi));
    return y;
}
__device__ __forceinline__ void st_split(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
// two sums, two fused multiply-adds: each rounded as the single ones are
__device__ __forceinline__ uint64_t st_add2(uint64_t a, uint64_t b)
{
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ uint64_t st_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}
// P = 2^(s scale + neg_m) of pairs [C0, C1) of the 64 scores from FIRST on, as bf16; the sums of P before that rounding go onto `sum`.
// The MMA takes P in 16 bits: each weight is off by half a step, 2^-8 of itself at most, to either side, which over many keys adds little to the rounding of the output (0.0020 to 0.0025
// of its rms in all for 0.0017).  A second half of every weight, as the walking kernel has it, would be some three instructions more to the
// four that each score takes here, which bound this kernel.
template <int FIRST, int C0, int C1>
__device__ __forceinline__ void st_exponentials(const float (&s)[ST_KB], float scale, float neg_m, uint64_t (&sum)[2], uint32_t (&pk)[32])
{
    const uint64_t scale2 = st_pair(scale, scale), neg2 = st_pair(neg_m, neg_m);
#pragma unroll
    for (int c = C0; c < C1; c++) {
        float p0, p1;
        st_split(st_fma2(st_pair(s[FIRST + 2 * c], s[FIRST + 2 * c + 1]), scale2, neg2), p0, p1);
        p0 = st_exp2(p0);
        p1 = st_exp2(p1);
        sum[c & 1] = st_add2(sum[c & 1], st_pair(p0, p1));
        pk[c] = ns_pack_bf16x2(p0, p1);
    }
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void st_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// a position in a ring of slots and the phase of its barriers
template <int SLOTS>
struct Ring {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next()
    {
        if (++s == SLOTS) { s = 0; phase ^= 1u; }
    }
};

template <int DH>
__global__ void __launch_bounds__(ST_THREADS, 1) ns_attention_shared_tile_kernel(const __grid_constant__ TileMaps maps, const TileParams p)
{
    using L = Layout<DH>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int abort_flag_storage;
    volatile int* abort_flag = &abort_flag_storage;
    const uint32_t smem_base = (ns_smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar_base = smem_base + L::BAR_AT;
    auto bar = [&](int i) { return bar_base + 8u * i; };
    const uint32_t tmem_slot = bar(L::COUNT);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    __shared__ uint32_t own_sums[ST_THREADS / 32];
    ns_pdl_wait();
    ns_pdl_trigger();
    // ---- this CTA's share, before anything else: the SMs of CTAs without one are the other kernel's
    const int n_keys = sh_clamp(p.s.prefix_len[0], p.s.prefix_pages, p.s.page_shift);
    uint32_t own = 0;                          // positions beside this kernel's, 16 at a time
    if (p.s.beside != nullptr)
        for (int b = threadIdx.x; b < p.s.batch; b += ST_THREADS) own = min(own + (uint32_t)(sh_clamp((int64_t)p.s.pos[b] + p.s.steps, p.s.max_pages, p.s.page_shift) >> 4), 1u << 26);
    own = __reduce_add_sync(0xffffffffu, own);
    if (lane == 0) own_sums[warp] = own;
    if (threadIdx.x == 0) {
        abort_flag_storage = 0;
        for (int i = 0; i < 2; i++) {
            ns_mbar_init(bar(L::Q_FULL + i), 4);
            ns_mbar_init(bar(L::S_FULL + i), 1);
            ns_mbar_init(bar(L::O_DONE + i), 1);
        }
        for (int i = 0; i < L::SLOTS; i++) {
            ns_mbar_init(bar(L::K_FULL + i), 1);
            ns_mbar_init(bar(L::K_EMPTY + i), 1);
            ns_mbar_init(bar(L::V_FULL + i), 1);
            ns_mbar_init(bar(L::V_EMPTY + i), 1);
        }
        for (int i = 0; i < 4; i++) ns_mbar_init(bar(L::P_FULL + i), 4);
        ns_mbar_init(bar(L::V_TAIL), 1);
        ns_fence_barrier_init();
        ns_fence_proxy_async();
        ns_prefetch_tensormap(&maps.k);
        ns_prefetch_tensormap(&maps.v);
        ns_prefetch_tensormap(&maps.o);
    }
    __syncthreads();
    float own_all = 0.0f;
#pragma unroll
    for (int w = 0; w < ST_THREADS / 32; w++) own_all += (float)own_sums[w];
    Share share(p, n_keys, 16.0f * own_all);
    Item t;
    if (share.at >= share.end && share.total != 0) return;
    if (warp == 1) {
        ns_tmem_alloc(tmem_slot, 512);
        ns_tmem_relinquish();
    }
    ns_tc_fence_before();
    __syncthreads();
    ns_tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));
    tmem_base = __shfl_sync(0xffffffffu, tmem_base, 0);
    const int code = 330;
    auto wait = [&](int i, uint32_t parity, int what) { return ns_mbar_wait_warp(bar(i), parity & 1u, abort_flag, p.s.status, code + what); };
    // whether group g has rows in a tile
    auto has_rows = [&](int g, const Item& t) { return p.turns != 0 || t.tile * 256 + 128 * g < p.rows; };
    // the page of box `lane` of a block: -1 behind the prefix
    const int boxes = ST_KB / p.box, shift = p.s.page_shift;
    auto box_page = [&](int j) {
        const int key = j * ST_KB + lane * p.box;
        return lane < boxes && key < n_keys ? p.s.prefix_table[key >> shift] : -1;
    };
    auto box_bad = [&](int j, int page) { return lane < boxes && j * ST_KB + lane * p.box < n_keys && (page < 0 || page >= p.s.num_pages); };

    // 168 registers a thread at launch; the softmax warps take what the other four give back: 72 + 2 x 216 = 3 x 168
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            // ------------------------------------------------------------ K and V
            const bool leader = ns_elect();
            Ring<L::SLOTS> ring;
            uint32_t tails = 0;
            bool ok = true, begun = false;
            while (ok && share.next(p, t)) {
                int page = t.b0 < t.b1 ? box_page(t.b0) : -1;
                for (int j = t.b0; j < t.b1; j++, ring.next()) {
                    const int next = j + 1 < t.b1 ? box_page(j + 1) : -1;
                    if (__any_sync(0xffffffffu, box_bad(j, page)) && lane == 0) *reinterpret_cast<volatile int*>(p.s.status) = SH_BAD_PAGE;
                    const int row = ((j * ST_KB) & ((1 << shift) - 1)) / L::KEYS;        // inside its page, where that is longer than a block
                    // a page that is none reads as zeros: its coordinate lies behind the pool
                    const int at = page < 0 || page >= p.s.num_pages ? p.s.num_pages : page;
                    auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t full) {
                        if (leader) ns_mbar_expect_tx(full, L::KV);
                        for (int i = 0; i < boxes; i++) {
                            const int pg = __shfl_sync(0xffffffffu, at, i);
                            if (leader) {
#pragma unroll
                                for (int h = 0; h < L::HALVES; h++) ns_tma_load_4d(dst + h * L::HALF + i * (p.box / L::KEYS) * 128, map, full, h * 64, row, t.kvh, pg);
                            }
                        }
                    };
                    ok = wait(L::K_EMPTY + ring.s, ring.phase ^ 1u, 1);
                    if (!ok) break;
                    load(&maps.k, smem_base + L::K_AT + ring.s * L::KV, bar(L::K_FULL + ring.s));
                    // at the start 128 KB of keys and values an SM would stand in the queue to memory before the queries (3 us): only the first keys do
                    if (!begun) {
                        begun = true;
                        ok = wait(L::Q_FULL, 0, 6);
                        if (ok && (p.turns ? t.b0 + 1 < t.b1 : has_rows(1, t))) ok = wait(L::Q_FULL + 1, 0, 6);
                        if (!ok) break;
                    }
                    ok = wait(L::V_EMPTY + ring.s, ring.phase ^ 1u, 2);
                    if (!ok) break;
                    const uint32_t v = smem_base + L::V_AT + ring.s * L::KV;
                    const int live = n_keys - j * ST_KB;
                    if (live >= ST_KB) {
                        load(&maps.v, v, bar(L::V_FULL + ring.s));
                    } else {
                        // the prefix ends inside the block: what lies behind it becomes zeros before anyone reads it
                        load(&maps.v, v, bar(L::V_TAIL));
                        ok = wait(L::V_TAIL, tails++, 3);
                        if (!ok) break;
                        const int rows = (live + L::KEYS - 1) / L::KEYS, gone = ST_KB / L::KEYS - rows;
                        for (int e = lane; e < gone * 8 * L::HALVES; e += 32) {
                            const int c = e & 7, r = rows + (e >> 3) % gone, h = (e >> 3) / gone;
                            ns_st_shared_v4(v + h * L::HALF + r * 128 + c * 16, 0, 0, 0, 0);
                        }
                        // (the second key of a row: its pieces 4 to 7, where the swizzle puts them)
                        if (L::TWO && (live & 1) != 0 && lane < 4) ns_st_shared_v4(v + (rows - 1) * 128 + (((4 + lane) ^ ((rows - 1) & 7)) * 16), 0, 0, 0, 0);
                        ns_fence_proxy_async();
                        __syncwarp();
                        if (leader) ns_mbar_arrive(bar(L::V_FULL + ring.s));
                    }
                    page = next;
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------ MMAs
            const bool leader = ns_elect();
            constexpr uint32_t idesc_qk = ns_idesc(1, 1, 0, 0, 128, ST_KB / L::KEYS), idesc_pv = ns_idesc(1, 1, 0, 1, 128, DH);
            const uint64_t desc_k = ns_desc_base(16, 1024);
            const uint64_t desc_v = ns_desc_base(L::HALF, 1024);      // MN-major: the halves of 64 columns, 8 key rows 1 KB apart
            Ring<L::SLOTS> kr, vr;
            uint32_t nq[2] = {0, 0}, kp[2] = {0, 0};                  // of each group: items and blocks so far
            bool ok = true;
            // the scores of group g for the block in the key ring's slot; `free`: the last ones that need it
            auto scores = [&](int g, bool free) {
                ns_tc_fence_after();
                if (leader) {
                    const uint32_t kb = smem_base + L::K_AT + kr.s * L::KV, qb = smem_base + L::Q * g, s_tmem = tmem_base + 256 * g + ST_S_COL;
#pragma unroll
                    for (int e = 0; e < L::KEYS; e++)
#pragma unroll
                        for (int kk = 0; kk < DH / 16; kk++)
                            ns_mma_f16(s_tmem + e * 64, ns_desc_at(desc_k, qb + (kk >> 2) * (128 * 128) + (kk & 3) * 32),
                                       ns_desc_at(desc_k, kb + (kk >> 2) * L::HALF + (kk & 3) * 32 + e * 64), idesc_qk, kk > 0 ? 1u : 0u);
                    ns_tc_commit(bar(L::S_FULL + g));
                    if (free) ns_tc_commit(bar(L::K_EMPTY + kr.s));
                }
                if (free) kr.next();
            };
            while (ok && share.next(p, t)) {
                const bool both = p.turns != 0 || has_rows(1, t);
                const int step = p.turns ? 2 : 1;
                // the first scores of each group: of one block, or of a block each
                for (int g = 0; g < (both ? 2 : 1) && ok; g++) {
                    if (p.turns && t.b0 + g >= t.b1) break;
                    ok = wait(L::Q_FULL + g, nq[g]++, 6);
                    if (ok && (g == 0 || p.turns)) ok = wait(L::K_FULL + kr.s, kr.phase, 4);
                    if (ok) scores(g, p.turns || g == (both ? 1 : 0));
                }
                for (int j = t.b0; j < t.b1 && ok; j++) {
                    const int g0 = p.turns ? (j - t.b0) & 1 : 0, g1 = p.turns ? g0 : both ? 1 : 0;
                    ok = wait(L::V_FULL + vr.s, vr.phase, 5);
                    for (int g = g0; g <= g1 && ok; g++) {
                        const uint32_t o_tmem = tmem_base + 256 * g, s_tmem = o_tmem + ST_S_COL;
#pragma unroll
                        for (int hf = 0; hf < 2; hf++) {
                            ok = ok && wait(L::P_FULL + 2 * g + hf, kp[g], 7);
                            if (!ok) break;
                            ns_tc_fence_after();
                            if (leader) {
                                const uint32_t vb = smem_base + L::V_AT + vr.s * L::KV + hf * (L::TWO ? 64 : 64 * 128), pa = s_tmem + hf * 32;
#pragma unroll
                                for (int kk = 0; kk < 4; kk++)
                                    st_mma_ts(o_tmem, pa + kk * 8, ns_desc_at(desc_v, vb + kk * (16 * 128)), idesc_pv, j - t.b0 >= step || hf > 0 || kk > 0 ? 1u : 0u);
                            }
                        }
                        if (!ok) break;
                        kp[g]++;
                        if (leader) {
                            ns_tc_commit(bar(L::O_DONE + g));
                            if (g == g1) ns_tc_commit(bar(L::V_EMPTY + vr.s));
                        }
                        if (j + step < t.b1) {
                            if (g == g0) ok = wait(L::K_FULL + kr.s, kr.phase, 4);
                            if (ok) scores(g, g == g1);
                        }
                    }
                    vr.next();
                }
            }
        }
    } else {
        // ------------------------------------------------------------ queries, softmax and output
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int g = (warp >> 2) - 1, quad = warp & 3;
        const int r = quad * 32 + lane;
        const uint32_t o_addr = tmem_base + (uint32_t(quad * 32) << 16) + 256 * g, s_addr = o_addr + ST_S_COL;
        const uint32_t stage = smem_base + L::STAGE_AT + (warp - 4) * ST_STAGE_BYTES;
        const uint32_t q_smem = smem_base + L::Q * g;
        const float scale = p.s.scale_log2;
        uint32_t k = 0;                          // blocks of this group so far, over all items
        bool ok = true;
        // parts [part, end) of row `row` hold nothing
        auto empty = [&](int part, int end, int kvh, int row) {
            if (row < p.rows)
                for (; part < end; part++) p.s.part_ml[((int64_t)part * p.s.kv_heads + kvh) * p.rows + row] = make_float2(-INFINITY, 0.0f);
        };
        const int turns = p.turns ? 2 : 1, parts = p.parts * turns;
        if (share.total == 0)
            for (int i = blockIdx.x; i < p.tiles * p.s.kv_heads; i += gridDim.x)
                if (p.turns == 0 || g == 0) empty(0, parts, i / p.tiles, i % p.tiles * 256 + (p.turns ? 0 : 128 * g) + r);
        while (ok && share.next(p, t)) {
            if (!has_rows(g, t)) continue;
            const int row = (p.turns ? 0 : t.tile * 256 + 128 * g) + r;
            const int part = t.part * turns + (p.turns ? g : 0);
            const int step = turns, first = t.b0 + (p.turns ? g : 0);
            // a tile's last part leaves the rest of them empty
            if (t.b1 == share.blocks && (p.turns == 0 || g == 0)) empty((t.part + 1) * turns, parts, t.kvh, row);
            if (first >= t.b1) {
                empty(part, part + 1, t.kvh, row);
                continue;
            }
            // whether a page of these blocks is none of the pool's (the answers are awaited behind the queries)
            bool any_bad = false;
            for (int key = t.b0 * ST_KB + lane * p.box; key < min(t.b1 * ST_KB, n_keys); key += 32 * p.box) {
                const int page = p.s.prefix_table[key >> shift];
                any_bad |= page < 0 || page >= p.s.num_pages;
            }
            // the warp's 32 queries, whole rows side by side: 16-byte piece c of row r at c ^ (r & 7).  (The group's scores before have all been computed: each warp
            // has waited for the last.)
            {
                constexpr int CH = DH / 8, PER = 32 / CH, UQ = 32 / PER < 8 ? 32 / PER : 8;      // pieces of a row, rows at a time, of those on their way
                const int c = lane % CH, r0 = quad * 32 + lane / CH, base = row - r;
                // (few instructions: this code is fetched cold, and unrolled with its divisions it took 7 000 cycles)
                const int64_t head = (int64_t)t.kvh * p.s.group * DH + c * 8;
#pragma unroll 1
                for (int i = 0; i < 32; i += UQ * PER) {
                    uint4 w[UQ];
#pragma unroll
                    for (int u = 0; u < UQ; u++) {
                        const int rr = base + r0 + i + u * PER, token = p.group.of(rr);
                        w[u] = make_uint4(0, 0, 0, 0);
                        if (rr < p.rows) w[u] = *reinterpret_cast<const uint4*>(p.s.q + head + (int64_t)token * p.s.q_stride + (rr - token * p.s.group) * DH);
                    }
#pragma unroll
                    for (int u = 0; u < UQ; u++) {
                        const int rr = r0 + i + u * PER;
                        ns_st_shared_v4(q_smem + (c >> 3) * (128 * 128) + rr * 128 + (((c & 7) ^ (rr & 7)) * 16), w[u].x, w[u].y, w[u].z, w[u].w);
                    }
                }
                ns_fence_proxy_async();
                __syncwarp();
                if (lane == 0) ns_mbar_arrive(bar(L::Q_FULL + g));
            }
            any_bad = __any_sync(0xffffffffu, any_bad);
            float m_ref = -INFINITY;             // reference maximum (raw score units)
            float l_run = 0.0f;                  // sum of the exponentials relative to m_ref
            for (int j = first; j < t.b1; j += step, k++) {
                ok = wait(L::S_FULL + g, k, 11);
                if (!ok) break;
                ns_tc_fence_after();
                float s[ST_KB];
                {
                    uint32_t s0[32], s1[32], s2[32], s3[32];
                    ns_tmem_ld32(s_addr, s0);
                    ns_tmem_ld32(s_addr + 32, s1);
                    ns_tmem_ld32(s_addr + 64, s2);
                    ns_tmem_ld32(s_addr + 96, s3);
                    ns_tc_wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; c++) {
                        s[c] = __uint_as_float(s0[c]); s[32 + c] = __uint_as_float(s1[c]);
                        s[64 + c] = __uint_as_float(s2[c]); s[96 + c] = __uint_as_float(s3[c]);
                    }
                }
                const int live = n_keys - j * ST_KB;
                if (__builtin_expect(live < ST_KB, 0)) {
#pragma unroll
                    for (int c = 0; c < ST_KB; c++)
                        if (L::key(c) >= live) s[c] = -INFINITY;
                }
                if (__builtin_expect(any_bad, 0)) {
                    const uint32_t bad = __ballot_sync(0xffffffffu, box_bad(j, box_page(j)));
                    const int box_shift = 31 - __clz(p.box);
#pragma unroll
                    for (int c = 0; c < ST_KB; c++)
                        if ((bad >> (L::key(c) >> box_shift)) & 1u) s[c] = -INFINITY;
                }
                // The reference maximum is raised only when the row maximum outgrew it by more than 8 in units of the exponent -- and in the first 512 keys
                // whenever it grew: the largest weight is then exactly 1, which counts where a row has few keys.
                const float mx = st_row_max(s);
                float alpha = 1.0f;
                bool rescale = false;
                if (mx != -INFINITY && (m_ref == -INFINITY || !((mx - m_ref) * scale <= (j - first < ST_EARLY * step ? 0.0f : 8.0f)))) {
                    alpha = m_ref == -INFINITY ? 0.0f : st_exp2((m_ref - mx) * scale);
                    rescale = m_ref != -INFINITY;
                    m_ref = mx;
                }
                // (these scores have followed the P.V before them through the tensor pipe: O is complete)
                if (__builtin_expect(j > first && __any_sync(0xffffffffu, rescale), 0)) {
#pragma unroll 1
                    for (int c = 0; c < DH / 32; c++) {
                        uint32_t ob[32];
                        ns_tmem_ld32(o_addr + c * 32, ob);
                        ns_tc_wait_ld();
#pragma unroll
                        for (int q = 0; q < 32; q++) ob[q] = __float_as_uint(__uint_as_float(ob[q]) * alpha);
                        ns_tmem_st32(o_addr + c * 32, ob);
                    }
                }
                // A score of NaN or +infinity makes a row NaN: both show in the maximum, which then makes every weight of the row NaN (0 m_ref is NaN,
                // else nothing).
                const float neg_m = m_ref == -INFINITY ? 0.0f : fmaf(m_ref, 0.0f, -m_ref * scale);
                uint64_t sum[2] = {0, 0};
                // P leaves for tensor memory half by half; the arrival of the first half is waited for inside the second's exponentials
                auto handed = [&](int hf) {
                    ns_tc_wait_st();
                    ns_tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ns_mbar_arrive(bar(L::P_FULL + 2 * g + hf));
                };
                uint32_t pk[32], pk2[32];
                st_exponentials<0, 0, 32>(s, scale, neg_m, sum, pk);
                __syncwarp();
                ns_tmem_st32(s_addr, pk);
                st_exponentials<64, 0, 8>(s, scale, neg_m, sum, pk2);
                handed(0);
                st_exponentials<64, 8, 32>(s, scale, neg_m, sum, pk2);
                ns_tmem_st32(s_addr + 32, pk2);
                handed(1);
                float l0, l1;
                st_split(st_add2(sum[0], sum[1]), l0, l1);
                l_run = l_run * alpha + (l0 + l1);
            }
            if (!ok) break;
            ok = wait(L::O_DONE + g, k - 1, 12);
            if (!ok) break;
            ns_tc_fence_after();
            if (row < p.rows) p.s.part_ml[((int64_t)part * p.s.kv_heads + t.kvh) * p.rows + row] = make_float2(m_ref * scale, l_run);
            // O -> shared memory (16-byte piece q of row r at q ^ (r & 7)) -> a TMA store a warp, 32 columns at a time; rows behind the last are clipped
            const int warp_row = row - lane;
#pragma unroll 1
            for (int c = 0; c < DH / 32; c++) {
                uint32_t ob[32];
                ns_tmem_ld32(o_addr + c * 32, ob);
                ns_tc_wait_ld();
                if (lane == 0) ns_bulk_wait_read<0>();   // the staging rows are still read by the store before
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 8; q++) ns_st_shared_v4(stage + lane * 128 + ((q ^ (lane & 7)) * 16), ob[4 * q], ob[4 * q + 1], ob[4 * q + 2], ob[4 * q + 3]);
                ns_fence_proxy_async();
                __syncwarp();
                if (lane == 0 && warp_row < p.rows) {
                    ns_tma_store_3d(&maps.o, stage, c * 32, warp_row, part * p.s.kv_heads + t.kvh);
                    ns_bulk_commit();
                }
                __syncwarp();
            }
            // the next item's first P.V overwrites O; it follows this warp's next P
            ns_tc_fence_before();
        }
        if (lane == 0) ns_bulk_wait_read<0>();
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    ns_tc_fence_before();
    __syncthreads();
    if (*abort_flag != 0 && threadIdx.x == 0) {
        // copies in flight land before the CTA's memory is given back
        long long t0 = clock64();
        while (clock64() - t0 < 400000) { }
    }
    __syncthreads();
    if (warp == 1) {
        ns_tc_fence_after();
        ns_tmem_dealloc(tmem_base, 512);
    }
}

// CTAs, by the longest prefix.
int tile_ctas(const NsDevice* d, const TileParams& p)
{
    const int64_t blocks = (((int64_t)p.s.prefix_pages << p.s.page_shift) + ST_KB - 1) / ST_KB, units = blocks * p.tiles * p.s.kv_heads;
    // (two units each where there are fewer than that: a part costs its results' way through memory)
    return (int)((units + 1) / 2 < d->sm_count ? (units + 1) / 2 : d->sm_count);
}

void tile_plan(const NsDevice* d, const SharedParams& s, TileParams& p)
{
    p.s = s;
    p.sms = d->sm_count;
    p.rows = s.batch * s.steps * s.group;
    p.group.by(s.group);
    p.turns = p.rows <= 128 ? 1 : 0;
    p.tiles = (p.rows + 255) / 256;
    p.box = s.page_shift < 7 ? 1 << s.page_shift : ST_KB;
    // a tile's units lie in the shares of at most one CTA more than fit into it, and one for a share that ends inside
    p.parts = tile_ctas(d, p) / (p.tiles * s.kv_heads) + 2;
}

template <int DH>
int launch_tiles(NsDevice* d, const TileParams& p)
{
    using L = Layout<DH>;
    TileMaps maps;
    const int page = 1 << p.s.page_shift;
    uint64_t dims[4] = {(uint64_t)DH * L::KEYS, (uint64_t)page / L::KEYS, (uint64_t)p.s.kv_heads, (uint64_t)p.s.num_pages};
    uint64_t bytes[3] = {(uint64_t)DH * 2 * L::KEYS, (uint64_t)page * DH * 2, (uint64_t)p.s.kv_heads * page * DH * 2};
    uint32_t box[4] = {64, (uint32_t)(p.box / L::KEYS), 1, 1};
    int rc = ns_make_tensor_map(&maps.k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, p.s.k_pool, dims, bytes, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == NS_OK) rc = ns_make_tensor_map(&maps.v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, p.s.v_pool, dims, bytes, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != NS_OK) return rc;
    uint64_t o_dims[3] = {(uint64_t)DH, (uint64_t)p.rows, (uint64_t)p.s.prefix_parts * p.s.kv_heads};
    uint64_t o_bytes[2] = {(uint64_t)DH * 4, (uint64_t)p.rows * DH * 4};
    uint32_t o_box[3] = {32, 32, 1};
    rc = ns_make_tensor_map(&maps.o, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, p.s.part_o, o_dims, o_bytes, o_box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != NS_OK) return rc;
    auto kernel = ns_attention_shared_tile_kernel<DH>;
    NS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::SMEM));
    kernel<<<tile_ctas(d, p), ST_THREADS, L::SMEM, d->stream>>>(maps, p);
    NS_CUDA(cudaGetLastError());
    return NS_OK;
}

}  // namespace

bool ns_attention_shared_tiles_fit(const NsDevice* d, const SharedParams& s, int head_dim, float scale, int* parts)
{
    // boxes of fewer than 8 rows would not begin on the swizzle's 1 KB; the reference maximum is one of raw scores, so their order has to be that of
    // the scaled ones
    if (s.page_shift < (head_dim == 32 ? 4 : 3) || !(scale > 0.0f) || s.prefix_pages == 0) return false;
    // Little to multiply is the walking kernel's, which starts at once; so is what few rows have to read of long keys, which it has on their way from more places.  Both sides of the
    // line, us, this kernel's way and the other's (rows of a key/value head x heads x keys x columns): 128 x 2 x 3333 x 128 22.6, 15.8; 64 x 8 x 2000 x 128 17.5, 17.2; 64 x 16 x 2500 x 64 21.0,
    // 18.3; 256 x 4 x 1600 x 128 24.8, 20.7; 256 x 8 x 700 x 128 20.0, 23.0; 256 x 2 x 4000 x 128 21.6, 23.2; 128 x 8 x 2500 x 128 27.2, 32.3; 64 x 16 x 5000 x 64 24.6, 27.9; 24 x 8 x 16000 x 128
    // 31.8, 33.6; 20 x 32 x 4000 x 128 42.0, 36.4; 20 x 16 x 16000 x 128 45.7, 54.8; 16 x 32 x 16000 x 128 67.6, 62.8; 8 x 8 x 64000 x 128 64.0, 51.3.
    // (One product for all leaves 256 x 8 x 700, 1 430 000, on the slower side: more rows pay earlier than fewer, 64 x 16 x 2500 x 64 at nearly the same product the other way round.)
    const int64_t rows = (int64_t)s.batch * s.steps * s.group;
    const double work = (double)rows * s.kv_heads * ((double)s.prefix_pages * (1 << s.page_shift)) * head_dim;
    if (rows <= 16 || work < (rows >= 24 ? 1.7e6 : 4e6) * 128) return false;
    TileParams p;
    tile_plan(d, s, p);
    *parts = p.parts * (p.turns ? 2 : 1);
    return true;
}

int ns_attention_shared_tiles(NsDevice* d, const SharedParams& s, int head_dim)
{
    TileParams p;
    tile_plan(d, s, p);
    return head_dim == 32 ? launch_tiles<32>(d, p) : head_dim == 64 ? launch_tiles<64>(d, p) : launch_tiles<128>(d, p);
}
