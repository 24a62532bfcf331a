// What the two kernels of ns_attention_shared share (ns_attention_shared.cu, ns_attention_shared_tc.cu).
#pragma once

#include "ns_cache.cuh"

constexpr int SH_BAD_PAGE = 520;           // status: a page-table entry that names no page of the pool

struct SharedParams {
    const uint16_t* q;
    int64_t q_stride;
    uint16_t* o;
    int64_t o_stride;
    const uint16_t* k_pool;
    const uint16_t* v_pool;
    const int32_t* prefix_table;
    const int32_t* prefix_len;
    const int32_t* page_table;
    const int32_t* pos;
    const int32_t* lens;
    int prefix_pages, max_pages, page_shift, num_pages;
    int batch, steps, heads, kv_heads, group;
    int prefix_parts, own_parts;           // a row's parts: of the prefix, then of its sequence's own positions
    int prefix_tiles, own_tiles;           // row tiles of the walking kernel: over all sequences (0: the other kernel reads the prefix), of a sequence
    float scale_log2;
    float* part_o;                         // [parts, kv_heads, rows, head_dim]: weighted values relative to the part's maximum
    float2* part_ml;                       // [parts, kv_heads, rows]: maximum in units of log2, sum; (-infinity, 0): nothing seen, and no values written
    int* status;
    uint32_t* beside;                      // the walking kernel runs beside the tensor-core kernel: a word that counts its CTAs, zero between kernels
};

// Whether the tensor-core kernel can read the prefix of such a cache, and its number of parts; ns_attention_shared_tiles queues it.
bool ns_attention_shared_tiles_fit(const NsDevice* d, const SharedParams& p, int head_dim, float scale, int* parts);
int ns_attention_shared_tiles(NsDevice* d, const SharedParams& p, int head_dim);

#ifdef __CUDACC__
// How many of n positions a table can name.
NS_DEVINL int sh_clamp(int64_t n, int pages, int shift)
{
    const int64_t most = (int64_t)pages << shift;
    return (int)(n < 0 ? 0 : n < most ? n : most);
}
#endif
