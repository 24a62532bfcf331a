// The pools and geometry of a paged key/value cache (ns_kv_cache_create), for kernels outside ns_attention_decode.cu.
#pragma once

#include "ns_common.cuh"

struct NsKvCacheView {
    uint16_t* k_pool;      // bf16 [num_pages, heads, page_size, head_dim]
    uint16_t* v_pool;
    int page_size, heads, head_dim, num_pages;
    int ordinal;           // of the device the pools lie on
};
int ns_kv_cache_view(ns_kv_cache_t cache, NsKvCacheView* out);   // ns_attention_decode.cu
