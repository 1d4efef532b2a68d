// pages.h — what the operators over the paged INT8 cache share (internal header).
//
//   K_pages, V_pages int8 [num_pages, kv_heads, page, D], scales fp32 [num_pages, kv_heads, page]
//   page a power of two in [16, 1024], D 64 or 128; a slot is page id * page + offset
#pragma once

#include "int8k_common.h"

namespace int8k {

inline int log2_of(int page) {
    int l = 0;
    while ((1 << l) < page) ++l;
    return l;
}

// Shared checks of the cache's shape: INT8K_OK or the status to return.
inline int check_pages(int num_pages, int page_size, int kv_heads, int head_dim) {
    if (num_pages <= 0 || kv_heads <= 0) return INT8K_ERR_INVALID_ARGUMENT;
    if (head_dim != 64 && head_dim != 128) return INT8K_ERR_UNSUPPORTED;
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
        return INT8K_ERR_UNSUPPORTED;
    // slots are int32
    if ((long long)num_pages * page_size > 0x7fffffffLL) return INT8K_ERR_UNSUPPORTED;
    if ((long long)num_pages * page_size >= (1LL << 40) / ((long long)kv_heads * head_dim))
        return INT8K_ERR_UNSUPPORTED;
    return INT8K_OK;
}

// Bad slots and page ids met on the current device, per translation unit (int8k_paged_bad_ids).
int append_bad_slots(unsigned int* count);   // heads.hip
int attend_bad_ids(unsigned int* count);     // paged.hip
int pages_bad_ids(unsigned int* count);      // pages.hip

// The selection of the blocks that a sparse decode reads (pages.hip): for each sequence and key
// head, from the scores of its blocks by their pages' mean keys,
//   selected [B, Hkv, top]   the blocks taken, ascending, -1 behind the last
//   pages [B, Hkv, top]      their page ids as the table has them
//   positions [B]            how many positions they hold, for every key head
struct Select {
    const int8_t *Q, *means;
    const float *sQ, *s_means;
    const int32_t *tables, *lens;
    uint64_t* keys;  // [B, Hkv, max_blocks]: the scores in an order that integers compare
    int32_t *selected, *pages, *positions;
    int B, Hq, Hkv, D, num_pages, log2_page, max_pages, max_context, max_blocks, top;
};
int launch_select(const Select& s, hipStream_t stream);

// Byte offsets of its arrays in a workspace, and their end.
struct SelectSpace {
    size_t keys, pages, positions, bytes;
};
inline SelectSpace select_space(int B, int kv_heads, int max_context, int page_size, int top) {
    const size_t rows = (size_t)B * kv_heads;
    SelectSpace s{};
    s.pages = round_up(rows * (size_t)ceil_div(max_context, page_size) * sizeof(uint64_t), kWorkspaceAlign);
    s.positions = s.pages + round_up(rows * top * sizeof(int32_t), kWorkspaceAlign);
    s.bytes = s.positions + round_up((size_t)B * sizeof(int32_t), kWorkspaceAlign);
    return s;
}

}  // namespace int8k
