// blocks.h - argument blocks and launchers of rotary positions on several axes, the pages' key bounds, the choice of pages
// and the attention over chosen pages.
#pragma once

#include "ffkv_internal.h"

namespace ffkv
{

constexpr int kMaxAxes = 4;

struct RopeAxesArgs
{
    const void*    q;  // [batch, seq_len, num_heads, head_dim], q_stride elements from token to token; null without q
    const void*    k;
    const void*    v;      // null: rotate only
    void*          q_out;  // the same (may be q), out_stride of its own
    void*          k_out;  // rotate only; null: the rotated key goes to the pages alone
    void*          k_cache;  // null: rotate only
    void*          v_cache;
    float*         k_scale;
    float*         v_scale;
    const int32_t* block_table;
    const int32_t* context_lens;
    const int32_t* positions;  // [axes, batch, seq_len]
    int64_t        q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    double         rate_log2;  // log2 of the ratio of neighbouring pairs' frequencies: -2 log2(theta) / head_dim
    int            section_end[kMaxAxes];  // sections: first pair past axis a's; interleaved: pairs of axis a
    int            axes;
    int            interleaved;
    int            src_dtype;
    int            cache_dtype;
    int            batch;
    int            seq_len;
    int            num_heads;
    int            num_kv_heads;
    int            head_dim;
    int            max_blocks;
    int            num_blocks;
};

struct KeyBoundsArgs
{
    const void*    k_cache;
    const float*   k_scale;
    void*          bounds;  // [num_blocks, num_kv_heads, 2, head_dim]
    const int32_t* block_table;
    const int32_t* context_lens;
    int            cache_dtype;
    int            batch;
    int            new_tokens;
    int            num_kv_heads;
    int            head_dim;
    int            max_blocks;
    int            num_blocks;
};

struct SelectArgs
{
    const void*    q;       // [batch, seq_len, num_heads, head_dim]
    const void*    bounds;  // [num_blocks, num_kv_heads, 2, head_dim]
    const int32_t* block_table;
    const int32_t* context_lens;
    int32_t*       blocks;  // [batch, lists, num_kv_heads, count]
    float*         scores;  // workspace [batch, lists, num_kv_heads, stride]
    double*        query_sums;  // workspace [batch, lists, num_kv_heads, 2, head_dim] (select_by_lists)
    int64_t        stride;
    int            q_dtype;
    int            bounds_dtype;
    int            batch;
    int            seq_len;
    int            num_heads;
    int            num_kv_heads;
    int            group;
    int            head_dim;
    int            max_blocks;
    int            num_blocks;
    int            most_pages;  // of a row
    int            query_block;
    int            lists;  // per row: blocks of queries
    int            count;
    int            sinks;
    int            recent;
};

struct BlocksArgs
{
    const void*    q;  // [batch, seq_len, num_heads, head_dim]
    void*          out;
    const void*    k_cache;
    const void*    v_cache;
    const float*   k_scale;
    const float*   v_scale;
    const int32_t* block_table;
    const int32_t* context_lens;
    const int32_t* blocks;  // [batch, lists, num_kv_heads, count]
    int            qo_dtype;
    int            cache_dtype;
    int            batch;
    int            seq_len;
    int            num_heads;
    int            num_kv_heads;
    int            group;
    int            head_dim;
    int            max_blocks;
    int            num_blocks;
    int            query_block;
    int            lists;
    int            count;
    int            splits;  // pieces of a list, each by a workgroup of its own
    int            waves;   // of a workgroup
    bool           pair;    // the prefill: whole lists, by two halves of a workgroup
    float          scale_log2;
    int32_t*       ws_pieces;  // the prefill's pieces of each block of query rows
    float2*        ws_ml;   // [batch * seq_len * num_heads, splits]: (max in the log2 domain, denominator)
    float*         ws_acc;  // [batch * seq_len * num_heads, splits, head_dim]: unnormalised output
};

// i / n and i % n, in 32 bits: a workgroup's index is one (an int64 division is a hundred instructions and a branch).
struct Split
{
    uint32_t div;
    int      rem;
};
__device__ __forceinline__ Split split_index(uint32_t i, int n)
{
    const uint32_t d = i / static_cast<uint32_t>(n);
    return Split{d, static_cast<int>(i - d * static_cast<uint32_t>(n))};
}

// Which kernel attends: the decode's on the matrix cores (token by token), the prefill's (lists that many tokens share, at
// head_dim 64, 128 and 256), or the vector kernel (fp32 caches, other head dims).
enum class BlocksKernel
{
    kDecode,
    kPrefill,
    kVector,
};
BlocksKernel blocks_kernel(const BlocksArgs& a);
struct BlocksLayout
{
    int64_t ml, acc, total;  // byte offsets in the workspace, and its size (0: none)
};
BlocksLayout plan_blocks(BlocksArgs& a);
bool         blocks_pairable(const BlocksArgs& a);
void         set_blocks_workspace(BlocksArgs& a, const BlocksLayout& l, void* ws);

hipError_t launch_rope_axes(const RopeAxesArgs& a, hipStream_t stream);
hipError_t launch_key_bounds(const KeyBoundsArgs& a, hipStream_t stream);
bool       select_by_lists(int seq_len, int lists, int group);  // whether the choice takes query_sums
constexpr int64_t kMostThreads = UINT32_MAX;  // of a launch
// Threads of a call's largest launch (sizes, and for the choice most_pages, set).
int64_t    key_bounds_threads(const KeyBoundsArgs& a);
int64_t    select_threads(const SelectArgs& a);
int64_t    blocks_threads(const BlocksArgs& a);
bool       select_in_one(const SelectArgs& a);  // in one launch, without a workspace (a's sizes and most_pages set)
hipError_t launch_select(const SelectArgs& a, hipStream_t stream);
hipError_t launch_blocks(const BlocksArgs& a, hipStream_t stream);
hipError_t launch_blocks_prefill(const BlocksArgs& a, hipStream_t stream);

}  // namespace ffkv
