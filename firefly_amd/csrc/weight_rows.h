// weight_rows.h - how the attention weights' query rows (tokens of a row times the heads of a KV head) are cut into the blocks
// that a workgroup stages: plain arithmetic that the launcher and the kernels share.
#pragma once

#include <stdint.h>

namespace ffkv
{

// Query rows of a block: as many whole tiles of 16 as the call has, up to `most` (a multiple of 16), and one tile where it
// has none (a call without queries, which decays the earlier weights: the kernel divides by this).
constexpr int weight_block_rows(int64_t query_rows, int most)
{
    const int64_t rows = (query_rows + 15) / 16 * 16;
    return rows < 16 ? 16 : (rows < most ? static_cast<int>(rows) : most);
}

// Blocks of them; none without queries.
constexpr int weight_row_blocks(int query_rows, int block_rows) { return (query_rows + block_rows - 1) / block_rows; }

}  // namespace ffkv
