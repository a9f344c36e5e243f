// The matrix-core path of tree attention: which calls it takes, how many items they have at most, and its launches.
#pragma once

#include "draft_tree.h"

namespace kvfp8 {

bool tree_mfma_supported(int32_t head_dim, int32_t block_size, int q_dtype, int kv_dtype);

struct TreePlan {
    int32_t block_rows, target;
    int64_t items;                    // at most
    int64_t part_l, part_acc, bytes;  // float32 states of block_rows pairs an item: m at 0, l and acc at these byte offsets
};
TreePlan tree_mfma_plan(int32_t seqs, int32_t max_nodes, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int q_dtype);

// Workgroups for so many items: whole runs of every XCD.
inline int64_t tree_grid(int64_t items) {
    const int64_t turn = kXcdCount * kXcdRun;
    return (items + turn - 1) / turn * turn;
}

// 16-bit q (tree_attention_blocks.hip).
template <int QT>
hipError_t launch_tree_blocks(const TreeArgs& a, int kv_dtype, int64_t items, hipStream_t s);

template <int QT>
hipError_t launch_tree_mfma(TreeArgs a, int kv_dtype, const TreePlan& p, void* workspace, hipStream_t s);

}  // namespace kvfp8
