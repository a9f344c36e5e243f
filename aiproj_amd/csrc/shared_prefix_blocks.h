// Row blocks of the shared-prefix kernels: which rows, tokens and KV head a workgroup takes.
#pragma once

#include "decode_mfma_kernels.h"
#include "shared_prefix.h"

namespace kvfp8 {

namespace {

constexpr int kXcds = 8;              // workgroups are dispatched round-robin over the XCDs

// A row block: rows [rs, re) of q in group g, from pair r0 on.
struct RowBlock {
    int32_t g;
    int64_t rs, re;
    int64_t r0;
};

// First q row of group boundary i (entry i of starts).
__device__ __forceinline__ int64_t group_row(const PrefixArgs& a, int i) {
    int64_t b = load_i(a.p_starts, a.p_starts64, i);
    const int64_t seqs = a.cu == nullptr ? a.rows : a.seqs;
    b = b < 0 ? 0 : (b > seqs ? seqs : b);
    if (a.cu == nullptr) return b;
    const int64_t row = load_i(a.cu, a.cu64, b);
    return row < 0 ? 0 : (row > a.rows ? a.rows : row);
}

// Row block `index` of the groups' blocks in their order; false past the last one. Whole waves.
__device__ __forceinline__ bool find_block(const PrefixArgs& a, int32_t index, int rows_per_block, int heads, RowBlock& out) {
    const int lane = threadIdx.x & 63;
    int64_t left = index;
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
        const int g = g0 + lane;
        int64_t rs = 0, re = 0;
        if (g < a.groups) {
            rs = group_row(a, g);
            re = group_row(a, g + 1);
        }
        const int64_t blocks = re > rs ? ((re - rs) * heads + rows_per_block - 1) / rows_per_block : 0;
        int64_t incl = blocks;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int64_t y = __shfl_up((long long)incl, off);
            if (lane >= off) incl += y;
        }
        const uint64_t over = __ballot(incl > left);
        if (over != 0) {
            const int at = __builtin_ctzll(over);
            out.g = g0 + at;
            out.rs = uniform64(__shfl((long long)rs, at));
            out.re = uniform64(__shfl((long long)re, at));
            out.r0 = uniform64((left - __shfl((long long)(incl - blocks), at)) * rows_per_block);
            return true;
        }
        left -= __shfl((long long)incl, 63);
    }
    return false;
}

// What a workgroup does: a row block, a KV head and the tokens [lo, hi) of its prefix.
struct PrefixItem {
    RowBlock rb;
    int h, split;
    int64_t lo, hi;
    const int32_t* table;             // block-table row of the prefix
    int64_t pairs;                    // (row, q head) pairs of the group
};

// The item of this workgroup, false without one. Each XCD takes one run of (split, KV head, row block), so
// that the blocks of one head and split meet their tokens in the same L2.
__device__ __forceinline__ bool prefix_item(const PrefixArgs& a, const PrefixGrid& grid, int rows_per_block, PrefixItem& it) {
    const int32_t local = (int32_t)(blockIdx.x / kXcds);
    const int32_t index = (int32_t)(blockIdx.x % kXcds) * grid.per_xcd + local;
    if (index >= grid.total || local >= grid.per_xcd) return false;
    const int32_t unit = index / grid.blocks;
    it.h = unit % a.d.num_kv_heads;
    it.split = unit / a.d.num_kv_heads;
    const int G = a.d.num_q_heads / a.d.num_kv_heads;
    if (!find_block(a, index - unit * grid.blocks, rows_per_block, G, it.rb)) return false;
    int64_t slot;
    const int64_t tokens = group_tokens(a, it.rb.g, &slot);
    split_range(tokens, a.split_step, a.splits, it.split, &it.lo, &it.hi);
    if (it.lo >= it.hi) return false;
    it.lo = uniform64(it.lo);
    it.hi = uniform64(it.hi);
    it.table = a.d.block_table + uniform64(slot) * a.d.bt_width;
    it.pairs = (it.rb.re - it.rb.rs) * G;
    return true;
}

}  // namespace

}  // namespace kvfp8
