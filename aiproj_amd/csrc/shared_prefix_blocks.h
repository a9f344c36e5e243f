// Row blocks of the shared-prefix kernels: which rows, tokens and KV head a workgroup takes.
#pragma once

#include "paged_operands.h"
#include "shared_prefix.h"

namespace kvfp8 {

namespace {

constexpr int kXcds = 8;              // workgroups are dispatched round-robin over the XCDs

// What a workgroup does: pairs (token of q, q head of a KV head) of a group or sequence from r0 on, against the
// tokens [lo, hi) of its prefix or own pages.
struct PrefixItem {
    int32_t h;                        // (first) KV head
    int32_t part;                     // where the states go
    int32_t tail;                     // number of the row block among those split at the end, else -1
    int32_t rs;                       // first q row of the group
    int32_t pairs;                    // its pairs
    int32_t r0;                       // first pair of the block
    int32_t lo, hi;
    const int32_t* table;             // block-table row
};

// First q row of group boundary i (entry i of starts).
__device__ __forceinline__ int32_t group_row(const PrefixArgs& a, int i) {
    int64_t b = load_i(a.p_starts, a.p_starts64, i);
    const int64_t seqs = a.cu == nullptr ? a.rows : a.seqs;
    b = b < 0 ? 0 : (b > seqs ? seqs : b);
    if (a.cu == nullptr) return (int32_t)b;
    const int64_t row = load_i(a.cu, a.cu64, b);
    return (int32_t)(row < 0 ? 0 : (row > a.rows ? a.rows : row));
}

// Item `index` of the prefixes with the tokens of one of its `parts` (part -1: of none); false without one (rows,
// pairs and tokens are int32, checked on the host). A wave looks through 64 groups at once, every value of a group in
// its lane.
__device__ __forceinline__ bool find_item(const PrefixArgs& a, const PrefixGrid& grid, int rows_per_block, int32_t index,
                                          int32_t tail_part, PrefixItem& it, int32_t* tokens_out) {
    const int32_t unit = (uint32_t)index / (uint32_t)grid.blocks;
    const int32_t split = (uint32_t)unit / (uint32_t)a.d.num_kv_heads;
    const int32_t splits = it.tail < 0 ? a.splits : grid.tail_splits;
    it.part = it.tail < 0 ? split : tail_part;
    it.h = unit - split * a.d.num_kv_heads;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    int32_t left = index - unit * grid.blocks;
    const int lane = threadIdx.x & 63;
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
        const int g = min(g0 + lane, a.groups - 1);
        int64_t slot;
        const int32_t tokens = (int32_t)group_tokens(a, g, &slot);
        const int32_t rs = group_row(a, g), re = group_row(a, g + 1);
        const int32_t pairs = g0 + lane < a.groups && re > rs ? (re - rs) * G : 0;
        const int32_t blocks = (pairs + rows_per_block - 1) / rows_per_block;
        int32_t incl = blocks;
        if (a.groups > 1) {
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int32_t y = __shfl_up(incl, off);
                if (lane >= off) incl += y;
            }
        }
        const uint64_t over = __ballot(incl > left);
        if (over != 0) {
            const int at = __builtin_ctzll(over);
            it.rs = __builtin_amdgcn_readlane(rs, at);
            it.pairs = __builtin_amdgcn_readlane(pairs, at);
            it.r0 = (left - __builtin_amdgcn_readlane(incl - blocks, at)) * rows_per_block;
            const int32_t n = __builtin_amdgcn_readlane(tokens, at);
            if (tokens_out != nullptr) *tokens_out = n;
            const int64_t per = split_tokens(n, a.step_shift, splits);
            const int64_t lo = it.part * per;
            if (lo >= n) return false;
            it.lo = uniform((int32_t)lo);
            it.hi = uniform((int32_t)min(lo + per, (int64_t)n));
            // A group with tokens has its slot inside the table (below 2^26 rows).
            it.table = a.d.block_table + (int64_t)__builtin_amdgcn_readlane((int32_t)slot, at) * a.d.bt_width;
            return true;
        }
        left -= __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}

// The item of this workgroup. Each XCD takes one run of (split, KV head, row block), so that the blocks of one head
// and split meet their tokens in the same L2; those of a run that would leave CUs idle at its end are split.
__device__ __forceinline__ bool prefix_item(const PrefixArgs& a, const PrefixGrid& grid, int rows_per_block, PrefixItem& it) {
    const int32_t xcd = (int32_t)(blockIdx.x % kXcds);
    int32_t local = (int32_t)(blockIdx.x / kXcds), part = 0;
    it.tail = -1;
    if (local >= grid.tail_from) {
        const int32_t x = local - grid.tail_from, at = (uint32_t)x / (uint32_t)grid.tail_splits;
        part = x - at * grid.tail_splits;
        local = grid.tail_from + at;
        it.tail = xcd * (grid.per_xcd - grid.tail_from) + at;
    }
    const int32_t index = xcd * grid.per_xcd + local;
    if (index >= grid.total || local >= grid.per_xcd) return false;
    return find_item(a, grid, rows_per_block, index, part, it, nullptr);
}

// Own tokens: block of 16 q heads, KV heads and split of a sequence. Neighbouring workgroups take the heads of the
// same tokens.
__device__ __forceinline__ bool own_item(const PrefixArgs& a, const PrefixGrid& grid, PrefixItem& it) {
    uint32_t index = blockIdx.x - grid.prefix_groups;
    const uint32_t head_groups = (uint32_t)a.d.num_kv_heads / (uint32_t)grid.own_heads;
    uint32_t rest = index / head_groups;
    it.h = (int32_t)(index - rest * head_groups) * grid.own_heads;
    index = rest;
    rest = index / (uint32_t)a.own_splits;
    const int32_t split = (int32_t)(index - rest * (uint32_t)a.own_splits);
    index = rest;
    rest = index / (uint32_t)grid.own_blocks;
    it.r0 = 16 * (int32_t)(index - rest * (uint32_t)grid.own_blocks);
    it.rs = (int32_t)rest;
    it.pairs = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    it.part = a.splits + split;
    int64_t slot;
    const int32_t n = (int32_t)seq_tokens(a.d, it.rs, &slot);
    const int64_t per = split_tokens(n, 5, a.own_splits);
    const int64_t lo = split * per;
    if (lo >= n) return false;
    it.lo = uniform((int32_t)lo);
    it.hi = uniform((int32_t)min(lo + per, (int64_t)n));
    it.table = a.d.block_table + uniform64(slot) * a.d.bt_width;
    return true;
}

}  // namespace

}  // namespace kvfp8
