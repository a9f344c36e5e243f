// Shared pieces of the shared-prefix attention kernels: arguments, the lookup of a row's group, and
// the softmax states that the kernels leave for the merge.
#pragma once

#include "kvfp8_decode_common.h"

namespace kvfp8 {

// Rows of q are the sequences' new tokens (decode form: row = sequence, `d.slots`/`d.ctx` name its own
// pages) or packed prompt tokens (prompt form: `cu` delimits the sequences; out and lse hold the
// attention over the prompts themselves). Group g holds sequences [starts[g], starts[g + 1]); its
// prefix is the first p_lens[g] tokens on block-table row p_slots[g].
struct PrefixArgs {
    DecodeArgs d;
    int64_t rows;
    const void* p_slots;
    const void* p_lens;
    const void* p_starts;
    int32_t p_slots64, p_lens64, p_starts64;
    int32_t groups;
    const void* cu;             // null: decode form
    int32_t cu64;
    int32_t seqs;
    int32_t max_len;            // prompt form: rows of a sequence past it are left alone
    int32_t splits;             // states per row of its prefix, and of its own tokens (matrix-core path, decode
    int32_t own_splits;         // form) behind them: [splits + own_splits][rows][Hq] in d.part_*
    int32_t step_shift;         // splits hold whole steps of 1 << step_shift tokens
    float* lse;                 // prompt form [rows, Hq]
};

// Prefix tokens of group g, clipped to what the block table addresses; 0 for a slot outside it.
__device__ __forceinline__ int64_t group_tokens(const PrefixArgs& a, int g, int64_t* slot_out) {
    const int64_t slot = load_i(a.p_slots, a.p_slots64, g);
    const int64_t raw = load_i(a.p_lens, a.p_lens64, g);
    const int64_t cap = a.d.bt_width * a.d.block_size;
    *slot_out = slot;
    if (slot < 0 || slot >= a.d.bt_rows || raw < 0) return 0;
    return raw < cap ? raw : cap;
}

// Last i in [0, n) with p[i] <= x (0 where there is none), p not decreasing.
__device__ __forceinline__ int last_at_most(const void* p, int is64, int n, int64_t x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (load_i(p, is64, mid) <= x) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// The group of sequence b, -1 where it is in none.
__device__ __forceinline__ int group_of_seq(const PrefixArgs& a, int64_t b) {
    if (a.groups <= 0) return -1;
    const int g = last_at_most(a.p_starts, a.p_starts64, a.groups, b);
    return load_i(a.p_starts, a.p_starts64, g) <= b && b < load_i(a.p_starts, a.p_starts64, g + 1) ? g : -1;
}

// The sequence of a row; -1 for a prompt row of no sequence or past max_len of its own.
__device__ __forceinline__ int64_t seq_of_row(const PrefixArgs& a, int64_t row) {
    if (a.cu == nullptr) return row;
    const int b = last_at_most(a.cu, a.cu64, a.seqs, row);
    const int64_t s0 = load_i(a.cu, a.cu64, b);
    return s0 <= row && row < load_i(a.cu, a.cu64, b + 1) && row - s0 < a.max_len ? b : -1;
}

// Tokens per split of n tokens: equal runs of whole steps (1 << step_shift tokens), the last ones shorter
// or empty. Splits from split_count on are empty.
__device__ __forceinline__ int64_t split_tokens(int64_t n, int step_shift, int splits) {
    const uint32_t steps = (uint32_t)((n + (1 << step_shift) - 1) >> step_shift);
    return (int64_t)((steps + splits - 1) / (uint32_t)splits) << step_shift;
}
__device__ __forceinline__ int split_count(int64_t n, int64_t per) { return n > 0 ? (int)((uint32_t)(n + per - 1) / (uint32_t)per) : 0; }

__device__ __forceinline__ int64_t prefix_part(const PrefixArgs& a, int64_t row, int s, int hq) {
    return (s * a.rows + row) * a.d.num_q_heads + hq;
}

// The matrix-core path: whether its prefix kernel takes these types and sizes (cache and q pointers are
// checked by the call), and where its workspace holds what (byte offsets).
bool prefix_mfma_supported(int32_t head_dim, int32_t block_size, int q_dtype, int kv_dtype);

struct PrefixMfmaPlan {
    int32_t rows;                     // pairs per row block: 16 or 256
    int32_t blocks;                   // row blocks, at most
    int32_t splits, step_shift;       // of a prefix
    int32_t own_groups, own_heads, own_blocks, own_splits;        // decode form, as in PrefixGrid
    int32_t per_xcd, tail_from, tail_splits;                      // as in PrefixGrid
    int64_t states;                   // float32 states: m at 0, l and acc at these byte offsets
    int64_t part_l, part_acc, bytes;
};
PrefixMfmaPlan prefix_mfma_plan(int64_t rows, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t groups,
                                int64_t bt_width, int32_t block_size, int q_dtype, bool prompt);

// Workgroups of the launch that leaves states: those of the prefixes, then those of the own tokens.
struct PrefixGrid {
    int32_t blocks;                   // row blocks, at most
    int32_t total;                    // items of the prefixes: blocks x KV heads x splits
    int32_t per_xcd;                  // total / 8, rounded up
    int32_t tail_from, tail_splits;   // an XCD's items from this one on are split (prompt form, else none: per_xcd, 1)
    int32_t prefix_groups;            // workgroups of the prefixes: 8 (tail_from + (per_xcd - tail_from) tail_splits)
    int32_t own_groups;               // workgroups of the own tokens
    int32_t own_heads;                // KV heads of one of them
    int32_t own_blocks;               // blocks of 16 q heads of a KV head
    int32_t q_vec;                    // q rows are 16-byte aligned
};

template <int QT>
hipError_t launch_prefix_wide(const PrefixArgs& a, int kv_dtype, const PrefixGrid& g, hipStream_t s);

template <int QT>
hipError_t launch_prefix_mfma(PrefixArgs a, int kv_dtype, const PrefixMfmaPlan& p, void* workspace, hipStream_t s);

}  // namespace kvfp8
