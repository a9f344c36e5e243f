// Shared pieces of the draft-tree kernels: arguments, a sequence's nodes and tokens, which nodes are above which, and how a
// batch is cut into work items on the device.
#pragma once

#include "paged_operands.h"
#include "kvfp8_decode_common.h"

namespace kvfp8 {

constexpr int kMaxNodes = 256;        // of a sequence
constexpr int kNodeWords = kMaxNodes / 32;

// Rows of q are the drafted nodes, packed: sequence b has rows [starts[b], starts[b + 1]), of which the first max_nodes are
// computed. d.slots and d.ctx: its block-table row, and its tokens in the cache with the nodes as the last ones.
struct TreeArgs {
    DecodeArgs d;
    int64_t rows;
    const void* starts;
    const void* parents;
    int32_t starts64, parents64;
    int32_t seqs, max_nodes;
    int32_t block_rows;               // (node, q head) pairs of a KV head in a row block
    int32_t target;                   // items that run at once
    int32_t q_vec;                    // q rows are 16-byte aligned
};

namespace {

constexpr int kStep = 64;             // chunks hold whole steps
constexpr int kXcdCount = 8;          // workgroups are dispatched round-robin over the XCDs
constexpr int kXcdRun = 8;            // neighbouring items of an XCD

struct TreeSeq {
    int32_t row0, nodes;              // first row, computed nodes
    int32_t tokens;                   // in the cache, as far as the block table addresses them
    int32_t held;                     // tokens before the nodes
    int64_t slot;                     // of a table of less than 2^31 rows, where there are tokens
};

// Element i of int32 or int64 numbers as two 32-bit loads without a branch, so that several are in flight at once.
__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
    const int32_t* const at = reinterpret_cast<const int32_t*>(p) + (is64 ? 2 * i : i);
    const int32_t lo = at[0], up = at[is64 ? 1 : 0];
    return ((int64_t)(is64 ? up : lo >> 31) << 32) | (uint32_t)lo;
}

__device__ __forceinline__ int64_t tree_row(const TreeArgs& a, int64_t i) {
    const int64_t x = index_at(a.starts, a.starts64, i);
    return x < 0 ? 0 : (x > a.rows ? a.rows : x);
}

// Sequence b. A slot outside the table, or fewer tokens than nodes: no tokens.
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& a, int b) {
    TreeSeq s;
    const int64_t r0 = tree_row(a, b), r1 = tree_row(a, b + 1), len = index_at(a.d.ctx, a.d.ctx64, b);
    const int64_t nodes = r1 > r0 ? r1 - r0 : 0, cap = a.d.bt_width * a.d.block_size;
    s.slot = index_at(a.d.slots, a.d.slots64, b);
    const bool ok = s.slot >= 0 && s.slot < a.d.bt_rows && len >= nodes;
    s.row0 = (int32_t)r0;
    s.nodes = (int32_t)(nodes < a.max_nodes ? nodes : a.max_nodes);
    s.tokens = (int32_t)(ok ? (len < cap ? len : cap) : 0);
    s.held = (int32_t)(ok ? (len - nodes < cap ? len - nodes : cap) : 0);
    return s;
}

// Which nodes are above which, as bits: node i sees the nodes of words[i]. Whole workgroup, at least kMaxNodes threads. A
// node's parent is a node before it; any other number makes it a root. Nodes above are found in rounds, each of which
// doubles how far up they are known, as many as the deepest needs.
struct TreeMasks {
    uint32_t words[kMaxNodes][kNodeWords + 1];           // (an odd stride: rows in different banks; the last word is 0)
    int32_t up[kMaxNodes];
};

__device__ __forceinline__ void build_masks(TreeMasks& m, const TreeArgs& a, const TreeSeq& s) {
    const int i = threadIdx.x;
    const bool mine = i < s.nodes;
    if (mine) {
        const int64_t p = load_i(a.parents, a.parents64, (int64_t)s.row0 + i);
        m.up[i] = p >= 0 && p < i ? (int32_t)p : -1;
#pragma unroll
        for (int w = 0; w <= kNodeWords; ++w) m.words[i][w] = w == i / 32 ? 1u << (i & 31) : 0u;
    }
    __syncthreads();
    for (;;) {
        const int up = mine ? m.up[i] : -1;
        uint32_t more[kNodeWords];
        int next = -1;
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < kNodeWords; ++w) more[w] = m.words[up][w];
            next = m.up[up];
        }
        if (!__syncthreads_or(up >= 0)) break;           // a node's root is reached in at most 8 rounds
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < kNodeWords; ++w) m.words[i][w] |= more[w];
            m.up[i] = next;
        }
        __syncthreads();
    }
}

// Bit t: token `first` + t counts for node i (t < 32; first and held are wave-uniform).
__device__ __forceinline__ uint32_t node_bits(const TreeMasks& m, int i, int32_t first, int32_t held) {
    const int32_t at = first - held;
    if (at <= -32) return ~0u;
    if (at < 0) return (m.words[i][0] << -at) | ((1u << -at) - 1u);
    const int w = at >> 5;
    if (w >= kNodeWords) return 0u;
    return (uint32_t)((((uint64_t)m.words[i][w + 1] << 32) | m.words[i][w]) >> (at & 31));
}

// How a batch is cut. A sequence has columns (row block, KV head) and steps of kStep tokens; a chunk is `chunk` steps of a
// column. Items are numbered sequence by sequence, in a sequence chunk by chunk, in a chunk head by head: the row blocks
// that read the same tokens are neighbours.
struct TreeCut {
    TreeSeq s;                        // lane's of the first 64 sequences
    int32_t chunk;                    // steps of a chunk
    int32_t total;                    // items
};
struct TreeItem {
    TreeSeq s;
    int32_t first;                    // number of the sequence's first item
    int32_t first_state;              // where the states of its items begin, which sequences of several chunks have
    int32_t blocks;                   // row blocks of the sequence
    int32_t chunks;                   // of its columns
};

// The sum of the lanes up to this one, by DPP: rows of 16 lanes, then their ends carried on (row_shr 1, 2, 4, 8, row_bcast 15, 31).
__device__ __forceinline__ int32_t sum_up_to(int32_t x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return x;
}
__device__ __forceinline__ int32_t lanes_sum(int32_t x) { return __builtin_amdgcn_readlane(sum_up_to(x), 63); }

__device__ __forceinline__ TreeSeq lane_seq(const TreeArgs& a, int b0) {
    const int b = b0 + (threadIdx.x & 63);
    TreeSeq s = tree_seq(a, min(b, a.seqs - 1));
    if (b >= a.seqs) s.nodes = s.tokens = 0;
    return s;
}
__device__ __forceinline__ int32_t tree_blocks(const TreeArgs& a, const TreeSeq& s) {
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    return s.tokens > 0 ? (int32_t)((uint32_t)(s.nodes * G + a.block_rows - 1) / (uint32_t)a.block_rows) : 0;
}
// 64 sequences, the longest ones first where they have more columns than run at once: items are dispatched in their order, and what
// begins last is to be short. Each lane finds its sequence's rank by comparison and hands it to the lane of that rank. (61 sequences
// of 1 to 3060 tokens and 1 to 60 nodes: 118 us in their own order, 105 in this. The sort costs 2 us, for nothing with fewer columns.)
__device__ __forceinline__ TreeSeq sorted_seq(const TreeArgs& a, int b0) {
    const int lane = threadIdx.x & 63, count = min(64, a.seqs - b0);
    const TreeSeq s = lane_seq(a, b0);
    if (lanes_sum(tree_blocks(a, s)) * a.d.num_kv_heads <= a.target) return s;
    const uint32_t key = (uint32_t)((s.tokens + kStep - 1) / kStep) * 64 + (63 - lane);        // below 2^32, no two alike
    int rank = 0;
    for (int i = 0; i < count; ++i) rank += (uint32_t)__builtin_amdgcn_readlane((int32_t)key, i) > key;
    if (lane >= count) rank = lane;
    TreeSeq sorted;
    sorted.row0 = __builtin_amdgcn_ds_permute(4 * rank, s.row0);
    sorted.nodes = __builtin_amdgcn_ds_permute(4 * rank, s.nodes);
    sorted.tokens = __builtin_amdgcn_ds_permute(4 * rank, s.tokens);
    sorted.held = __builtin_amdgcn_ds_permute(4 * rank, s.held);
    sorted.slot = __builtin_amdgcn_ds_permute(4 * rank, (int32_t)s.slot);
    return sorted;
}
__device__ __forceinline__ int32_t tree_chunks(const TreeSeq& s, int32_t chunk) {
    return (int32_t)((uint32_t)((s.tokens + kStep - 1) / kStep + chunk - 1) / (uint32_t)chunk);
}

// A wave looks through 64 sequences at once, each in its lane; every wave of the call finds the same. Chunks are as short
// as the work divided by the items that run at once, and up to 1.5 times that while there are more items than those (up to
// 64 sequences).
__device__ __forceinline__ TreeCut cut_batch(const TreeArgs& a) {
    TreeCut c;
    c.s = sorted_seq(a, 0);
    uint64_t work = 0;
    TreeSeq s = c.s;
    for (int b0 = 0;;) {
        const uint64_t mine = (uint64_t)tree_blocks(a, s) * (uint32_t)tree_chunks(s, 1);       // below 2^48
        work += (uint32_t)lanes_sum((int32_t)(mine & 0xFFFFFFu)) + ((uint64_t)(uint32_t)lanes_sum((int32_t)(mine >> 24)) << 24);
        b0 += 64;
        if (b0 >= a.seqs) break;
        s = sorted_seq(a, b0);
    }
    work *= (uint32_t)a.d.num_kv_heads;
    const uint64_t even = (work + a.target - 1) / (uint32_t)a.target;
    // (Never more than a table's 2^25 steps.)
    const int32_t least = (int32_t)(even < 1 ? 1 : (even < (1ull << 25) ? even : 1ull << 25));
    auto items = [&](int32_t chunk) __attribute__((always_inline)) {
        int32_t n = 0;
        TreeSeq s = c.s;
        for (int b0 = 0;;) {
            n += tree_blocks(a, s) * tree_chunks(s, chunk);
            b0 += 64;
            if (b0 >= a.seqs) break;
            s = sorted_seq(a, b0);
        }
        return lanes_sum(n) * a.d.num_kv_heads;
    };
    c.chunk = least;
    c.total = items(least);
    // With as many columns as that no chunk helps.
    if (a.seqs <= 64 && c.total > a.target && lanes_sum(tree_blocks(a, c.s)) * a.d.num_kv_heads <= a.target) {
        for (int i = 1; i <= 8; ++i) {
            const int32_t chunk = least + (least * i + 15) / 16, n = items(chunk);
            if (n > a.target) continue;
            c.chunk = chunk;
            c.total = n;
            break;
        }
    }
    return c;
}

// The sequence that holds item `index` (kByRow: that computes row `index`); false without one.
template <bool kByRow>
__device__ __forceinline__ bool find_tree_item(const TreeArgs& a, const TreeCut& c, int32_t index, TreeItem& it) {
    int32_t before = 0, before_states = 0;
    TreeSeq s = c.s;
    for (int b0 = 0;;) {
        const int32_t blocks = tree_blocks(a, s), chunks = tree_chunks(s, c.chunk), items = blocks * a.d.num_kv_heads * chunks;
        const int32_t states = chunks > 1 ? items : 0;
        const int32_t incl = sum_up_to(items), incl_states = sum_up_to(states);
        const int32_t first = before + incl - items;
        const uint64_t hit = __ballot(kByRow ? index >= s.row0 && index - s.row0 < s.nodes : index >= first && index - first < items);
        if (hit != 0) {
            const int at = __builtin_ctzll(hit);
            it.s.row0 = __builtin_amdgcn_readlane(s.row0, at);
            it.s.nodes = __builtin_amdgcn_readlane(s.nodes, at);
            it.s.tokens = __builtin_amdgcn_readlane(s.tokens, at);
            it.s.held = __builtin_amdgcn_readlane(s.held, at);
            it.s.slot = __builtin_amdgcn_readlane((int32_t)s.slot, at);
            it.blocks = __builtin_amdgcn_readlane(blocks, at);
            it.chunks = __builtin_amdgcn_readlane(chunks, at);
            it.first = __builtin_amdgcn_readlane(first, at);
            it.first_state = before_states + __builtin_amdgcn_readlane(incl_states - states, at);
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
        before_states += __builtin_amdgcn_readlane(incl_states, 63);
        b0 += 64;
        if (b0 >= a.seqs) return false;
        s = sorted_seq(a, b0);
    }
}

// What a workgroup does: pairs (node, q head of KV head h) from r0 on against the tokens [lo, hi).
struct TreeWork {
    TreeItem it;
    int32_t state;                    // number of the item's states, where its sequence has several chunks
    int32_t h, r0, pairs, lo, hi;
    const int32_t* table;             // block-table row
};

// The item of this workgroup; false without one. Each XCD takes runs of neighbouring items in turn: row blocks meet their tokens in
// the same L2, and long sequences spread over all XCDs. (Single items: 427 us instead of 415 for 8 sequences of 32768 tokens and
// four row blocks; one run an XCD: 111 instead of 100 for 61 ragged ones.)
__device__ __forceinline__ bool tree_work(const TreeArgs& a, TreeWork& w) {
    const TreeCut c = cut_batch(a);
    const uint32_t local = blockIdx.x / kXcdCount, turn = local / (uint32_t)kXcdRun;
    const int32_t index = (int32_t)((turn * kXcdCount + blockIdx.x % kXcdCount) * kXcdRun + (local - turn * kXcdRun));
    if (index >= uniform(c.total) || !find_tree_item<false>(a, c, index, w.it)) return false;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    uint32_t rest = (uint32_t)(index - w.it.first);
    w.state = w.it.first_state + (int32_t)rest;
    const uint32_t column = rest / (uint32_t)w.it.blocks;
    w.r0 = (int32_t)(rest - column * (uint32_t)w.it.blocks) * a.block_rows;
    rest = column / (uint32_t)a.d.num_kv_heads;
    w.h = (int32_t)(column - rest * (uint32_t)a.d.num_kv_heads);
    w.pairs = w.it.s.nodes * G;
    const int64_t per = (int64_t)uniform(c.chunk) * kStep, lo = rest * per;
    w.lo = uniform((int32_t)lo);
    w.hi = uniform((int32_t)min(lo + per, (int64_t)w.it.s.tokens));
    w.table = a.d.block_table + uniform64(w.it.s.slot) * a.d.bt_width;
    return true;
}

// Whether a dword holds a value that is not finite: codes 0x7F and 0xFF, or a 16-bit exponent of ones.
template <int ES, bool kF16>
__device__ __forceinline__ bool not_finite(uint32_t x) {
    if constexpr (ES == 1) return (((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
    constexpr uint32_t kInf = kF16 ? 0x7C00u : 0x7F80u;
    return (x & 0x7FFFu) >= kInf || ((x >> 16) & 0x7FFFu) >= kInf;
}

// Pages of the two 16-token tiles of a step. They are read a step before their rows (scalar loads, whose wait leaves the
// rows in flight alone), and there is no branch around the loads of a step: with one, the compiler could not count the
// loads in flight and would wait for all of them. A tile past the end has the chunk's first page, and counts nothing.
struct StepPages {
    int32_t a, b;
};
struct StepRefs {
    TileRef a, b;
};
__device__ __forceinline__ StepPages step_pages(const TreeArgs& a, const TreeWork& w, int32_t t0) {
    auto page = [&](int32_t tok) __attribute__((always_inline)) {
        const int64_t addr = uniform64((int64_t)(uintptr_t)(w.table + ((tok < w.hi ? tok : w.lo) >> a.d.bs_shift)));
        return *(const_i32_ptr)(uintptr_t)addr;
    };
    t0 = uniform(t0);
    return StepPages{page(t0), page(t0 + 16)};
}
__device__ __forceinline__ StepRefs step_refs(const TreeArgs& a, const TreeWork& w, const StepPages& p, int32_t t0) {
    auto ref = [&](int32_t page, int32_t tok) __attribute__((always_inline)) {
        page = uniform(page);
        const bool ok = page >= 0 && page < a.d.num_blocks && tok < w.hi;
        return TileRef{ok ? (int64_t)page * a.d.block_size + (tok & (a.d.block_size - 1)) : 0, ok};
    };
    t0 = uniform(t0);
    return StepRefs{ref(p.a, t0), ref(p.b, t0 + 16)};
}

}  // namespace

}  // namespace kvfp8
