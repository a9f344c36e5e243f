// The drafted tokens that a model agrees with, and their cache rows moved together (gfx950).
//
// Node 0 of a sequence is its last chosen token and counts always. From it a walk goes down: to the child, lowest number
// first, whose token is the model's choice at the node. The c nodes of the walk, in order i_0 = 0 < i_1 < ..., keep
// their keys and values: cache row held + i_j moves to held + j, codes and scales, in every layer.
//
// A workgroup takes a sequence in a layer, walks by itself (a wave tests 64 nodes at once; a step is some fifty cycles) and
// moves the rows: each thread a column of all rows, in order, so that no row is written before it is read (held + j <= held +
// i_j, and i grows). Bound by latency: the walk waits for its parents and tokens, the moves for their pages (one sequence of 8
// nodes in 16 layers 5.7 us; 128 sequences in 32 layers 27 us, 2.2 TB/s).
#include "draft_tree.h"

namespace kvfp8 {

namespace {

constexpr int kAcceptThreads = 256;
constexpr int kAcceptLayers = 64;     // of a launch: their addresses are arguments of 2 KB

struct AcceptArgs {
    TreeArgs t;
    const void* tokens;
    const void* best;
    int32_t tokens64, best64;
    int32_t layers;
    int32_t answers;                  // this launch writes counts, path and next tokens
    int64_t row_bytes, scale_bytes;   // of a token in k and v, in their scales
    int32_t unit;                     // bytes of an access to k and v: 16, 4 or 1
    int32_t* counts;
    int32_t* path;
    int64_t* next;
    void* cache[kAcceptLayers][4];    // k, v, k scales, v scales
};

// Rows src -> dst of a column `unit` bytes wide at byte `at`, eight rows of the path at a time.
template <typename U>
__device__ __forceinline__ void move_column(uint8_t* base, int64_t row_bytes, int64_t at, const int64_t* src, const int64_t* dst,
                                            int n) {
    for (int i = 0; i < n; i += 8) {
        U x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + k < n && src[i + k] >= 0) x[k] = *reinterpret_cast<const U*>(base + src[i + k] * row_bytes + at);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + k < n && src[i + k] >= 0) *reinterpret_cast<U*>(base + dst[i + k] * row_bytes + at) = x[k];
    }
}

__global__ void __launch_bounds__(kAcceptThreads)
accept_kernel(AcceptArgs a) {
    constexpr int kWords = kMaxNodes / 64;
    __shared__ int64_t src[kMaxNodes], dst[kMaxNodes];
    const int b = blockIdx.x, layer = blockIdx.y, lane = threadIdx.x & 63;
    const int64_t r0 = tree_row(a.t, b), r1 = tree_row(a.t, b + 1), raw = r1 > r0 ? r1 - r0 : 0;
    const int32_t nodes = (int32_t)(raw < a.t.max_nodes ? raw : a.t.max_nodes);
    // Node 64 w + lane of the sequence.
    int32_t parent[kWords];
    int64_t token[kWords], choice[kWords];
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
        const int i = 64 * w + lane;
        parent[w] = -1;
        token[w] = choice[w] = 0;
        if (i < nodes) {
            const int64_t p = load_i(a.t.parents, a.t.parents64, r0 + i);
            parent[w] = p >= 0 && p < i ? (int32_t)p : -1;
            token[w] = load_i(a.tokens, a.tokens64, r0 + i);
            choice[w] = load_i(a.best, a.best64, r0 + i);
        }
    }
    uint64_t kept[kWords] = {};
    int32_t count = 0, at = nodes > 0 ? 0 : -1;
    int64_t wanted = -1;
    while (at >= 0) {                                    // at grows: at most `nodes` steps
        int64_t here = 0;
#pragma unroll
        for (int w = 0; w < kWords; ++w)
            if (at >> 6 == w) {
                kept[w] |= 1ull << (at & 63);
                here = choice[w];
            }
        wanted = __shfl((long long)here, at & 63);
        ++count;
        int32_t child = -1;
#pragma unroll
        for (int w = kWords - 1; w >= 0; --w) {
            const uint64_t hit = __ballot(parent[w] == at && token[w] == wanted);
            if (hit != 0) child = 64 * w + __builtin_ctzll(hit);
        }
        at = uniform(child);
    }
    if (a.answers && layer == 0) {
        if (threadIdx.x == 0) {
            a.counts[b] = count;
            a.next[b] = wanted;
        }
        // Entry j of the path is the number of its j-th bit: each kept node writes its own.
        for (int i = threadIdx.x; i < a.t.max_nodes; i += kAcceptThreads)
            if (i >= count) a.path[(int64_t)b * a.t.max_nodes + i] = -1;
    }
    const int64_t len = load_i(a.t.d.ctx, a.t.d.ctx64, b), slot = load_i(a.t.d.slots, a.t.d.slots64, b);
    const int64_t held = len - raw, cap = a.t.d.bt_width * a.t.d.block_size;
    const bool ok = slot >= 0 && slot < a.t.d.bt_rows && held >= 0;
    auto row_of = [&](int64_t pos) -> int64_t {
        if (!ok || pos >= cap) return -1;
        const int64_t page = a.t.d.block_table[slot * a.t.d.bt_width + (pos >> a.t.d.bs_shift)];
        return page >= 0 && page < a.t.d.num_blocks ? page * a.t.d.block_size + (pos & (a.t.d.block_size - 1)) : -1;
    };
    {
        const int i = threadIdx.x;                       // a node each
        uint64_t mine = 0;
        int before = 0;
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            if (w < i >> 6) before += __builtin_popcountll(kept[w]);
            if (w == i >> 6) mine = kept[w];
        }
        if ((mine >> (i & 63)) & 1) {
            before += __builtin_popcountll(mine & ((1ull << (i & 63)) - 1));
            if (a.answers && layer == 0) a.path[(int64_t)b * a.t.max_nodes + before] = i;
            int64_t from = -1, to = -1;
            if (a.layers > 0 && before != i) {
                from = row_of(held + i);
                to = row_of(held + before);
            }
            src[before] = to >= 0 ? from : -1;           // negative: stays
            dst[before] = to;
        }
    }
    __syncthreads();
    if (layer >= a.layers) return;
    const int64_t columns = a.row_bytes / a.unit, scales = a.scale_bytes / 4;
    for (int64_t c = threadIdx.x; c < 2 * (columns + scales); c += kAcceptThreads) {
        if (c < 2 * columns) {
            const int tensor = c >= columns;
            uint8_t* const base = reinterpret_cast<uint8_t*>(a.cache[layer][tensor]);
            const int64_t x = (tensor ? c - columns : c) * a.unit;
            if (a.unit == 16) move_column<uint4>(base, a.row_bytes, x, src, dst, count);
            else if (a.unit == 4) move_column<uint32_t>(base, a.row_bytes, x, src, dst, count);
            else move_column<uint8_t>(base, a.row_bytes, x, src, dst, count);
        } else {
            const int64_t y = c - 2 * columns;
            const int tensor = y >= scales;
            move_column<uint32_t>(reinterpret_cast<uint8_t*>(a.cache[layer][2 + tensor]), a.scale_bytes, 4 * (tensor ? y - scales : y), src,
                                  dst, count);
        }
    }
}

bool accept_index(int t) { return t == KVFP8_I32 || t == KVFP8_I64; }

}  // namespace

}  // namespace kvfp8

using namespace kvfp8;

extern "C" int kvfp8_accept_draft(const void* tokens, int tokens_dtype, const void* best, int best_dtype, const void* starts,
                                  int starts_dtype, const void* parents, int parents_dtype, int64_t rows, int32_t seqs,
                                  int32_t max_nodes, const void* slots, int slots_dtype, const void* context_lengths,
                                  int ctx_dtype, const int32_t* block_table, int64_t bt_rows, int64_t bt_width,
                                  int64_t num_blocks, int32_t block_size, void* const* caches, int32_t layers,
                                  int64_t row_bytes, int64_t scale_bytes, int32_t* counts, int32_t* path,
                                  int64_t* next_tokens, void* stream) {
    if (!accept_index(tokens_dtype) || !accept_index(best_dtype) || !accept_index(starts_dtype) || !accept_index(parents_dtype) ||
        !accept_index(slots_dtype) || !accept_index(ctx_dtype))
        return KVFP8_EDTYPE;
    if (rows < 0 || seqs < 0 || max_nodes <= 0 || layers < 0 || bt_rows <= 0 || bt_width <= 0 || num_blocks <= 0 || block_size <= 0 ||
        (block_size & (block_size - 1)) != 0 || row_bytes <= 0 || scale_bytes < 0 || scale_bytes % 4 != 0)
        return KVFP8_ESHAPE;
    // A launch has fewer than 2^32 threads, of 256 for each sequence and layer.
    if (max_nodes > kMaxNodes || rows > INT32_MAX || seqs >= 1 << 17 || bt_width > INT64_MAX / block_size ||
        num_blocks > INT64_MAX / block_size / row_bytes)
        return KVFP8_ELIMIT;
    if (seqs == 0) return KVFP8_OK;
    if (!starts || !slots || !context_lengths || !block_table || !counts || !path || !next_tokens || (layers > 0 && !caches))
        return KVFP8_ENULL;
    if (rows > 0 && (!tokens || !best || !parents)) return KVFP8_ENULL;
    uintptr_t bits = (uintptr_t)row_bytes;
    for (int32_t i = 0; i < layers; ++i) {
        for (int t = 0; t < (scale_bytes > 0 ? 4 : 2); ++t)
            if (caches[4 * i + t] == nullptr) return KVFP8_ENULL;
        bits |= (uintptr_t)caches[4 * i] | (uintptr_t)caches[4 * i + 1];
        if (scale_bytes > 0 && (((uintptr_t)caches[4 * i + 2] | (uintptr_t)caches[4 * i + 3]) & 3) != 0) return KVFP8_ESTRIDE;
    }
    AcceptArgs a = {};
    a.t.rows = rows;
    a.t.starts = starts;
    a.t.parents = parents;
    a.t.starts64 = starts_dtype == KVFP8_I64;
    a.t.parents64 = parents_dtype == KVFP8_I64;
    a.t.seqs = seqs;
    a.t.max_nodes = max_nodes;
    a.t.d.num_blocks = num_blocks;
    a.t.d.block_size = block_size;
    while ((1 << a.t.d.bs_shift) < block_size) ++a.t.d.bs_shift;
    a.t.d.block_table = block_table;
    a.t.d.bt_rows = bt_rows;
    a.t.d.bt_width = bt_width;
    a.t.d.slots = slots;
    a.t.d.ctx = context_lengths;
    a.t.d.slots64 = slots_dtype == KVFP8_I64;
    a.t.d.ctx64 = ctx_dtype == KVFP8_I64;
    a.tokens = tokens;
    a.best = best;
    a.tokens64 = tokens_dtype == KVFP8_I64;
    a.best64 = best_dtype == KVFP8_I64;
    a.row_bytes = row_bytes;
    a.scale_bytes = scale_bytes;
    a.unit = bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 1);
    a.counts = counts;
    a.path = path;
    a.next = next_tokens;
    int32_t done = 0;
    do {
        a.layers = layers - done < kAcceptLayers ? layers - done : kAcceptLayers;
        a.answers = done == 0;
        for (int32_t i = 0; i < a.layers; ++i)
            for (int t = 0; t < 4; ++t) a.cache[i][t] = scale_bytes > 0 || t < 2 ? caches[4 * (done + i) + t] : nullptr;
        hipLaunchKernelGGL(accept_kernel, dim3((unsigned)seqs, (unsigned)(a.layers > 0 ? a.layers : 1)), dim3(kAcceptThreads), 0,
                           reinterpret_cast<hipStream_t>(stream), a);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return (int)err;
        done += a.layers;
    } while (done < layers);
    return KVFP8_OK;
}
