// Attention of drafted trees on the gfx950 matrix cores: float32 queries, and the join of all types.
//
// A call is two launches. In the first a workgroup takes an item: pairs (node, q head of a KV head) of a sequence against
// a chunk of its tokens. Its waves take steps of 32 tokens in turn, each with the pairs in registers, join in LDS and leave
// a softmax state, or the output where the sequence is one chunk. The second launch joins the states of a row. (16-bit queries:
// tree_attention_blocks.hip.)
#include "joined_state.h"
#include "shared_prefix_narrow.h"
#include "tree_attention.h"

namespace kvfp8 {

namespace {

constexpr int kTreeWaves = 8;

// Counts of a step that reaches the nodes: of the tokens that are there (FirstTokens) those whose bit is set for the row.
struct NodeTokens {
    FirstTokens first;
    uint32_t bits;                    // token t of the step
    static constexpr bool kByRow = true;
    __device__ __forceinline__ bool held(int i) const { return first.held(i); }
    __device__ __forceinline__ bool row(int i) const {
        return held(i) && ((bits >> (16 * (i >> 2) + 4 * first.j + (i & 3))) & 1u) != 0;
    }
};

// V of a step that some rows do not count: with a value that is not finite in it the products go token by token, and a
// row adds those of its own tokens alone.
template <int C>
struct NodeProducts {
    const DecodeArgs& d;
    int64_t row_a, row_b;             // first cache rows of the tiles
    int h, lane;

    template <int VW>
    __device__ __forceinline__ bool fits(const uint32_t (&v)[8][VW]) const {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int w = 0; w < VW; ++w) odd = odd || not_finite<1, false>(v[i][w]);
        return __ballot(odd) == 0;
    }
    __device__ __forceinline__ void add(RowState<C>& st, const float (&weight)[8], const bool (&live)[8]) const {
        constexpr int NB = 4 * C;
        const int m16 = lane & 15, j = lane >> 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            for (int g = 0; g < 4; ++g) {
                const float w = __shfl(weight[i], 16 * g + m16);
                if (__shfl((int)live[i], 16 * g + m16) == 0) continue;
                const int64_t row = (i < 4 ? row_a : row_b) + 4 * g + (i & 3);
                const int64_t at = (row * d.num_kv_heads + h) * d.head_dim;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const int dim = NB * (4 * j + e) + nb;
                        if (dim >= d.head_dim) continue;
                        st.o[nb][e] += w * decode_e4m3fn(reinterpret_cast<const uint8_t*>(d.v_cache)[at + dim]);
                    }
            }
        }
    }
};

// Blocks of 16 pairs, for float32 queries: in three bf16 parts, whose operands leave no registers for more pairs. Bound by
// the six products of a step: 32 sequences of 16 nodes and 4080 tokens, 32 / 8 heads of 128, 217 us (16-bit queries: 86).
template <int C>
__global__ void __launch_bounds__(64 * kTreeWaves)
tree_narrow_kernel(TreeArgs a) {
    constexpr int QT = KVFP8_F32, ES = 1;                // 16-bit caches come with q of their type
    using K = Kinds<QT, ES>;
    constexpr int NB = 4 * C, NW = kTreeWaves;
    __shared__ NarrowLds<C, NW> lds;
    __shared__ TreeMasks masks;
    TreeWork w;
    if (!tree_work(a, w)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int m16 = lane & 15, j = lane >> 4;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int D = a.d.head_dim;
    const int32_t hi = w.hi, held = w.it.s.held;

    PrefixStep<C, ES> buf0, buf1;
    constexpr int32_t stride = 32 * NW;
    int32_t tok = w.lo + 32 * wave;
    StepRefs r0 = step_refs(a, w, step_pages(a, w, tok), tok), r1;
    load_prefix_step<C, ES>(buf0, a.d, w.h, r0.a, r0.b, lane);
    StepPages next = step_pages(a, w, tok + stride);

    const int32_t pair = min(w.r0 + m16, w.pairs - 1), node = (uint32_t)pair / (uint32_t)G;
    const int hq = w.h * G + (pair - node * G);
    OpT<K::kF16> q[K::kQParts][2 * C];
    load_narrow_q<C, QT, ES>(reinterpret_cast<const float*>(a.d.q) + (int64_t)(w.it.s.row0 + node) * a.d.q_stride_b + hq * a.d.q_stride_h,
                             D, j, a.q_vec, q);
    if (hi > held) build_masks(masks, a, w.it.s);

    RowState<C> st;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) st.o[nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    st.m = kNegInf;
    st.l = 0.0f;
    // The steps before the nodes, then those that reach them.
    auto compute = [&](const PrefixStep<C, ES>& cur) __attribute__((always_inline)) {
        prefix_step<C, QT, ES, true>(st, cur, q, lds.stage[wave], lane, FirstTokens{j, 16, 16}, a.d.score_scale);
    };
    auto issue = [&](PrefixStep<C, ES>& dst, StepRefs& refs, int32_t t0) __attribute__((always_inline)) {
        refs = step_refs(a, w, next, t0);
        load_prefix_step<C, ES>(dst, a.d, w.h, refs.a, refs.b, lane);
        next = step_pages(a, w, t0 + stride);
    };
    const int32_t before = min(hi, held) - 31;           // steps that begin below it end before the nodes
    while (tok < before && r0.a.valid && r0.b.valid) {
        issue(buf1, r1, tok + stride);
        compute(buf0);
        tok += stride;
        if (tok >= before || !r1.a.valid || !r1.b.valid) {
            buf0 = buf1;
            r0 = r1;
            break;
        }
        issue(buf0, r0, tok + stride);
        compute(buf1);
        tok += stride;
    }
    while (tok < hi) {
        issue(buf1, r1, tok + stride);
        const FirstTokens first{j, r0.a.valid ? min(16, hi - tok) : 0, r0.b.valid ? min(16, hi - tok - 16) : 0};
        const NodeTokens counts{first, hi > held ? node_bits(masks, node, tok, held) : ~0u};
        const NodeProducts<C> products{a.d, r0.a.row0, r0.b.row0, w.h, lane};
        prefix_step<C, QT, ES, false>(st, buf0, q, lds.stage[wave], lane, counts, a.d.score_scale, products);
        tok += stride;
        buf0 = buf1;
        r0 = r1;
    }
    join_waves<C, NW>(st, lds, wave, 0, NW, (hi - w.lo + 31) >> 5, lane);
    if (wave != 0) return;
    const float l = sum_across_rows(st.l);
    if (w.r0 + m16 >= w.pairs) return;
    if (w.it.chunks > 1) {
        store_state<C>(a.d, (int64_t)w.state * a.block_rows + m16, st, l, D, j);
        return;
    }
    float* const out = reinterpret_cast<float*>(a.d.out) + ((int64_t)(w.it.s.row0 + node) * a.d.num_q_heads + hq) * D;
    const bool ok = l > 0.0f || l != l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int d0 = NB * (4 * j + e);
        if (d0 >= D) continue;
        float y[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) y[nb] = ok ? st.o[nb][e] / l : 0.0f;
        store_run<QT, NB>(out + d0, y);
    }
}

// The states of sequences of several chunks, zeros where a sequence has no tokens. A wave takes `run` pairs (row, q head), so
// that few waves look for their sequence, and up to four pairs of a row at once, so that their states are read together.
template <int C, int QT>
__global__ void __launch_bounds__(256)
tree_join_kernel(TreeArgs a, int32_t run) {
    constexpr int kLanes = 16 * C, kPass = 64 / kLanes, kPairs = 4;
    using T = typename Elem<QT>::T;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int D = a.d.head_dim;
    const int32_t units = (int32_t)a.rows * a.d.num_q_heads, begin = ((int32_t)blockIdx.x * 4 + wave) * run;
    const int32_t end = min(begin + run, units);
    if (begin >= end) return;
    const TreeCut c = cut_batch(a);
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int d4 = min(lane % kLanes, D / 4 - 1), po = lane / kLanes;
    TreeItem it;
    bool found = false;
    int32_t last = -1;
    for (int32_t unit = begin; unit < end;) {
        const int32_t row = (uint32_t)unit / (uint32_t)a.d.num_q_heads, hq = unit - row * a.d.num_q_heads;
        const int32_t count = min(min(kPairs, end - unit), a.d.num_q_heads - hq);
        if (row != last && !(found && row - it.s.row0 < it.s.nodes)) found = find_tree_item<true>(a, c, row, it);
        last = row;
        if (!found || it.chunks == 1) {
            unit += count;
            continue;
        }
        const int64_t stride = (int64_t)a.d.num_kv_heads * it.blocks * a.block_rows;
        int64_t first[kPairs];
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
            const int32_t q = hq + min(u, count - 1), h = (uint32_t)q / (uint32_t)G, pair = (row - it.s.row0) * G + (q - h * G);
            const int32_t block = (uint32_t)pair / (uint32_t)a.block_rows;
            first[u] = ((int64_t)it.first_state + (int64_t)h * it.blocks + block) * a.block_rows + (pair - block * a.block_rows);
        }
        JoinedState st[kPairs];
#pragma unroll 2
        for (int i = po; i < it.chunks; i += kPass) {
#pragma unroll
            for (int u = 0; u < kPairs; ++u) {
                const int64_t at = first[u] + i * stride;
                st[u].add(a.d.part_m[at], a.d.part_l[at], reinterpret_cast<const float4*>(a.d.part_acc + at * D)[d4]);
            }
        }
#pragma unroll
        for (int u = 0; u < kPairs; ++u) {
            if (u >= count) break;
            st[u].template across<kLanes>();
            if (po == 0 && 4 * (lane % kLanes) < D) st[u].template store<QT>(reinterpret_cast<T*>(a.d.out) + (int64_t)(unit + u) * D + 4 * d4);
        }
        unit += count;
    }
}

size_t tree_align(size_t x) { return (x + 255) & ~(size_t)255; }

hipError_t launch_tree_narrow(const TreeArgs& a, int64_t items, hipStream_t s) {
    const dim3 grid((unsigned)tree_grid(items));
    if (a.d.head_dim == 64) hipLaunchKernelGGL(tree_narrow_kernel<1>, grid, dim3(64 * kTreeWaves), 0, s, a);
    else hipLaunchKernelGGL(tree_narrow_kernel<2>, grid, dim3(64 * kTreeWaves), 0, s, a);
    return hipGetLastError();
}

}  // namespace

bool tree_mfma_supported(int32_t head_dim, int32_t block_size, int q_dtype, int kv_dtype) {
    if (block_size < 16) return false;
    if (kv_dtype == KVFP8_E4M3FN) return head_dim == 64 || head_dim == 80 || head_dim == 96 || head_dim == 112 || head_dim == 128;
    return (head_dim == 64 || head_dim == 128) && (kv_dtype == KVFP8_BF16 || kv_dtype == KVFP8_F16) && q_dtype == kv_dtype;
}

TreePlan tree_mfma_plan(int32_t seqs, int32_t max_nodes, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int q_dtype) {
    TreePlan p = {};
    const int64_t pairs = (int64_t)max_nodes * (num_q_heads / num_kv_heads);
    const bool narrow = q_dtype == KVFP8_F32;
    p.block_rows = narrow ? 16 : 64;
    p.target = device_cus() * (narrow ? 1 : 2);          // workgroups that a CU holds
    const int64_t columns = (int64_t)seqs * ((pairs + p.block_rows - 1) / p.block_rows) * num_kv_heads;
    // A chunk is at least the work divided by the target, so there are that many whole ones at most, and a column's last. Columns
    // of several chunks, whose items alone leave states, have fewer than two for each whole one.
    p.items = p.target + columns;
    const int64_t states = (p.items < 2 * p.target ? p.items : 2 * p.target) * p.block_rows;
    p.part_l = (int64_t)tree_align((size_t)states * 4);
    p.part_acc = 2 * p.part_l;
    p.bytes = p.part_acc + (int64_t)tree_align((size_t)states * head_dim * 4);
    return p;
}

template <int QT>
hipError_t launch_tree_mfma(TreeArgs a, int kv_dtype, const TreePlan& p, void* workspace, hipStream_t s) {
    char* const ws = reinterpret_cast<char*>(workspace);
    a.d.part_m = reinterpret_cast<float*>(ws);
    a.d.part_l = reinterpret_cast<float*>(ws + p.part_l);
    a.d.part_acc = reinterpret_cast<float*>(ws + p.part_acc);
    a.block_rows = p.block_rows;
    a.target = p.target;
    const int64_t q_size = QT == KVFP8_F32 ? 4 : 2;
    a.q_vec = (uintptr_t)a.d.q % 16 == 0 && a.d.q_stride_b * q_size % 16 == 0 && a.d.q_stride_h * q_size % 16 == 0;
    hipError_t err;
    if constexpr (QT == KVFP8_F32) err = launch_tree_narrow(a, p.items, s);
    else err = launch_tree_blocks<QT>(a, kv_dtype, p.items, s);
    if (err != hipSuccess) return err;
    // Sixteen waves a CU at most: each looks for its sequence, which takes longer than a row (ragged sequences: 19 us with 8, 16 with
    // 16, 23 with a wave for every row).
    const int64_t units = a.rows * a.d.num_q_heads, waves = 16 * (int64_t)device_cus();
    const int32_t run = (int32_t)((units + waves - 1) / waves);
    const dim3 grid((unsigned)((units + 4 * run - 1) / (4 * run)));
    if (a.d.head_dim == 64) hipLaunchKernelGGL((tree_join_kernel<1, QT>), grid, dim3(256), 0, s, a, run);
    else hipLaunchKernelGGL((tree_join_kernel<2, QT>), grid, dim3(256), 0, s, a, run);
    return hipGetLastError();
}

template hipError_t launch_tree_mfma<KVFP8_F32>(TreeArgs, int, const TreePlan&, void*, hipStream_t);
template hipError_t launch_tree_mfma<KVFP8_F16>(TreeArgs, int, const TreePlan&, void*, hipStream_t);
template hipError_t launch_tree_mfma<KVFP8_BF16>(TreeArgs, int, const TreePlan&, void*, hipStream_t);

}  // namespace kvfp8
