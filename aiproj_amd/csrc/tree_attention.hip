// Attention of trees of drafted tokens, each behind its sequence's tokens in the paged cache (gfx950).
//
// A sequence of L tokens in the cache has n drafted nodes as the last of them. Row i (node i) attends the L - n tokens
// before the nodes, the nodes above it and itself:
//   out[i] = sum_t w_t vhat_t / sum_t w_t,  w_t = e^(s_t - max s),  s_t = sm_scale q_i . khat_t
// over those tokens t, khat and vhat the cache's rows, dequantized. float32 sums, scores base 2; zeros for a row without
// tokens.
//
// Its floor is the cache's bytes up to about 64 pairs (node, q head) of a KV head, each token being read once a KV head, and the
// products behind that; the kernels on the matrix cores are bound by the vector ALU beside them. tree_generic_kernel takes every
// cache, head size (up to 512) and page size on the vector ALU (8 sequences of 16 nodes and 1016 tokens, 32 / 8 heads of 80: 389 us
// against 32 there): a workgroup reads a sequence's tokens for one row alone.
#include "tree_attention.h"

namespace kvfp8 {

namespace {

constexpr int kGenericWaves = 4;
constexpr int kGenericDim = 512;

template <int KVT>
__device__ __forceinline__ float cached(const void* p, int64_t i) {
    if constexpr (KVT == KVFP8_E4M3FN) return decode_e4m3fn(reinterpret_cast<const uint8_t*>(p)[i]);
    else return Elem<KVT>::load(reinterpret_cast<const typename Elem<KVT>::T*>(p)[i]);
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off);
    return x;
}

// A workgroup per (row, q head). Its waves take steps of 64 tokens in turn: each lane scores a token, then the lanes add
// the weighted values of the dims l, l + 64, ... token by token (those that do not count are passed over).
template <int KVT, int QT, int ND>
__global__ void __launch_bounds__(64 * kGenericWaves)
tree_generic_kernel(TreeArgs a) {
    using T = typename Elem<QT>::T;
    __shared__ float qs[64 * ND];
    __shared__ int32_t parents[kMaxNodes];
    __shared__ uint32_t above[kNodeWords];
    __shared__ float join_m[kGenericWaves], join_l[kGenericWaves], join_o[kGenericWaves][64 * ND];
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int D = a.d.head_dim;
    const int32_t row = (int32_t)(blockIdx.x / (uint32_t)a.d.num_q_heads), hq = (int32_t)(blockIdx.x - (uint32_t)row * a.d.num_q_heads);
    const int32_t h = hq / (a.d.num_q_heads / a.d.num_kv_heads);
    // The row's sequence: a wave looks through 64 at once.
    TreeSeq s = {};
    bool found = false;
    for (int b0 = 0; b0 < a.seqs && !found; b0 += 64) {
        const TreeSeq x = lane_seq(a, b0);
        const uint64_t hit = __ballot(row >= x.row0 && row - x.row0 < x.nodes);
        if (hit == 0) continue;
        const int at = __builtin_ctzll(hit);
        s.row0 = __builtin_amdgcn_readlane(x.row0, at);
        s.nodes = __builtin_amdgcn_readlane(x.nodes, at);
        s.tokens = __builtin_amdgcn_readlane(x.tokens, at);
        s.held = __builtin_amdgcn_readlane(x.held, at);
        s.slot = __builtin_amdgcn_readlane((int32_t)x.slot, at);
        found = true;
    }
    if (!found) return;
    const int32_t node = row - s.row0;
    for (int d = threadIdx.x; d < 64 * ND; d += 64 * kGenericWaves)
        qs[d] = d < D ? load_q<QT>(a.d, row, hq, d) * a.d.score_scale : 0.0f;
    if ((int32_t)threadIdx.x <= node) {                  // (kMaxNodes threads)
        const int64_t p = load_i(a.parents, a.parents64, (int64_t)s.row0 + threadIdx.x);
        parents[threadIdx.x] = p >= 0 && p < (int64_t)threadIdx.x ? (int32_t)p : -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kNodeWords; ++i) above[i] = 0;
        for (int i = node; i >= 0; i = parents[i]) above[i >> 5] |= 1u << (i & 31);
    }
    __syncthreads();
    float m = kNegInf, l = 0.0f, o[ND];
#pragma unroll
    for (int e = 0; e < ND; ++e) o[e] = 0.0f;
    const int32_t* const table = a.d.block_table + s.slot * a.d.bt_width;
    for (int32_t t0 = 64 * wave; t0 < s.tokens; t0 += 64 * kGenericWaves) {
        const int32_t tok = t0 + lane, n = tok - s.held;
        const int64_t page = tok < s.tokens ? table[tok >> a.d.bs_shift] : -1;
        bool live = page >= 0 && page < a.d.num_blocks;
        if (n >= 0) live = live && n < kMaxNodes && ((above[n >> 5] >> (n & 31)) & 1u) != 0;
        const int64_t at = live ? (page * a.d.block_size + (tok & (a.d.block_size - 1))) * a.d.num_kv_heads + h : 0;
        float score = kNegInf, vscale = 1.0f;
        if (live) {
            float dot = 0.0f;
            for (int d = 0; d < D; ++d) dot += qs[d] * cached<KVT>(a.d.k_cache, at * D + d);
            score = KVT == KVFP8_E4M3FN ? dot * a.d.k_scales[at] : dot;
            if (KVT == KVFP8_E4M3FN) vscale = a.d.v_scales[at];
        }
        float top = score;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
        const float mn = fmaxf(m, top), mu = mn == kNegInf ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - mu), p = live ? __builtin_amdgcn_exp2f(score - mu) : 0.0f;
        m = mn;
        l = l * alpha + wave_sum(p);
#pragma unroll
        for (int e = 0; e < ND; ++e) o[e] *= alpha;
        const float weight = p * vscale;
        uint64_t left = __ballot(live);
        while (left != 0) {
            const int i = __builtin_ctzll(left);
            left &= left - 1;
            const float w = __shfl(weight, i);
            const int64_t v = __shfl((long long)at, i) * D;
#pragma unroll
            for (int e = 0; e < ND; ++e)
                if (lane + 64 * e < D) o[e] += w * cached<KVT>(a.d.v_cache, v + lane + 64 * e);
        }
    }
    if (lane == 0) {
        join_m[wave] = m;
        join_l[wave] = l;
    }
#pragma unroll
    for (int e = 0; e < ND; ++e) join_o[wave][lane + 64 * e] = o[e];
    __syncthreads();
    float top = kNegInf;
#pragma unroll
    for (int i = 0; i < kGenericWaves; ++i) top = fmaxf(top, join_m[i]);
    const float mu = top == kNegInf ? 0.0f : top;
    float den = 0.0f;
#pragma unroll
    for (int i = 0; i < kGenericWaves; ++i) den += join_l[i] * __builtin_amdgcn_exp2f(join_m[i] - mu);
    T* const out = reinterpret_cast<T*>(a.d.out) + ((int64_t)row * a.d.num_q_heads + hq) * D;
    for (int d = threadIdx.x; d < D; d += 64 * kGenericWaves) {
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < kGenericWaves; ++i) y += join_o[i][d] * __builtin_amdgcn_exp2f(join_m[i] - mu);
        out[d] = Elem<QT>::store(den > 0.0f || den != den ? y / den : 0.0f);
    }
}

template <int KVT, int QT>
hipError_t launch_tree_generic(const TreeArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.rows * a.d.num_q_heads)), block(64 * kGenericWaves);
    if (a.d.head_dim <= 128) hipLaunchKernelGGL((tree_generic_kernel<KVT, QT, 2>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((tree_generic_kernel<KVT, QT, kGenericDim / 64>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <int QT>
hipError_t launch_tree_generic(const TreeArgs& a, int kv_dtype, hipStream_t s) {
    switch (kv_dtype) {
        case KVFP8_E4M3FN: return launch_tree_generic<KVFP8_E4M3FN, QT>(a, s);
        case KVFP8_BF16: return launch_tree_generic<KVFP8_BF16, QT>(a, s);
        case KVFP8_F16: return launch_tree_generic<KVFP8_F16, QT>(a, s);
        default: return launch_tree_generic<KVFP8_F32, QT>(a, s);
    }
}

bool tree_index(int t) { return t == KVFP8_I32 || t == KVFP8_I64; }
bool tree_float(int t) { return t == KVFP8_F32 || t == KVFP8_F16 || t == KVFP8_BF16; }

// Sizes from which nothing overflows: token numbers are int32 and run up to a chunk past the last, and a launch has
// fewer than 2^32 threads, of which a workgroup of 512 may go to every pair.
bool tree_limits(int64_t rows, int32_t seqs, int32_t max_nodes, int32_t hq, int32_t d, int64_t bt_rows, int64_t bt_width,
                 int32_t block_size) {
    constexpr int64_t kPairs = (int64_t)1 << 22;
    return d <= kGenericDim && max_nodes <= kMaxNodes && rows < kPairs / hq && seqs < kPairs / hq / max_nodes &&
           bt_rows <= INT32_MAX && bt_width <= (INT32_MAX - 65536) / block_size;
}

bool tree_on_mfma(int32_t hkv, int32_t d, int32_t block_size, int q_dtype, int kv_dtype) {
    // Byte offsets within 16 tokens are int32 (elements of 2 bytes at most).
    return (int64_t)hkv * d <= (int64_t)1 << 25 && tree_mfma_supported(d, block_size, q_dtype, kv_dtype);
}

int tree_shift(int32_t x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

template <int QT>
int run_tree(const TreeArgs& a, int kv_dtype, void* workspace, int64_t workspace_bytes, hipStream_t s) {
    const bool aligned = (((uintptr_t)a.d.k_cache | (uintptr_t)a.d.v_cache | (uintptr_t)a.d.out) & 15) == 0;
    if (!aligned || a.d.score_scale == 0.0f || !tree_on_mfma(a.d.num_kv_heads, a.d.head_dim, a.d.block_size, QT, kv_dtype))
        return (int)launch_tree_generic<QT>(a, kv_dtype, s);
    const TreePlan p = tree_mfma_plan(a.seqs, a.max_nodes, a.d.num_q_heads, a.d.num_kv_heads, a.d.head_dim, QT);
    if (!workspace || workspace_bytes < p.bytes) return KVFP8_EWORKSPACE;
    return (int)launch_tree_mfma<QT>(a, kv_dtype, p, workspace, s);
}

}  // namespace

}  // namespace kvfp8

using namespace kvfp8;

extern "C" int64_t kvfp8_tree_attention_workspace_bytes(int32_t seqs, int32_t max_nodes, int32_t num_q_heads,
                                                        int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                                        int kv_dtype) {
    if (seqs <= 0 || max_nodes <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
        num_q_heads % num_kv_heads != 0 || !tree_limits(0, seqs, max_nodes, num_q_heads, head_dim, 0, 0, block_size))
        return 0;                                        // the call refuses these
    int64_t bytes = 0;
    for (const int q_dtype : {KVFP8_F32, KVFP8_F16, KVFP8_BF16})
        if (tree_on_mfma(num_kv_heads, head_dim, block_size, q_dtype, kv_dtype)) {
            const int64_t need = tree_mfma_plan(seqs, max_nodes, num_q_heads, num_kv_heads, head_dim, q_dtype).bytes;
            bytes = bytes > need ? bytes : need;
        }
    return bytes;
}

extern "C" int kvfp8_tree_attention(const void* q, int q_dtype, int64_t q_stride_r, int64_t q_stride_h, int64_t rows,
                                    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const void* k_cache,
                                    const void* v_cache, int kv_dtype, const float* k_scales, const float* v_scales,
                                    int64_t num_blocks, int32_t block_size, const int32_t* block_table, int64_t bt_rows,
                                    int64_t bt_width, const void* slots, int slots_dtype, const void* context_lengths,
                                    int ctx_dtype, const void* starts, int starts_dtype, const void* parents,
                                    int parents_dtype, int32_t seqs, int32_t max_nodes, float sm_scale, void* out,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
    if (!tree_float(q_dtype) || (!tree_float(kv_dtype) && kv_dtype != KVFP8_E4M3FN) || !tree_index(slots_dtype) ||
        !tree_index(ctx_dtype) || !tree_index(starts_dtype) || !tree_index(parents_dtype))
        return KVFP8_EDTYPE;
    if (rows < 0 || seqs < 0 || max_nodes < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 ||
        head_dim <= 0 || num_blocks <= 0 || bt_rows <= 0 || bt_width <= 0 || block_size <= 0 || (block_size & (block_size - 1)) != 0)
        return KVFP8_ESHAPE;
    if (!tree_limits(rows, seqs, max_nodes > 0 ? max_nodes : 1, num_q_heads, head_dim, bt_rows, bt_width, block_size))
        return KVFP8_ELIMIT;
    if (rows == 0 || seqs == 0 || max_nodes == 0) return KVFP8_OK;
    if (!q || !k_cache || !v_cache || !block_table || !slots || !context_lengths || !starts || !parents || !out) return KVFP8_ENULL;
    if (kv_dtype == KVFP8_E4M3FN && (!k_scales || !v_scales)) return KVFP8_ENULL;
    TreeArgs a = {};
    a.d.q = q;
    a.d.q_stride_b = q_stride_r;
    a.d.q_stride_h = q_stride_h;
    a.d.batch = seqs;
    a.d.num_q_heads = num_q_heads;
    a.d.num_kv_heads = num_kv_heads;
    a.d.head_dim = head_dim;
    a.d.k_cache = k_cache;
    a.d.v_cache = v_cache;
    a.d.k_scales = k_scales;
    a.d.v_scales = v_scales;
    a.d.num_blocks = num_blocks;
    a.d.block_size = block_size;
    a.d.bs_shift = tree_shift(block_size);
    a.d.block_table = block_table;
    a.d.bt_rows = bt_rows;
    a.d.bt_width = bt_width;
    a.d.slots = slots;
    a.d.ctx = context_lengths;
    a.d.slots64 = slots_dtype == KVFP8_I64;
    a.d.ctx64 = ctx_dtype == KVFP8_I64;
    a.d.score_scale = sm_scale * kLog2e;
    a.d.out = out;
    a.d.q_dtype = q_dtype;
    a.rows = rows;
    a.starts = starts;
    a.parents = parents;
    a.starts64 = starts_dtype == KVFP8_I64;
    a.parents64 = parents_dtype == KVFP8_I64;
    a.seqs = seqs;
    a.max_nodes = max_nodes;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (q_dtype) {
        case KVFP8_F32: return run_tree<KVFP8_F32>(a, kv_dtype, workspace, workspace_bytes, s);
        case KVFP8_F16: return run_tree<KVFP8_F16>(a, kv_dtype, workspace, workspace_bytes, s);
        default: return run_tree<KVFP8_BF16>(a, kv_dtype, workspace, workspace_bytes, s);
    }
}
