// Attention of a batch whose sequences share long prefixes in the paged cache (gfx950).
//
// A row's keys are the tokens of its group's prefix and then its own: in the decode form the tokens on
// its sequence's pages, in the prompt form the keys of its packed prompt up to itself. With
// s_t = sm_scale q . khat_t a set of tokens has the softmax state
//   m = max s_t,  l = sum e^(s_t - m),  acc = sum e^(s_t - m) vhat_t,
// and states of disjoint sets join exactly: M = max(m1, m2), l = l1 e^(m1 - M) + l2 e^(m2 - M), acc
// likewise; the output is acc / l, 0 for a row without tokens. States are float32, scores base 2.
//
// The matrix-core kernels are in shared_prefix_mfma.hip. prefix_generic_kernel takes every cache, head size (up to 512)
// and page size: one wave per (row, q head, split of the row's tokens), on the vector ALU. Every row reads its prefix by
// itself there: 32 rows x 32 heads behind 4096 tokens take 1200 us at head size 80 of a bf16 cache and 2030 at 128 of a
// float32 one, where the matrix cores take 24 to 33.
#include "shared_prefix.h"

namespace kvfp8 {

namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr int kGenWaves = 4;
constexpr int kGenMaxD = 512;

template <int KVT>
__device__ __forceinline__ float cache_element(const void* p, int64_t i) {
    if constexpr (KVT == KVFP8_E4M3FN) return decode_e4m3fn(reinterpret_cast<const uint8_t*>(p)[i]);
    else return Elem<KVT>::load(reinterpret_cast<const typename Elem<KVT>::T*>(p)[i]);
}

// A row's state over part of its tokens joins what the prompt form's out and lse hold (one state
// with l = 1: out is the weighted mean and lse the log of its denominator). out comes rounded to q's type and is rounded
// again: the first rounding counts by the prompt's share of the weight. lse is float32, so the weights of prefix
// and prompt against each other are off by up to |lse| 2^-23, which shows from scores of about 1e4 on.
template <int QT, int ND>
__device__ __forceinline__ void finish_row(const PrefixArgs& a, int64_t row, int hq, int lane, float m, float l,
                                           float (&acc)[ND]) {
    using T = typename Elem<QT>::T;
    const int D = a.d.head_dim;
    const int64_t at = row * a.d.num_q_heads + hq;
    T* out = reinterpret_cast<T*>(a.d.out) + at * D;
    if (a.cu != nullptr) {
        const float mo = a.lse[at] * kLog2e;
        const float mn = fmaxf(m, mo);
        const float mu = mn == kNegInf ? 0.0f : mn;
        const float wp = __builtin_amdgcn_exp2f(m - mu), wo = __builtin_amdgcn_exp2f(mo - mu);
        l = l * wp + wo;
#pragma unroll
        for (int e = 0; e < ND; ++e) {
            const int d = lane + 64 * e;
            if (d < D) acc[e] = acc[e] * wp + Elem<QT>::load(out[d]) * wo;
        }
        if (lane == 0) a.lse[at] = (mu + __builtin_log2f(l)) * kLn2;
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int e = 0; e < ND; ++e) {
        const int d = lane + 64 * e;
        if (d < D) out[d] = Elem<QT>::store(l > 0.0f || l != l ? acc[e] * inv : 0.0f);
    }
}

template <int KVT, int QT, int ND>
__global__ void __launch_bounds__(64 * kGenWaves)
prefix_generic_kernel(PrefixArgs a) {
    constexpr bool kQuant = KVT == KVFP8_E4M3FN;
    __shared__ float q_lds[kGenWaves][kGenMaxD];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int D = a.d.head_dim, hkv = a.d.num_kv_heads;
    const int64_t units = a.rows * a.d.num_q_heads * a.splits;
    for (int64_t unit = (int64_t)blockIdx.x * kGenWaves + wave; unit < units; unit += (int64_t)gridDim.x * kGenWaves) {
        const int split = (int)(unit % a.splits);
        const int64_t rest = unit / a.splits;
        const int hq = (int)(rest % a.d.num_q_heads);
        const int64_t row = rest / a.d.num_q_heads;
        const int64_t seq = seq_of_row(a, row);
        if (seq < 0) continue;
        const int g = group_of_seq(a, seq);
        int64_t p_slot = 0, o_slot = 0, own = 0;
        const int64_t prefix = g >= 0 ? group_tokens(a, g, &p_slot) : 0;
        if (a.cu == nullptr) own = seq_tokens(a.d, (int)seq, &o_slot);
        else if (prefix == 0) continue;                  // out and lse stand
        const int32_t* p_table = a.d.block_table + p_slot * a.d.bt_width;
        const int32_t* o_table = a.d.block_table + o_slot * a.d.bt_width;
        const int64_t per = split_tokens(prefix + own, a.step_shift, a.splits);
        const int64_t lo = split * per, hi = min(lo + per, prefix + own);
        const int h = hq / (a.d.num_q_heads / hkv);
        float* q = q_lds[wave];
        for (int d = lane; d < D; d += 64)
            q[d] = Elem<QT>::load(reinterpret_cast<const typename Elem<QT>::T*>(a.d.q)[row * a.d.q_stride_b + hq * a.d.q_stride_h + d]);
        __builtin_amdgcn_wave_barrier();                 // one wave's LDS operations complete in order
        float m = kNegInf, l = 0.0f, acc[ND];
#pragma unroll
        for (int e = 0; e < ND; ++e) acc[e] = 0.0f;
        for (int64_t t0 = lo; t0 < hi; t0 += 64) {
            // One token per lane; at: its cache row, -1 past the end and on pages outside the pool.
            const int64_t tok = t0 + lane;
            int64_t at = -1;
            if (tok < hi) {
                const int64_t pos = tok < prefix ? tok : tok - prefix;
                const int64_t page = (tok < prefix ? p_table : o_table)[pos >> a.d.bs_shift];
                if (page >= 0 && page < a.d.num_blocks)
                    at = ((page << a.d.bs_shift) + (pos & (a.d.block_size - 1))) * hkv + h;
            }
            float s = kNegInf, vs = 1.0f;
            if (at >= 0) {
                float dot = 0.0f;
                for (int d = 0; d < D; ++d) dot += q[d] * cache_element<KVT>(a.d.k_cache, at * D + d);
                if (kQuant) {
                    dot *= a.d.k_scales[at];
                    vs = a.d.v_scales[at];
                }
                s = dot * a.d.score_scale;
            }
            float mx = s;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
            const float mn = fmaxf(m, mx);
            const float mu = mn == kNegInf ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - mu);
            const float p = at >= 0 ? __builtin_amdgcn_exp2f(s - mu) : 0.0f;
            float sum = p;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
            l = l * alpha + sum;
            m = mn;
#pragma unroll
            for (int e = 0; e < ND; ++e) acc[e] *= alpha;
            const float pv = p * vs;
            for (int j = 0; j < 64; ++j) {
                const uint32_t lo32 = __builtin_amdgcn_readlane((int)(uint32_t)(uint64_t)at, j);
                const uint32_t hi32 = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)at >> 32), j);
                const int64_t vrow = (int64_t)(((uint64_t)hi32 << 32) | lo32);
                if (vrow < 0) continue;
                const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, pv), j));
#pragma unroll
                for (int e = 0; e < ND; ++e) {
                    const int d = lane + 64 * e;
                    if (d < D) acc[e] += w * cache_element<KVT>(a.d.v_cache, vrow * D + d);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
        if (a.splits == 1) {
            finish_row<QT, ND>(a, row, hq, lane, m, l, acc);
            continue;
        }
        const int64_t pi = prefix_part(a, row, split, hq);
        if (lane == 0) {
            a.d.part_m[pi] = m;
            a.d.part_l[pi] = l;
        }
#pragma unroll
        for (int e = 0; e < ND; ++e) {
            const int d = lane + 64 * e;
            if (d < D) a.d.part_acc[pi * D + d] = acc[e];
        }
    }
}

// One wave per (row, q head) joins the states of its splits (and, in the prompt form, out and lse).
template <int QT, int ND>
__global__ void __launch_bounds__(64 * kGenWaves)
prefix_generic_join_kernel(PrefixArgs a) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int D = a.d.head_dim;
    const int64_t units = a.rows * a.d.num_q_heads;
    for (int64_t unit = (int64_t)blockIdx.x * kGenWaves + wave; unit < units; unit += (int64_t)gridDim.x * kGenWaves) {
        const int64_t row = unit / a.d.num_q_heads;
        const int hq = (int)(unit - row * a.d.num_q_heads);
        const int64_t seq = seq_of_row(a, row);
        if (seq < 0) continue;
        if (a.cu != nullptr) {
            const int g = group_of_seq(a, seq);
            int64_t slot;
            if (g < 0 || group_tokens(a, g, &slot) == 0) continue;
        }
        float m = kNegInf, l = 0.0f, acc[ND];
#pragma unroll
        for (int e = 0; e < ND; ++e) acc[e] = 0.0f;
        for (int s = 0; s < a.splits; ++s) {
            const int64_t pi = prefix_part(a, row, s, hq);
            const float mi = a.d.part_m[pi];
            const float mn = fmaxf(m, mi);
            const float mu = mn == kNegInf ? 0.0f : mn;
            const float sa = __builtin_amdgcn_exp2f(m - mu), sb = __builtin_amdgcn_exp2f(mi - mu);
            l = l * sa + a.d.part_l[pi] * sb;
#pragma unroll
            for (int e = 0; e < ND; ++e) {
                const int d = lane + 64 * e;
                if (d < D) acc[e] = acc[e] * sa + a.d.part_acc[pi * D + d] * sb;
            }
            m = mn;
        }
        finish_row<QT, ND>(a, row, hq, lane, m, l, acc);
    }
}

// ------------------------------------------------------------------ host

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int ilog2(int64_t x) {
    int s = 0;
    while ((int64_t)1 << s < x) ++s;
    return s;
}

struct PrefixPlan {
    int32_t splits;
    int64_t bytes;              // workspace
};

// States of `splits` per row and q head.
int64_t state_bytes(int64_t rows, int32_t hq, int32_t d, int32_t splits) {
    const size_t states = (size_t)rows * hq * splits;
    return (int64_t)(2 * align256(states * sizeof(float)) + align256(states * d * sizeof(float)));
}

PrefixPlan make_plan(int64_t rows, int32_t hq, int32_t d, int64_t bt_width, int32_t block_size, bool prompt) {
    // Enough waves for every SIMD of the chip, none with fewer than 256 tokens of the longest row.
    const int64_t longest = bt_width * block_size * (prompt ? 1 : 2);
    int64_t splits = (4 * 4 * (int64_t)device_cus()) / (rows * hq);
    splits = splits < longest / 256 ? splits : longest / 256;
    splits = splits < 1 ? 1 : (splits > 64 ? 64 : splits);
    PrefixPlan p;
    p.splits = (int32_t)splits;
    p.bytes = p.splits > 1 ? state_bytes(rows, hq, d, p.splits) : 0;
    return p;
}

constexpr int64_t kMaxGrid = 1 << 20;

template <typename F>
hipError_t launch_units(F kernel, int64_t units, const PrefixArgs& a, hipStream_t s) {
    int64_t blocks = (units + kGenWaves - 1) / kGenWaves;
    blocks = blocks < kMaxGrid ? blocks : kMaxGrid;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * kGenWaves), 0, s, a);
    return hipGetLastError();
}

template <int KVT, int QT, int ND>
hipError_t launch_generic_nd(const PrefixArgs& a, hipStream_t s) {
    const int64_t pairs = a.rows * a.d.num_q_heads;
    const hipError_t err = launch_units(prefix_generic_kernel<KVT, QT, ND>, pairs * a.splits, a, s);
    if (err != hipSuccess || a.splits == 1) return err;
    return launch_units(prefix_generic_join_kernel<QT, ND>, pairs, a, s);
}

template <int KVT, int QT>
hipError_t launch_generic(const PrefixArgs& a, hipStream_t s) {
    if (a.d.head_dim <= 128) return launch_generic_nd<KVT, QT, 2>(a, s);
    return launch_generic_nd<KVT, QT, 8>(a, s);
}

template <int QT>
hipError_t launch_generic_kv(const PrefixArgs& a, int kv_dtype, hipStream_t s) {
    switch (kv_dtype) {
        case KVFP8_E4M3FN: return launch_generic<KVFP8_E4M3FN, QT>(a, s);
        case KVFP8_BF16: return launch_generic<KVFP8_BF16, QT>(a, s);
        case KVFP8_F16: return launch_generic<KVFP8_F16, QT>(a, s);
        default: return launch_generic<KVFP8_F32, QT>(a, s);
    }
}

bool index_dtype(int t) { return t == KVFP8_I32 || t == KVFP8_I64; }
bool float_dtype(int t) { return t == KVFP8_F32 || t == KVFP8_F16 || t == KVFP8_BF16; }

// Sizes (none negative) that the kernels take, from which nothing on the host overflows. Their token numbers are int32
// and run up to three blocks past the last.
bool within_limits(int64_t rows, int32_t hq, int32_t d, int64_t bt_width, int32_t block_size) {
    return d <= kGenMaxD && rows <= INT32_MAX && rows * hq <= INT32_MAX && bt_width <= (INT32_MAX - 8192) / block_size;
}

// What the two forms check alike; fills the shared arguments.
int shared_args(PrefixArgs& a, const void* q, int q_dtype, int64_t q_stride_t, int64_t q_stride_h, int64_t rows,
                int32_t hq, int32_t hkv, int32_t d, const void* k_cache, const void* v_cache, int kv_dtype,
                const float* k_scales, const float* v_scales, int64_t num_blocks, int32_t block_size,
                const int32_t* block_table, int64_t bt_rows, int64_t bt_width, const void* p_slots, int p_slots_dtype,
                const void* p_lens, int p_lens_dtype, const void* p_starts, int p_starts_dtype, int32_t groups,
                float sm_scale, void* out) {
    if (!float_dtype(q_dtype) || (!float_dtype(kv_dtype) && kv_dtype != KVFP8_E4M3FN) || !index_dtype(p_slots_dtype) ||
        !index_dtype(p_lens_dtype) || !index_dtype(p_starts_dtype))
        return KVFP8_EDTYPE;
    if (rows < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || d <= 0 || num_blocks <= 0 || bt_rows <= 0 || bt_width <= 0 ||
        block_size <= 0 || (block_size & (block_size - 1)) != 0 || groups < 0)
        return KVFP8_ESHAPE;
    if (!within_limits(rows, hq, d, bt_width, block_size)) return KVFP8_ELIMIT;
    if (rows == 0) return KVFP8_OK;
    if (!q || !k_cache || !v_cache || !block_table || !out || (groups > 0 && (!p_slots || !p_lens || !p_starts)))
        return KVFP8_ENULL;
    if (kv_dtype == KVFP8_E4M3FN && (!k_scales || !v_scales)) return KVFP8_ENULL;
    a = PrefixArgs{};
    a.d.q = q;
    a.d.q_stride_b = q_stride_t;
    a.d.q_stride_h = q_stride_h;
    a.d.batch = (int32_t)rows;
    a.d.num_q_heads = hq;
    a.d.num_kv_heads = hkv;
    a.d.head_dim = d;
    a.d.k_cache = k_cache;
    a.d.v_cache = v_cache;
    a.d.k_scales = k_scales;
    a.d.v_scales = v_scales;
    a.d.num_blocks = num_blocks;
    a.d.block_size = block_size;
    a.d.bs_shift = ilog2(block_size);
    a.d.block_table = block_table;
    a.d.bt_rows = bt_rows;
    a.d.bt_width = bt_width;
    a.d.score_scale = sm_scale * kLog2e;
    a.d.out = out;
    a.d.q_dtype = q_dtype;
    a.rows = rows;
    a.p_slots = p_slots;
    a.p_lens = p_lens;
    a.p_starts = p_starts;
    a.p_slots64 = p_slots_dtype == KVFP8_I64;
    a.p_lens64 = p_lens_dtype == KVFP8_I64;
    a.p_starts64 = p_starts_dtype == KVFP8_I64;
    a.groups = groups;
    return KVFP8_OK;
}

int run_generic(PrefixArgs& a, const PrefixPlan& p, int q_dtype, int kv_dtype, void* workspace, hipStream_t s) {
    a.splits = p.splits;
    a.step_shift = 6;
    const size_t states = (size_t)a.rows * a.d.num_q_heads * p.splits;
    char* ws = reinterpret_cast<char*>(workspace);
    a.d.part_m = reinterpret_cast<float*>(ws);
    a.d.part_l = reinterpret_cast<float*>(ws + align256(states * sizeof(float)));
    a.d.part_acc = reinterpret_cast<float*>(ws + 2 * align256(states * sizeof(float)));
    switch (q_dtype) {
        case KVFP8_F32: return (int)launch_generic_kv<KVFP8_F32>(a, kv_dtype, s);
        case KVFP8_F16: return (int)launch_generic_kv<KVFP8_F16>(a, kv_dtype, s);
        default: return (int)launch_generic_kv<KVFP8_BF16>(a, kv_dtype, s);
    }
}

// Whether a call runs on the matrix cores.
bool mfma_shape(int64_t rows, int32_t hq, int32_t hkv, int32_t d, int32_t groups, int32_t bs, int q_dtype, int kv_dtype) {
    if (!prefix_mfma_supported(d, bs, q_dtype, kv_dtype)) return false;
    // Byte offsets within 16 tokens are int32 (elements of 2 bytes at most).
    if ((int64_t)hkv * d > (int64_t)1 << 25) return false;
    // A launch has fewer than 2^32 threads, and the decode form may take a workgroup of 512 for every pair's own tokens
    // (one q head a KV head). The prompt form has the same limit, though it launches a sixteenth of that or less: a call
    // of 2^22 pairs (131072 tokens of 32 heads) goes row by row, and callers with more split theirs.
    return rows * hq < ((int64_t)1 << 22) && (int64_t)groups * hkv < ((int64_t)1 << 21);
}

template <int QT>
int run(PrefixArgs& a, int kv_dtype, void* workspace, int64_t workspace_bytes, hipStream_t s) {
    const bool prompt = a.cu != nullptr;
    const bool aligned = (((uintptr_t)a.d.k_cache | (uintptr_t)a.d.v_cache | (uintptr_t)a.d.out) & 15) == 0;
    if (aligned && a.d.bt_rows < ((int64_t)1 << 26) &&
        mfma_shape(a.rows, a.d.num_q_heads, a.d.num_kv_heads, a.d.head_dim, a.groups, a.d.block_size, QT, kv_dtype)) {
        const PrefixMfmaPlan p = prefix_mfma_plan(a.rows, a.d.num_q_heads, a.d.num_kv_heads, a.d.head_dim, a.groups,
                                                  a.d.bt_width, a.d.block_size, QT, prompt);
        if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return KVFP8_EWORKSPACE;
        return (int)launch_prefix_mfma<QT>(a, kv_dtype, p, workspace, s);
    }
    const PrefixPlan p = make_plan(a.rows, a.d.num_q_heads, a.d.head_dim, a.d.bt_width, a.d.block_size, prompt);
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return KVFP8_EWORKSPACE;
    return run_generic(a, p, QT, kv_dtype, workspace, s);
}

int run(PrefixArgs& a, int q_dtype, int kv_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (q_dtype) {
        case KVFP8_F32: return run<KVFP8_F32>(a, kv_dtype, workspace, workspace_bytes, s);
        case KVFP8_F16: return run<KVFP8_F16>(a, kv_dtype, workspace, workspace_bytes, s);
        default: return run<KVFP8_BF16>(a, kv_dtype, workspace, workspace_bytes, s);
    }
}

}  // namespace

}  // namespace kvfp8

using namespace kvfp8;

extern "C" int64_t kvfp8_shared_prefix_workspace_bytes(int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                                                       int32_t head_dim, int32_t groups, int64_t bt_width,
                                                       int32_t block_size, int kv_dtype, int prompt) {
    if (rows <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || groups < 0 || bt_width <= 0 ||
        block_size <= 0 || !within_limits(rows, num_q_heads, head_dim, bt_width, block_size))
        return 0;                                        // the calls refuse these
    // The larger of what the paths need that a call of these shapes may take (its pointers decide).
    int64_t bytes = make_plan(rows, num_q_heads, head_dim, bt_width, block_size, prompt != 0).bytes;
    if (num_q_heads % num_kv_heads == 0)
        for (const int q_dtype : {KVFP8_F32, KVFP8_F16, KVFP8_BF16})
            if (mfma_shape(rows, num_q_heads, num_kv_heads, head_dim, groups, block_size, q_dtype, kv_dtype)) {
                const int64_t need = prefix_mfma_plan(rows, num_q_heads, num_kv_heads, head_dim, groups, bt_width, block_size,
                                                      q_dtype, prompt != 0).bytes;
                bytes = bytes > need ? bytes : need;
            }
    return bytes;
}

extern "C" int kvfp8_shared_prefix_decode(
    const void* q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h, int32_t batch, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, const void* k_cache, const void* v_cache, int kv_dtype,
    const float* k_scales, const float* v_scales, int64_t num_blocks, int32_t block_size, const int32_t* block_table,
    int64_t bt_rows, int64_t bt_width, const void* slots, int slots_dtype, const void* context_lengths, int ctx_dtype,
    float sm_scale, void* out, void* workspace, int64_t workspace_bytes, void* stream, const void* prefix_slots,
    int prefix_slots_dtype, const void* prefix_lengths, int prefix_lengths_dtype, const void* prefix_starts,
    int prefix_starts_dtype, int32_t groups) {
    PrefixArgs a;
    if (!index_dtype(slots_dtype) || !index_dtype(ctx_dtype)) return KVFP8_EDTYPE;
    const int bad = shared_args(a, q, q_dtype, q_stride_b, q_stride_h, batch, num_q_heads, num_kv_heads, head_dim,
                                k_cache, v_cache, kv_dtype, k_scales, v_scales, num_blocks, block_size, block_table,
                                bt_rows, bt_width, prefix_slots, prefix_slots_dtype, prefix_lengths,
                                prefix_lengths_dtype, prefix_starts, prefix_starts_dtype, groups, sm_scale, out);
    if (bad != KVFP8_OK || batch == 0) return bad;
    if (!slots || !context_lengths) return KVFP8_ENULL;
    a.d.slots = slots;
    a.d.ctx = context_lengths;
    a.d.slots64 = slots_dtype == KVFP8_I64;
    a.d.ctx64 = ctx_dtype == KVFP8_I64;
    return run(a, q_dtype, kv_dtype, workspace, workspace_bytes, stream);
}

extern "C" int kvfp8_shared_prefix_prefill(
    const void* q, int q_dtype, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    const void* k_cache, const void* v_cache, int kv_dtype, const float* k_scales, const float* v_scales,
    int64_t num_blocks, int32_t block_size, const int32_t* block_table, int64_t bt_rows, int64_t bt_width,
    const void* prefix_slots, int prefix_slots_dtype, const void* prefix_lengths, int prefix_lengths_dtype,
    const void* prefix_starts, int prefix_starts_dtype, int32_t groups, const void* cu_seqlens, int cu_dtype,
    int32_t batch, int32_t max_seq_len, float scale, void* out, float* lse, void* workspace, int64_t workspace_bytes,
    void* stream) {
    PrefixArgs a;
    if (!index_dtype(cu_dtype)) return KVFP8_EDTYPE;
    if (batch < 0 || max_seq_len < 0) return KVFP8_ESHAPE;
    const int bad = shared_args(a, q, q_dtype, (int64_t)num_q_heads * head_dim, head_dim, rows, num_q_heads,
                                num_kv_heads, head_dim, k_cache, v_cache, kv_dtype, k_scales, v_scales, num_blocks,
                                block_size, block_table, bt_rows, bt_width, prefix_slots, prefix_slots_dtype,
                                prefix_lengths, prefix_lengths_dtype, prefix_starts, prefix_starts_dtype, groups, scale,
                                out);
    if (bad != KVFP8_OK || rows == 0 || batch == 0 || max_seq_len == 0 || groups == 0) return bad;
    if (!cu_seqlens || !lse) return KVFP8_ENULL;
    a.cu = cu_seqlens;
    a.cu64 = cu_dtype == KVFP8_I64;
    a.seqs = batch;
    a.max_len = max_seq_len;
    a.lse = lse;
    return run(a, q_dtype, kv_dtype, workspace, workspace_bytes, stream);
}
