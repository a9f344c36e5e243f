// Norms of the query and key heads with the position rotation, in one pass over fused projection rows, the
// cache write of the keys and values on the way, and the gradients (gfx950).
//
// Rows are [q heads | k heads | v heads] of head_dim elements each. For head row x of token t, pair i < head_dim / 2:
//   inv = 1 / sqrt(mean_d x[d]^2 + eps),  y[d] = (x[d] inv) w[d]          (w: q_weight or k_weight; no weights: y = x)
//   c, s = cos_table[pos[t], i], sin_table[pos[t], i]                      (1, 0 for a position outside the tables)
//   out[2 i] = c y[2 i] - s y[2 i + 1],  out[2 i + 1] = s y[2 i] + c y[2 i + 1]
// in float32 with one rounding to the outputs' type; values are copied. k (as float32, before that rounding) and v go
// to (blocks[t], offsets[t]) of a paged cache by the rule of kvfp8_quantize_append or kvfp8_store_append.
// Backward, with g the gradient of out: h = g turned back, dw = sum over rows of h x inv,
//   dx = inv (h w - (x inv) mean_d(h w x inv)),  and the gradient of the values as it is.
//
// Layout: a head row is held by LPR lanes with eight elements (four pairs) each, so that 128 dims take 16 lanes and one
// 16-byte load a lane. A group of LPR lanes takes a run of up to kHeads heads of one section (q, k or v), the same heads of one
// token after another: the weights and their gradients' sums stay in registers, the heads of a token share the angles, and their
// loads are issued together.
//
// Bound by HBM: 16384 tokens of 32 + 8 heads of 128 in bfloat16 take 73 us forward (403 MB, 5.5 TB/s) and 118 us backward (570 MB,
// 4.8 TB/s); 65536 tokens of 16 + 4 heads with packed outputs and an e4m3fn cache 187 us (873 MB, 4.7 TB/s). Sums across a row's
// lanes by DPP, the hardware's reciprocal root and 16-bit roundings in pairs keep the vector ALU below that.
#include "kvfp8_decode_common.h"
#include "mfma_tiles.h"

namespace kvfp8 {

namespace {

constexpr int kNrThreads = 256;
constexpr int kNrElems = 8;
constexpr int kNrTokens = 4;

struct NormRopeArgs {
    const void* x;
    int64_t rows, row_stride;
    int32_t num_q_heads, num_kv_heads, head_dim;
    uint32_t q_runs, kv_runs;             // of heads, per section
    uint32_t step;                        // tokens taken at once: group g begins with run g % runs of token g / runs
    const void* positions;
    int32_t pos64;
    const void* cos_table;
    const void* sin_table;
    int32_t table_dtype;
    int64_t table_rows;
    const void* q_weight;                 // null: no norm
    const void* k_weight;
    int32_t w_dtype;
    float eps;
    // forward
    void* q_out;
    void* k_out;                          // null where only the cache is written
    void* v_out;
    const void* blocks;                   // null: no cache
    const void* offsets;
    int32_t blocks64, offsets64;
    int64_t num_blocks;
    int32_t block_size, cache_dtype;
    void* k_cache;
    void* v_cache;
    float* k_scales;
    float* v_scales;
    // backward
    const void* gq;                       // null: zeros
    const void* gk;
    const void* gv;
    void* dx;                             // null: not wanted
    float* part;                          // [workgroups][2][head_dim] sums for the weights, null: not wanted
};

// Elements d0 .. d0 + N - 1 of a row of type DT as they are stored, zeros past D. VEC: the row starts at a multiple of the access
// and D is a multiple of N.
template <int DT, int N>
struct alignas(sizeof(typename Elem<DT>::T) * N < 16 ? sizeof(typename Elem<DT>::T) * N : 16) Raw {
    typename Elem<DT>::T e[N];
};
template <int DT, int N, bool VEC>
__device__ __forceinline__ Raw<DT, N> load_raw(const typename Elem<DT>::T* row, int d0, int D) {
    Raw<DT, N> raw = {};
    if constexpr (VEC) {
        if (d0 < D) raw = *reinterpret_cast<const Raw<DT, N>*>(row + d0);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (d0 + i < D) raw.e[i] = row[d0 + i];
    }
    return raw;
}
template <int DT, int N, bool VEC>
__device__ __forceinline__ void store_raw(typename Elem<DT>::T* row, int d0, int D, const Raw<DT, N>& raw) {
    if constexpr (VEC) {
        if (d0 < D) *reinterpret_cast<Raw<DT, N>*>(row + d0) = raw;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (d0 + i < D) row[d0 + i] = raw.e[i];
    }
}
template <int DT, int N>
__device__ __forceinline__ void widen(const Raw<DT, N>& raw, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = Elem<DT>::load(raw.e[i]);
}

template <int N, bool VEC>
__device__ __forceinline__ void load_any(const void* row, int dtype, int d0, int D, float (&x)[N]) {
    if (dtype == KVFP8_F32) widen(load_raw<KVFP8_F32, N, VEC>(reinterpret_cast<const float*>(row), d0, D), x);
    else if (dtype == KVFP8_F16) widen(load_raw<KVFP8_F16, N, VEC>(reinterpret_cast<const uint16_t*>(row), d0, D), x);
    else widen(load_raw<KVFP8_BF16, N, VEC>(reinterpret_cast<const uint16_t*>(row), d0, D), x);
}

template <int DT, bool VEC>
__device__ __forceinline__ void store_run8(typename Elem<DT>::T* row, int d0, int D, const float (&x)[kNrElems]) {
    Raw<DT, kNrElems> raw;
    if constexpr (DT == KVFP8_F32) {
#pragma unroll
        for (int i = 0; i < kNrElems; ++i) raw.e[i] = x[i];
    } else {
#pragma unroll
        for (int i = 0; i < kNrElems; i += 2) {
            const uint32_t two = pack2<DT == KVFP8_F16>(x[i], x[i + 1]);
            raw.e[i] = (uint16_t)two;
            raw.e[i + 1] = (uint16_t)(two >> 16);
        }
    }
    store_raw<DT, kNrElems, VEC>(row, d0, D, raw);
}

// Sum (largest) of the LPR lanes of a row, the same in each: 16 lanes by DPP (quads, half rows and rows mirrored).
template <int CTRL>
__device__ __forceinline__ uint32_t row_dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true);
}
template <int LPR, typename Fold>
__device__ __forceinline__ uint32_t row_fold(uint32_t x, Fold fold) {
    x = fold(x, row_dpp<0xB1>(x));
    x = fold(x, row_dpp<0x4E>(x));
    x = fold(x, row_dpp<0x141>(x));
    if constexpr (LPR >= 16) x = fold(x, row_dpp<0x140>(x));
    if constexpr (LPR >= 32) x = fold(x, (uint32_t)__shfl_xor((int)x, 16, 64));
    if constexpr (LPR >= 64) x = fold(x, (uint32_t)__shfl_xor((int)x, 32, 64));
    return x;
}
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
    return bits_f32(row_fold<LPR>(f32_bits(x), [](uint32_t a, uint32_t b) { return f32_bits(bits_f32(a) + bits_f32(b)); }));
}

// 1 / sqrt(x): the hardware's estimate (one unit in the last place) but for subnormal numbers, which it takes for zeros. A root and a
// division instead would round twice, half a unit each. It moves a quantized row's scale by as much, and a code only where a value lies
// that close to a border (none of 524288 codes of normal rows on the CPU, for a root one unit off).
__device__ __forceinline__ float inverse_root(float x) {
    return x < 1.17549435e-38f ? 1.0f / sqrtf(x) : __builtin_amdgcn_rsqf(x);
}

// The heads of a group: `count` ones from `first` on of a section (0 q, 1 k, 2 v) of `heads`, behind `before` others in a row of x.
struct HeadRun {
    int section, first, count, heads, before;
    uint32_t token;
};
template <int LPR, int kHeads>
__device__ __forceinline__ HeadRun head_run(const NormRopeArgs& a) {
    HeadRun r;
    const uint32_t runs = a.q_runs + 2 * a.kv_runs, group = blockIdx.x * (kNrThreads / LPR) + threadIdx.x / LPR;
    r.token = group / runs;
    uint32_t run = group - r.token * runs;
    if (r.token >= a.step) r.token = (uint32_t)a.rows;   // the last workgroup's groups past the last whole token: none
    r.section = run < a.q_runs ? 0 : (run < a.q_runs + a.kv_runs ? 1 : 2);
    run -= r.section == 0 ? 0 : (r.section == 1 ? a.q_runs : a.q_runs + a.kv_runs);
    r.heads = r.section == 0 ? a.num_q_heads : a.num_kv_heads;
    r.first = (int)run * kHeads;
    r.count = min(kHeads, r.heads - r.first);
    r.before = r.section == 0 ? 0 : a.num_q_heads + (r.section == 2 ? a.num_kv_heads : 0);
    return r;
}

// The four angles of a lane's pairs.
struct Angles {
    float c[4], s[4];
};

template <bool VEC>
__device__ __forceinline__ Angles load_angles(const NormRopeArgs& a, int64_t pos, int d0) {
    Angles g;
    const int half = a.head_dim / 2;
    if (pos >= 0 && pos < a.table_rows) {
        const int64_t es = a.table_dtype == KVFP8_F32 ? 4 : 2;
        load_any<4, VEC>(reinterpret_cast<const char*>(a.cos_table) + pos * half * es, a.table_dtype, d0 / 2, half, g.c);
        load_any<4, VEC>(reinterpret_cast<const char*>(a.sin_table) + pos * half * es, a.table_dtype, d0 / 2, half, g.s);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            g.c[i] = 1.0f;
            g.s[i] = 0.0f;
        }
    }
    return g;
}

// Codes of one lane's eight elements (largest magnitude of the row as bits in amax), the rule of kvfp8_quantize_append.
__device__ __forceinline__ uint2 encode_run(const float (&x)[kNrElems], uint32_t amax, float scale) {
    const RowDivider div(scale);
    uint32_t w[2];
    if (div.fast && amax < 0x7F800000u) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int v = __builtin_amdgcn_cvt_pk_fp8_f32(div.corrected(x[4 * i]), div.corrected(x[4 * i + 1]), 0, false);
            v = __builtin_amdgcn_cvt_pk_fp8_f32(div.corrected(x[4 * i + 2]), div.corrected(x[4 * i + 3]), v, true);
            w[i] = (uint32_t)v;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            w[i] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i] |= (uint32_t)clamp_encode(x[4 * i + e] / scale) << (8 * e);
        }
    }
    return make_uint2(w[0], w[1]);
}

template <int DT, int LPR, bool VEC, int kHeads>
__global__ void __launch_bounds__(kNrThreads)
norm_rope_kernel(NormRopeArgs a) {
    using T = typename Elem<DT>::T;
    const int D = a.head_dim, lane = threadIdx.x % LPR, d0 = kNrElems * lane;
    const HeadRun r = head_run<LPR, kHeads>(a);
    if (r.token >= a.rows) return;
    const bool is_v = r.section == 2, cached = r.section != 0 && a.blocks != nullptr;
    const float per_dim = 1.0f / (float)D;
    float w[kNrElems] = {};
    if (a.q_weight != nullptr && !is_v) load_any<kNrElems, VEC>(r.section == 0 ? a.q_weight : a.k_weight, a.w_dtype, d0, D, w);
    T* const outs = reinterpret_cast<T*>(r.section == 0 ? a.q_out : (is_v ? a.v_out : a.k_out));
    for (int64_t token = r.token; token < a.rows; token += a.step) {
        const int64_t pos = is_v ? 0 : load_i(a.positions, a.pos64, token);
        const T* const src = reinterpret_cast<const T*>(a.x) + token * a.row_stride + (int64_t)(r.before + r.first) * D;
        Raw<DT, kNrElems> raw[kHeads];
#pragma unroll
        for (int u = 0; u < kHeads; ++u) raw[u] = load_raw<DT, kNrElems, VEC>(src + (int64_t)min(u, r.count - 1) * D, d0, D);
        int64_t block = -1, offset = -1;
        if (cached) {
            block = load_i(a.blocks, a.blocks64, token);
            offset = load_i(a.offsets, a.offsets64, token);
        }
        const bool inside = block >= 0 && block < a.num_blocks && offset >= 0 && offset < a.block_size;
        Angles g = {};
        if (!is_v) g = load_angles<VEC>(a, pos, d0);
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            if (u >= r.count) break;                     // the same for the lanes of a row
            T* const out = outs == nullptr ? nullptr : outs + (token * r.heads + r.first + u) * D;
            float x[kNrElems];
            widen(raw[u], x);
            if (is_v) {
                if (out != nullptr) store_raw<DT, kNrElems, VEC>(out, d0, D, raw[u]);
            } else {
                if (a.q_weight != nullptr) {
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < kNrElems; ++i) sum += x[i] * x[i];
                    const float inv = inverse_root(row_sum<LPR>(sum) * per_dim + a.eps);
#pragma unroll
                    for (int i = 0; i < kNrElems; ++i) x[i] = (x[i] * inv) * w[i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y0 = x[2 * i], y1 = x[2 * i + 1];
                    x[2 * i] = g.c[i] * y0 - g.s[i] * y1;
                    x[2 * i + 1] = g.s[i] * y0 + g.c[i] * y1;
                }
                if (out != nullptr) store_run8<DT, VEC>(out, d0, D, x);
            }
            if (!cached) continue;
            const int64_t slot = (block * a.block_size + offset) * r.heads + r.first + u;
            void* const cache = is_v ? a.v_cache : a.k_cache;
            if (a.cache_dtype == KVFP8_E4M3FN) {
                uint32_t amax = 0;
#pragma unroll
                for (int i = 0; i < kNrElems; ++i) amax = max(amax, abs_bits(x[i]));
                amax = row_fold<LPR>(amax, [](uint32_t p, uint32_t q) { return max(p, q); });
                if (!inside) continue;
                const float scale = row_scale(amax);
                const uint2 codes = encode_run(x, amax, scale);
                uint8_t* const dst = reinterpret_cast<uint8_t*>(cache) + slot * D + d0;
                if constexpr (VEC) {
                    if (d0 < D) *reinterpret_cast<uint2*>(dst) = codes;
                } else {
#pragma unroll
                    for (int i = 0; i < kNrElems; ++i)
                        if (d0 + i < D) dst[i] = (uint8_t)((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)));
                }
                if (lane == 0) (is_v ? a.v_scales : a.k_scales)[slot] = scale;
            } else if (inside) {
                if (a.cache_dtype == KVFP8_F32) store_run8<KVFP8_F32, VEC>(reinterpret_cast<float*>(cache) + slot * D, d0, D, x);
                else if (a.cache_dtype == KVFP8_F16) store_run8<KVFP8_F16, VEC>(reinterpret_cast<uint16_t*>(cache) + slot * D, d0, D, x);
                else store_run8<KVFP8_BF16, VEC>(reinterpret_cast<uint16_t*>(cache) + slot * D, d0, D, x);
            }
        }
    }
}

// Gradients. The weights' sums stay in registers over a group's tokens, join across the workgroup's groups of a section in LDS
// in a fixed order, and leave as one partial sum a workgroup and weight.
template <int DT, int LPR, bool VEC, int kHeads>
__global__ void __launch_bounds__(kNrThreads, 4)
norm_rope_backward_kernel(NormRopeArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int kGroups = kNrThreads / LPR;
    __shared__ float sums[kGroups][LPR * kNrElems];
    const int D = a.head_dim, lane = threadIdx.x % LPR, group = threadIdx.x / LPR, d0 = kNrElems * lane;
    const HeadRun r = head_run<LPR, kHeads>(a);
    const int heads = a.num_q_heads + 2 * a.num_kv_heads;
    const bool is_v = r.section == 2, normed = a.q_weight != nullptr && !is_v, summed = a.part != nullptr;
    const float per_dim = 1.0f / (float)D;
    float w[kNrElems] = {}, dw[kNrElems] = {};
    if (normed) load_any<kNrElems, VEC>(r.section == 0 ? a.q_weight : a.k_weight, a.w_dtype, d0, D, w);
    const T* const grads = reinterpret_cast<const T*>(r.section == 0 ? a.gq : (is_v ? a.gv : a.gk));
    for (int64_t token = r.token; token < a.rows; token += a.step) {
        const int64_t pos = is_v ? 0 : load_i(a.positions, a.pos64, token);
        const T* const src = reinterpret_cast<const T*>(a.x) + token * a.row_stride + (int64_t)(r.before + r.first) * D;
        Raw<DT, kNrElems> rx[kHeads], rg[kHeads];
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            const int at = min(u, r.count - 1);
            rx[u] = rg[u] = {};
            if (grads != nullptr) rg[u] = load_raw<DT, kNrElems, VEC>(grads + (token * r.heads + r.first + at) * D, d0, D);
            if (normed) rx[u] = load_raw<DT, kNrElems, VEC>(src + (int64_t)at * D, d0, D);
        }
        Angles t = {};
        if (!is_v) t = load_angles<VEC>(a, pos, d0);
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            if (u >= r.count) break;
            T* const dx = a.dx == nullptr ? nullptr : reinterpret_cast<T*>(a.dx) + (token * heads + r.before + r.first + u) * D;
            if (is_v) {
                if (dx != nullptr) store_raw<DT, kNrElems, VEC>(dx, d0, D, rg[u]);
                continue;
            }
            float g[kNrElems];
            widen(rg[u], g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float y0 = g[2 * i], y1 = g[2 * i + 1];
                g[2 * i] = t.c[i] * y0 + t.s[i] * y1;
                g[2 * i + 1] = t.c[i] * y1 - t.s[i] * y0;
            }
            if (normed) {
                float x[kNrElems], sum = 0.0f, dot = 0.0f;
                widen(rx[u], x);
#pragma unroll
                for (int i = 0; i < kNrElems; ++i) {
                    sum += x[i] * x[i];
                    dot += (g[i] * w[i]) * x[i];
                }
                const float inv = inverse_root(row_sum<LPR>(sum) * per_dim + a.eps);
                const float mean = row_sum<LPR>(dot) * inv * per_dim;
#pragma unroll
                for (int i = 0; i < kNrElems; ++i) {
                    const float xh = x[i] * inv;
                    dw[i] += g[i] * xh;
                    g[i] = inv * (g[i] * w[i] - xh * mean);
                }
            }
            if (dx != nullptr) store_run8<DT, VEC>(dx, d0, D, g);
        }
    }
    if (!summed) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kNrElems; ++i) sums[group][d0 + i] = r.section == k ? dw[i] : 0.0f;
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kNrThreads) {
            float total = 0.0f;
#pragma unroll
            for (int r = 0; r < kGroups; ++r) total += sums[r][d];
            a.part[((int64_t)blockIdx.x * 2 + k) * D + d] = total;
        }
    }
}

// Column d of both weights' sums over the workgroups: eight columns a workgroup, 32 threads down each.
__global__ void __launch_bounds__(kNrThreads)
norm_rope_weight_grad_kernel(const float* part, int32_t blocks, int32_t D, int32_t w_dtype, void* dq, void* dk) {
    __shared__ float sums[32][8];
    const int col = threadIdx.x & 7, group = threadIdx.x >> 3, at = blockIdx.x * 8 + col;
    float total = 0.0f;
    if (at < 2 * D) {
#pragma unroll 8
        for (int b = group; b < blocks; b += 32) total += part[(int64_t)b * 2 * D + at];
    }
    sums[group][col] = total;
    __syncthreads();
    if (threadIdx.x >= 8 || at >= 2 * D) return;
    total = 0.0f;
#pragma unroll
    for (int g = 0; g < 32; ++g) total += sums[g][col];
    void* const dst = at < D ? dq : dk;
    const int d = at < D ? at : at - D;
    if (dst == nullptr) return;
    if (w_dtype == KVFP8_F32) reinterpret_cast<float*>(dst)[d] = total;
    else reinterpret_cast<uint16_t*>(dst)[d] = w_dtype == KVFP8_F16 ? f32_to_f16(total) : f32_to_bf16(total);
}

bool nr_float(int d) { return d == KVFP8_F32 || d == KVFP8_F16 || d == KVFP8_BF16; }
bool nr_index(int d) { return d == KVFP8_I32 || d == KVFP8_I64; }
int64_t nr_size(int d) { return d == KVFP8_F32 ? 4 : 2; }

constexpr int kNrMaxDim = 64 * kNrElems;
constexpr int64_t kNrMaxHeads = 4096;
constexpr int64_t kNrMaxBlocks = (int64_t)1 << 20;        // of a launch, which holds less than 2^32 threads

int check_norm_rope(const void* x, int dtype, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                    int64_t row_stride, const void* positions, int pos_dtype, const void* cos_table, const void* sin_table,
                    int table_dtype, int64_t table_rows, const void* q_weight, const void* k_weight, int w_dtype) {
    if (!nr_float(dtype) || !nr_float(table_dtype) || !nr_float(w_dtype) || !nr_index(pos_dtype)) return KVFP8_EDTYPE;
    if (rows < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || head_dim % 2 != 0 || table_rows <= 0)
        return KVFP8_ESHAPE;
    const int64_t heads = (int64_t)num_q_heads + 2 * (int64_t)num_kv_heads;
    if (head_dim > kNrMaxDim || heads > kNrMaxHeads || rows >= ((int64_t)1 << 31) / heads) return KVFP8_ELIMIT;
    if (rows > 0 && row_stride < 0) return KVFP8_ESTRIDE;
    if ((q_weight == nullptr) != (k_weight == nullptr)) return KVFP8_ENULL;
    if (rows > 0 && (!x || !positions || !cos_table || !sin_table)) return KVFP8_ENULL;
    return KVFP8_OK;
}

// Whether the rows, tables and weights fit eight-element accesses.
bool nr_vectors(const NormRopeArgs& a, int dtype) {
    const int64_t ts = nr_size(a.table_dtype);
    return a.head_dim % kNrElems == 0 && (uintptr_t)a.x % 16 == 0 && a.row_stride * nr_size(dtype) % 16 == 0 &&
           ((uintptr_t)a.cos_table | (uintptr_t)a.sin_table) % (4 * ts) == 0 &&
           ((uintptr_t)a.q_weight | (uintptr_t)a.k_weight) % 16 == 0;
}

int lanes_of(int head_dim) {
    int lpr = 8;
    while (lpr * kNrElems < head_dim) lpr <<= 1;
    return lpr;
}

// Heads of a run. With rows enough for every lane of the device and 16-byte accesses of 16-bit elements four, else one. Forward in
// microseconds with runs of 1 / 4, bfloat16, 32 + 8 heads of 128: 512 rows 5.6 / 5.5 (below: 1.0 less with one), 1024 rows 8.2 / 6.8,
// 16384 rows 93 / 73; backward of 16384 rows 139 / 118. float32, whose runs of four need twice the registers: 4096 rows 32 / 36, and
// backward 56 / 79.
constexpr int kNrRun = 4;
int run_of(int64_t rows, int64_t heads, int dtype, bool vec, int lanes) {
    return vec && dtype != KVFP8_F32 && rows * heads * lanes >= (int64_t)device_cus() * 8 * kNrThreads ? kNrRun : 1;
}

template <bool kBackward, int DT, int LPR, bool VEC, int kHeads>
hipError_t launch_norm_rope(const NormRopeArgs& a, unsigned blocks, hipStream_t s) {
    if constexpr (kBackward) hipLaunchKernelGGL((norm_rope_backward_kernel<DT, LPR, VEC, kHeads>), dim3(blocks), dim3(kNrThreads), 0, s, a);
    else hipLaunchKernelGGL((norm_rope_kernel<DT, LPR, VEC, kHeads>), dim3(blocks), dim3(kNrThreads), 0, s, a);
    return hipGetLastError();
}

template <bool kBackward, int DT, int LPR>
hipError_t launch_norm_rope(const NormRopeArgs& a, int run, unsigned blocks, hipStream_t s) {
    if constexpr (DT != KVFP8_F32)
        if (run != 1) return launch_norm_rope<kBackward, DT, LPR, true, kNrRun>(a, blocks, s);
    return launch_norm_rope<kBackward, DT, LPR, true, 1>(a, blocks, s);
}

template <bool kBackward, int DT>
hipError_t launch_norm_rope(const NormRopeArgs& a, bool vec, int lanes, int run, unsigned blocks, hipStream_t s) {
    if (!vec) return launch_norm_rope<kBackward, DT, 64, false, 1>(a, blocks, s);
    if (lanes == 8) return launch_norm_rope<kBackward, DT, 8>(a, run, blocks, s);
    if (lanes == 16) return launch_norm_rope<kBackward, DT, 16>(a, run, blocks, s);
    if (lanes == 32) return launch_norm_rope<kBackward, DT, 32>(a, run, blocks, s);
    return launch_norm_rope<kBackward, DT, 64>(a, run, blocks, s);
}

template <bool kBackward>
hipError_t launch_norm_rope(const NormRopeArgs& a, int dtype, bool vec, int lanes, int run, int64_t blocks, hipStream_t s) {
    switch (dtype) {
        case KVFP8_F32: return launch_norm_rope<kBackward, KVFP8_F32>(a, vec, lanes, run, (unsigned)blocks, s);
        case KVFP8_F16: return launch_norm_rope<kBackward, KVFP8_F16>(a, vec, lanes, run, (unsigned)blocks, s);
        default: return launch_norm_rope<kBackward, KVFP8_BF16>(a, vec, lanes, run, (unsigned)blocks, s);
    }
}

// Workgroups of the backward: at most what the device holds at once, as each leaves partial sums, and groups for every head of a
// token. By sizes alone (64 lanes a row, runs of one head), as the workspace is asked for without pointers.
int64_t backward_blocks(int64_t rows, int64_t heads) {
    const int64_t per = kNrThreads / 64, held = (int64_t)device_cus() * 4, most = held > heads / per + 1 ? held : heads / per + 1;
    const int64_t wanted = (rows * heads + per - 1) / per;
    return wanted < most ? wanted : most;
}

// The runs and how many tokens so many workgroups take at once.
void set_runs(NormRopeArgs& a, int run, int lanes, int64_t blocks) {
    a.q_runs = (uint32_t)((a.num_q_heads + run - 1) / run);
    a.kv_runs = (uint32_t)((a.num_kv_heads + run - 1) / run);
    a.step = (uint32_t)(blocks * (kNrThreads / lanes) / (a.q_runs + 2 * a.kv_runs));
}

}  // namespace

}  // namespace kvfp8

using namespace kvfp8;

extern "C" int kvfp8_norm_rope(const void* x, int dtype, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                               int32_t head_dim, int64_t row_stride, const void* positions, int pos_dtype,
                               const void* cos_table, const void* sin_table, int table_dtype, int64_t table_rows,
                               const void* q_weight, const void* k_weight, int w_dtype, float eps, void* q_out,
                               void* k_out, void* v_out, const void* blocks, int blocks_dtype, const void* offsets,
                               int offsets_dtype, int64_t num_blocks, int32_t block_size, void* k_cache, void* v_cache,
                               int cache_dtype, float* k_scales, float* v_scales, void* stream) {
    const int rc = check_norm_rope(x, dtype, rows, num_q_heads, num_kv_heads, head_dim, row_stride, positions, pos_dtype,
                                   cos_table, sin_table, table_dtype, table_rows, q_weight, k_weight, w_dtype);
    if (rc != KVFP8_OK) return rc;
    const bool cached = blocks != nullptr || offsets != nullptr;
    if (cached) {
        if (!nr_index(blocks_dtype) || !nr_index(offsets_dtype)) return KVFP8_EDTYPE;
        if (cache_dtype != KVFP8_E4M3FN && !nr_float(cache_dtype)) return KVFP8_EDTYPE;
        if (num_blocks <= 0 || block_size <= 0) return KVFP8_ESHAPE;
        if (!blocks || !offsets || !k_cache || !v_cache) return KVFP8_ENULL;
        if (cache_dtype == KVFP8_E4M3FN && (!k_scales || !v_scales)) return KVFP8_ENULL;
    }
    if (rows == 0) return KVFP8_OK;
    if (!q_out || (k_out == nullptr) != (v_out == nullptr) || (!cached && !k_out)) return KVFP8_ENULL;
    NormRopeArgs a = {};
    a.x = x;
    a.rows = rows;
    a.row_stride = row_stride;
    a.num_q_heads = num_q_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.positions = positions;
    a.pos64 = pos_dtype == KVFP8_I64;
    a.cos_table = cos_table;
    a.sin_table = sin_table;
    a.table_dtype = table_dtype;
    a.table_rows = table_rows;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.w_dtype = w_dtype;
    a.eps = eps;
    a.q_out = q_out;
    a.k_out = k_out;
    a.v_out = v_out;
    if (cached) {
        a.blocks = blocks;
        a.offsets = offsets;
        a.blocks64 = blocks_dtype == KVFP8_I64;
        a.offsets64 = offsets_dtype == KVFP8_I64;
        a.num_blocks = num_blocks;
        a.block_size = block_size;
        a.cache_dtype = cache_dtype;
        a.k_cache = k_cache;
        a.v_cache = v_cache;
        a.k_scales = k_scales;
        a.v_scales = v_scales;
    }
    const bool vec = nr_vectors(a, dtype) && ((uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)a.k_cache |
                                              (uintptr_t)a.v_cache) % 16 == 0;
    const int lanes = vec ? lanes_of(head_dim) : 64;
    const int64_t heads = (int64_t)num_q_heads + 2 * (int64_t)num_kv_heads;
    const int run = run_of(rows, heads, dtype, vec, lanes);
    const int64_t runs = (num_q_heads + run - 1) / run + 2 * (int64_t)((num_kv_heads + run - 1) / run), per = kNrThreads / lanes;
    // A group takes up to kNrTokens tokens, so that the weights are read seldom, while there are workgroups enough.
    int64_t tokens = rows * runs / (per * device_cus() * 16);
    tokens = tokens < 1 ? 1 : (tokens > kNrTokens ? kNrTokens : tokens);
    int64_t wanted = ((rows + tokens - 1) / tokens * runs + per - 1) / per;
    wanted = wanted < kNrMaxBlocks ? wanted : kNrMaxBlocks;
    set_runs(a, run, lanes, wanted);
    return (int)launch_norm_rope<false>(a, dtype, vec, lanes, run, wanted, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int64_t kvfp8_norm_rope_backward_workspace_bytes(int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                                                            int32_t head_dim) {
    if (rows <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    const int64_t heads = (int64_t)num_q_heads + 2 * (int64_t)num_kv_heads;
    if (head_dim > kNrMaxDim || heads > kNrMaxHeads || rows >= ((int64_t)1 << 31) / heads) return 0;
    return backward_blocks(rows, heads) * 2 * head_dim * 4;
}

extern "C" int kvfp8_norm_rope_backward(const void* x, int dtype, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                                        int32_t head_dim, int64_t row_stride, const void* positions, int pos_dtype,
                                        const void* cos_table, const void* sin_table, int table_dtype, int64_t table_rows,
                                        const void* q_weight, const void* k_weight, int w_dtype, float eps,
                                        const void* grad_q, const void* grad_k, const void* grad_v, void* dx,
                                        void* dq_weight, void* dk_weight, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
    const int rc = check_norm_rope(x, dtype, rows, num_q_heads, num_kv_heads, head_dim, row_stride, positions, pos_dtype,
                                   cos_table, sin_table, table_dtype, table_rows, q_weight, k_weight, w_dtype);
    if (rc != KVFP8_OK) return rc;
    const bool summed = dq_weight != nullptr || dk_weight != nullptr;
    if (summed && q_weight == nullptr) return KVFP8_ENULL;
    const int64_t need = summed ? kvfp8_norm_rope_backward_workspace_bytes(rows, num_q_heads, num_kv_heads, head_dim) : 0;
    if (need > 0 && !workspace) return KVFP8_ENULL;
    if (workspace_bytes < need) return KVFP8_EWORKSPACE;
    if (need > 0 && (uintptr_t)workspace % 4 != 0) return KVFP8_ESTRIDE;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const int64_t heads = (int64_t)num_q_heads + 2 * (int64_t)num_kv_heads;
    const int64_t blocks = rows > 0 ? backward_blocks(rows, heads) : 0;
    if (rows > 0 && (dx != nullptr || summed)) {
        NormRopeArgs a = {};
        a.x = x;
        a.rows = rows;
        a.row_stride = row_stride;
        a.num_q_heads = num_q_heads;
        a.num_kv_heads = num_kv_heads;
        a.head_dim = head_dim;
        a.positions = positions;
        a.pos64 = pos_dtype == KVFP8_I64;
        a.cos_table = cos_table;
        a.sin_table = sin_table;
        a.table_dtype = table_dtype;
        a.table_rows = table_rows;
        a.q_weight = q_weight;
        a.k_weight = k_weight;
        a.w_dtype = w_dtype;
        a.eps = eps;
        a.gq = grad_q;
        a.gk = grad_k;
        a.gv = grad_v;
        a.dx = dx;
        a.part = summed ? reinterpret_cast<float*>(workspace) : nullptr;
        const bool vec = nr_vectors(a, dtype) &&
                         ((uintptr_t)grad_q | (uintptr_t)grad_k | (uintptr_t)grad_v | (uintptr_t)dx) % 16 == 0;
        const int lanes = vec ? lanes_of(head_dim) : 64;
        const int run = run_of(rows, heads, dtype, vec, lanes);
        set_runs(a, run, lanes, blocks);
        const hipError_t err = launch_norm_rope<true>(a, dtype, vec, lanes, run, blocks, s);
        if (err != hipSuccess) return (int)err;
    }
    if (!summed) return KVFP8_OK;
    hipLaunchKernelGGL(norm_rope_weight_grad_kernel, dim3((unsigned)((2 * head_dim + 7) / 8)), dim3(kNrThreads), 0, s,
                       reinterpret_cast<const float*>(workspace), (int32_t)blocks, head_dim, w_dtype, dq_weight, dk_weight);
    return (int)hipGetLastError();
}
