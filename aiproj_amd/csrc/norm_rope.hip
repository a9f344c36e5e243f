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
// 16-byte load a lane. A group of LPR lanes takes a run of kHeads heads of one token, whose loads are issued together
// and which share the position, the angles and the weights' cache lines.
#include "kvfp8_common.h"

namespace kvfp8 {

namespace {

constexpr int kNrThreads = 256;
constexpr int kNrElems = 8;

struct NormRopeArgs {
    const void* x;
    int64_t rows, row_stride;
    int32_t num_q_heads, num_kv_heads, head_dim;
    uint32_t runs;                        // of heads, per token
    uint32_t total;                       // rows x runs, below 2^31
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

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
    return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}

// Elements d0 .. d0 + N - 1 of a row of type DT, zeros past D. VEC: the row starts at a multiple of the access and D is a
// multiple of N.
template <int DT, int N, bool VEC>
__device__ __forceinline__ void load_run(const void* row, int d0, int D, float (&x)[N]) {
    using T = typename Elem<DT>::T;
    const T* p = reinterpret_cast<const T*>(row) + d0;
    if constexpr (VEC) {
        struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Run { T e[N]; };
        Run raw = {};
        if (d0 < D) raw = *reinterpret_cast<const Run*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = Elem<DT>::load(raw.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = d0 + i < D ? Elem<DT>::load(p[i]) : 0.0f;
    }
}

template <int N, bool VEC>
__device__ __forceinline__ void load_any(const void* row, int dtype, int d0, int D, float (&x)[N]) {
    if (dtype == KVFP8_F32) load_run<KVFP8_F32, N, VEC>(row, d0, D, x);
    else if (dtype == KVFP8_F16) load_run<KVFP8_F16, N, VEC>(row, d0, D, x);
    else load_run<KVFP8_BF16, N, VEC>(row, d0, D, x);
}

template <int DT, bool VEC>
__device__ __forceinline__ void store_run8(void* row, int d0, int D, const float (&x)[kNrElems]) {
    using T = typename Elem<DT>::T;
    T* p = reinterpret_cast<T*>(row) + d0;
    if constexpr (VEC) {
        struct alignas(16) Run { T e[kNrElems]; };
        Run raw;
#pragma unroll
        for (int i = 0; i < kNrElems; ++i) raw.e[i] = Elem<DT>::store(x[i]);
        if (d0 < D) *reinterpret_cast<Run*>(p) = raw;
    } else {
#pragma unroll
        for (int i = 0; i < kNrElems; ++i)
            if (d0 + i < D) p[i] = Elem<DT>::store(x[i]);
    }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
    for (int s = 1; s < LPR; s <<= 1) x += __shfl_xor(x, s, 64);
    return x;
}

// The four angles of a lane's pairs.
struct Angles {
    float c[4], s[4];
};

template <bool VEC>
__device__ __forceinline__ Angles load_angles(const NormRopeArgs& a, int64_t token, int d0) {
    Angles g;
    const int64_t pos = index_at(a.positions, a.pos64, token);
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
    const int heads = a.num_q_heads + 2 * a.num_kv_heads, first_v = a.num_q_heads + a.num_kv_heads;
    const uint32_t stride = gridDim.x * (kNrThreads / LPR);
    for (uint32_t unit = blockIdx.x * (kNrThreads / LPR) + threadIdx.x / LPR; unit < a.total; unit += stride) {
        const uint32_t token = unit / a.runs;
        const int h0 = (int)(unit - token * a.runs) * kHeads;
        const T* const src = reinterpret_cast<const T*>(a.x) + (int64_t)token * a.row_stride;
        float x[kHeads][kNrElems];
#pragma unroll
        for (int u = 0; u < kHeads; ++u) load_run<DT, kNrElems, VEC>(src + (int64_t)min(h0 + u, heads - 1) * D, d0, D, x[u]);
        int64_t block = -1, offset = -1;
        if (a.blocks != nullptr && h0 + kHeads > a.num_q_heads) {
            block = index_at(a.blocks, a.blocks64, token);
            offset = index_at(a.offsets, a.offsets64, token);
        }
        Angles g;
        if (h0 < first_v) g = load_angles<VEC>(a, token, d0);
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            const int h = h0 + u;
            if (h >= heads) break;                       // the same for the lanes of a row
            if (h < first_v) {
                if (a.q_weight != nullptr) {
                    float w[kNrElems], sum = 0.0f;
                    load_any<kNrElems, VEC>(h < a.num_q_heads ? a.q_weight : a.k_weight, a.w_dtype, d0, D, w);
#pragma unroll
                    for (int i = 0; i < kNrElems; ++i) sum += x[u][i] * x[u][i];
                    const float inv = 1.0f / sqrtf(row_sum<LPR>(sum) / (float)D + a.eps);
#pragma unroll
                    for (int i = 0; i < kNrElems; ++i) x[u][i] = (x[u][i] * inv) * w[i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y0 = x[u][2 * i], y1 = x[u][2 * i + 1];
                    x[u][2 * i] = g.c[i] * y0 - g.s[i] * y1;
                    x[u][2 * i + 1] = g.s[i] * y0 + g.c[i] * y1;
                }
            }
            const bool is_q = h < a.num_q_heads, is_v = h >= first_v;
            const int nh = is_q ? a.num_q_heads : a.num_kv_heads, hh = is_q ? h : (is_v ? h - first_v : h - a.num_q_heads);
            T* const out = reinterpret_cast<T*>(is_q ? a.q_out : (is_v ? a.v_out : a.k_out));
            if (out != nullptr) store_run8<DT, VEC>(out + ((int64_t)token * nh + hh) * D, d0, D, x[u]);
            if (is_q || a.blocks == nullptr) continue;
            const bool inside = block >= 0 && block < a.num_blocks && offset >= 0 && offset < a.block_size;
            const int64_t slot = (block * a.block_size + offset) * nh + hh;
            void* const cache = is_v ? a.v_cache : a.k_cache;
            if (a.cache_dtype == KVFP8_E4M3FN) {
                uint32_t amax = 0;
#pragma unroll
                for (int i = 0; i < kNrElems; ++i) amax = max(amax, abs_bits(x[u][i]));
#pragma unroll
                for (int s = 1; s < LPR; s <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, s, 64));
                if (!inside) continue;
                const float scale = row_scale(amax);
                const uint2 codes = encode_run(x[u], amax, scale);
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
                if (a.cache_dtype == KVFP8_F32) store_run8<KVFP8_F32, VEC>(reinterpret_cast<float*>(cache) + slot * D, d0, D, x[u]);
                else if (a.cache_dtype == KVFP8_F16) store_run8<KVFP8_F16, VEC>(reinterpret_cast<uint16_t*>(cache) + slot * D, d0, D, x[u]);
                else store_run8<KVFP8_BF16, VEC>(reinterpret_cast<uint16_t*>(cache) + slot * D, d0, D, x[u]);
            }
        }
    }
}

// Gradients. The weights' sums stay in registers over a workgroup's units, join across its rows in LDS in a fixed
// order, and leave as one partial sum a workgroup and weight.
template <int DT, int LPR, bool VEC, int kHeads>
__global__ void __launch_bounds__(kNrThreads)
norm_rope_backward_kernel(NormRopeArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int kGroups = kNrThreads / LPR;
    __shared__ float sums[kGroups][LPR * kNrElems];
    const int D = a.head_dim, lane = threadIdx.x % LPR, group = threadIdx.x / LPR, d0 = kNrElems * lane;
    const int heads = a.num_q_heads + 2 * a.num_kv_heads, first_v = a.num_q_heads + a.num_kv_heads;
    const bool normed = a.q_weight != nullptr, summed = a.part != nullptr;
    float dw[2][kNrElems];
#pragma unroll
    for (int i = 0; i < kNrElems; ++i) dw[0][i] = dw[1][i] = 0.0f;
    const uint32_t stride = gridDim.x * kGroups;
    for (uint32_t unit = blockIdx.x * kGroups + group; unit < a.total; unit += stride) {
        const uint32_t token = unit / a.runs;
        const int h0 = (int)(unit - token * a.runs) * kHeads;
        const T* const src = reinterpret_cast<const T*>(a.x) + (int64_t)token * a.row_stride;
        float x[kHeads][kNrElems], g[kHeads][kNrElems];
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            const int h = min(h0 + u, heads - 1);
            const bool is_q = h < a.num_q_heads, is_v = h >= first_v;
            const int nh = is_q ? a.num_q_heads : a.num_kv_heads, hh = is_q ? h : (is_v ? h - first_v : h - a.num_q_heads);
            const T* const grad = reinterpret_cast<const T*>(is_q ? a.gq : (is_v ? a.gv : a.gk));
            if (grad != nullptr) {
                load_run<DT, kNrElems, VEC>(grad + ((int64_t)token * nh + hh) * D, d0, D, g[u]);
            } else {
#pragma unroll
                for (int i = 0; i < kNrElems; ++i) g[u][i] = 0.0f;
            }
            if (normed && !is_v) load_run<DT, kNrElems, VEC>(src + (int64_t)h * D, d0, D, x[u]);
        }
        Angles t;
        if (h0 < first_v) t = load_angles<VEC>(a, token, d0);
#pragma unroll
        for (int u = 0; u < kHeads; ++u) {
            const int h = h0 + u;
            if (h >= heads) break;
            if (h < first_v) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y0 = g[u][2 * i], y1 = g[u][2 * i + 1];
                    g[u][2 * i] = t.c[i] * y0 + t.s[i] * y1;
                    g[u][2 * i + 1] = t.c[i] * y1 - t.s[i] * y0;
                }
                if (normed) {
                    const bool is_q = h < a.num_q_heads;
                    float w[kNrElems], sum = 0.0f, dot = 0.0f;
                    load_any<kNrElems, VEC>(is_q ? a.q_weight : a.k_weight, a.w_dtype, d0, D, w);
#pragma unroll
                    for (int i = 0; i < kNrElems; ++i) {
                        sum += x[u][i] * x[u][i];
                        dot += (g[u][i] * w[i]) * x[u][i];
                    }
                    const float inv = 1.0f / sqrtf(row_sum<LPR>(sum) / (float)D + a.eps);
                    const float mean = row_sum<LPR>(dot) * inv / (float)D;
#pragma unroll
                    for (int i = 0; i < kNrElems; ++i) {
                        const float xh = x[u][i] * inv, s = g[u][i] * xh;
                        if (summed) {
                            dw[0][i] += is_q ? s : 0.0f;
                            dw[1][i] += is_q ? 0.0f : s;
                        }
                        g[u][i] = inv * (g[u][i] * w[i] - xh * mean);
                    }
                }
            }
            if (a.dx != nullptr)
                store_run8<DT, VEC>(reinterpret_cast<T*>(a.dx) + ((int64_t)token * heads + h) * D, d0, D, g[u]);
        }
    }
    if (!summed) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kNrElems; ++i) sums[group][d0 + i] = dw[k][i];
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
constexpr int64_t kNrMaxBlocks = (int64_t)1 << 20;

int check_norm_rope(const void* x, int dtype, int64_t rows, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                    int64_t row_stride, const void* positions, int pos_dtype, const void* cos_table, const void* sin_table,
                    int table_dtype, int64_t table_rows, const void* q_weight, const void* k_weight, int w_dtype) {
    if (!nr_float(dtype) || !nr_float(table_dtype) || !nr_float(w_dtype) || !nr_index(pos_dtype)) return KVFP8_EDTYPE;
    if (rows < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || head_dim % 2 != 0 || table_rows <= 0)
        return KVFP8_ESHAPE;
    const int64_t heads = (int64_t)num_q_heads + 2 * (int64_t)num_kv_heads;
    if (head_dim > kNrMaxDim || heads >= ((int64_t)1 << 24) || rows >= ((int64_t)1 << 31) / heads) return KVFP8_ELIMIT;
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

// Heads of a run. Few rows: one, for as many workgroups as there are; many: four.
constexpr int kNrRun = 4;
int run_of(int64_t rows, int64_t heads, int lanes) {
    return rows * heads * lanes >= (int64_t)device_cus() * 8 * kNrThreads ? kNrRun : 1;
}

template <bool kBackward, int DT, int LPR, bool VEC>
hipError_t launch_norm_rope(const NormRopeArgs& a, int run, unsigned blocks, hipStream_t s) {
    if constexpr (kBackward) {
        if (run == 1) hipLaunchKernelGGL((norm_rope_backward_kernel<DT, LPR, VEC, 1>), dim3(blocks), dim3(kNrThreads), 0, s, a);
        else hipLaunchKernelGGL((norm_rope_backward_kernel<DT, LPR, VEC, kNrRun>), dim3(blocks), dim3(kNrThreads), 0, s, a);
    } else {
        if (run == 1) hipLaunchKernelGGL((norm_rope_kernel<DT, LPR, VEC, 1>), dim3(blocks), dim3(kNrThreads), 0, s, a);
        else hipLaunchKernelGGL((norm_rope_kernel<DT, LPR, VEC, kNrRun>), dim3(blocks), dim3(kNrThreads), 0, s, a);
    }
    return hipGetLastError();
}

template <bool kBackward, int DT>
hipError_t launch_norm_rope(const NormRopeArgs& a, bool vec, int lanes, int run, unsigned blocks, hipStream_t s) {
    if (!vec) return launch_norm_rope<kBackward, DT, 64, false>(a, run, blocks, s);
    if (lanes == 8) return launch_norm_rope<kBackward, DT, 8, true>(a, run, blocks, s);
    if (lanes == 16) return launch_norm_rope<kBackward, DT, 16, true>(a, run, blocks, s);
    if (lanes == 32) return launch_norm_rope<kBackward, DT, 32, true>(a, run, blocks, s);
    return launch_norm_rope<kBackward, DT, 64, true>(a, run, blocks, s);
}

template <bool kBackward>
hipError_t launch_norm_rope(const NormRopeArgs& a, int dtype, bool vec, int lanes, int run, int64_t blocks, hipStream_t s) {
    switch (dtype) {
        case KVFP8_F32: return launch_norm_rope<kBackward, KVFP8_F32>(a, vec, lanes, run, (unsigned)blocks, s);
        case KVFP8_F16: return launch_norm_rope<kBackward, KVFP8_F16>(a, vec, lanes, run, (unsigned)blocks, s);
        default: return launch_norm_rope<kBackward, KVFP8_BF16>(a, vec, lanes, run, (unsigned)blocks, s);
    }
}

// Workgroups of the backward: at most what the device holds at once, as each leaves partial sums. By sizes alone
// (64 lanes a row, runs of one head), as the workspace is asked for without pointers.
int64_t backward_blocks(int64_t rows, int64_t heads) {
    const int64_t per = kNrThreads / 64, most = (int64_t)device_cus() * 4, wanted = (rows * heads + per - 1) / per;
    return wanted < most ? wanted : most;
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
    const int run = run_of(rows, heads, lanes);
    a.runs = (uint32_t)((heads + run - 1) / run);
    a.total = (uint32_t)(rows * a.runs);
    const int64_t per = kNrThreads / lanes, wanted = (a.total + per - 1) / per;
    return (int)launch_norm_rope<false>(a, dtype, vec, lanes, run, wanted < kNrMaxBlocks ? wanted : kNrMaxBlocks,
                                        reinterpret_cast<hipStream_t>(stream));
}

extern "C" int64_t kvfp8_norm_rope_backward_workspace_bytes(int64_t rows, int32_t num_q_heads, int32_t num_kv_heads,
                                                            int32_t head_dim) {
    if (rows <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    const int64_t heads = (int64_t)num_q_heads + 2 * (int64_t)num_kv_heads;
    if (head_dim > kNrMaxDim || heads >= ((int64_t)1 << 24) || rows >= ((int64_t)1 << 31) / heads) return 0;
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
        const int run = run_of(rows, heads, lanes);
        a.runs = (uint32_t)((heads + run - 1) / run);
        a.total = (uint32_t)(rows * a.runs);
        const hipError_t err = launch_norm_rope<true>(a, dtype, vec, lanes, run, blocks, s);
        if (err != hipSuccess) return (int)err;
    }
    if (!summed) return KVFP8_OK;
    hipLaunchKernelGGL(norm_rope_weight_grad_kernel, dim3((unsigned)((2 * head_dim + 7) / 8)), dim3(kNrThreads), 0, s,
                       reinterpret_cast<const float*>(workspace), (int32_t)blocks, head_dim, w_dtype, dq_weight, dk_weight);
    return (int)hipGetLastError();
}
