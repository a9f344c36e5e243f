// Log probabilities of given tokens, entropy and the most probable tokens of logit rows, and
// the gradient of the logits (gfx950).
//
// For a row x[0 .. V) with m = max x and S = sum e^(x - m):
//   logprob of token y   (x_y - m) - ln S
//   entropy              ln S - (1 / S) sum e^(x - m) (x - m)      (both terms are >= 0)
//   alternatives         the `top` largest x, ties to the lowest index, as (x - m) - ln S
//   gradient             dx_j = g ([j = y] - p_j) - h p_j (ln p_j + H),  p_j = e^((x_j - m) - ln S)
// with g, h the gradients of the log probability and the entropy. x - m is formed before the
// exponent's scale, so the largest entry weighs exactly 1 whatever its size.
//
// A token outside [0, V) has log probability 0 and no gradient of its own (a row without a
// target). Entries of -inf weigh nothing. A row of -inf alone has log probability -inf, entropy 0,
// alternatives of -inf at indices 0, 1, .. and gradient 0. NaN or +inf anywhere gives NaN
// (alternatives: NaN counts as the largest value).
//
// One workgroup per row. Pass 1 keeps (m, S, sum e^d d) per thread, online, and the thread's largest
// value. Alternatives: each wave finds the `top`-th largest of its 64 thread maxima by a search over
// the bits of the value (ballots); the largest such bound over the waves is one that at least
// `top` entries of the row reach. Pass 2 collects the entries that reach it in LDS and ranks them by
// counting. Rows with more such entries than the list holds (long runs of equal logits), and rows
// with NaN, are searched entry by entry instead.
#include "kvfp8_common.h"

namespace kvfp8 {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kList = 1024;           // entries of the alternatives' list
constexpr int kMaxTop = 64;           // a wave's thread maxima

struct LogprobArgs {
    const void* x;
    int64_t stride;                   // elements between rows
    int64_t row0;                     // first row of the launch
    int32_t vocab;
    int32_t top;
    const void* tokens;
    int32_t tokens64;
    float* logprobs;
    float* entropy;
    float2* stats;                    // (m, ln S) of every row
    float* top_logprobs;              // [rows, top]
    int64_t* top_tokens;
};

// Sixteen bytes at any element-aligned address (one unaligned vector access).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec16 {
    uint32_t w[4];
};

template <int DT>
__device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&v)[16 / sizeof(typename Elem<DT>::T)]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == KVFP8_F32) {
            v[i] = bits_f32(w[i]);
        } else if constexpr (DT == KVFP8_BF16) {
            v[2 * i] = bits_f32(w[i] << 16);
            v[2 * i + 1] = bits_f32(w[i] & 0xFFFF0000u);
        } else {
            v[2 * i] = f16_to_f32((uint16_t)w[i]);
            v[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16));
        }
    }
}

// Order of values as unsigned integers: NaN above +inf, -0 as +0. 0 is below every value.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = f32_bits(x + 0.0f);
    if (x != x) return 0xFFFFFFFFu;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
    return k == 0xFFFFFFFFu ? bits_f32(0x7FC00000u) : bits_f32((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
// Larger value first, then the lower index.
__device__ __forceinline__ uint64_t entry_key(uint32_t value, int32_t index) {
    return ((uint64_t)value << 32) | (uint32_t)~index;
}

struct Sums {
    float m, s, t;      // max, sum e^(x - m), sum e^(x - m) (x - m)
};

// The state with its maximum moved up to m (finite or -inf, at least s.m).
__device__ __forceinline__ Sums moved(Sums a, float m) {
    const float d = a.m == kNegInf ? 0.0f : a.m - m;     // an empty state has s = t = 0
    const float f = __builtin_amdgcn_exp2f(d * kLog2e);
    return Sums{m, a.s * f, (a.t + d * a.s) * f};
}
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    a = moved(a, m);
    b = moved(b, m);
    return Sums{m, a.s + b.s, a.t + b.t};
}

// Adds e^d and e^d d of d = x - m. Below -200 e^d is 0, and d is kept finite for the product.
__device__ __forceinline__ void add_entry(Sums& a, float x, float m) {
    const float d = x - m;
    const float e = __builtin_amdgcn_exp2f(d * kLog2e);
    a.s += e;
    a.t += e * fmaxf(d, -200.0f);
}

template <int DT, int NT>
__global__ void __launch_bounds__(NT)
token_logprobs_kernel(LogprobArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int kPer = 16 / (int)sizeof(T);
    constexpr int kWaves = NT / 64;
    __shared__ Sums wave_sums[kWaves];
    __shared__ uint32_t wave_bound[kWaves];
    __shared__ uint64_t list[kList];
    __shared__ int32_t listed;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = a.row0 + blockIdx.x;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.stride;
    const int32_t vectors = a.vocab / kPer, rest = a.vocab - vectors * kPer;

    Sums st = {kNegInf, 0.0f, 0.0f};
    uint32_t best = 0;
    for (int32_t i = tid; i < vectors; i += NT) {
        float v[kPer];
        unpack<DT>(reinterpret_cast<const Vec16<T>*>(x)[i].w, v);
        float mx = v[0];
#pragma unroll
        for (int e = 1; e < kPer; ++e) mx = fmaxf(mx, v[e]);
        if (mx > st.m) st = moved(st, mx);
        const float m = st.m == kNegInf ? 0.0f : st.m;
#pragma unroll
        for (int e = 0; e < kPer; ++e) add_entry(st, v[e], m);
    }
    if (tid < rest) {
        const float v = Elem<DT>::load(x[vectors * kPer + tid]);
        if (v > st.m) st = moved(st, v);
        add_entry(st, v, st.m == kNegInf ? 0.0f : st.m);
    }
    if (a.top > 0) {
        // The wave's bound: the top-th largest thread maximum (0 where fewer threads hold entries).
        best = tid < vectors || tid < rest ? ordered(st.m) : 0u;
        uint32_t bound = 0;
        for (int bit = 31; bit >= (DT == KVFP8_BF16 ? 16 : 0); --bit) {
            const uint32_t trial = bound | (1u << bit);
            if (__popcll(__ballot(best >= trial)) >= a.top) bound = trial;
        }
        if (lane == 0) wave_bound[wave] = bound;
        if (tid == 0) listed = 0;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1)
        st = joined(st, Sums{__shfl_xor(st.m, off), __shfl_xor(st.s, off), __shfl_xor(st.t, off)});
    if (lane == 0) wave_sums[wave] = st;
    __syncthreads();
    st = wave_sums[0];
    uint32_t bound = a.top > 0 ? wave_bound[0] : 0u;
    for (int w = 1; w < kWaves; ++w) {
        st = joined(st, wave_sums[w]);
        if (a.top > 0) bound = max(bound, wave_bound[w]);
    }
    const bool empty = st.m == kNegInf && st.s == 0.0f;      // every entry is -inf
    const float log_s = empty ? kNegInf : __builtin_logf(st.s);
    if (tid == 0) {
        const int64_t token = a.tokens64 ? reinterpret_cast<const int64_t*>(a.tokens)[row]
                                         : (int64_t)reinterpret_cast<const int32_t*>(a.tokens)[row];
        float lp = 0.0f;
        if (token >= 0 && token < a.vocab) lp = empty ? kNegInf : (Elem<DT>::load(x[token]) - st.m) - log_s;
        a.logprobs[row] = lp;
        a.entropy[row] = empty ? 0.0f : log_s - st.t / st.s;
        a.stats[row] = make_float2(st.m, log_s);
    }
    if (a.top == 0) return;

    auto emit = [&](int32_t rank, uint64_t key) {
        const float v = from_ordered((uint32_t)(key >> 32));
        a.top_logprobs[row * a.top + rank] = empty ? kNegInf : (v - st.m) - log_s;
        a.top_tokens[row * a.top + rank] = (int64_t)(int32_t)~(uint32_t)key;
    };
    // Every entry whose value reaches the bound, once.
    auto scan = [&](auto&& visit) {
        for (int32_t i = tid; i < vectors; i += NT) {
            float v[kPer];
            unpack<DT>(reinterpret_cast<const Vec16<T>*>(x)[i].w, v);
#pragma unroll
            for (int e = 0; e < kPer; ++e) visit(ordered(v[e]), i * kPer + e);
        }
        if (tid < rest) visit(ordered(Elem<DT>::load(x[vectors * kPer + tid])), vectors * kPer + tid);
    };
    const bool clean = st.s == st.s;         // no NaN and no +inf
    if (clean)
        scan([&](uint32_t value, int32_t index) {
            if (value >= bound) {
                const int32_t at = atomicAdd(&listed, 1);
                if (at < kList) list[at] = entry_key(value, index);
            }
        });
    __syncthreads();
    if (clean && listed <= kList) {
        // The list's order is that of arrival; a rank counts keys, which are distinct.
        const int32_t n = listed;
        for (int32_t i = tid; i < n; i += NT) {
            const uint64_t key = list[i];
            int32_t rank = 0;
            for (int32_t j = 0; j < n; ++j) rank += list[j] > key;
            if (rank < a.top) emit(rank, key);
        }
        return;
    }
    // One alternative per round: the largest key below the last one.
    uint64_t last = 0;
    for (int32_t r = 0; r < a.top; ++r) {
        uint64_t mine = 0;
        scan([&](uint32_t value, int32_t index) {
            const uint64_t key = entry_key(value, index);
            if ((r == 0 || key < last) && key > mine) mine = key;
        });
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint64_t other = (uint64_t)__shfl_xor((long long)mine, off);
            mine = other > mine ? other : mine;
        }
        __syncthreads();
        if (lane == 0) list[wave] = mine;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) mine = list[w] > mine ? list[w] : mine;
        if (tid == 0) emit(r, mine);
        last = mine;
    }
}

struct LogprobGradArgs {
    const void* x;
    int64_t stride;
    int64_t row0;
    int32_t vocab;
    const void* tokens;
    int32_t tokens64;
    const float* entropy;
    const float2* stats;
    const float* grad_logprobs;       // either may be null
    const float* grad_entropy;
    void* dx;                         // [rows, vocab] contiguous
};

constexpr int kGradThreads = 256;

template <int DT>
__global__ void __launch_bounds__(kGradThreads)
token_logprobs_grad_kernel(LogprobGradArgs a, int32_t pieces) {
    using T = typename Elem<DT>::T;
    constexpr int kPer = 16 / (int)sizeof(T);
    const int32_t local = (int32_t)(blockIdx.x / pieces), piece = (int32_t)(blockIdx.x - local * pieces);
    const int64_t row = a.row0 + local;
    const T* x = reinterpret_cast<const T*>(a.x) + row * a.stride;
    T* dx = reinterpret_cast<T*>(a.dx) + row * a.vocab;
    const float2 st = a.stats[row];
    const int64_t token64 = a.tokens64 ? reinterpret_cast<const int64_t*>(a.tokens)[row]
                                       : (int64_t)reinterpret_cast<const int32_t*>(a.tokens)[row];
    const bool given = token64 >= 0 && token64 < a.vocab;
    const int32_t token = given ? (int32_t)token64 : -1;
    const float g = given && a.grad_logprobs != nullptr ? a.grad_logprobs[row] : 0.0f;
    const float h = a.grad_entropy != nullptr ? a.grad_entropy[row] : 0.0f;
    const float entropy = a.entropy[row];
    const bool empty = st.y == kNegInf;              // every entry is -inf
    auto grad = [&](float v, int32_t index) {
        const float logp = (v - st.x) - st.y;
        const float p = __builtin_amdgcn_exp2f(logp * kLog2e);
        const float d = -p * (g + h * (fmaxf(logp, -200.0f) + entropy));
        return empty ? 0.0f : (index == token ? d + g : d);
    };
    const int32_t vectors = a.vocab / kPer, rest = a.vocab - vectors * kPer;
    for (int32_t i = piece * kGradThreads + threadIdx.x; i < vectors; i += pieces * kGradThreads) {
        float v[kPer];
        unpack<DT>(reinterpret_cast<const Vec16<T>*>(x)[i].w, v);
        Vec16<T> out;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if constexpr (DT == KVFP8_F32) {
                out.w[w] = f32_bits(grad(v[w], i * kPer + w));
            } else {
                out.w[w] = (uint32_t)Elem<DT>::store(grad(v[2 * w], i * kPer + 2 * w)) |
                           ((uint32_t)Elem<DT>::store(grad(v[2 * w + 1], i * kPer + 2 * w + 1)) << 16);
            }
        }
        reinterpret_cast<Vec16<T>*>(dx)[i] = out;
    }
    if (piece == 0 && (int32_t)threadIdx.x < rest) {
        const int32_t index = vectors * kPer + threadIdx.x;
        dx[index] = Elem<DT>::store(grad(Elem<DT>::load(x[index]), index));
    }
}

int check_rows(int dtype, int64_t stride, int64_t rows, int64_t vocab, int tok_dtype) {
    if (dtype != KVFP8_F32 && dtype != KVFP8_F16 && dtype != KVFP8_BF16) return KVFP8_EDTYPE;
    if (tok_dtype != KVFP8_I32 && tok_dtype != KVFP8_I64) return KVFP8_EDTYPE;
    if (rows < 0 || vocab <= 0 || stride < 0) return KVFP8_ESHAPE;
    if (vocab >= ((int64_t)1 << 30)) return KVFP8_ELIMIT;
    return KVFP8_OK;
}

bool aligned(const void* p, int dtype) { return (uintptr_t)p % (dtype == KVFP8_F32 ? 4 : 2) == 0; }

// A launch has fewer than 2^32 threads: rows go in runs of this many workgroups.
constexpr int64_t kMaxGroups = (int64_t)1 << 21;

template <int DT>
hipError_t launch_logprobs(LogprobArgs a, int64_t rows, hipStream_t s) {
    for (a.row0 = 0; a.row0 < rows; a.row0 += kMaxGroups) {
        const dim3 grid((unsigned)(rows - a.row0 < kMaxGroups ? rows - a.row0 : kMaxGroups));
        if (a.vocab <= 8192)
            hipLaunchKernelGGL((token_logprobs_kernel<DT, 256>), grid, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((token_logprobs_kernel<DT, 1024>), grid, dim3(1024), 0, s, a);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

template <int DT>
hipError_t launch_logprobs_grad(LogprobGradArgs a, int64_t rows, hipStream_t s) {
    // Eight vectors a thread; vocab < 2^30 keeps the pieces of a row below kMaxGroups.
    const int64_t vectors = a.vocab / (DT == KVFP8_F32 ? 4 : 8);
    const int32_t pieces = (int32_t)((vectors + 8 * kGradThreads - 1) / (8 * kGradThreads)) + (vectors == 0);
    const int64_t run = kMaxGroups / pieces;
    for (a.row0 = 0; a.row0 < rows; a.row0 += run) {
        const int64_t n = rows - a.row0 < run ? rows - a.row0 : run;
        hipLaunchKernelGGL((token_logprobs_grad_kernel<DT>), dim3((unsigned)(n * pieces)), dim3(kGradThreads), 0, s, a, pieces);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

}  // namespace

}  // namespace kvfp8

using namespace kvfp8;

extern "C" int kvfp8_token_logprobs(const void* logits, int dtype, int64_t row_stride, int64_t rows, int64_t vocab,
                                    const void* tokens, int tok_dtype, int32_t top, float* logprobs, float* entropy,
                                    float* stats, float* top_logprobs, int64_t* top_tokens, void* stream) {
    const int bad = check_rows(dtype, row_stride, rows, vocab, tok_dtype);
    if (bad != KVFP8_OK) return bad;
    if (top < 0 || top > vocab) return KVFP8_ESHAPE;
    if (top > kMaxTop) return KVFP8_ELIMIT;
    if (rows == 0) return KVFP8_OK;
    if (!logits || !tokens || !logprobs || !entropy || !stats || (top > 0 && (!top_logprobs || !top_tokens)))
        return KVFP8_ENULL;
    if (!aligned(logits, dtype) || (uintptr_t)stats % 8 != 0) return KVFP8_ESTRIDE;
    const LogprobArgs a = {logits, row_stride, 0, (int32_t)vocab, top, tokens, tok_dtype == KVFP8_I64,
                           logprobs, entropy, reinterpret_cast<float2*>(stats), top_logprobs, top_tokens};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (dtype) {
        case KVFP8_F32: return (int)launch_logprobs<KVFP8_F32>(a, rows, s);
        case KVFP8_F16: return (int)launch_logprobs<KVFP8_F16>(a, rows, s);
        default: return (int)launch_logprobs<KVFP8_BF16>(a, rows, s);
    }
}

extern "C" int kvfp8_token_logprobs_backward(const void* logits, int dtype, int64_t row_stride, int64_t rows,
                                             int64_t vocab, const void* tokens, int tok_dtype, const float* entropy,
                                             const float* stats, const float* grad_logprobs, const float* grad_entropy,
                                             void* grad_logits, void* stream) {
    const int bad = check_rows(dtype, row_stride, rows, vocab, tok_dtype);
    if (bad != KVFP8_OK) return bad;
    if (rows == 0) return KVFP8_OK;
    if (!logits || !tokens || !entropy || !stats || !grad_logits) return KVFP8_ENULL;
    if (!aligned(logits, dtype) || !aligned(grad_logits, dtype) || (uintptr_t)stats % 8 != 0) return KVFP8_ESTRIDE;
    const LogprobGradArgs a = {logits, row_stride, 0, (int32_t)vocab, tokens, tok_dtype == KVFP8_I64, entropy,
                               reinterpret_cast<const float2*>(stats), grad_logprobs, grad_entropy, grad_logits};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (dtype) {
        case KVFP8_F32: return (int)launch_logprobs_grad<KVFP8_F32>(a, rows, s);
        case KVFP8_F16: return (int)launch_logprobs_grad<KVFP8_F16>(a, rows, s);
        default: return (int)launch_logprobs_grad<KVFP8_BF16>(a, rows, s);
    }
}
