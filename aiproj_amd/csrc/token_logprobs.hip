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
// One workgroup per row. Rows of up to 131072 16-bit entries (65536 of float32) stay in registers: every load is
// issued at once, the maximum is known before the first exponential, and the row is read once. Longer rows
// keep (m, S, sum e^d d) per thread online and are read again for the alternatives.
//
// Alternatives: with A waves that hold entries in all lanes, every wave finds the n-th largest of its 64 thread maxima,
// n = ceil(top / A); the ceil(top / n)-th largest of these is a bound that at least `top` entries of the row reach,
// and not many more. The entries that reach it are collected in LDS and ranked by counting. Where more reach it than
// the list holds (runs of equal logits, masked rows, sorted rows), the bound is raised to the largest over the waves of
// the `top`-th thread maximum, only entries above it are collected, and those equal to it follow by index. What still
// does not fit, and rows with NaN, are searched entry by entry.
#include "mfma_tiles.h"

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
    float2* stats;                    // (m, ln S) of every row, or null
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

// DPP lane permutations inside rows of 16 lanes; together they reach all 16.
constexpr int kDppXor1 = 0xB1;          // quad_perm [1, 0, 3, 2]
constexpr int kDppXor2 = 0x4E;          // quad_perm [2, 3, 0, 1]
constexpr int kDppHalfMirror = 0x141;   // lane i <-> 7 - i within each 8 lanes
constexpr int kDppMirror = 0x140;       // lane i <-> 15 - i within each row
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_bits(x), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, dpp<kDppXor1>(x));
    x = fmaxf(x, dpp<kDppXor2>(x));
    x = fmaxf(x, dpp<kDppHalfMirror>(x));
    return fmaxf(x, dpp<kDppMirror>(x));
}
__device__ __forceinline__ float row_sum(float x) {
    x += dpp<kDppXor1>(x);
    x += dpp<kDppXor2>(x);
    x += dpp<kDppHalfMirror>(x);
    return x + dpp<kDppMirror>(x);
}
__device__ __forceinline__ float wave_max(float x) { return max_across_rows(row_max(x)); }
__device__ __forceinline__ float wave_sum(float x) { return sum_across_rows(row_sum(x)); }

__device__ __forceinline__ float first_lane(float x) { return bits_f32((uint32_t)__builtin_amdgcn_readfirstlane((int)f32_bits(x))); }

struct Sums {
    float m, s, t;      // max, sum e^(x - m), sum e^(x - m) (x - m)
};

// The state with its maximum moved up to m (finite or -inf, at least a.m). Below -200 f is 0, and d is kept finite for
// the product: entries of a type's lowest value are some 1e38 below the others, which the number of them takes past
// float32's range.
__device__ __forceinline__ Sums moved(Sums a, float m) {
    const float d = a.m == kNegInf ? 0.0f : a.m - m;     // an empty state has s = t = 0
    const float f = __builtin_amdgcn_exp2f(d * kLog2e);
    return Sums{m, a.s * f, (a.t + fmaxf(d, -200.0f) * a.s) * f};
}

// Adds e^d and e^d d of d = x - m. Below -200 e^d is 0, and d is kept finite for the product.
__device__ __forceinline__ void add_entry(Sums& a, float x, float m) {
    const float d = x - m;
    const float e = __builtin_amdgcn_exp2f(d * kLog2e);
    a.s += e;
    a.t += e * fmaxf(d, -200.0f);
}

// Two entries of -inf (one of float32).
template <int DT>
constexpr uint32_t kNegInfBits = DT == KVFP8_F32 ? 0xFF800000u : (DT == KVFP8_BF16 ? 0xFF80FF80u : 0xFC00FC00u);
// Lowest bit of the wave's first search for a bound: the values' own last bit, or 20 bits of float32 (a bound that is
// a little low only lets more entries into the list; in the order of negative values the bits left out are ones, so it
// lies below the value itself). The second bound has all bits: it has to be a value of the row, which entries equal.
template <int DT>
constexpr int kLastBit = DT == KVFP8_BF16 ? 16 : (DT == KVFP8_F16 ? 13 : 12);

// R: vectors of 16 bytes a thread holds; 0: the row is read in passes.
template <int DT, int NT, int R>
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
    const int64_t token = a.tokens64 ? reinterpret_cast<const int64_t*>(a.tokens)[row]
                                     : (int64_t)reinterpret_cast<const int32_t*>(a.tokens)[row];
    const bool given = token >= 0 && token < a.vocab;

    uint32_t raw[R > 0 ? R : 1][4];
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int32_t i = r * NT + tid;
            if (i < vectors) {
                const Vec16<T> v = reinterpret_cast<const Vec16<T>*>(x)[i];
#pragma unroll
                for (int w = 0; w < 4; ++w) raw[r][w] = v.w[w];
            } else {
#pragma unroll
                for (int w = 0; w < 4; ++w) raw[r][w] = kNegInfBits<DT>;
            }
        }
    }
    // The entries behind the last whole vector, one a thread.
    const float tail = tid < rest ? Elem<DT>::load(x[vectors * kPer + tid]) : kNegInf;
    const float chosen = tid == 0 && given ? Elem<DT>::load(x[token]) : 0.0f;
    if (tid == 0) listed = 0;

    // Between the passes over the registers: the words stay packed (else every unpacked value is kept).
    auto keep_packed = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int w = 0; w < 4; ++w) __asm__ volatile("" : "+v"(raw[r][w]));
    };
    Sums st = {kNegInf, 0.0f, 0.0f};
    float best = tail;                                    // this thread's largest value
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[kPer];
            unpack<DT>(raw[r], v);
#pragma unroll
            for (int e = 0; e < kPer; ++e) best = fmaxf(best, v[e]);
        }
        st.m = wave_max(best);
        keep_packed();
        const float m = st.m == kNegInf ? 0.0f : st.m;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[kPer];
            unpack<DT>(raw[r], v);
#pragma unroll
            for (int e = 0; e < kPer; ++e) add_entry(st, v[e], m);
        }
        if (tid < rest) add_entry(st, tail, m);
    } else {
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
            if (tail > st.m) st = moved(st, tail);
            add_entry(st, tail, st.m == kNegInf ? 0.0f : st.m);
        }
        best = fmaxf(best, st.m);
        st = moved(st, wave_max(st.m));
    }
    // The n-th largest thread maximum of the wave, as an order of values (0 where fewer threads hold entries).
    const uint32_t mine = tid < vectors || tid < rest ? ordered(best) : 0u;
    auto nth_of_wave = [&](int n, int last_bit) __attribute__((always_inline)) {
        uint32_t bound = 0;
        for (int bit = 31; bit >= last_bit; --bit) {
            const uint32_t trial = bound | (1u << bit);
            if (__popcll(__ballot(mine >= trial)) >= n) bound = trial;
        }
        return bound;
    };
    const int full = min(vectors / 64, kWaves);          // waves that hold entries in all lanes
    if (a.top > 0) {
        uint32_t bound = 0;
        const int n = full > 0 ? (a.top + full - 1) / full : 0;
        if (n == 1) bound = ordered(st.m);
        else if (n > 1) bound = nth_of_wave(n, kLastBit<DT>);
        if (lane == 0) wave_bound[wave] = bound;
    }
    st.s = wave_sum(st.s);
    st.t = wave_sum(st.t);
    if (lane == 0) wave_sums[wave] = st;
    __syncthreads();
    // Every row of 16 lanes joins the waves' states, one a lane; all take lane 0's result (a fused multiply in the sums
    // rounds differently per lane, and the alternatives are written by threads in order of arrival).
    const bool holds = (lane & 15) < kWaves;
    st = holds ? wave_sums[lane & (kWaves - 1)] : Sums{kNegInf, 0.0f, 0.0f};
    st = moved(st, row_max(st.m));
    st.s = first_lane(row_sum(st.s));
    st.t = first_lane(row_sum(st.t));
    const bool empty = st.m == kNegInf && st.s == 0.0f;  // every entry is -inf
    const float log_s = empty ? kNegInf : __builtin_logf(st.s);
    if (tid == 0) {
        a.logprobs[row] = !given ? 0.0f : (empty ? kNegInf : (chosen - st.m) - log_s);
        a.entropy[row] = empty ? 0.0f : log_s - st.t / st.s;
        if (a.stats != nullptr) a.stats[row] = make_float2(st.m, log_s);
    }
    if (a.top == 0) return;

    auto emit = [&](int32_t rank, uint64_t key) {
        const float v = from_ordered((uint32_t)(key >> 32));
        a.top_logprobs[row * a.top + rank] = empty ? kNegInf : (v - st.m) - log_s;
        a.top_tokens[row * a.top + rank] = (int64_t)(int32_t)~(uint32_t)key;
    };
    // Every entry of this thread, with its index.
    auto scan_memory = [&](auto&& visit) __attribute__((always_inline)) {
        for (int32_t i = tid; i < vectors; i += NT) {
            float v[kPer];
            unpack<DT>(reinterpret_cast<const Vec16<T>*>(x)[i].w, v);
#pragma unroll
            for (int e = 0; e < kPer; ++e) visit(v[e], i * kPer + e);
        }
        if (tid < rest) visit(tail, vectors * kPer + tid);
    };
    auto scan = [&](auto&& visit) __attribute__((always_inline)) {
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int32_t i = r * NT + tid;
                if (i < vectors) {
                    float v[kPer];
                    unpack<DT>(raw[r], v);
#pragma unroll
                    for (int e = 0; e < kPer; ++e) visit(v[e], i * kPer + e);
                }
            }
            if (tid < rest) visit(tail, vectors * kPer + tid);
        } else {
            scan_memory(visit);
        }
    };
    // The least value of an order bound. (Shortened to its upper bits, the order of -inf is that of no value.)
    auto value_of = [&](uint32_t bound) __attribute__((always_inline)) { return bound <= 0x007FFFFFu ? kNegInf : from_ordered(bound); };
    // Collects the entries above `least` (and those equal to it) and returns their number; all threads.
    auto collect = [&](float least, bool equal) __attribute__((always_inline)) {
        if (equal ? best >= least : best > least)
            scan([&](float v, int32_t index) {
                if (v > least || (equal && v == least)) {
                    const int32_t at = atomicAdd(&listed, 1);
                    if (at < kList) list[at] = entry_key(ordered(v), index);
                }
            });
        __syncthreads();
        return listed;
    };
    // The list's order is that of arrival; a rank counts keys, which are distinct. Sixteen lanes count for a key.
    auto rank_list = [&](int32_t n) __attribute__((always_inline)) {
        for (int32_t i = tid >> 4; i < n; i += NT / 16) {
            const uint64_t key = list[i];
            int32_t above = 0;
            for (int32_t j = tid & 15; j < n; j += 16) above += list[j] > key;
            const int32_t rank = (int32_t)row_sum((float)above);           // at most kList: exact
            if (rank < a.top && (tid & 15) == 0) emit(rank, key);
        }
    };
    const bool clean = st.s == st.s;                     // no NaN and no +inf
    if (clean) {
        keep_packed();
        uint32_t bound = 0;
        if (full > 0) {
            const int each = (a.top + full - 1) / full, rank = (a.top + each - 1) / each - 1;
            const int w = lane & (kWaves - 1);
            const uint32_t b = w < full ? wave_bound[w] : 0u;
            int above = 0;
#pragma unroll
            for (int v = 0; v < kWaves; ++v) {
                const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)b, v);
                above += v < full && (other > b || (other == b && v < w));
            }
            bound = (uint32_t)__builtin_amdgcn_readlane((int)b, (int)__builtin_ctzll(__ballot(w < full && above == rank)));
        }
        int32_t n = collect(value_of(bound), true);
        if (n <= kList) {
            rank_list(n);
            return;
        }
        __syncthreads();                                 // all have read the bounds and the count
        const uint32_t higher = nth_of_wave(a.top, 0);
        if (lane == 0) wave_bound[wave] = higher;
        if (tid == 0) listed = 0;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) bound = max(bound, wave_bound[w]);
        const float least = value_of(bound);
        n = collect(least, false);
        if (n <= kList) {
            if (n < a.top) {
                // The first entries equal to the bound, in the order of their index.
                if (wave == 0) {
                    for (int32_t i = lane; n < a.top && i - lane < a.vocab; i += 64) {
                        const bool hit = i < a.vocab && Elem<DT>::load(x[i]) == least;
                        const uint64_t hits = __ballot(hit);
                        const int32_t at = n + __popcll(hits & (((uint64_t)1 << lane) - 1));
                        if (hit && at < a.top) list[at] = entry_key(ordered(least), i);
                        n += __popcll(hits);
                    }
                }
                __syncthreads();
                n = a.top;
            }
            rank_list(n);
            return;
        }
        __syncthreads();                                 // all have read the count
    }
    // One alternative per round: the largest key below the last one.
    uint64_t last = 0;
    for (int32_t r = 0; r < a.top; ++r) {
        uint64_t most = 0;
        scan_memory([&](float v, int32_t index) {
            const uint64_t key = entry_key(ordered(v), index);
            if ((r == 0 || key < last) && key > most) most = key;
        });
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint64_t other = (uint64_t)__shfl_xor((long long)most, off);
            most = other > most ? other : most;
        }
        __syncthreads();
        if (lane == 0) list[wave] = most;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) most = list[w] > most ? list[w] : most;
        if (tid == 0) emit(r, most);
        last = most;
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

// Bound by HBM: a piece of a row per workgroup, its logits read and the gradient written 16 bytes a lane, nothing
// exchanged (the row's m, ln S and entropy come from the forward). 4096 x 32000 bf16: 84-90 us, 5.8-6.2 TB/s; 333 x 32000
// float32: 15 us.
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

template <int DT, int NT, int R>
void launch_rows(const LogprobArgs& a, int64_t rows, hipStream_t s) {
    hipLaunchKernelGGL((token_logprobs_kernel<DT, NT, R>), dim3((unsigned)rows), dim3(NT), 0, s, a);
}

// Threads and vectors a thread by the row's length. More rows than two per CU are bound by the loads that are in flight
// between the workgroups' barriers, and take more, smaller workgroups. Measured, 4096 rows of 32000 bf16, no, 1, 5
// and 20 alternatives: 1024 threads 49, 74, 71 and 81 us, 512 threads 43, 54, 57 and 63, 256 threads 42, 56, 63
// and 63 (262 MB: 6.1 TB/s without alternatives). A few rows are bound by latency: one row, 1024 threads, 4.1, 6.9,
// 7.0 and 7.9 us.
template <int DT>
hipError_t launch_logprobs(LogprobArgs a, int64_t rows, hipStream_t s) {
    const int64_t vectors = a.vocab / (DT == KVFP8_F32 ? 4 : 8);
    for (a.row0 = 0; a.row0 < rows; a.row0 += kMaxGroups) {
        const int64_t n = rows - a.row0 < kMaxGroups ? rows - a.row0 : kMaxGroups;
        const bool many = n > 2 * device_cus();
        if (vectors <= 256) launch_rows<DT, 256, 1>(a, n, s);
        else if (vectors <= 1024) launch_rows<DT, 256, 4>(a, n, s);
        else if (many && vectors <= 2048) launch_rows<DT, 512, 4>(a, n, s);
        else if (many && vectors <= 4096) launch_rows<DT, 512, 8>(a, n, s);
        else if (many && vectors <= 8192) launch_rows<DT, 512, 16>(a, n, s);
        else if (vectors <= 2048) launch_rows<DT, 1024, 2>(a, n, s);
        else if (vectors <= 4096) launch_rows<DT, 1024, 4>(a, n, s);
        else if (vectors <= 8192) launch_rows<DT, 1024, 8>(a, n, s);
        else if (vectors <= 16384) launch_rows<DT, 1024, 16>(a, n, s);
        else launch_rows<DT, 1024, 0>(a, n, s);
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
    if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_logprobs || !top_tokens)))
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
