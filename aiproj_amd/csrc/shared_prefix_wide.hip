// Shared prefixes for many rows: blocks of 256 (row, q head) pairs against a prefix, gfx950.
//
// A workgroup takes one (row block, KV head, split of the prefix). Its eight waves hold 32 rows each and share the
// prefix's tokens through LDS in blocks of 64: the codes are widened to 16 bits once per workgroup on their way
// there (exact), instead of once per wave, and the tokens' bytes cross L2 once per 256 rows. A wave takes a block in
// two halves of 32 tokens (MFMA 32x32x16: A[row = l % 32][k = 8 (l / 32) + i], B likewise, D[row = 8 (i / 4) + 4 (l / 32)
// + i % 4][col = l % 32]):
//   S^T[token, row] = K Q^T     A = K rows from LDS, B = Q^T from registers
//   softmax                     t = score x (k_scale[token] x sm_scale x log2(e)), e2(t - reference), float32, online, base
//                               2; the reference follows a row's maximum only where that exceeds it by 2^8. The product
//                               is rounded before the reference is taken off: fused, an equal key in a later block would
//                               differ by up to half a step of the reference, which at scores of 1e8 is a factor of 16
//                               (the operation more costs 1.1% to 1.6% of a call)
//   O^T[d, row] += V^T P'^T     P' = e2() v_scale[token] from the score registers; A = V^T by transposing LDS reads
//
// One stretch of code without a branch holds, for half s, the products of the scores of half s + 1, the weights of half
// s and the products with V of half s - 1, which are independent of each other; scheduling groups spread the products
// over the vector operations and start the LDS reads ahead. The staging of later blocks lies in the stretch of a block's
// first half, a barrier behind it:
//   first half of g     scores K(g) second half, V(g - 1) second half;  V(g) and K(g + 1) to LDS, loads of V(g + 1), K(g + 2)
//   second half of g    scores K(g + 1) first half, V(g) first half
// so two buffers of each do: K(g + 1) replaces K(g - 1) and V(g) replaces V(g - 2), both last read before the barrier of
// block g - 1. Scales and counts, of which a wave that lags may still read those of g - 1, have four buffers.
//
// What bounds it (256 x 64 heads, 16384 tokens of 8 KV heads x 128, bf16 on e4m3fn: 157-175 us without the own tokens, 800-870
// TFLOP/s): a block takes 5300 cycles of which the matrix cores work 2050 and the vector ALU 2500 (seven operations a score,
// the exponential counts two), and one hides little of the other: next to 16x16x32 products vector operations of
// another wave took 70% of their time on top, next to 32x32x16 ones 37% (both alone in a loop). LDS reads fill 1600 cycles
// (256 bytes each), the widened writes 500. Measured on 9216 rows x 16 heads x 4096 tokens: two half-workgroups in turn on
// products and softmax 480 us, this order with 16x16x32 products 463, with 32x32x16 445.
//
// LDS rows are 16-byte chunks in an order by row in which neither the 32 rows of a K read nor the 4 x 4 chunks of a
// transposing read meet in a bank (4.4 and 3.7 cycles an instruction; chunk ^ (row % 16) 4.4 and, for these blocks, 7.9).
#include "shared_prefix_narrow.h"

namespace kvfp8 {

namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr int kKeys = 64;             // tokens per block
constexpr int kWideWaves = 8;
// log2 of how far a row's maximum may exceed its reference. Weights reach 2^8 so, and the largest is not 1 in general: it
// is rounded to the products' type like the others, by at most half a step relatively, while their sum is not.
constexpr float kLag = 8.0f;

typedef __attribute__((address_space(3))) const uint8_t lds_u8;
typedef __attribute__((address_space(3))) const u32x4_t lds_u32x4;
typedef __attribute__((address_space(3))) const u32x2_t lds_u32x2;
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

typedef float f32x16_t __attribute__((ext_vector_type(16)));

// c += a b of 32 x 16 and 16 x 32 (lane l: A[l % 32][8 (l / 32) + i], B likewise, c[8 (i / 4) + 4 (l / 32) + i % 4][l % 32]).
template <bool kF16>
__device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    if constexpr (kF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Over the two lanes of a row.
__device__ __forceinline__ float max_across_halves(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return fmaxf(as_float(a[0]), as_float(a[1]));
}
__device__ __forceinline__ float sum_across_halves(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return as_float(a[0]) + as_float(a[1]);
}

// Two codes -> two 16-bit values in a dword.
template <bool kF16, bool kHi>
__device__ __forceinline__ uint32_t widen2(uint32_t x) {
    if constexpr (kF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, kHi));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, kHi));
}

template <int kD>
struct WideLds {
    static constexpr int kRow = kD <= 64 ? 128 : 256;    // bytes of an LDS row
    uint8_t k[2][kKeys * kRow];
    uint8_t v[2][kKeys * kRow];
    float scale[4][2][kKeys];
    int32_t count[4][4];                                 // tokens of each tile that count
    __attribute__((aligned(16))) uint8_t spare[16 + 256];  // what lanes without a value write
};

template <int kD, int QT, int ES>
__global__ void __launch_bounds__(64 * kWideWaves)
prefix_wide_kernel(PrefixArgs a, PrefixGrid grid) {
    static_assert(kD % 16 == 0 && kD >= 64 && kD <= 128 && (ES == 1 || kD % 64 == 0), "head sizes of this kernel");
    using T = typename Elem<QT>::T;
    constexpr bool kF16 = QT == KVFP8_F16;               // K and Q^T operands
    constexpr bool kF16V = kF16 && ES == 2;              // V^T and P operands; f16 q over codes: two bf16 parts of P
    constexpr int kParts = kF16 && ES == 1 ? 2 : 1;
    constexpr int NW = kWideWaves, kThreads = 64 * NW;
    constexpr int ROW = WideLds<kD>::kRow;
    constexpr int CPR = ROW / 16;                        // 16-byte chunks of an LDS row
    constexpr int NB = (kD + 31) / 32, KS = kD / 16;     // blocks of 32 dims of O, steps of 16 dims of Q K^T
    // Staging: a row of K or V is `SLOTS` runs of 16 bytes of cache; slot x of the block's 2 x 64 x SLOTS goes to
    // thread x % kThreads. A wave's rows of one load lie in one 16-token tile, so its page is wave-uniform.
    constexpr int SLOTS = ES == 1 ? CPR / 2 : CPR;
    constexpr int RUNS = kD * ES / 16;                   // of them used
    constexpr int PER = kKeys * SLOTS;                   // slots per tensor
    constexpr int LOADS = 2 * PER / kThreads;
    constexpr int TILES = LOADS > 1 ? LOADS / 2 : 1;     // loads of K, each from a tile of its own, then those of V
    constexpr int RPW = 64 / SLOTS;                      // rows of one load of a wave
    union Lds {
        WideLds<kD> wide;
        NarrowLds<(kD <= 64 ? 1 : 2), NW> narrow;
    };
    __shared__ __attribute__((aligned(16))) Lds lds;
    if ((int32_t)blockIdx.x >= grid.prefix_groups) {
        PrefixItem own;
        if (own_item(a, grid, own)) narrow_run<(kD <= 64 ? 1 : 2), QT, ES, NW>(a, own, grid.own_heads, grid.q_vec, lds.narrow);
        return;
    }
    auto& lds_k = lds.wide.k;
    auto& lds_v = lds.wide.v;
    auto& lds_scale = lds.wide.scale;
    auto& lds_count = lds.wide.count;

    PrefixItem it;
    if (!prefix_item(a, grid, 32 * NW, it)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int col = lane & 31, hi = lane >> 5;           // the lane's row of a wave's, and half
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int h = it.h;
    const int32_t blocks = (it.hi - it.lo + kKeys - 1) / kKeys;
    const int32_t r0 = it.r0 + 32 * wave;                // first pair of the wave
    const bool active = r0 < it.pairs;

    // Where chunk c of an LDS row stands.
    auto swizzle = [](int row, int c) __attribute__((always_inline)) {
        return 16 * (c ^ (CPR == 16 ? ((row & 3) << 2) | ((row >> 2) & 3) : (row >> 1) & 7));
    };
    // Row and tensor of load i of this thread; the tile of its wave's rows.
    auto row_of = [&](int i) __attribute__((always_inline)) { return ((int)threadIdx.x + kThreads * i) % PER / SLOTS; };
    auto wave_row = [&](int i) __attribute__((always_inline)) { return (64 * wave + kThreads * i) % PER / SLOTS; };
    const int run = threadIdx.x % SLOTS;
    const int64_t row_bytes = (int64_t)a.d.num_kv_heads * kD * ES;
    // Scales: 2 RPW lanes of a wave that loads K load those of its rows, of K and of V.
    constexpr bool kByWave = LOADS == 1;                 // the first half of the waves loads K, the other V
    const bool loads_v = kByWave && wave >= NW / 2;
    const int s_tensor = (lane / RPW) & 1, s_row = lane % RPW;
    const bool s_mine = !loads_v && lane < 2 * RPW;

    // The page of the tile of load i in block g; past the prefix one of its own (no branch), which counts nothing.
    auto fetch_page = [&](int32_t g, int i) __attribute__((always_inline)) -> int32_t {
        const int32_t tok = it.lo + g * kKeys + (wave_row(i) & ~15);
        const int64_t addr = uniform64((int64_t)(uintptr_t)(it.table + ((tok < it.hi ? tok : it.lo) >> a.d.bs_shift)));
        return *(const_i32_ptr)(uintptr_t)addr;
    };
    int32_t page[TILES];
    auto fetch = [&](int32_t g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < TILES; ++u) page[u] = fetch_page(g, u);
    };
    const uint32_t pages = (uint32_t)min(a.d.num_blocks, (int64_t)INT32_MAX);
    // A thread's rows have one place in their tiles, and so one offset behind a tile's first row.
    const uint32_t row_off = (uint32_t)((row_of(0) & 15) * (int32_t)row_bytes + 16 * (run < RUNS ? run : 0));
    const uint32_t scale_off = (uint32_t)(((wave_row(0) & 15) + s_row) * a.d.num_kv_heads);
    u32x4_t raw[LOADS];
    float scale[TILES];
    int64_t base[TILES];                                 // first cache row of the wave's tiles: of the K block in flight
    int32_t count_k[TILES], count_v[TILES];              // tokens that count in them, of the K and the V block in flight
    auto locate = [&](int32_t g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
            const int32_t tok = it.lo + g * kKeys + (wave_row(u) & ~15);
            const bool ok = (uint32_t)page[u] < pages && tok < it.hi;
            count_k[u] = ok ? min(16, it.hi - tok) : 0;
            base[u] = (int64_t)(ok ? page[u] : 0) * a.d.block_size + (ok ? tok & (a.d.block_size - 1) : 0);
        }
    };
    auto is_v = [&](int i) __attribute__((always_inline)) { return kByWave ? loads_v : kThreads * i >= PER; };
    auto issue = [&](bool v) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            if (is_v(i) != v) continue;
            const uint8_t* src = reinterpret_cast<const uint8_t*>(v ? a.d.v_cache : a.d.k_cache) + base[i % TILES] * row_bytes + h * kD * ES;
            raw[i] = *reinterpret_cast<const u32x4_t*>(src + row_off);
        }
        if (v) {
#pragma unroll
            for (int u = 0; u < TILES; ++u) count_v[u] = count_k[u];
        } else if constexpr (ES == 1) {
#pragma unroll
            for (int u = 0; u < TILES; ++u)
                scale[u] = ((s_tensor ? a.d.v_scales : a.d.k_scales) + base[u] * a.d.num_kv_heads + h)[scale_off];
        }
    };
    // Rows that do not count become zeros (their bytes may be anything).
    auto publish = [&](bool v, int buf, int32_t g) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            if (is_v(i) != v) continue;
            const int row = row_of(i);
            const bool live = (row & 15) < (v ? count_v : count_k)[i % TILES];
            uint8_t* dst = (v ? lds_v[buf] : lds_k[buf]) + row * ROW;
            const bool held = run < RUNS;                // else to where nobody reads
            if constexpr (ES == 1) {
                u32x4_t x[2];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t c = live ? raw[i][w] : 0u;
                    if (kF16 && !v) {
                        x[w >> 1][2 * (w & 1)] = widen2<kF16, false>(c);
                        x[w >> 1][2 * (w & 1) + 1] = widen2<kF16, true>(c);
                    } else {
                        x[w >> 1][2 * (w & 1)] = widen2<false, false>(c);
                        x[w >> 1][2 * (w & 1) + 1] = widen2<false, true>(c);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<u32x4_t*>(held ? dst + swizzle(row, 2 * run + e) : lds.wide.spare) = x[e];
            } else {
                *reinterpret_cast<u32x4_t*>(held ? dst + swizzle(row, run) : lds.wide.spare) = live ? raw[i] : u32x4_t{0u, 0u, 0u, 0u};
            }
        }
        if (v) return;
        if constexpr (ES == 1) {
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                const int row = wave_row(u) + s_row;
                const float x = (row & 15) < count_k[u] ? scale[u] : 0.0f;
                *(s_mine ? &lds_scale[g & 3][s_tensor][row] : reinterpret_cast<float*>(lds.wide.spare) + 4 + lane) = s_tensor ? x : x * a.d.score_scale;
            }
        }
#pragma unroll
        for (int u = 0; u < TILES; ++u)
            *(lane == 0 && !loads_v && wave_row(u) % 16 == 0 ? &lds_count[g & 3][wave_row(u) / 16]
                                                             : reinterpret_cast<int32_t*>(lds.wide.spare) + 4 + lane) = count_k[u];
    };

    // Q^T operands: lane (row l % 32, l / 32) holds dims 16 s + 8 (l / 32) .. + 7 (pairs past the last repeat it: their
    // rows are never stored).
    u32x4_t qop[KS];
    auto load_q = [&]() __attribute__((always_inline)) {
        const int32_t pair = min(r0 + col, it.pairs - 1);
        const int32_t t = (uint32_t)pair / (uint32_t)G;
        const T* src = reinterpret_cast<const T*>(a.d.q) + (int64_t)(it.rs + t) * a.d.q_stride_b + (h * G + (pair - t * G)) * a.d.q_stride_h;
        auto element2 = [&](int d) __attribute__((always_inline)) { return (uint32_t)src[d] | ((uint32_t)src[d + 1] << 16); };
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * hi;
            if (grid.q_vec) qop[s] = *reinterpret_cast<const u32x4_t*>(src + d);
            else qop[s] = u32x4_t{element2(d), element2(d + 2), element2(d + 4), element2(d + 6)};
        }
    };

    // Per-lane byte offsets of the operand reads: K row l % 32, chunk 2 s + l / 32. V^T by the transposing read
    // ds_read_b64_tr_b16: of 16 lanes lane i reads dims 4 (i % 4) .. + 3 of key i / 4 of a block of 4 keys x 16 dims and
    // receives dim i of the four keys. Lanes 0..15 and 16..31 (32..47, 48..63) take the two halves of 32 dims, lanes
    // below 32 keys 0..3 and 8..11 (two reads) of 16, the others 4..7 and 12..15: what their scores belong to. Dims
    // past the head size are read from chunks that nobody writes and end in rows of O that nobody stores.
    int k_off[KS], v_off[NB][2];
#pragma unroll
    for (int s = 0; s < KS; ++s) k_off[s] = col * ROW + swizzle(col, 2 * s + hi);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int vrow = 8 * e + 4 * hi + ((lane & 15) >> 2), chunk = 4 * nb + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
            v_off[nb][e] = vrow * ROW + swizzle(vrow, chunk) + 8 * (lane & 1);
        }

    f32x16_t o[NB];
    float ref = 0.0f, lim = kNegInf, l = 0.0f;           // a row's reference (0 before its first score), what scores may reach
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nb][i] = 0.0f;

    // Scores and P'^T operands of a block's halves of 32 tokens. Score i of a row: token 8 (i / 4) + 4 (l / 32) + i % 4.
    f32x16_t sacc[2];
    u32x4_t pop[2][kParts][2];
    // Steps of K operands that are read before the products of a half, the others among them (weights of two parts leave
    // no registers for that).
    constexpr int kPre = kParts == 2 ? 0 : KS / 2;
    u32x4_t kop[KS];
    auto read_k = [&](auto buf_c, auto half_c, int first, int last) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value, half = decltype(half_c)::value;
        lds_u8* const kl = (lds_u8*)&lds_k[buf][32 * half * ROW];
#pragma unroll
        for (int s = first; s < last; ++s) kop[s] = *(lds_u32x4*)(kl + k_off[s]);
    };
    auto qk = [&](auto half_c) __attribute__((always_inline)) {
        constexpr int half = decltype(half_c)::value;
#pragma unroll
        for (int s = 0; s < KS; ++s) sacc[half] = mma32<kF16>(kop[s], qop[s], s == 0 ? f32x16_t{} : sacc[half]);
    };
    auto pv = [&](auto buf_c, auto half_c) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value, half = decltype(half_c)::value;
        lds_u8* const vl = (lds_u8*)&lds_v[buf][32 * half * ROW];
#pragma unroll
        for (int pp = 0; pp < 2; ++pp)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                u32x4_t av;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vl + v_off[nb][e] + 16 * pp * ROW));
                    const uint2 w = __builtin_bit_cast(uint2, x);
                    av[2 * e] = w.x;
                    av[2 * e + 1] = w.y;
                }
#pragma unroll
                for (int part = 0; part < kParts; ++part) o[nb] = mma32<kF16V>(av, pop[half][part][pp], o[nb]);
            }
    };
    // Scores of a half with their scales.
    float mx;
    int2 counts;                                         // tokens of the half's tiles that count
    auto scale_scores = [&](int32_t g, auto half_c) __attribute__((always_inline)) {
#pragma clang fp contract(off)
        constexpr int half = decltype(half_c)::value;
        counts = *reinterpret_cast<const int2*>(&lds_count[g & 3][2 * half]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4_t ks = {a.d.score_scale, a.d.score_scale, a.d.score_scale, a.d.score_scale};
            if constexpr (ES == 1) ks = *reinterpret_cast<const f32x4_t*>(&lds_scale[g & 3][0][32 * half + 8 * q + 4 * hi]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sacc[half][4 * q + i] *= ks[i];
        }
    };
    auto largest = [&](auto half_c) __attribute__((always_inline)) {
        constexpr int half = decltype(half_c)::value;
        mx = sacc[half][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sacc[half][i]);
    };
    // Tokens of the half that do not count, and references that have to move: where some row's maximum passes its
    // own by 2^8 (each lane tests its 16 tokens). `alpha` is then the factor of what has been summed relative to the
    // old reference: l at once, O one half later, when the last products of such weights have been added.
    float alpha = 1.0f;
    auto settle = [&](auto half_c) __attribute__((always_inline)) -> bool {
        constexpr int half = decltype(half_c)::value;
        const int n0 = uniform(counts.x), n1 = uniform(counts.y);
        if (n0 + n1 < 32) {                              // wave-uniform
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i / 4 % 2) + 4 * hi + i % 4 >= (i < 8 ? n0 : n1)) sacc[half][i] = kNegInf;
            largest(half_c);
        }
        if (!__ballot(mx > lim)) return false;
        const float top = max_across_halves(mx);
        const bool fresh = lim == kNegInf;
        const float to = fresh ? (top == kNegInf ? 0.0f : top) : fmaxf(top, ref);
        alpha = fresh ? 0.0f : __builtin_amdgcn_exp2f(ref - to);
        lim = fresh && top == kNegInf ? kNegInf : to + kLag;
        ref = to;
        l *= alpha;
        return true;
    };
    auto weigh = [&](int32_t g, auto half_c) __attribute__((always_inline)) {
#pragma clang fp contract(off)
        constexpr int half = decltype(half_c)::value;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            f32x4_t vs = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (ES == 1) vs = *reinterpret_cast<const f32x4_t*>(&lds_scale[g & 3][1][32 * half + 8 * q + 4 * hi]);
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(sacc[half][4 * q + i] - ref);
                l += p;
                x[i] = ES == 1 ? p * vs[i] : p;
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t top = pack2<kF16V>(x[2 * w], x[2 * w + 1]);
                pop[half][0][q / 2][2 * (q % 2) + w] = top;
                if constexpr (kParts == 2)
                    pop[half][1][q / 2][2 * (q % 2) + w] =
                        pack2<false>(x[2 * w] - bits_f32(top << 16), x[2 * w + 1] - bits_f32(top & 0xFFFF0000u));
            }
        }
    };
    // The products are spread over the softmax's operations, V's operand reads run ahead of them. What the region
    // leaves is kept in its place: the compiler would sink it to its use behind the next branch, away from the products.
    constexpr int kReads = 4 * NB + KS - kPre, kProducts = 2 * NB * kParts + KS, kAhead = (ES == 1 ? 8 : 0) + 1;
    auto interleave = [&](auto half_c) __attribute__((always_inline)) {
        constexpr int half = decltype(half_c)::value;
        constexpr bool stages = half == 0;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);                      // LDS reads of scales and counts
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                       // matrix products
            __builtin_amdgcn_sched_group_barrier(0x402, stages ? 10 : 7, 0);          // softmax, widening
            if (2 * i < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            else if (stages) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
        }
#pragma unroll
        for (int pp = 0; pp < 2; ++pp)
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                u32x4_t& weights = pop[half][part][pp];
                __asm__ volatile("" : "+v"(weights));
            }
        float &sum = l, &most = mx;
        __asm__ volatile("" : "+v"(sum), "+v"(most));
    };

    // A barrier that waits for this wave's LDS operations and leaves its loads in flight.
    auto barrier = [&]() __attribute__((always_inline)) {
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);              // lgkmcnt(0) alone
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
    };
    constexpr std::integral_constant<int, 0> c0{};
    constexpr std::integral_constant<int, 1> c1{};
    fetch(0);
    locate(0);
    issue(false);
    issue(true);
    fetch(1);
    load_q();
    publish(false, 0, 0);
    locate(1);
    issue(false);
    fetch(2);
    barrier();
    bool moved = false;
    if (active) {
        read_k(c0, c0, 0, KS);
        qk(c0);
        scale_scores(0, c0);
        largest(c0);
        read_k(c0, c1, 0, kPre);
        settle(c0);                                      // O and l are zeros yet
    }
    // Half `half` of block g, whose scores are there: its weights; the scores of the next half (of block gn,
    // buffer kbuf); the products with V of the half before (buffer vbuf). All three are independent of each other.
    auto part = [&](int32_t g, auto half_c, int32_t gn, auto kbuf_c, auto vbuf_c, bool first) __attribute__((always_inline)) {
        constexpr std::integral_constant<int, 1 - decltype(half_c)::value> next{};
        read_k(kbuf_c, next, kPre, KS);
        qk(next);
        weigh(g, half_c);
        if (!first) pv(vbuf_c, next);
        scale_scores(gn, next);
        largest(next);
    };
    auto rest = [&](auto half_c) __attribute__((always_inline)) {
        if (moved) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[nb] *= alpha;
        }
        constexpr std::integral_constant<int, 1 - decltype(half_c)::value> next{};
        moved = settle(next);
    };
    // Step g (buffer of K(g), V(g): g % 2). Past the last block the staging moves rows that count nothing, so that
    // there is no branch around it.
    auto step = [&](int32_t g, auto buf_c, bool first) __attribute__((always_inline)) {
        constexpr std::integral_constant<int, 1 - decltype(buf_c)::value> other{};
        auto stage = [&]() __attribute__((always_inline)) {
            publish(true, decltype(buf_c)::value, g);
            publish(false, other.value, g + 1);
            issue(true);
            locate(g + 2);
            issue(false);
            fetch(g + 3);
        };
        if (!active) {
            stage();
            barrier();
            return;
        }
        part(g, c0, g, buf_c, other, first);
        stage();
        interleave(c0);
        barrier();
        read_k(other, c0, 0, kPre);
        rest(c0);
        part(g, c1, g + 1, other, buf_c, false);
        interleave(c1);
        read_k(other, c1, 0, kPre);
        rest(c1);
    };
    step(0, c0, true);
    for (int32_t g = 1; g < blocks; g += 2) {
        step(g, c1, false);
        if (g + 1 < blocks) step(g + 1, c0, false);
    }
    if (!active) return;
    if ((blocks & 1) != 0) pv(c0, c1);
    else pv(c1, c1);
    // Nothing moves behind the last block: its scores do not count.
    const float m = lim == kNegInf ? kNegInf : ref;
    const float lt = sum_across_halves(l);
    const int32_t pair = r0 + col;
    if (pair >= it.pairs) return;
    const int32_t t = (uint32_t)pair / (uint32_t)G;
    const int64_t row = it.rs + t;
    const int hq = h * G + (pair - t * G);
    // Element 4 q + i of block nb: dim 32 nb + 8 q + 4 hi + i of the row.
    if (a.cu != nullptr && a.splits == 1 && it.tail < 0) {
        // The prompt form's only state of the row: joined with out and lse at once (out has been rounded once before).
        if (seq_of_row(a, row) < 0) return;
        const int64_t at = row * a.d.num_q_heads + hq;
        const float mo = a.lse[at] * kLog2e;
        const float mn = fmaxf(m, mo), mu = mn == kNegInf ? 0.0f : mn;
        const float wp = fast_exp2(m - mu), wo = fast_exp2(mo - mu);
        const float den = lt * wp + wo;
        const float inv = den > 0.0f || den != den ? 1.0f / den : 0.0f;
        T* out = reinterpret_cast<T*>(a.d.out) + at * kD + 4 * hi;
#pragma unroll
        for (int d = 0; d < kD; d += 8) {
            uint2* dst = reinterpret_cast<uint2*>(out + d);
            const uint2 x = *dst;
            const float y[4] = {Elem<QT>::load((T)(x.x & 0xFFFFu)), Elem<QT>::load((T)(x.x >> 16)),
                                Elem<QT>::load((T)(x.y & 0xFFFFu)), Elem<QT>::load((T)(x.y >> 16))};
            float z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = (o[d / 32][d % 32 / 2 + i] * wp + y[i] * wo) * inv;
            *dst = make_uint2(pack2<kF16>(z[0], z[1]), pack2<kF16>(z[2], z[3]));
        }
        // The row's two lanes run in step: both have read lse.
        if (hi == 0) a.lse[at] = (mu + __builtin_log2f(den)) * kLn2;
        return;
    }
    const int64_t pi = it.tail < 0 ? prefix_part(a, row, it.part, hq)
                                   : ((int64_t)it.tail * (32 * NW) + (pair - it.r0)) * grid.tail_splits + it.part;
    if (hi == 0) {
        a.d.part_m[pi] = m;
        a.d.part_l[pi] = lt;
    }
#pragma unroll
    for (int d = 0; d < kD; d += 8) {
        const int i = d % 32 / 2;
        *reinterpret_cast<float4*>(a.d.part_acc + pi * kD + d + 4 * hi) = make_float4(o[d / 32][i], o[d / 32][i + 1], o[d / 32][i + 2], o[d / 32][i + 3]);
    }
}

template <int kD, int QT, int ES>
hipError_t launch_wide(const PrefixArgs& a, const PrefixGrid& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.prefix_groups + g.own_groups));
    hipLaunchKernelGGL((prefix_wide_kernel<kD, QT, ES>), grid, dim3(64 * kWideWaves), 0, s, a, g);
    return hipGetLastError();
}

}  // namespace

template <int QT>
hipError_t launch_prefix_wide(const PrefixArgs& a, int kv_dtype, const PrefixGrid& g, hipStream_t s) {
    if (kv_dtype != KVFP8_E4M3FN) return a.d.head_dim == 64 ? launch_wide<64, QT, 2>(a, g, s) : launch_wide<128, QT, 2>(a, g, s);
    switch (a.d.head_dim) {
        case 64: return launch_wide<64, QT, 1>(a, g, s);
        case 80: return launch_wide<80, QT, 1>(a, g, s);
        case 96: return launch_wide<96, QT, 1>(a, g, s);
        case 112: return launch_wide<112, QT, 1>(a, g, s);
        default: return launch_wide<128, QT, 1>(a, g, s);
    }
}

template hipError_t launch_prefix_wide<KVFP8_F16>(const PrefixArgs&, int, const PrefixGrid&, hipStream_t);
template hipError_t launch_prefix_wide<KVFP8_BF16>(const PrefixArgs&, int, const PrefixGrid&, hipStream_t);

}  // namespace kvfp8
