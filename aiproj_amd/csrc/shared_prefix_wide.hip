// Shared prefixes for many rows: blocks of 256 or 128 (row, q head) pairs against a prefix, gfx950.
//
// A workgroup takes one (row block, KV head, split of the prefix). Its eight or four waves hold 32 rows each and
// share the prefix's tokens through LDS in blocks of 64: the codes are widened to 16 bits once per
// workgroup on their way there (exact), instead of once per wave, and the tokens' bytes cross L2 once per
// 256 rows. Per block and wave (MFMA 16x16x32, layouts in mfma_tiles.h):
//   S^T[token, row] = K Q^T     A = K rows from LDS, B = Q^T from registers
//   softmax                     scores x k_scale[token] x sm_scale x log2(e) in float32, online, base 2; the
//                               reference follows a row's maximum only where that exceeds it by 2^8
//   O^T[d, row] += V^T P'^T     P' = p v_scale[token] from the score registers; A = V^T by transposing LDS reads
// The vector ALU bounds it: nine operations a score, one of them the exponential at a quarter rate.
//
// LDS rows are 16-byte chunks at position chunk ^ (row % chunks per row), so that the 16 rows of an operand
// read lie in different bank groups.
//
// The two halves of the waves alternate between a phase on the matrix cores (PV of block g - 1, QK of
// block g) and one on the vector ALU (softmax of block g), half a step apart, with a barrier after each phase:
//   phase 2 g       waves 0..3: PV(g - 1), QK(g)    waves 4..7: softmax(g - 1)
//   phase 2 g + 1   waves 0..3: softmax(g)          waves 4..7: PV(g - 1), QK(g)
// so K(g) and V(g - 1) are read in phases 2 g and 2 g + 1. In its matrix phase of step g a wave moves its part of
// K(g + 1) and V(g) from registers to the buffers that K(g - 1) and V(g - 2) have left, and issues the loads of
// K(g + 2) and V(g + 1). Scales and counts (softmax(g) of waves 4..7 reads them in phase 2 g + 2, when waves 0..3
// write those of g + 2) have four buffers.
#include "shared_prefix_narrow.h"

namespace kvfp8 {

namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr int kKeys = 64;             // tokens per block
constexpr float kLag = 8.0f;          // log2 of how far a row's maximum may exceed its reference

typedef __attribute__((address_space(3))) const uint8_t lds_u8;
typedef __attribute__((address_space(3))) const u32x4_t lds_u32x4;
typedef __attribute__((address_space(3))) const u32x2_t lds_u32x2;
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

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
};

// NW waves, 32 rows each.
template <int kD, int QT, int ES, int NW>
__global__ void __launch_bounds__(64 * NW)
prefix_wide_kernel(PrefixArgs a, PrefixGrid grid) {
    static_assert(kD % 16 == 0 && kD >= 64 && kD <= 128 && (ES == 1 || kD % 64 == 0), "head sizes of this kernel");
    using T = typename Elem<QT>::T;
    constexpr bool kF16 = QT == KVFP8_F16;               // K and Q^T operands
    constexpr bool kF16V = kF16 && ES == 2;              // V^T and P operands; f16 q over codes: two bf16 parts of P
    constexpr int kParts = kF16 && ES == 1 ? 2 : 1;
    constexpr int kThreads = 64 * NW;
    constexpr int ROW = WideLds<kD>::kRow;
    constexpr int CPR = ROW / 16;                        // 16-byte chunks of an LDS row
    constexpr int NB = kD / 16, KS = kD / 32;
    constexpr bool kHalf = kD % 32 != 0;                 // and one step of 16 dims
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
    const int m16 = lane & 15, j = lane >> 4;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int h = it.h;
    const int32_t blocks = (it.hi - it.lo + kKeys - 1) / kKeys;
    const int32_t r0 = it.r0 + 32 * wave;                // first pair of the wave
    const bool active = r0 < it.pairs;

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
    u32x4_t raw[LOADS];
    float scale[TILES];
    int64_t base[TILES];                                 // first cache row of the wave's tiles: of the K block in flight
    int32_t count_k[TILES], count_v[TILES];              // tokens that count in them, of the K and the V block in flight
    auto locate = [&](int32_t g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
            const int32_t tok = it.lo + g * kKeys + (wave_row(u) & ~15);
            const bool ok = page[u] >= 0 && page[u] < a.d.num_blocks && tok < it.hi;
            count_k[u] = ok ? min(16, it.hi - tok) : 0;
            base[u] = ok ? (int64_t)page[u] * a.d.block_size + (tok & (a.d.block_size - 1)) : 0;
        }
    };
    auto is_v = [&](int i) __attribute__((always_inline)) { return kByWave ? loads_v : kThreads * i >= PER; };
    auto issue = [&](bool v) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            if (is_v(i) != v) continue;
            const uint8_t* src = reinterpret_cast<const uint8_t*>(v ? a.d.v_cache : a.d.k_cache) +
                                 (base[i % TILES] + (row_of(i) & 15)) * row_bytes + h * kD * ES + 16 * (run < RUNS ? run : 0);
            raw[i] = *reinterpret_cast<const u32x4_t*>(src);
        }
        if (v) {
#pragma unroll
            for (int u = 0; u < TILES; ++u) count_v[u] = count_k[u];
        } else if constexpr (ES == 1) {
#pragma unroll
            for (int u = 0; u < TILES; ++u)
                scale[u] = (s_tensor ? a.d.v_scales : a.d.k_scales)[(base[u] + (wave_row(u) & 15) + s_row) * a.d.num_kv_heads + h];
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
            if (run >= RUNS) continue;
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
                    *reinterpret_cast<u32x4_t*>(dst + 16 * ((2 * run + e) ^ (row % CPR))) = x[e];
            } else {
                *reinterpret_cast<u32x4_t*>(dst + 16 * (run ^ (row % CPR))) = live ? raw[i] : u32x4_t{0u, 0u, 0u, 0u};
            }
        }
        if (v) return;
        if constexpr (ES == 1) {
#pragma unroll
            for (int u = 0; u < TILES; ++u) {
                const float x = (wave_row(u) & 15) + s_row < count_k[u] ? scale[u] : 0.0f;
                if (s_mine) lds_scale[g & 3][s_tensor][wave_row(u) + s_row] = s_tensor ? x : x * a.d.score_scale;
            }
        }
#pragma unroll
        for (int u = 0; u < TILES; ++u)
            if (lane == 0 && !loads_v && wave_row(u) % 16 == 0) lds_count[g & 3][wave_row(u) / 16] = count_k[u];
    };

    // Q^T operands: lane (row 16 qt + l % 16, l / 16) holds dims 32 s + 8 (l / 16) .. + 7 (pairs past the last
    // repeat it: their rows are never stored).
    u32x4_t qop[2][KS];
    uint2 qhalf[2];
    auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) {
            const int32_t pair = min(r0 + 16 * qt + m16, it.pairs - 1);
            const int32_t t = (uint32_t)pair / (uint32_t)G;
            const T* src = reinterpret_cast<const T*>(a.d.q) + (int64_t)(it.rs + t) * a.d.q_stride_b + (h * G + (pair - t * G)) * a.d.q_stride_h;
            auto element2 = [&](int d) __attribute__((always_inline)) { return (uint32_t)src[d] | ((uint32_t)src[d + 1] << 16); };
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 32 * s + 8 * j;
                if (grid.q_vec) qop[qt][s] = *reinterpret_cast<const u32x4_t*>(src + d);
                else qop[qt][s] = u32x4_t{element2(d), element2(d + 2), element2(d + 4), element2(d + 6)};
            }
            if constexpr (kHalf) {
                const int d = 32 * KS + 4 * j;
                if (grid.q_vec) qhalf[qt] = *reinterpret_cast<const uint2*>(src + d);
                else qhalf[qt] = make_uint2(element2(d), element2(d + 2));
            }
        }
    };

    // Per-lane byte offsets of the operand reads: K row m16, chunk 4 s + j; V^T as in the transposing read
    // ds_read_b64_tr_b16: lane (j, m16) reads dims 16 nb + 4 (m16 % 4) .. + 3 of key 4 j + m16 / 4 of a 16-key
    // tile and receives V[4 j + r][16 nb + m16], r = 0..3.
    int k_off[KS], k_half = 0, v_off[NB];
#pragma unroll
    for (int s = 0; s < KS; ++s) k_off[s] = m16 * ROW + 16 * ((4 * s + j) ^ (m16 % CPR));
    if constexpr (kHalf) k_half = m16 * ROW + 16 * ((4 * KS + (j >> 1)) ^ (m16 % CPR)) + 8 * (j & 1);
    {
        const int vrow = 4 * j + (m16 >> 2);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            v_off[nb] = vrow * ROW + 16 * ((2 * nb + ((m16 >> 1) & 1)) ^ (vrow % CPR)) + 8 * (m16 & 1);
    }

    f32x4_t o[2][NB];
    float m[2], l[2];
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[qt][nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m[qt] = kNegInf;
        l[qt] = 0.0f;
    }

    f32x4_t sacc[4][2];
    auto qk = [&](auto buf_c) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value;
        lds_u8* const kl = (lds_u8*)&lds_k[buf][0];
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                const u32x4_t kop = *(lds_u32x4*)(kl + k_off[s] + 16 * kt * ROW);
#pragma unroll
                for (int qt = 0; qt < 2; ++qt)
                    sacc[kt][qt] = mma16<kF16>(kop, qop[qt][s], s == 0 ? f32x4_t{0.0f, 0.0f, 0.0f, 0.0f} : sacc[kt][qt]);
            }
        if constexpr (kHalf) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                const uint2 kop = __builtin_bit_cast(uint2, *(lds_u32x2*)(kl + k_half + 16 * kt * ROW));
#pragma unroll
                for (int qt = 0; qt < 2; ++qt) sacc[kt][qt] = mma16_half<kF16>(kop, qhalf[qt], sacc[kt][qt]);
            }
        }
    };
    // P'^T operands; pp holds tokens 16 (2 pp + i / 4) + 4 j + i % 4.
    u32x4_t pop[2][kParts][2];
    auto softmax = [&](int32_t g) __attribute__((always_inline)) {
        const float(*scales)[kKeys] = lds_scale[g & 3];
        // Scaled scores (score i of a row: token 16 (i / 4) + 4 j + i % 4).
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            float4 ks = make_float4(a.d.score_scale, a.d.score_scale, a.d.score_scale, a.d.score_scale);
            if constexpr (ES == 1) {
                ks = *reinterpret_cast<const float4*>(&scales[0][16 * kt + 4 * j]);
            }
#pragma unroll
            for (int qt = 0; qt < 2; ++qt) {
                sacc[kt][qt][0] *= ks.x;
                sacc[kt][qt][1] *= ks.y;
                sacc[kt][qt][2] *= ks.z;
                sacc[kt][qt][3] *= ks.w;
            }
        }
        const int4 counts = *reinterpret_cast<const int4*>(&lds_count[g & 3][0]);
        const int n[4] = {uniform(counts.x), uniform(counts.y), uniform(counts.z), uniform(counts.w)};
        if (n[0] + n[1] + n[2] + n[3] < kKeys) {         // wave-uniform
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
                    if (4 * j + jj >= n[kt]) sacc[kt][0][jj] = sacc[kt][1][jj] = kNegInf;
        }
        float neg_m[2];
#pragma unroll
        for (int qt = 0; qt < 2; ++qt) {
            float mx = sacc[0][qt][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sacc[i / 4][qt][i % 4]);
            // The reference moves where some row's maximum passes it by 2^8; each lane tests its 16 tokens.
            if (__ballot(mx > m[qt] + kLag)) {
                const float m_new = fmaxf(m[qt], max_across_rows(mx));
                const float alpha = __builtin_amdgcn_exp2f(m[qt] - (m_new == kNegInf ? 0.0f : m_new));
                l[qt] *= alpha;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[qt][nb] *= alpha;
                m[qt] = m_new;
            }
            neg_m[qt] = m[qt] == kNegInf ? 0.0f : -m[qt];
        }
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            f32x4_t vs = {1.0f, 1.0f, 1.0f, 1.0f};
            if constexpr (ES == 1) vs = *reinterpret_cast<const f32x4_t*>(&scales[1][16 * kt + 4 * j]);
#pragma unroll
            for (int qt = 0; qt < 2; ++qt) {
                float x[4];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) {
                    const float p = __builtin_amdgcn_exp2f(sacc[kt][qt][jj] + neg_m[qt]);
                    l[qt] += p;
                    x[jj] = ES == 1 ? p * vs[jj] : p;
                }
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t top = pack2<kF16V>(x[2 * w], x[2 * w + 1]);
                    pop[qt][0][kt >> 1][2 * (kt & 1) + w] = top;
                    if constexpr (kParts == 2)
                        pop[qt][1][kt >> 1][2 * (kt & 1) + w] =
                            pack2<false>(x[2 * w] - bits_f32(top << 16), x[2 * w + 1] - bits_f32(top & 0xFFFF0000u));
                }
            }
        }
    };
    auto pv = [&](auto buf_c) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_c)::value;
        lds_u8* const vl = (lds_u8*)&lds_v[buf][0];
#pragma unroll
        for (int pp = 0; pp < 2; ++pp)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                u32x4_t av;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vl + v_off[nb] + 16 * (2 * pp + half) * ROW));
                    const uint2 w = __builtin_bit_cast(uint2, x);
                    av[2 * half] = w.x;
                    av[2 * half + 1] = w.y;
                }
#pragma unroll
                for (int qt = 0; qt < 2; ++qt)
#pragma unroll
                    for (int part = 0; part < kParts; ++part) o[qt][nb] = mma16<kF16V>(av, pop[qt][part][pp], o[qt][nb]);
            }
    };

    // A barrier that waits for this wave's LDS operations and leaves its loads in flight.
    auto barrier = [&]() __attribute__((always_inline)) {
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);              // lgkmcnt(0) alone
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
    };
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
    constexpr std::integral_constant<int, 0> b0{};
    constexpr std::integral_constant<int, 1> b1{};
    // The matrix phase of step g (buffer of K(g), V(g): g % 2). Past the last block the staging moves rows that count
    // nothing, so that there is no branch around it.
    // Operand reads run ahead of the products by up to 16 (an LDS read under this load takes some 200 cycles, a
    // product 16); left alone, the compiler reads each operand right before its use.
    constexpr int kReads = 4 * NB + 4 * KS + (kHalf ? 4 : 0), kProducts = 4 * NB * kParts + 8 * KS + (kHalf ? 8 : 0);
    constexpr int kAhead = 16, kPace = (kProducts - kAhead) / ((kReads - kAhead) / 2);
    auto matrix = [&](int32_t g, auto buf_c, bool first) __attribute__((always_inline)) {
        constexpr std::integral_constant<int, 1 - decltype(buf_c)::value> other{};
        publish(true, decltype(buf_c)::value, g);
        publish(false, other.value, g + 1);
        issue(true);
        locate(g + 2);
        issue(false);
        fetch(g + 3);
        if (!active) return;
        if (first) {
            qk(buf_c);
            return;
        }
        pv(other);
        qk(buf_c);
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);              // LDS reads
#pragma unroll
        for (int i = 0; i < (kReads - kAhead) / 2; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, kPace, 0);           // matrix products
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, kProducts, 0);
    };
    // Both halves run the same 2 * blocks barriers.
    if (wave < NW / 2) {
        matrix(0, b0, true);
        barrier();
        if (active) softmax(0);
        barrier();
        for (int32_t g = 1; g < blocks; g += 2) {
            matrix(g, b1, false);
            barrier();
            if (active) softmax(g);
            barrier();
            if (g + 1 < blocks) {
                matrix(g + 1, b0, false);
                barrier();
                if (active) softmax(g + 1);
                barrier();
            }
        }
    } else {
        barrier();
        matrix(0, b0, true);
        barrier();
        for (int32_t g = 1; g < blocks; g += 2) {
            if (active) softmax(g - 1);
            barrier();
            matrix(g, b1, false);
            barrier();
            if (g + 1 < blocks) {
                if (active) softmax(g);
                barrier();
                matrix(g + 1, b0, false);
                barrier();
            }
        }
        if (active) softmax(blocks - 1);
    }
    if (active) {
        if ((blocks & 1) != 0) pv(b0);
        else pv(b1);
    }
    if (!active) return;

    // Lane (row, j) holds dims 16 nb + 4 j + jj of its row.
#pragma unroll
    for (int qt = 0; qt < 2; ++qt) {
        const float lt = sum_across_rows(l[qt]);
        const int32_t pair = r0 + 16 * qt + m16;
        if (pair >= it.pairs) continue;
        const int32_t t = (uint32_t)pair / (uint32_t)G;
        const int64_t row = it.rs + t;
        const int hq = h * G + (pair - t * G);
        if (a.cu != nullptr && a.splits == 1) {
            // The prompt form's only state of the row: joined with out and lse at once.
            if (seq_of_row(a, row) < 0) continue;
            const int64_t at = row * a.d.num_q_heads + hq;
            const float mo = a.lse[at] * kLog2e;
            const float mn = fmaxf(m[qt], mo), mu = mn == kNegInf ? 0.0f : mn;
            const float wp = fast_exp2(m[qt] - mu), wo = fast_exp2(mo - mu);
            const float den = lt * wp + wo;
            const float inv = den > 0.0f || den != den ? 1.0f / den : 0.0f;
            T* out = reinterpret_cast<T*>(a.d.out) + at * kD + 4 * j;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                uint2* dst = reinterpret_cast<uint2*>(out + 16 * nb);
                const uint2 x = *dst;
                const float y[4] = {Elem<QT>::load((T)(x.x & 0xFFFFu)), Elem<QT>::load((T)(x.x >> 16)),
                                    Elem<QT>::load((T)(x.y & 0xFFFFu)), Elem<QT>::load((T)(x.y >> 16))};
                float z[4];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) z[jj] = (o[qt][nb][jj] * wp + y[jj] * wo) * inv;
                *dst = make_uint2(pack2<kF16>(z[0], z[1]), pack2<kF16>(z[2], z[3]));
            }
            // The row's four lanes run in step: all have read lse.
            if (j == 0) a.lse[at] = (mu + __builtin_log2f(den)) * kLn2;
            continue;
        }
        const int64_t pi = prefix_part(a, row, it.part, hq);
        if (j == 0) {
            a.d.part_m[pi] = m[qt];
            a.d.part_l[pi] = lt;
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
            *reinterpret_cast<float4*>(a.d.part_acc + pi * kD + 16 * nb + 4 * j) =
                make_float4(o[qt][nb][0], o[qt][nb][1], o[qt][nb][2], o[qt][nb][3]);
    }
}

template <int kD, int QT, int ES>
hipError_t launch_wide(const PrefixArgs& a, int rows, const PrefixGrid& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.prefix_groups + g.own_groups));
    if (rows == 256) hipLaunchKernelGGL((prefix_wide_kernel<kD, QT, ES, 8>), grid, dim3(512), 0, s, a, g);
    else hipLaunchKernelGGL((prefix_wide_kernel<kD, QT, ES, 4>), grid, dim3(256), 0, s, a, g);
    return hipGetLastError();
}

}  // namespace

template <int QT>
hipError_t launch_prefix_wide(const PrefixArgs& a, int kv_dtype, int rows, const PrefixGrid& g, hipStream_t s) {
    if (kv_dtype != KVFP8_E4M3FN) return a.d.head_dim == 64 ? launch_wide<64, QT, 2>(a, rows, g, s) : launch_wide<128, QT, 2>(a, rows, g, s);
    switch (a.d.head_dim) {
        case 64: return launch_wide<64, QT, 1>(a, rows, g, s);
        case 80: return launch_wide<80, QT, 1>(a, rows, g, s);
        case 96: return launch_wide<96, QT, 1>(a, rows, g, s);
        case 112: return launch_wide<112, QT, 1>(a, rows, g, s);
        default: return launch_wide<128, QT, 1>(a, rows, g, s);
    }
}

template hipError_t launch_prefix_wide<KVFP8_F16>(const PrefixArgs&, int, int, const PrefixGrid&, hipStream_t);
template hipError_t launch_prefix_wide<KVFP8_BF16>(const PrefixArgs&, int, int, const PrefixGrid&, hipStream_t);

}  // namespace kvfp8
