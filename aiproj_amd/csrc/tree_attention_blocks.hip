// Drafted trees with 16-bit queries: blocks of 64 (node, q head) pairs of a KV head, gfx950.
//
// Four waves are two tiles of 32 pairs, times two groups that take steps of 32 tokens of the chunk in turn and join at the end. A
// group's tokens come from the cache straight into LDS, a ring of steps, as they are stored, up to three steps ahead; every wave
// widens the codes on the way from there. Per step (MFMA 32x32x16: A[row = l % 32][k = 8 (l / 32) + i], B likewise,
// D[row = 8 (i / 4) + 4 (l / 32) + i % 4][col = l % 32]):
//   S^T[token, pair] = K Q^T    A = K rows, 16 bytes a lane and read; B = Q^T, loaded once
//   softmax                     t = (score x sm_scale x log2(e)) x k_scale, e2(t - reference), float32, online, base 2; the
//                               reference follows a pair's maximum only where that exceeds it by 2^8. The product is rounded
//                               before the reference, which is such a product, is taken off: fused, the largest key's weight
//                               would be 2^(what its rounding took off), infinite or 0 from scores of 2^31 on (the operation
//                               more costs 0 to 2% of a call; with k_scale x sm_scale first, 2% to 6% for f16 q)
//   O^T[d, pair] += V^T P'^T    P' = e2() v_scale from the score registers: score i of lane l is token 8 (i / 4) + 4 (l / 32)
//                               + i % 4, so a product of 16 tokens takes scores 8 pp .. + 7 of both halves; V^T by transposing
//                               reads of those rows
// Operand types as in shared_prefix_narrow.h.
//
// Two workgroups share a CU (237 VGPRs, 77 KB of LDS each), so that one computes while the other begins or joins. Microseconds of
// a call when that was chosen, four waves on 64 pairs, against blocks of 16 pairs from registers (as tree_attention_mfma.hip has them
// for float32 queries; that form for 16-bit ones is gone) and against blocks of 32, 64 and 128 of eight waves, alone on their CU;
// cache in e4m3fn, head size 128, and last the present kernel, behind later steps:
//   sequences, nodes, tokens, q / KV heads           16    8 x 32    8 x 64   8 x 128    4 x 64    now
//   64, 2, 2000, 64 / 8                              88        92       114       139        80
//   32, 16, 4080, 32 / 8                            184       118        83       116        88     86
//   61, 1 to 60, 1 to 3060, 16 / 4 (float16 q)      221       153       144       163       118    104
//   8, 64, 32768, 32 / 8                            951       576       419       402       399    390
// The vector ALU and the matrix cores bound it where there are rows enough: per step 225 and 16 instructions, of which two waves a
// SIMD hide little from each other. Steps since that table: the waves' priority is higher at the loads and the products (8 sequences of
// 32768 tokens: 399 us without it, 377 with it), and all of a step's operands leave LDS at its begin (403, 393). With one row block
// the same bounds it before HBM does: 32 sequences of 4096 tokens take 78 us without the join, 269 MB at 3.4 TB/s, where one row a
// sequence (kvfp8_decode_mfma.hip) takes 48: both tiles' waves read and widen every code, and every workgroup makes the plan.
#include "joined_state.h"
#include "shared_prefix_narrow.h"
#include "tree_attention.h"

namespace kvfp8 {

namespace {

constexpr int kTiles = 2, kGroups = 2, kBlockWaves = kTiles * kGroups;
constexpr int kRingBytes = 68 * 1024;
constexpr float kTreeLag = 8.0f;      // log2 of how far a maximum may exceed its reference

typedef __attribute__((address_space(3))) const uint8_t lds_u8;
typedef __attribute__((address_space(3))) const u32x4_t lds_u32x4;
typedef int v2i_t __attribute__((ext_vector_type(2)));
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v2i_t lds_v2i;
typedef __attribute__((address_space(3))) v4s_t lds_v4s;

// One step of a group in LDS: 32 rows of K, 32 of V, of 64 C elements each, then e4m3fn scales ([k|v][token]). A row is 16-byte
// runs in an order by row (run r in slot r ^ order(row)), in which neither the 16 rows of a K read nor the rows of a transposing
// read meet in a bank.
template <int C, int ES>
struct Ring {
    static constexpr int kRow = 64 * C * ES, kSlots = kRow / 16, kRows = 64 / kSlots;     // bytes, runs; rows of one load
    static constexpr int kLoads = 2 * 32 / kRows;                                         // of K, then of V
    static constexpr int kOffsets = 16 / kRows;                                           // different ones by lane: rows of a tile
    static constexpr int kScales = ES == 1 ? 1 : 0;
    static constexpr int kStepBytes = 64 * kRow + 256 * kScales;
    static constexpr int kSteps = kGroups * kStepBytes * 4 <= kRingBytes ? 4 : 2;
    static constexpr int kMine = kLoads / kTiles;             // loads of a wave, a step
    static constexpr int kPerStep = kMine + kScales;
    static_assert(kGroups * kStepBytes * kSteps <= kRingBytes, "two steps of every group fit into LDS");
    static __device__ __forceinline__ int order(int row) {
        if constexpr (kSlots == 4) return (row >> 2) & 3;
        const int u = (row >> 1) & 7;
        if constexpr (kSlots == 8) return ES == 1 ? ((u & 1) << 1) | ((u >> 1) & 1) | (u & 4) : ((u & 1) << 2) | (u >> 1);
        return ((row & 3) << 2) | ((row >> 2) & 3);
    }
};

// Tokens of the chunk whose pages are all there, from its start on: a wave looks at 64 pages at once.
__device__ __forceinline__ int32_t paged_until(const TreeArgs& a, const TreeWork& w) {
    const int32_t first = w.lo >> a.d.bs_shift, last = (w.hi - 1) >> a.d.bs_shift;
    for (int32_t p = first; p <= last; p += 64) {
        const int32_t page = w.table[min(p + (int32_t)(threadIdx.x & 63), last)];
        const uint64_t missing = __ballot(page < 0 || page >= a.d.num_blocks);
        if (missing != 0) return max(w.lo, (p + (int32_t)__builtin_ctzll(missing)) << a.d.bs_shift);
    }
    return w.hi;
}

// Which tokens of a step count: those of the tiles that are there, and of nodes those whose bit is set for the lane's pair.
struct BlockTokens {
    int hi, lim_a, lim_b;
    uint32_t bits;
    __device__ __forceinline__ bool held(int x) const { return 8 * ((x >> 2) & 1) + 4 * hi + (x & 3) < (x < 8 ? lim_a : lim_b); }
    __device__ __forceinline__ bool row(int x) const { return held(x) && ((bits >> (8 * (x >> 2) + 4 * hi + (x & 3))) & 1u) != 0; }
};

template <int C, int QT, int ES>
__global__ void __launch_bounds__(64 * kBlockWaves, 2)
tree_block_kernel(TreeArgs a) {
    using T = typename Elem<QT>::T;
    using K = Kinds<QT, ES>;
    using R = Ring<C, ES>;
    constexpr int N = 2 * C, KS = 4 * C, S = R::kSteps;
    constexpr bool kF16 = K::kF16, kF16V = K::kF16V;
    constexpr int kParts = K::kPParts;
    struct Lds {
        union {
            uint8_t ring[kGroups][S][R::kStepBytes];
            float merge[kTiles][16 * N + 2][64];     // once the rings are empty
        };
        TreeMasks masks;
    };
    __shared__ __attribute__((aligned(16))) Lds lds;
    TreeWork w;
    if (!tree_work(a, w)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int group = wave / kTiles, tile = wave % kTiles;
    const int col = lane & 31, hi = lane >> 5;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int D = a.d.head_dim;
    const int32_t end = w.hi, held = w.it.s.held;
    constexpr int32_t stride = 32 * kGroups;             // tokens of a round
    const bool active = w.r0 + 32 * tile < w.pairs;

    // A wave's part of the loads of its group's next step. As inline assembly: the compiler would wait for all of them before any
    // read of LDS. The waits are those before each round's barrier; the compiler holds nothing in m0 across a statement. Every
    // step has the same number of loads, past the chunk's end too (rows of its first page, which count nothing). Lane l of load i
    // of a tensor writes slot l % kSlots of row kRows i + l / kSlots.
    typedef __attribute__((address_space(3))) void* lds_ptr;
    const uint32_t ring0 = uniform((int32_t)(uint32_t)(uintptr_t)(lds_ptr)(&lds.ring[group][0][0]));
    uint32_t off[R::kOffsets];
    const int32_t row_stride = a.d.num_kv_heads * D * ES;
#pragma unroll
    for (int i = 0; i < R::kOffsets; ++i) {
        const int row = R::kRows * i + lane / R::kSlots;
        off[i] = (uint32_t)(row * row_stride + 16 * min((lane % R::kSlots) ^ R::order(row), D * ES / 16 - 1));
    }
    int32_t next_tok = w.lo + 32 * group;
    StepPages next = step_pages(a, w, next_tok);
    auto push = [&](int slot) __attribute__((always_inline)) {
        const StepRefs refs = step_refs(a, w, next, next_tok);
        next_tok += stride;
        next = step_pages(a, w, next_tok);
        const uint32_t to = ring0 + (uint32_t)(slot * R::kStepBytes);
        const int64_t at_a = (refs.a.row0 * a.d.num_kv_heads + w.h) * D * ES, at_b = (refs.b.row0 * a.d.num_kv_heads + w.h) * D * ES;
#pragma unroll
        for (int j = 0; j < R::kMine; ++j) {
            const int i = (tile * R::kMine + j) % R::kLoads, v = i / (R::kLoads / 2), t = i / R::kOffsets & 1;
            const uint64_t from = uniform64((int64_t)(uintptr_t)(v ? a.d.v_cache : a.d.k_cache) + (t ? at_b : at_a));
            uint32_t by_lane = off[0];
#pragma unroll
            for (int o = 1; o < R::kOffsets; ++o) by_lane = i % R::kOffsets == o ? off[o] : by_lane;
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(uniform(to + 1024u * (uint32_t)i)), "v"(by_lane),
                             "s"(from)
                             : "memory");
        }
        if constexpr (R::kScales != 0) {
            const float* p = (hi ? a.d.v_scales : a.d.k_scales) + ((col < 16 ? refs.a.row0 : refs.b.row0) + (col & 15)) * a.d.num_kv_heads + w.h;
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(uniform(to + 64 * R::kRow)), "v"(p) : "memory");
        }
    };
#pragma unroll
    for (int i = 0; i + 1 < S; ++i) push(i);

    // Q^T operands: lane (pair l % 32 of the tile, l / 32); pairs past the last repeat it and are never stored.
    u32x4_t q[KS];
    const int32_t pair = min(w.r0 + 32 * tile + col, w.pairs - 1), node = (uint32_t)pair / (uint32_t)G;
    const int32_t hq = w.h * G + (pair - node * G);
    {
        const T* src = reinterpret_cast<const T*>(a.d.q) + (int64_t)(w.it.s.row0 + node) * a.d.q_stride_b + hq * a.d.q_stride_h;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = ES == 1 ? 32 * (s >> 1) + 16 * hi + 8 * (s & 1) : 16 * s + 8 * hi;
            const bool inside = d < D;
            const T* p = src + (inside ? d : 0);
            u32x4_t x;
            if (a.q_vec) {
                x = *reinterpret_cast<const u32x4_t*>(p);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (uint32_t)p[2 * e] | ((uint32_t)p[2 * e + 1] << 16);
            }
            q[s] = inside ? x : u32x4_t{0u, 0u, 0u, 0u};
        }
    }
    if (end > held) build_masks(lds.masks, a, w.it.s);

    // Per-lane byte offsets of the operand reads in a step. K: row l % 32, run 2 u + l / 32. V^T of e4m3fn by the transposing read
    // of bytes: of 16 lanes lane i reads dims 8 (i % 2) .. + 7 of row i / 2 of a block of 8 rows x 16 dims and receives dim i of the
    // eight rows; of 16 bits: dims 4 (i % 4) .. + 3 of row i / 4 of 4 rows x 16 dims. Lanes 16..31 of a half take the next 16 dims.
    const uint32_t k_off = (uint32_t)(col * R::kRow + 16 * (hi ^ R::order(col)));
    uint32_t v_off[ES];
    if constexpr (ES == 1) {
        const int row = 8 * ((lane >> 3) & 1) + 4 * hi + ((lane >> 1) & 3);
        v_off[0] = (uint32_t)(32 * R::kRow + row * R::kRow + 16 * (((lane >> 4) & 1) ^ R::order(row)) + 8 * (lane & 1));
    } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = 8 * e + 4 * hi + ((lane >> 2) & 3);
            v_off[e] = (uint32_t)(32 * R::kRow + row * R::kRow + 16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ R::order(row)) + 8 * (lane & 1));
        }
    }

    f32x16_t o[N];                                       // O^T[d = 32 nb + 8 (i / 4) + 4 (l / 32) + i % 4][pair l % 32] in o[nb][i]
#pragma unroll
    for (int nb = 0; nb < N; ++nb) o[nb] = f32x16_t{};
    float ref = 0.0f, lim = kNegInf, l = 0.0f;           // reference (0 before the first score), what scores may reach, the lane's sum

    // The step in `slot`, from token t0 on. kWhole: all 32 tokens count for every pair.
    auto compute = [&](int slot, auto whole_c, int32_t t0) __attribute__((always_inline)) {
#pragma clang fp contract(off)
        constexpr bool kWhole = decltype(whole_c)::value;
        const uint8_t* const here = &lds.ring[group][0][0] + slot * R::kStepBytes;
        lds_u8* const at = (lds_u8*)here;
        const float4* const scales = reinterpret_cast<const float4*>(here + 64 * R::kRow);
        // All operands are asked for at once: two waves a SIMD hide little of LDS' latency.
        u32x4_t kx[2 * C * ES], vx[2][N];
#pragma unroll
        for (int u = 0; u < 2 * C * ES; ++u) kx[u] = *(lds_u32x4*)(at + (k_off ^ (32u * u)));
        f32x4_t ks[4], vs[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if constexpr (ES == 1) ks[g] = __builtin_bit_cast(f32x4_t, scales[2 * g + hi]);
            if constexpr (ES == 1) vs[g] = __builtin_bit_cast(f32x4_t, scales[8 + 2 * g + hi]);
        }
#pragma unroll
        for (int pp = 0; pp < 2; ++pp)
#pragma unroll
            for (int nb = 0; nb < N; ++nb) {
                if constexpr (ES == 1) {
                    const v2i_t x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(at + ((v_off[0] ^ (32u * nb)) + 16 * pp * R::kRow)));
                    vx[pp][nb] = u32x4_t{(uint32_t)x.x, (uint32_t)x.y, 0u, 0u};
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint2 x = __builtin_bit_cast(
                            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + ((v_off[e] ^ (64u * nb)) + 16 * pp * R::kRow))));
                        vx[pp][nb][2 * e] = x.x;
                        vx[pp][nb][2 * e + 1] = x.y;
                    }
                }
            }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
        f32x16_t sc;
#pragma unroll
        for (int u = 0; u < 2 * C * ES; ++u) {
            if constexpr (ES == 1) {
                sc = mma32<kF16>(__builtin_bit_cast(u32x4_t, widen8<kF16>(kx[u][0], kx[u][1])), q[2 * u], u == 0 ? f32x16_t{} : sc);
                sc = mma32<kF16>(__builtin_bit_cast(u32x4_t, widen8<kF16>(kx[u][2], kx[u][3])), q[2 * u + 1], sc);
            } else {
                sc = mma32<kF16>(kx[u], q[u], u == 0 ? f32x16_t{} : sc);
            }
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int x = 0; x < 16; ++x) sc[x] *= a.d.score_scale;
        if constexpr (ES == 1) {
#pragma unroll
            for (int x = 0; x < 16; ++x) sc[x] *= ks[x >> 2][x & 3];
        }
        // Rows of V that count for no pair (stale pages may hold NaN) and those with a value that is not finite are zeros in the
        // products, and their scales zeros: a weight of 0 would not keep them from a pair. The latter (`odd`) come one by one.
        StepRefs refs;
        BlockTokens counts{hi, 16, 16, ~0u};
        uint32_t odd = 0, gone = 0;                      // by token
        if constexpr (!kWhole) {
            refs = step_refs(a, w, step_pages(a, w, t0), t0);
            counts.lim_a = refs.a.valid ? max(0, min(16, end - t0)) : 0;
            counts.lim_b = refs.b.valid ? max(0, min(16, end - t0 - 16)) : 0;
            gone = ~(((1u << counts.lim_a) - 1u) | (((1u << counts.lim_b) - 1u) << 16));
#pragma unroll
            for (int i = 0; i < R::kLoads / 2; ++i) {
                const u32x4_t x = *(lds_u32x4*)(at + 32 * R::kRow + 1024 * i + 16 * lane);
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) bad = bad || not_finite<ES, kF16V>(x[e]);
                const uint64_t found = __ballot(bad);
                if (found != 0) {
#pragma unroll 1
                    for (int k = 0; k < R::kRows; ++k)
                        if (((found >> (R::kSlots * k)) & ((1ull << (R::kSlots - 1) << 1) - 1)) != 0) odd |= 1u << (R::kRows * i + k);
                }
            }
            if constexpr (ES == 1) {
                const float x = reinterpret_cast<const float*>(scales)[lane];
                odd |= (uint32_t)(__ballot((f32_bits(x) & 0x7F800000u) == 0x7F800000u) >> 32);
            }
            odd &= ~gone;
            gone |= odd;
            if (end > held) counts.bits = node_bits(lds.masks, node, t0, held);
#pragma unroll
            for (int x = 0; x < 16; ++x)
                if (!counts.row(x)) sc[x] = kNegInf;
        }
        float mx = sc[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) mx = fmaxf(mx, sc[x]);
        if (__ballot(mx > lim)) {
            const float top = max_across_halves(mx);
            const bool fresh = lim == kNegInf;
            const float to = fresh ? (top == kNegInf ? 0.0f : top) : fmaxf(top, ref);
            const float alpha = fresh ? 0.0f : fast_exp2(ref - to);
            // From 2^27 on the sum may round to 2^4 more, and a weight of 2^16 is past float16's numbers.
            const float most = to + kTreeLag;
            lim = fresh && top == kNegInf ? kNegInf : (most - to > kTreeLag ? to : most);
            ref = to;
            l *= alpha;
#pragma unroll
            for (int nb = 0; nb < N; ++nb) o[nb] *= alpha;
        }
        u32x4_t pop[kParts][2];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                float y[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float p = fast_exp2(sc[4 * g + 2 * v + e] - ref);
                    l += p;
                    y[e] = ES == 1 ? p * vs[g][2 * v + e] : p;
                    if (!kWhole && ((gone >> (8 * g + 4 * hi + 2 * v + e)) & 1) != 0) y[e] = 0.0f;
                }
#pragma unroll
                for (int part = 0; part < kParts; ++part) {
                    const uint32_t top = pack2<kF16V>(y[0], y[1]);
                    pop[part][g >> 1][2 * (g & 1) + v] = top;
                    if (part + 1 < kParts) {
                        y[0] -= bits_f32(top << 16);
                        y[1] -= bits_f32(top & 0xFFFF0000u);
                    }
                }
            }
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int pp = 0; pp < 2; ++pp) {
            u32x4_t keep = {~0u, ~0u, ~0u, ~0u};         // bytes or 16-bit values by token
            if constexpr (!kWhole) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t part = ES == 1 ? 0xFFu << (8 * (e & 3)) : 0xFFFFu << (16 * (e & 1));
                    if (((gone >> (16 * pp + 8 * (e >> 2) + 4 * hi + (e & 3))) & 1) != 0) keep[ES == 1 ? e >> 2 : e >> 1] &= ~part;
                }
            }
#pragma unroll
            for (int nb = 0; nb < N; ++nb) {
                u32x4_t av;
                if constexpr (ES == 1) av = __builtin_bit_cast(u32x4_t, fp8x8(vx[pp][nb][0] & keep[0], vx[pp][nb][1] & keep[1]));
                else av = vx[pp][nb] & keep;
#pragma unroll
                for (int part = 0; part < kParts; ++part) o[nb] = mma32<kF16V>(av, pop[part][pp], o[nb]);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (!kWhole) {
#pragma unroll 1
            for (uint32_t left = odd; left != 0; left &= left - 1) {
                const int tt = __builtin_ctz(left);
                float s = kNegInf;
#pragma unroll
                for (int x = 0; x < 16; ++x) s = 4 * (tt >> 3) + (tt & 3) == x ? sc[x] : s;
                s = __shfl(s, 32 * ((tt >> 2) & 1) + col);
                if (s == kNegInf) continue;              // it does not count for the pair (or at a weight of 0)
                const int64_t row = ((tt < 16 ? refs.a.row0 : refs.b.row0) + (tt & 15)) * a.d.num_kv_heads + w.h;
                const float weight = fast_exp2(s - ref) * (ES == 1 ? a.d.v_scales[row] : 1.0f);
#pragma unroll
                for (int nb = 0; nb < N; ++nb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int dim = 32 * nb + 8 * (i >> 2) + 4 * hi + (i & 3);
                        if (dim >= D) continue;
                        float y;
                        if constexpr (ES == 1) y = decode_e4m3fn(reinterpret_cast<const uint8_t*>(a.d.v_cache)[row * D + dim]);
                        else y = Elem<kF16V ? KVFP8_F16 : KVFP8_BF16>::load(reinterpret_cast<const uint16_t*>(a.d.v_cache)[row * D + dim]);
                        o[nb][i] += weight * y;
                    }
            }
        }
    };
    // A round: each group's step n, when its loads are there and every wave is done with step n - 1, whose place takes step
    // n + S - 1. First the rounds whose tokens all lie on pages before the nodes.
    auto begin_round = [&](int32_t n) __attribute__((always_inline)) {
        __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(R::kPerStep * (S - 2)) : "memory");
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_setprio(2);
        push((int)((uint32_t)(n + S - 1) % (uint32_t)S));
        __builtin_amdgcn_s_setprio(0);
    };
    const int32_t rounds = (end - w.lo + stride - 1) / stride;
    const int32_t plain = uniform((min(min(end, held), paged_until(a, w)) - w.lo) / stride);
    int32_t n = 0;
    for (; n < plain; ++n) {
        begin_round(n);
        if (active) compute((int)((uint32_t)n % (uint32_t)S), std::integral_constant<bool, true>{}, 0);
    }
    for (; n < rounds; ++n) {
        begin_round(n);
        const int32_t tok = w.lo + n * stride + 32 * group;
        if (active && tok < end) compute((int)((uint32_t)n % (uint32_t)S), std::integral_constant<bool, false>{}, tok);
    }
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");

    // The second group's states join the first one's in LDS.
    float m = lim == kNegInf ? kNegInf : ref;
    if (end - w.lo > 32) {                               // (workgroup-uniform)
        __syncthreads();                                 // both rings are empty
        float(*const other)[64] = lds.merge[tile];
        if (group == 1) {
#pragma unroll
            for (int nb = 0; nb < N; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) other[16 * nb + i][lane] = o[nb][i];
            other[16 * N][lane] = m;
            other[16 * N + 1][lane] = l;
        }
        __syncthreads();
        if (group == 0) {
            const float mo = other[16 * N][lane];
            const float mn = fmaxf(m, mo), mu = mn == kNegInf ? 0.0f : mn;
            const float wa = fast_exp2(m - mu), wb = fast_exp2(mo - mu);
#pragma unroll
            for (int nb = 0; nb < N; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[nb][i] = o[nb][i] * wa + other[16 * nb + i][lane] * wb;
            l = l * wa + other[16 * N + 1][lane] * wb;
            m = mn;
        }
    }
    if (group != 0) return;
    l = sum_across_halves(l);
    if (w.r0 + 32 * tile + col >= w.pairs) return;
    if (w.it.chunks > 1) {
        const int64_t at = (int64_t)w.state * a.block_rows + 32 * tile + col;
        if (hi == 0) {
            a.d.part_m[at] = m;
            a.d.part_l[at] = l;
        }
#pragma unroll
        for (int d = 0; d < 64 * C; d += 8) {
            const int i = d % 32 / 2;
            if (d + 4 * hi >= D) continue;
            *reinterpret_cast<float4*>(a.d.part_acc + at * D + d + 4 * hi) = make_float4(o[d / 32][i], o[d / 32][i + 1], o[d / 32][i + 2], o[d / 32][i + 3]);
        }
        return;
    }
    T* const out = reinterpret_cast<T*>(a.d.out) + ((int64_t)(w.it.s.row0 + node) * a.d.num_q_heads + hq) * D;
    const bool ok = l > 0.0f || l != l;
#pragma unroll
    for (int d = 0; d < 64 * C; d += 8) {
        const int i = d % 32 / 2;
        if (d + 4 * hi >= D) continue;
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = ok ? o[d / 32][i + e] / l : 0.0f;
        store_run<QT, 4>(out + d + 4 * hi, y);
    }
}

template <int C, int QT, int ES>
hipError_t launch_blocks(const TreeArgs& a, int64_t items, hipStream_t s) {
    const dim3 grid((unsigned)tree_grid(items));
    hipLaunchKernelGGL((tree_block_kernel<C, QT, ES>), grid, dim3(64 * kBlockWaves), 0, s, a);
    return hipGetLastError();
}

}  // namespace

template <int QT>
hipError_t launch_tree_blocks(const TreeArgs& a, int kv_dtype, int64_t items, hipStream_t s) {
    if (kv_dtype == KVFP8_E4M3FN) return a.d.head_dim == 64 ? launch_blocks<1, QT, 1>(a, items, s) : launch_blocks<2, QT, 1>(a, items, s);
    return a.d.head_dim == 64 ? launch_blocks<1, QT, 2>(a, items, s) : launch_blocks<2, QT, 2>(a, items, s);
}

template hipError_t launch_tree_blocks<KVFP8_F16>(const TreeArgs&, int, int64_t, hipStream_t);
template hipError_t launch_tree_blocks<KVFP8_BF16>(const TreeArgs&, int, int64_t, hipStream_t);

}  // namespace kvfp8
