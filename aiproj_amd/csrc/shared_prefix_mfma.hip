// Shared prefixes on the gfx950 matrix cores.
//
// Rows of a group are the pairs (token of q, q head of one KV head), so a prefix is one product of
// [rows, D] with [tokens, D] per KV head and its bytes are read once for a block of 16 RT rows. A
// workgroup takes one (row block, KV head, split of the prefix); its eight waves take steps of 32
// tokens in turn, each with the whole row block in registers, and join their states at the end.
//
// Per step (MFMA 16x16x32: A[row = l % 16][k = 8 (l / 16) + i], B[k][col = l % 16], D[row = 4 (l / 16) +
// j][col = l % 16]):
//   S^T[token, row] = K Q^T     A = K codes widened in registers (exact), B = Q^T, loaded once;
//                               then x k_scale[token] x sm_scale x log2(e) in float32
//   softmax                     online, base 2, float32, per row (column l % 16)
//   O^T[d, row] += V^T P'^T     P' = p v_scale[token]; V^T by byte transposes of eight token rows
// Operand types: bf16 q over e4m3fn codes bf16 throughout; f16 q multiplies codes widened to f16 (exact),
// its P' enters as two bf16 parts (an f16 P' would lose scales outside f16's range); float32 q and its P'
// as three bf16 parts; bf16 and f16 caches with q of their type are operands as they are.
#include "shared_prefix_blocks.h"

namespace kvfp8 {

namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;

template <int QT, int ES>
struct Kinds {
    static constexpr bool kF16 = QT == KVFP8_F16;                 // K and Q^T operands
    static constexpr bool kF16V = kF16 && ES == 2;                // V^T and P operands
    static constexpr int kQParts = QT == KVFP8_F32 ? 3 : 1;
    static constexpr int kPParts = ES == 2 || QT == KVFP8_BF16 ? 1 : (QT == KVFP8_F16 ? 2 : 3);
};

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// Eight codes -> eight 16-bit values in byte order.
template <bool kF16>
__device__ __forceinline__ OpT<kF16> widen8(uint32_t x0, uint32_t x1) {
    if constexpr (kF16) {
        const f16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x0, 1.0f, false);
        const f16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x0, 1.0f, true);
        const f16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x1, 1.0f, false);
        const f16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x1, 1.0f, true);
        return f16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    } else {
        return fp8x8(x0, x1);
    }
}

// One step of 32 tokens of one KV head: tile A is tokens 0..15, tile B 16..31.
template <int C, int ES>
struct PrefixStep {
    u32x4_t ka[C * ES], kb[C * ES];   // token l % 16, 16-byte runs at bytes 64 r + 16 (l / 16)
    uint32_t v[8][C * ES];            // token 4 (l / 16) + i % 4 of tile i / 4, 4 C elements at 4 C (l % 16)
    float sc;                         // e4m3fn: lane l holds the [k|v][tile A|B][token l % 16] scale
};

template <int C, int ES>
__device__ __forceinline__ void load_prefix_step(PrefixStep<C, ES>& s, const DecodeArgs& d, int h, const TileRef& ta,
                                                 const TileRef& tb, int lane) {
    constexpr int NB = 4 * C, KR = C * ES, VW = C * ES;
    const int m16 = lane & 15, j = lane >> 4;
    const int D = d.head_dim;
    const int32_t row_stride = d.num_kv_heads * D * ES;
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(d.k_cache);
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(d.v_cache);
    const int64_t ea = (ta.row0 * d.num_kv_heads + h) * D * ES, eb = (tb.row0 * d.num_kv_heads + h) * D * ES;
#pragma unroll
    for (int r = 0; r < KR; ++r) {
        // Head sizes between 64 and 128 end inside the second run: its last 16 bytes again (q is 0 there).
        const uint32_t off = (uint32_t)(m16 * row_stride + min(64 * r + 16 * j, D * ES - 16));
        s.ka[r] = *reinterpret_cast<const u32x4_t*>(kc + ea + off);
        s.kb[r] = *reinterpret_cast<const u32x4_t*>(kc + eb + off);
    }
    const int col = min(NB * m16, D - NB) * ES;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint8_t* p = vc + (i < 4 ? ea : eb) + (uint32_t)((4 * j + (i & 3)) * row_stride + col);
        if constexpr (VW == 1) {
            s.v[i][0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (VW == 2) {
            const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p);
            s.v[i][0] = x.x;
            s.v[i][1] = x.y;
        } else {
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
            for (int w = 0; w < 4; ++w) s.v[i][w] = x[w];
        }
    }
    if constexpr (ES == 1) {
        const int64_t row = ((lane & 16) ? tb.row0 : ta.row0) + m16;
        s.sc = ((lane & 32) ? d.v_scales : d.k_scales)[row * d.num_kv_heads + h];
    }
}

template <int C, int RT>
struct RowState {
    f32x4_t o[RT][4 * C];             // O^T[d = 4 C (4 (l / 16) + j) + nb][row l % 16 of tile rt] in o[rt][nb][j]
    float m[RT], l[RT];               // maximum; this lane's share of the sum
};

template <int C, int QT, int ES, int RT>
__device__ __forceinline__ void prefix_step(RowState<C, RT>& st, const PrefixStep<C, ES>& s,
                                            const OpT<Kinds<QT, ES>::kF16> (&q)[RT][Kinds<QT, ES>::kQParts][2 * C],
                                            float4* stage, int lane, int lim_a, int lim_b, float score_scale) {
    using K = Kinds<QT, ES>;
    constexpr int VW = C * ES, NB = 4 * C;
    const int j = lane >> 4;
    const bool full = lim_a == 16 && lim_b == 16;        // wave-uniform
    float ks[8], vs[8];
    if constexpr (ES == 1) {
        // Lane l's scale goes to slot l of the wave's 64; every lane reads its eight tokens'.
        reinterpret_cast<float*>(stage)[lane] = lane < 32 ? s.sc * score_scale : s.sc;
        __builtin_amdgcn_wave_barrier();
        const float4 k0 = stage[j], k1 = stage[4 + j], v0 = stage[8 + j], v1 = stage[12 + j];
        __builtin_amdgcn_wave_barrier();
        ks[0] = k0.x; ks[1] = k0.y; ks[2] = k0.z; ks[3] = k0.w;
        ks[4] = k1.x; ks[5] = k1.y; ks[6] = k1.z; ks[7] = k1.w;
        vs[0] = v0.x; vs[1] = v0.y; vs[2] = v0.z; vs[3] = v0.w;
        vs[4] = v1.x; vs[5] = v1.y; vs[6] = v1.z; vs[7] = v1.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ks[i] = score_scale;
            vs[i] = 1.0f;
        }
    }
    f32x4_t sa[RT], sb[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) sa[rt] = sb[rt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kb = 0; kb < 2 * C; ++kb) {
        OpT<K::kF16> xa, xb;
        if constexpr (ES == 1) {
            xa = widen8<K::kF16>(s.ka[kb >> 1][2 * (kb & 1)], s.ka[kb >> 1][2 * (kb & 1) + 1]);
            xb = widen8<K::kF16>(s.kb[kb >> 1][2 * (kb & 1)], s.kb[kb >> 1][2 * (kb & 1) + 1]);
        } else {
            xa = __builtin_bit_cast(OpT<K::kF16>, s.ka[kb]);
            xb = __builtin_bit_cast(OpT<K::kF16>, s.kb[kb]);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int p = 0; p < K::kQParts; ++p) {
                sa[rt] = mma(xa, q[rt][p][kb], sa[rt]);
                sb[rt] = mma(xb, q[rt][p][kb], sb[rt]);
            }
        }
    }
    // Score i is token 4 j + i % 4 of tile i / 4.
    bool live[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) live[i] = full || 4 * j + (i & 3) < (i < 4 ? lim_a : lim_b);
    OpT<K::kF16V> pp[RT][K::kPParts];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float sc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = (i < 4 ? sa[rt][i & 3] : sb[rt][i & 3]) * ks[i];
            sc[i] = full || live[i] ? x : kNegInf;
        }
        float mx = sc[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = fmaxf(st.m[rt], mx);
        const float m_use = m_new == kNegInf ? 0.0f : m_new;
        const float alpha = fast_exp2(st.m[rt] - m_use);
        if (__ballot(alpha != 1.0f)) {
            st.l[rt] *= alpha;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) st.o[rt][nb] *= alpha;
        }
        st.m[rt] = m_new;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = fast_exp2(sc[i] - m_use);
            st.l[rt] += p;
            float x = p * vs[i];
            if (!full && !live[i]) x = 0.0f;             // a stale scale may be NaN
#pragma unroll
            for (int part = 0; part < K::kPParts; ++part) {
                const OpE<K::kF16V> hi = (OpE<K::kF16V>)x;
                pp[rt][part][i] = hi;
                x -= (float)hi;
            }
        }
    }
    // V rows of masked tokens are zero (stale pages may hold NaN).
    uint32_t vr[8][VW];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) vr[i][w] = full || live[i] ? s.v[i][w] : 0u;
    auto product = [&](OpT<K::kF16V> av, int nb) __attribute__((always_inline)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int part = 0; part < K::kPParts; ++part) st.o[rt][nb] = mma(av, pp[rt][part], st.o[rt][nb]);
    };
    if constexpr (ES == 1) {
        // Byte transpose: the codes of rows (2 p, 2 p + 1) at one column side by side, widened.
#pragma unroll
        for (int c = 0; c < C; ++c) {
            bf16x2_t e[4][4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const uint32_t x = __builtin_amdgcn_perm(vr[2 * p + 1][c], vr[2 * p][c], 0x05010400u);
                const uint32_t y = __builtin_amdgcn_perm(vr[2 * p + 1][c], vr[2 * p][c], 0x07030602u);
                e[0][p] = fp8x2_lo(x);
                e[1][p] = fp8x2_hi(x);
                e[2][p] = fp8x2_lo(y);
                e[3][p] = fp8x2_hi(y);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) product(cat8(e[x][0], e[x][1], e[x][2], e[x][3]), 4 * c + x);
        }
    } else {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const uint32_t sel = (nb & 1) ? 0x07060302u : 0x05040100u;
            u32x4_t w;
#pragma unroll
            for (int p = 0; p < 4; ++p) w[p] = __builtin_amdgcn_perm(vr[2 * p + 1][nb >> 1], vr[2 * p][nb >> 1], sel);
            product(__builtin_bit_cast(OpT<K::kF16V>, w), nb);
        }
    }
}

// Elements [d0, d0 + n) of an output row.
template <int QT, int N>
__device__ __forceinline__ void store_run(typename Elem<QT>::T* dst, const float (&x)[N]) {
    if constexpr (QT == KVFP8_F32) {
#pragma unroll
        for (int w = 0; w < N / 4; ++w)
            reinterpret_cast<float4*>(dst)[w] = make_float4(x[4 * w], x[4 * w + 1], x[4 * w + 2], x[4 * w + 3]);
    } else {
#pragma unroll
        for (int w = 0; w < N / 4; ++w) {
            const uint32_t lo = (uint32_t)Elem<QT>::store(x[4 * w]) | ((uint32_t)Elem<QT>::store(x[4 * w + 1]) << 16);
            const uint32_t hi = (uint32_t)Elem<QT>::store(x[4 * w + 2]) | ((uint32_t)Elem<QT>::store(x[4 * w + 3]) << 16);
            reinterpret_cast<uint2*>(dst)[w] = make_uint2(lo, hi);
        }
    }
}

template <int C, int QT, int ES, int RT>
__global__ void __launch_bounds__(kThreads)
prefix_mfma_kernel(PrefixArgs a, PrefixGrid grid, int q_vec) {
    using K = Kinds<QT, ES>;
    using T = typename Elem<QT>::T;
    constexpr int NB = 4 * C;
    constexpr int kVals = 4 * NB + 2;
    __shared__ float4 stage_all[kWaves][16];
    __shared__ float merge[kWaves / 2][kVals][64];
    PrefixItem it;
    if (!prefix_item(a, grid, 16 * RT, it)) return;
    const int h = it.h, split = it.split;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int32_t lo = it.lo, hi = it.hi;
    const int32_t* table = it.table;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int m16 = lane & 15, j = lane >> 4;
    const int D = a.d.head_dim;

    auto issue = [&](PrefixStep<C, ES>& dst, int32_t t0, TileRef& ra, TileRef& rb2) __attribute__((always_inline)) {
        auto ref = [&](int32_t tok) __attribute__((always_inline)) {
            // Wave-uniform scalar load of the table: its wait leaves the loads in flight alone.
            const int64_t addr = uniform64((int64_t)(uintptr_t)(table + (tok >> a.d.bs_shift)));
            const int64_t phys = *(const_i32_ptr)(uintptr_t)addr;
            const bool ok = phys >= 0 && phys < a.d.num_blocks;
            return TileRef{ok ? phys * a.d.block_size + (tok & (a.d.block_size - 1)) : 0, ok};
        };
        ra = ref(t0);
        rb2 = t0 + 16 < hi ? ref(t0 + 16) : TileRef{0, 0};
        load_prefix_step<C, ES>(dst, a.d, h, ra, rb2, lane);
    };
    PrefixStep<C, ES> buf0, buf1;
    TileRef r0a, r0b, r1a, r1b;
    const int32_t stride = 32 * kWaves;
    int32_t tok = lo + 32 * wave;
    if (tok < hi) issue(buf0, tok, r0a, r0b);

    // Q^T operands: column l % 16 of tile rt is pair r0 + 16 rt + l % 16 (rows past the last repeat it).
    OpT<K::kF16> q[RT][K::kQParts][2 * C];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int32_t pair = min(it.r0 + 16 * rt + m16, it.pairs - 1);
        const int32_t t = (uint32_t)pair / (uint32_t)G;
        const T* src = reinterpret_cast<const T*>(a.d.q) + (int64_t)(it.rs + t) * a.d.q_stride_b + (h * G + (pair - t * G)) * a.d.q_stride_h;
#pragma unroll
        for (int kb = 0; kb < 2 * C; ++kb) {
            const int dim = ES == 1 ? 64 * (kb >> 1) + 16 * j + 8 * (kb & 1) : 32 * kb + 8 * j;
            const bool inside = dim < D;
            const T* p = src + (inside ? dim : 0);
            float x[8];
            if (q_vec) {
                constexpr int kW = 8 * sizeof(T) / 16;
                uint32_t w[4 * kW];
#pragma unroll
                for (int u = 0; u < kW; ++u) {
                    const u32x4_t y = reinterpret_cast<const u32x4_t*>(p)[u];
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[4 * u + e] = y[e];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (QT == KVFP8_F32) x[i] = bits_f32(w[i]);
                    else x[i] = Elem<QT>::load((T)((w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = Elem<QT>::load(p[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float y = inside ? x[i] : 0.0f;
#pragma unroll
                for (int part = 0; part < K::kQParts; ++part) {
                    const OpE<K::kF16> top = (OpE<K::kF16>)y;
                    q[rt][part][kb][i] = top;
                    y = __builtin_isinf(y) ? 0.0f : y - (float)top;      // an infinite q is its first part alone
                }
            }
        }
    }

    RowState<C, RT> st;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) st.o[rt][nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        st.m[rt] = kNegInf;
        st.l[rt] = 0.0f;
    }
    auto compute = [&](const PrefixStep<C, ES>& cur, int32_t t0, const TileRef& ra, const TileRef& rb2) __attribute__((always_inline)) {
        const int lim_a = ra.valid ? min(16, hi - t0) : 0;
        const int lim_b = rb2.valid ? min(16, hi - t0 - 16) : 0;
        prefix_step<C, QT, ES, RT>(st, cur, q, stage_all[wave], lane, lim_a, lim_b, a.d.score_scale);
    };
    while (tok < hi) {
        if (tok + stride < hi) issue(buf1, tok + stride, r1a, r1b);
        compute(buf0, tok, r0a, r0b);
        tok += stride;
        if (tok >= hi) break;
        if (tok + stride < hi) issue(buf0, tok + stride, r0a, r0b);
        compute(buf1, tok, r1a, r1b);
        tok += stride;
    }

    // The waves' states join pairwise in LDS, one row tile at a time, into wave 0.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int half = kWaves / 2; half > 0; half >>= 1) {
            if (wave >= half && wave < 2 * half) {
                float(*mine)[64] = merge[wave - half];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mine[4 * nb + i][lane] = st.o[rt][nb][i];
                mine[4 * NB][lane] = st.m[rt];
                mine[4 * NB + 1][lane] = st.l[rt];
            }
            __syncthreads();
            if (wave < half) {
                const float(*other)[64] = merge[wave];
                const float mo = other[4 * NB][lane];
                const float mn = fmaxf(st.m[rt], mo);
                const float mu = mn == kNegInf ? 0.0f : mn;
                const float wa = fast_exp2(st.m[rt] - mu), wb = fast_exp2(mo - mu);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 4; ++i) st.o[rt][nb][i] = st.o[rt][nb][i] * wa + other[4 * nb + i][lane] * wb;
                st.l[rt] = st.l[rt] * wa + other[4 * NB + 1][lane] * wb;
                st.m[rt] = mn;
            }
            __syncthreads();
        }
    }
    if (wave != 0) return;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float l = st.l[rt] + __shfl_xor(st.l[rt], 16);
        l += __shfl_xor(l, 32);
        float m = st.m[rt];
        const int32_t pair = it.r0 + 16 * rt + m16;
        if (pair >= it.pairs) continue;
        const int32_t t = (uint32_t)pair / (uint32_t)G;
        const int64_t row = it.rs + t;
        const int hq = h * G + (pair - t * G);
        if (a.cu != nullptr && a.splits == 1) {
            // The prompt form's only state of the row: joined with out and lse at once.
            if (seq_of_row(a, row) < 0) continue;
            const int64_t at = row * a.d.num_q_heads + hq;
            const float mo = a.lse[at] * kLog2e;
            const float mn = fmaxf(m, mo), mu = mn == kNegInf ? 0.0f : mn;
            const float wp = fast_exp2(m - mu), wo = fast_exp2(mo - mu);
            const float den = l * wp + wo;
            const float inv = den > 0.0f || den != den ? 1.0f / den : 0.0f;
            T* out = reinterpret_cast<T*>(a.d.out) + at * D;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d0 = NB * (4 * j + i);
                if (d0 >= D) continue;
                float y[NB];
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) y[nb] = (st.o[rt][nb][i] * wp + Elem<QT>::load(out[d0 + nb]) * wo) * inv;
                store_run<QT, NB>(out + d0, y);
            }
            if (j == 0) a.lse[at] = (mu + __builtin_log2f(den)) * kLn2;
            continue;
        }
        const int64_t pi = prefix_part(a, row, split, hq);
        if (j == 0) {
            a.d.part_m[pi] = m;
            a.d.part_l[pi] = l;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d0 = NB * (4 * j + i);
            if (d0 >= D) continue;
            float* acc = a.d.part_acc + pi * D + d0;
#pragma unroll
            for (int w = 0; w < NB / 4; ++w)
                reinterpret_cast<float4*>(acc)[w] =
                    make_float4(st.o[rt][4 * w][i], st.o[rt][4 * w + 1][i], st.o[rt][4 * w + 2][i], st.o[rt][4 * w + 3][i]);
        }
    }
}

// One wave per (row, q head) joins the prefix's states and, in the decode form (kOwn), those of the row's
// own tokens that the decode kernel left (pieces as in combine_mfma_kernel, or a whole state), in the
// prompt form out and lse. Lanes take 16 C float4 columns; 4 / C states are read side by side.
template <int C, int QT, bool kOwn>
__global__ void __launch_bounds__(256)
prefix_mfma_join_kernel(PrefixArgs a, MfmaArgs own) {
    constexpr int kLanes = 16 * C, kPass = 64 / kLanes;
    using T = typename Elem<QT>::T;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int D = a.d.head_dim;
    const int32_t unit = (int32_t)blockIdx.x * 4 + wave;      // below 2^26
    if (unit >= (int32_t)a.rows * a.d.num_q_heads) return;
    const int32_t row = (uint32_t)unit / (uint32_t)a.d.num_q_heads;
    const int32_t hq = unit - row * a.d.num_q_heads;
    const int64_t seq = seq_of_row(a, row);
    if (seq < 0) return;
    const int g = group_of_seq(a, seq);
    int64_t slot;
    const int64_t tokens = g >= 0 ? group_tokens(a, g, &slot) : 0;
    if (!kOwn && tokens == 0) return;                    // out and lse stand
    const int d4 = min(lane % kLanes, D / 4 - 1), po = lane / kLanes;

    float mr = kNegInf, den = 0.0f;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float mi, float li, float4 x) __attribute__((always_inline)) {
        const float mn = fmaxf(mr, mi);
        const float mu = mn == kNegInf ? 0.0f : mn;
        const float wa = fast_exp2(mr - mu), wb = fast_exp2(mi - mu);
        num.x = num.x * wa + x.x * wb;
        num.y = num.y * wa + x.y * wb;
        num.z = num.z * wa + x.z * wb;
        num.w = num.w * wa + x.w * wb;
        den = den * wa + li * wb;
        mr = mn;
    };
    auto add_state = [&](const float* m, const float* l, const float* acc, int64_t i) __attribute__((always_inline)) {
        add(m[i], l[i], reinterpret_cast<const float4*>(acc + i * D)[d4]);
    };
    if constexpr (kOwn) {
        const int32_t t0 = own.plan[row], t1 = own.plan[row + 1];
        if (t1 != t0) {
            const int64_t total = own.plan[a.d.batch], groups = own.plan[a.d.batch + 1];
            const int32_t w0 = uniform(group_of(t0, total, groups)), w1 = uniform(group_of(t1 - 1, total, groups));
            if (w0 == w1) {
                if (po == 0) add_state(own.seq_m, own.seq_l, own.seq_acc, unit);
            } else {
                const int32_t cut0 = floor_div((int64_t)w0 * total, groups) < t0 ? 1 : 0;
#pragma unroll 4
                for (int32_t i = po; i <= w1 - w0; i += kPass)
                    add_state(own.part_m, own.part_l, own.part_acc,
                              (2 * (int64_t)(w0 + i) + (i == 0 ? cut0 : 0)) * a.d.num_q_heads + hq);
            }
        }
    }
    // Splits without tokens left no state.
    const int held = split_count(tokens, split_tokens(tokens, a.step_shift, a.splits));
#pragma unroll 4
    for (int s = po; s < held; s += kPass) add_state(a.d.part_m, a.d.part_l, a.d.part_acc, prefix_part(a, row, s, hq));
#pragma unroll
    for (int off = kLanes; off < 64; off <<= 1)
        add(__shfl_xor(mr, off), __shfl_xor(den, off),
            make_float4(__shfl_xor(num.x, off), __shfl_xor(num.y, off), __shfl_xor(num.z, off), __shfl_xor(num.w, off)));
    if (po != 0 || 4 * (lane % kLanes) >= D) return;
    const int64_t at = unit;
    T* out = reinterpret_cast<T*>(a.d.out) + at * D + 4 * d4;
    if constexpr (!kOwn) {
        add(a.lse[at] * kLog2e, 1.0f,
            make_float4(Elem<QT>::load(out[0]), Elem<QT>::load(out[1]), Elem<QT>::load(out[2]), Elem<QT>::load(out[3])));
        __builtin_amdgcn_wave_barrier();                 // every lane has read lse before lane 0 writes it
        if (lane == 0) a.lse[at] = ((mr == kNegInf ? 0.0f : mr) + __builtin_log2f(den)) * kLn2;
    }
    const bool ok = den > 0.0f || den != den;
    const float y[4] = {ok ? num.x / den : 0.0f, ok ? num.y / den : 0.0f, ok ? num.z / den : 0.0f, ok ? num.w / den : 0.0f};
    store_run<QT, 4>(out, y);
}

// ------------------------------------------------------------------ host

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Pairs of an average group from which blocks of 256 rows are taken.
constexpr int64_t kWidePairs = 128;

template <int C, int QT> constexpr int kTiles = C == 2 || QT == KVFP8_F32 ? 1 : 2;

template <int C, int QT, int ES>
hipError_t launch_prefix(const PrefixArgs& a, const PrefixGrid& g, int q_vec, hipStream_t s) {
    hipLaunchKernelGGL((prefix_mfma_kernel<C, QT, ES, kTiles<C, QT>>), dim3((unsigned)(kXcds * g.per_xcd)), dim3(kThreads), 0, s,
                       a, g, q_vec);
    return hipGetLastError();
}

template <int QT>
hipError_t launch_prefix_kv(const PrefixArgs& a, int kv_dtype, const PrefixGrid& g, int q_vec, hipStream_t s) {
    if (kv_dtype == KVFP8_E4M3FN)
        return a.d.head_dim == 64 ? launch_prefix<1, QT, 1>(a, g, q_vec, s) : launch_prefix<2, QT, 1>(a, g, q_vec, s);
    if constexpr (QT != KVFP8_F32)
        return a.d.head_dim == 64 ? launch_prefix<1, QT, 2>(a, g, q_vec, s) : launch_prefix<2, QT, 2>(a, g, q_vec, s);
    else return hipErrorInvalidValue;                    // 16-bit caches come with q of their type
}

template <int QT, bool kOwn>
hipError_t launch_join(const PrefixArgs& a, const MfmaArgs& own, hipStream_t s) {
    const int64_t units = a.rows * a.d.num_q_heads;
    const dim3 grid((unsigned)((units + 3) / 4));
    if (a.d.head_dim == 64) hipLaunchKernelGGL((prefix_mfma_join_kernel<1, QT, kOwn>), grid, dim3(256), 0, s, a, own);
    else hipLaunchKernelGGL((prefix_mfma_join_kernel<2, QT, kOwn>), grid, dim3(256), 0, s, a, own);
    return hipGetLastError();
}

int rows_per_block(int32_t head_dim, int q_dtype, bool wide) {
    return wide ? kWideRows : (head_dim > 64 || q_dtype == KVFP8_F32 ? 16 : 32);
}

// At most this many row blocks: every group may leave its last one unfilled.
int64_t row_blocks(int64_t rows, int32_t heads, int32_t groups, int per_block) { return rows * heads / per_block + groups; }

}  // namespace

bool prefix_mfma_supported(int32_t head_dim, int32_t block_size, int q_dtype, int kv_dtype) {
    if (block_size < 16) return false;
    if (kv_dtype == KVFP8_E4M3FN) return head_dim == 64 || head_dim == 128 || narrow_head(head_dim);
    return (head_dim == 64 || head_dim == 128) && (kv_dtype == KVFP8_BF16 || kv_dtype == KVFP8_F16) && q_dtype == kv_dtype;
}

PrefixMfmaPlan prefix_mfma_plan(int64_t rows, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t groups,
                                int64_t bt_width, int32_t block_size, int q_dtype, bool prompt) {
    PrefixMfmaPlan p;
    const int heads = num_q_heads / num_kv_heads;
    p.wide = q_dtype != KVFP8_F32 && groups > 0 && rows * heads / groups >= kWidePairs;
    p.step_shift = p.wide ? 6 : 5;
    const int64_t columns = row_blocks(rows, heads, groups, rows_per_block(head_dim, q_dtype, p.wide)) * num_kv_heads;
    // One workgroup per CU, each with at least 256 tokens of the longest prefix.
    int64_t splits = columns > 0 ? (device_cus() + columns / 2) / columns : 1;      // no group: no column
    const int64_t most = bt_width * block_size / 256;
    splits = splits < most ? splits : most;
    p.splits = (int32_t)(splits < 1 ? 1 : splits);
    p.states = prompt && p.splits == 1 ? 0 : rows * num_q_heads * p.splits;
    int64_t off = 0;
    auto take = [&](int64_t bytes) {
        const int64_t at = off;
        off += (int64_t)align256((size_t)bytes);
        return at;
    };
    const int64_t own = prompt ? 0 : rows * num_q_heads;
    int64_t unused[4];
    p.own_plan = take(prompt ? 0 : mfma_workspace_layout((int32_t)rows, num_q_heads, num_kv_heads, head_dim, unused));
    p.seq_m = take(own * 4);
    p.seq_l = take(own * 4);
    p.seq_acc = take(own * head_dim * 4);
    p.part_m = take(p.states * 4);
    p.part_l = take(p.states * 4);
    p.part_acc = take(p.states * head_dim * 4);
    p.bytes = off;
    return p;
}

template <int QT>
hipError_t launch_prefix_mfma(PrefixArgs a, int kv_dtype, const PrefixMfmaPlan& p, void* workspace, hipStream_t s) {
    char* ws = reinterpret_cast<char*>(workspace);
    a.splits = p.splits;
    a.step_shift = p.step_shift;
    a.d.part_m = reinterpret_cast<float*>(ws + p.part_m);
    a.d.part_l = reinterpret_cast<float*>(ws + p.part_l);
    a.d.part_acc = reinterpret_cast<float*>(ws + p.part_acc);
    MfmaArgs own = {};
    if (a.cu == nullptr) {
        const DecodeStates states = {reinterpret_cast<float*>(ws + p.seq_m), reinterpret_cast<float*>(ws + p.seq_l),
                                     reinterpret_cast<float*>(ws + p.seq_acc)};
        const hipError_t err = launch_mfma_states<QT>(a.d, kv_dtype, ws + p.own_plan, states, s);
        if (err != hipSuccess) return err;
        int64_t off[4];
        mfma_workspace_layout(a.d.batch, a.d.num_q_heads, a.d.num_kv_heads, a.d.head_dim, off);
        own.plan = reinterpret_cast<int32_t*>(ws + p.own_plan + off[0]);
        own.part_m = reinterpret_cast<float*>(ws + p.own_plan + off[1]);
        own.part_l = reinterpret_cast<float*>(ws + p.own_plan + off[2]);
        own.part_acc = reinterpret_cast<float*>(ws + p.own_plan + off[3]);
        own.seq_m = states.m;
        own.seq_l = states.l;
        own.seq_acc = states.acc;
    }
    if (a.groups > 0) {
        PrefixGrid g;
        g.blocks = (int32_t)row_blocks(a.rows, a.d.num_q_heads / a.d.num_kv_heads, a.groups,
                                       rows_per_block(a.d.head_dim, QT, p.wide));
        const int64_t total = (int64_t)g.blocks * a.d.num_kv_heads * p.splits;
        g.total = (int32_t)total;
        g.per_xcd = (int32_t)((total + kXcds - 1) / kXcds);
        const int64_t q_size = QT == KVFP8_F32 ? 4 : 2;
        const int q_vec = (uintptr_t)a.d.q % 16 == 0 && a.d.q_stride_b * q_size % 16 == 0 && a.d.q_stride_h * q_size % 16 == 0;
        hipError_t err;
        if constexpr (QT == KVFP8_F32) err = launch_prefix_kv<QT>(a, kv_dtype, g, q_vec, s);
        else err = p.wide ? launch_prefix_wide<QT>(a, kv_dtype, g, q_vec, s) : launch_prefix_kv<QT>(a, kv_dtype, g, q_vec, s);
        if (err != hipSuccess) return err;
    }
    if (a.cu == nullptr) return launch_join<QT, true>(a, own, s);
    return p.splits == 1 ? hipSuccess : launch_join<QT, false>(a, own, s);
}

template hipError_t launch_prefix_mfma<KVFP8_F32>(PrefixArgs, int, const PrefixMfmaPlan&, void*, hipStream_t);
template hipError_t launch_prefix_mfma<KVFP8_F16>(PrefixArgs, int, const PrefixMfmaPlan&, void*, hipStream_t);
template hipError_t launch_prefix_mfma<KVFP8_BF16>(PrefixArgs, int, const PrefixMfmaPlan&, void*, hipStream_t);

}  // namespace kvfp8
