// Up to 16 (row, q head) pairs against runs of cached tokens on the matrix cores: the prefix of a group with
// few rows, and every sequence's own tokens.
//
// A workgroup's waves are divided over `heads` KV heads; the waves of one head take steps of 32 tokens in turn,
// each with the 16 pairs in registers, and join their states at the end. Per step (MFMA 16x16x32: A[row = l %
// 16][k = 8 (l / 16) + i], B[k][col = l % 16], D[row = 4 (l / 16) + j][col = l % 16]):
//   S^T[token, row] = K Q^T     A = K codes widened in registers (exact), B = Q^T, loaded once;
//                               then x k_scale[token] x sm_scale x log2(e) in float32
//   softmax                     online, base 2, float32, per row (column l % 16)
//   O^T[d, row] += V^T P'^T     P' = p v_scale[token]; V^T by byte transposes of eight token rows
// Operand types: bf16 q over e4m3fn codes bf16 throughout; f16 q multiplies codes widened to f16 (exact),
// its P' enters as two bf16 parts (an f16 P' would lose scales outside f16's range); float32 q and its P'
// as three bf16 parts; bf16 and f16 caches with q of their type are operands as they are. A P' of one part is off by up to
// half a step of its type and the sum of weights is not: for bf16 an error of 2.3e-3 of the output's norm against the 1.7e-3
// that its own rounding makes. A second part would cost a product more for each.
// Bound by latency where there are few tokens (a step's loads wait for its pages, the first ones for the group's search:
// 4 x 8 heads, 500 tokens: 6.1 us), by the widening and transposing of V's codes and the loads' latency where there are
// many: own tokens of 256 sequences, 520 on average, 8 KV heads x 128: 82 us, 3.4 TB/s (decode without prefixes takes
// 76 us for the same tokens). Page numbers read a step ahead and loads without a branch around them did not change that.
#pragma once

#include "mfma_tiles.h"
#include "shared_prefix_blocks.h"

namespace kvfp8 {

namespace {

template <int QT, int ES>
struct Kinds {
    static constexpr bool kF16 = QT == KVFP8_F16;                 // K and Q^T operands
    static constexpr bool kF16V = kF16 && ES == 2;                // V^T and P operands
    static constexpr int kQParts = QT == KVFP8_F32 ? 3 : 1;
    static constexpr int kPParts = ES == 2 || QT == KVFP8_BF16 ? 1 : (QT == KVFP8_F16 ? 2 : 3);
};

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

template <int C>
struct RowState {
    f32x4_t o[4 * C];                 // O^T[d = 4 C (4 (l / 16) + j) + nb][row l % 16] in o[nb][j]
    float m, l;                       // maximum; this lane's share of the sum
};

// Which tokens of a step count, of token i = 0..7 of a lane: token 4 (l / 16) + i % 4 of tile i / 4. Here the first lim_a of
// tile A and lim_b of tile B, for every row.
struct FirstTokens {
    int j, lim_a, lim_b;              // j: l / 16
    static constexpr bool kByRow = false;
    __device__ __forceinline__ bool row(int i) const { return held(i); }        // for the lane's row
    __device__ __forceinline__ bool held(int i) const { return 4 * j + (i & 3) < (i < 4 ? lim_a : lim_b); }   // for any row
};

// What takes the place of the products with V where tokens count for some of the rows only (0 times a value that is not
// finite would reach the others).
struct MatrixProducts {};

// kFull: all 32 tokens count. Else those that `counts` says do. `products`: MatrixProducts, or with counts by row what says
// whether a step's V fits them and adds it otherwise.
template <int C, int QT, int ES, bool kFull, typename Counts, typename Products = MatrixProducts>
__device__ __forceinline__ void prefix_step(RowState<C>& st, const PrefixStep<C, ES>& s,
                                            const OpT<Kinds<QT, ES>::kF16> (&q)[Kinds<QT, ES>::kQParts][2 * C],
                                            float4* stage, int lane, const Counts& counts, float score_scale,
                                            const Products& products = Products{}) {
    using K = Kinds<QT, ES>;
    constexpr int VW = C * ES, NB = 4 * C;
    const int j = lane >> 4;
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
    f32x4_t sa = {0.0f, 0.0f, 0.0f, 0.0f}, sb = sa;
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
        for (int p = 0; p < K::kQParts; ++p) {
            sa = mma(xa, q[p][kb], sa);
            sb = mma(xb, q[p][kb], sb);
        }
    }
    // Score i is token 4 j + i % 4 of tile i / 4.
    bool live[8];
    float sc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        live[i] = kFull || counts.row(i);
        const float x = (i < 4 ? sa[i & 3] : sb[i & 3]) * ks[i];
        sc[i] = live[i] ? x : kNegInf;
    }
    float mx = sc[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i]);
    const float m_new = fmaxf(st.m, max_across_rows(mx));
    const float m_use = m_new == kNegInf ? 0.0f : m_new;
    const float alpha = fast_exp2(st.m - m_use);
    if (__ballot(alpha != 1.0f)) {
        st.l *= alpha;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) st.o[nb] *= alpha;
    }
    st.m = m_new;
    OpT<K::kF16V> pp[K::kPParts];
    float weight[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float p = fast_exp2(sc[i] - m_use);
        st.l += p;
        float x = live[i] ? p * vs[i] : 0.0f;            // a stale scale may be NaN
        weight[i] = x;
#pragma unroll
        for (int part = 0; part < K::kPParts; ++part) {
            const OpE<K::kF16V> hi = (OpE<K::kF16V>)x;
            pp[part][i] = hi;
            x -= (float)hi;
        }
    }
    // V rows of masked tokens are zero (stale pages may hold NaN).
    uint32_t vr[8][VW];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) vr[i][w] = kFull || counts.held(i) ? s.v[i][w] : 0u;
    if constexpr (!kFull && Counts::kByRow) {
        if (!products.fits(vr)) {                        // wave-uniform
            products.add(st, weight, live);
            return;
        }
    }
    auto product = [&](OpT<K::kF16V> av, int nb) __attribute__((always_inline)) {
#pragma unroll
        for (int part = 0; part < K::kPParts; ++part) st.o[nb] = mma(av, pp[part], st.o[nb]);
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

// LDS of narrow_run: the waves' scales, then the states that half of them publish.
template <int C, int NW>
struct NarrowLds {
    float4 stage[NW][16];
    float merge[NW / 2][4 * (4 * C) + 2][64];
};

// Q^T operands of the lane's row at src; j: l / 16.
template <int C, int QT, int ES>
__device__ __forceinline__ void load_narrow_q(const typename Elem<QT>::T* src, int D, int j, int q_vec,
                                              OpT<Kinds<QT, ES>::kF16> (&q)[Kinds<QT, ES>::kQParts][2 * C]) {
    using K = Kinds<QT, ES>;
    using T = typename Elem<QT>::T;
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
                q[part][kb][i] = top;
                y = __builtin_isinf(y) ? 0.0f : y - (float)top;      // an infinite q is its first part alone
            }
        }
    }
}

// The states of a head's waves join pairwise in LDS into its first one; waves without a step have nothing. Wave tw of
// per_head of head hw; all waves of the workgroup.
template <int C, int NW>
__device__ __forceinline__ void join_waves(RowState<C>& st, NarrowLds<C, NW>& lds, int tw, int hw, int per_head, int steps, int lane) {
    constexpr int NB = 4 * C;
    for (int half = per_head >> 1; half > 0; half >>= 1) {
        if (half >= steps) continue;                     // the upper half has no step (workgroup-uniform)
        if (tw >= half && tw < 2 * half) {
            float(*mine)[64] = lds.merge[hw * half + tw - half];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[4 * nb + i][lane] = st.o[nb][i];
            mine[4 * NB][lane] = st.m;
            mine[4 * NB + 1][lane] = st.l;
        }
        __syncthreads();
        if (tw < half) {
            const float(*other)[64] = lds.merge[hw * half + tw];
            const float mo = other[4 * NB][lane];
            const float mn = fmaxf(st.m, mo);
            const float mu = mn == kNegInf ? 0.0f : mn;
            const float wa = fast_exp2(st.m - mu), wb = fast_exp2(mo - mu);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 4; ++i) st.o[nb][i] = st.o[nb][i] * wa + other[4 * nb + i][lane] * wb;
            st.l = st.l * wa + other[4 * NB + 1][lane] * wb;
            st.m = mn;
        }
        __syncthreads();
    }
}

// A lane's part of state `at`; l: the sum over the row's lanes.
template <int C>
__device__ __forceinline__ void store_state(const DecodeArgs& d, int64_t at, const RowState<C>& st, float l, int D, int j) {
    constexpr int NB = 4 * C;
    if (j == 0) {
        d.part_m[at] = st.m;
        d.part_l[at] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d0 = NB * (4 * j + i);
        if (d0 >= D) continue;
        float* acc = d.part_acc + at * D + d0;
#pragma unroll
        for (int w = 0; w < NB / 4; ++w)
            reinterpret_cast<float4*>(acc)[w] = make_float4(st.o[4 * w][i], st.o[4 * w + 1][i], st.o[4 * w + 2][i], st.o[4 * w + 3][i]);
    }
}

// The states of an item's pairs, written to part `it.part`. NW waves, all of the workgroup.
template <int C, int QT, int ES, int NW>
__device__ __forceinline__ void narrow_run(const PrefixArgs& a, const PrefixItem& it, int heads, int q_vec, NarrowLds<C, NW>& lds) {
    using K = Kinds<QT, ES>;
    using T = typename Elem<QT>::T;
    constexpr int NB = 4 * C;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int m16 = lane & 15, j = lane >> 4;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int D = a.d.head_dim;
    const int per_head = NW / heads;                     // waves of one KV head (powers of two)
    const int tw = wave & (per_head - 1), hw = (wave - tw) / per_head;
    const int h = it.h + hw;
    const int32_t lo = it.lo, hi = it.hi;

    auto issue = [&](PrefixStep<C, ES>& dst, int32_t t0, TileRef& ra, TileRef& rb) __attribute__((always_inline)) {
        auto ref = [&](int32_t tok) __attribute__((always_inline)) {
            // Wave-uniform scalar load of the table: its wait leaves the loads in flight alone.
            const int64_t addr = uniform64((int64_t)(uintptr_t)(it.table + (tok >> a.d.bs_shift)));
            const int64_t phys = *(const_i32_ptr)(uintptr_t)addr;
            const bool ok = phys >= 0 && phys < a.d.num_blocks;
            return TileRef{ok ? phys * a.d.block_size + (tok & (a.d.block_size - 1)) : 0, ok};
        };
        ra = ref(t0);
        rb = t0 + 16 < hi ? ref(t0 + 16) : TileRef{0, 0};
        load_prefix_step<C, ES>(dst, a.d, h, ra, rb, lane);
    };
    PrefixStep<C, ES> buf0, buf1;
    TileRef r0a, r0b, r1a, r1b;
    const int32_t stride = 32 * per_head;
    int32_t tok = lo + 32 * tw;
    if (tok < hi) issue(buf0, tok, r0a, r0b);

    // Q^T operands: column l % 16 is pair r0 + l % 16 (those past the last repeat it).
    OpT<K::kF16> q[K::kQParts][2 * C];
    {
        const int32_t pair = min(it.r0 + m16, it.pairs - 1);
        const int32_t t = (uint32_t)pair / (uint32_t)G;
        load_narrow_q<C, QT, ES>(reinterpret_cast<const T*>(a.d.q) + (int64_t)(it.rs + t) * a.d.q_stride_b +
                                     (h * G + (pair - t * G)) * a.d.q_stride_h, D, j, q_vec, q);
    }

    RowState<C> st;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) st.o[nb] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    st.m = kNegInf;
    st.l = 0.0f;
    auto compute = [&](const PrefixStep<C, ES>& cur, int32_t t0, const TileRef& ra, const TileRef& rb) __attribute__((always_inline)) {
        const int lim_a = ra.valid ? min(16, hi - t0) : 0;
        const int lim_b = rb.valid ? min(16, hi - t0 - 16) : 0;
        const FirstTokens counts{j, lim_a, lim_b};
        if (lim_a + lim_b == 32) prefix_step<C, QT, ES, true>(st, cur, q, lds.stage[wave], lane, counts, a.d.score_scale);
        else prefix_step<C, QT, ES, false>(st, cur, q, lds.stage[wave], lane, counts, a.d.score_scale);
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

    join_waves<C, NW>(st, lds, tw, hw, per_head, (hi - lo + 31) >> 5, lane);
    if (tw != 0) return;
    const float l = sum_across_rows(st.l);
    const int32_t pair = it.r0 + m16;
    if (pair >= it.pairs) return;
    const int32_t t = (uint32_t)pair / (uint32_t)G;
    const int hq = h * G + (pair - t * G);
    const int64_t pi = prefix_part(a, it.rs + t, it.part, hq);
    store_state<C>(a.d, pi, st, l, D, j);
}

}  // namespace

}  // namespace kvfp8
