// Shared prefixes on the gfx950 matrix cores: the kernel for groups of few rows, the join and the launches.
//
// A call is two launches. The first leaves softmax states: its first workgroups take the prefixes, (row block,
// KV head, split of the prefix) each, the others the sequences' own tokens, (sequence, block of 16 q heads, KV
// heads, split) each. Groups of many rows take blocks of 256 rows (shared_prefix_wide.hip), others
// blocks of 16 (shared_prefix_narrow.h). The second launch joins a row's states.
#include "shared_prefix_narrow.h"

namespace kvfp8 {

namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr int kWaves = 8;

template <int C, int QT, int ES>
__global__ void __launch_bounds__(64 * kWaves)
prefix_narrow_kernel(PrefixArgs a, PrefixGrid grid) {
    __shared__ NarrowLds<C, kWaves> lds;
    PrefixItem it;
    const bool own = (int32_t)blockIdx.x >= grid.prefix_groups;
    if (!(own ? own_item(a, grid, it) : prefix_item(a, grid, 16, it))) return;
    narrow_run<C, QT, ES, kWaves>(a, it, own ? grid.own_heads : 1, grid.q_vec, lds);
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

// Four columns of a softmax state in the making.
struct JoinedState {
    float mr = kNegInf, den = 0.0f;
    float4 num = {0.0f, 0.0f, 0.0f, 0.0f};

    __device__ __forceinline__ void add(float mi, float li, float4 x) {
        const float mn = fmaxf(mr, mi);
        const float mu = mn == kNegInf ? 0.0f : mn;
        const float wa = fast_exp2(mr - mu), wb = fast_exp2(mi - mu);
        num.x = num.x * wa + x.x * wb;
        num.y = num.y * wa + x.y * wb;
        num.z = num.z * wa + x.z * wb;
        num.w = num.w * wa + x.w * wb;
        den = den * wa + li * wb;
        mr = mn;
    }
    // The states of the lanes kLanes apart.
    template <int kLanes>
    __device__ __forceinline__ void across() {
#pragma unroll
        for (int off = kLanes; off < 64; off <<= 1)
            add(__shfl_xor(mr, off), __shfl_xor(den, off),
                make_float4(__shfl_xor(num.x, off), __shfl_xor(num.y, off), __shfl_xor(num.z, off), __shfl_xor(num.w, off)));
    }
    // The row's attention over its prompt, out and *lse; *lse becomes that of both.
    template <int QT>
    __device__ __forceinline__ void with_prompt(const typename Elem<QT>::T* out, float* lse, int lane) {
        add(*lse * kLog2e, 1.0f,
            make_float4(Elem<QT>::load(out[0]), Elem<QT>::load(out[1]), Elem<QT>::load(out[2]), Elem<QT>::load(out[3])));
        __builtin_amdgcn_wave_barrier();                 // every lane has read lse before lane 0 writes it
        if (lane == 0) *lse = ((mr == kNegInf ? 0.0f : mr) + __builtin_log2f(den)) * kLn2;
    }
    template <int QT>
    __device__ __forceinline__ void store(typename Elem<QT>::T* out) const {
        const bool ok = den > 0.0f || den != den;
        const float y[4] = {ok ? num.x / den : 0.0f, ok ? num.y / den : 0.0f, ok ? num.z / den : 0.0f, ok ? num.w / den : 0.0f};
        store_run<QT, 4>(out, y);
    }
};

// One wave per (row, q head) joins the states of its prefix and own tokens, in the prompt form with out and lse
// in place of the latter. Lanes take 16 C float4 columns; 4 / C states are read side by side. Bound by the search for
// the row's group and a chain of three loads where there are few rows (32 x 32 heads: 5.6 us, 16 + 1 states), by the
// states' bytes where there are many (256 x 64 heads, 5 states: 16 us, 2.7 TB/s).
template <int C, int QT, bool kOwn>
__global__ void __launch_bounds__(256)
prefix_join_kernel(PrefixArgs a) {
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
    const int64_t mine = kOwn ? seq_tokens(a.d, row, &slot) : 0;
    // Splits without tokens left no state.
    const int held = split_count(tokens, split_tokens(tokens, a.step_shift, a.splits));
    const int held_own = kOwn ? split_count(mine, split_tokens(mine, 5, a.own_splits)) : 0;
    const int d4 = min(lane % kLanes, D / 4 - 1), po = lane / kLanes;

    JoinedState st;
#pragma unroll 4
    for (int i = po; i < held + held_own; i += kPass) {
        const int64_t pi = prefix_part(a, row, i < held ? i : a.splits + i - held, hq);
        st.add(a.d.part_m[pi], a.d.part_l[pi], reinterpret_cast<const float4*>(a.d.part_acc + pi * D)[d4]);
    }
    st.across<kLanes>();
    if (po != 0 || 4 * (lane % kLanes) >= D) return;
    const int64_t at = unit;
    T* out = reinterpret_cast<T*>(a.d.out) + at * D + 4 * d4;
    if constexpr (!kOwn) st.with_prompt<QT>(out, a.lse + at, lane);
    st.store<QT>(out);
}

// Prompt form: the states of the row blocks that were split at the end, with out and lse. One wave per four
// pairs (often of one row: one search for its sequence). 64 blocks of 256 pairs in four parts, D 128: 16 us (20 with a
// search for every pair).
template <int C, int QT>
__global__ void __launch_bounds__(256)
prefix_tail_kernel(PrefixArgs a, PrefixGrid grid, int rows_per_block) {
    constexpr int kLanes = 16 * C, kPass = 64 / kLanes;
    using T = typename Elem<QT>::T;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int D = a.d.head_dim;
    const uint32_t per_block = (uint32_t)rows_per_block / 16;
    const int32_t tails = grid.per_xcd - grid.tail_from;
    PrefixItem it;
    it.tail = blockIdx.x / per_block;
    const int32_t first_pair = 16 * (int32_t)(blockIdx.x - it.tail * per_block) + 4 * wave;
    const int32_t xcd = (uint32_t)it.tail / (uint32_t)tails, index = xcd * grid.per_xcd + grid.tail_from + (it.tail - xcd * tails);
    int32_t tokens;
    if (index >= grid.total || !find_item(a, grid, rows_per_block, index, 0, it, &tokens)) return;
    const int32_t G = (uint32_t)a.d.num_q_heads / (uint32_t)a.d.num_kv_heads;
    const int held = split_count(tokens, split_tokens(tokens, a.step_shift, grid.tail_splits));
    const int d4 = min(lane % kLanes, D / 4 - 1), po = lane / kLanes;
    int32_t last = -1;
    bool inside = false;
    for (int p = 0; p < 4; ++p) {
        const int32_t pair = it.r0 + first_pair + p;
        if (pair >= it.pairs) return;
        const int32_t t = (uint32_t)pair / (uint32_t)G;
        const int64_t row = it.rs + t;
        if (t != last) inside = seq_of_row(a, row) >= 0;
        last = t;
        if (!inside) continue;
        JoinedState st;
        const int64_t first = ((int64_t)it.tail * rows_per_block + first_pair + p) * grid.tail_splits;
#pragma unroll 4
        for (int i = po; i < held; i += kPass)
            st.add(a.d.part_m[first + i], a.d.part_l[first + i], reinterpret_cast<const float4*>(a.d.part_acc + (first + i) * D)[d4]);
        st.across<kLanes>();
        if (po != 0 || 4 * (lane % kLanes) >= D) continue;
        const int64_t at = row * a.d.num_q_heads + it.h * G + (pair - t * G);
        T* out = reinterpret_cast<T*>(a.d.out) + at * D + 4 * d4;
        st.with_prompt<QT>(out, a.lse + at, lane);
        st.store<QT>(out);
    }
}

// ------------------------------------------------------------------ host

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

template <int C, int QT, int ES>
hipError_t launch_narrow(const PrefixArgs& a, const PrefixGrid& g, hipStream_t s) {
    hipLaunchKernelGGL((prefix_narrow_kernel<C, QT, ES>), dim3((unsigned)(g.prefix_groups + g.own_groups)), dim3(64 * kWaves), 0, s, a, g);
    return hipGetLastError();
}

template <int QT>
hipError_t launch_narrow_kv(const PrefixArgs& a, int kv_dtype, const PrefixGrid& g, hipStream_t s) {
    if (kv_dtype == KVFP8_E4M3FN)
        return a.d.head_dim == 64 ? launch_narrow<1, QT, 1>(a, g, s) : launch_narrow<2, QT, 1>(a, g, s);
    if constexpr (QT != KVFP8_F32)
        return a.d.head_dim == 64 ? launch_narrow<1, QT, 2>(a, g, s) : launch_narrow<2, QT, 2>(a, g, s);
    else return hipErrorInvalidValue;                    // 16-bit caches come with q of their type
}

template <int QT, bool kOwn>
hipError_t launch_join(const PrefixArgs& a, hipStream_t s) {
    const int64_t units = a.rows * a.d.num_q_heads;
    const dim3 grid((unsigned)((units + 3) / 4));
    if (a.d.head_dim == 64) hipLaunchKernelGGL((prefix_join_kernel<1, QT, kOwn>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((prefix_join_kernel<2, QT, kOwn>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

// Pairs of an average group from which blocks of 256 rows are taken, and in block tables that address no more than
// kShortTable tokens. Whole calls of 32 q and 8 KV heads x 128, blocks of 16 against 256 rows, us:
//   pairs x tokens    48 x 1024  14.5  16.4    128 x 1024  16.6  19.7    256 x 1024  19.8  25.0    512 x 1024  29.2  29.1
//                     48 x 4096  16.8  18.3     64 x 4096  20.1  19.0    128 x 4096  26.9  23.6    256 x 4096  39.1  32.2
//                     48 x 16384 30.5  32.0     64 x 16384 42.3  35.0    128 x 16384 68.1  37.9    256 x 16384  117  51.5
// Blocks of 128 rows lay between the two or behind both (64 x 4096 21.3, 128 x 4096 26.1, 128 x 16384 40.5).
// Measured on e4m3 alone, and taken for the other sizes and 16-bit caches too. Lengths and groups are on the device, so
// the rule goes by the block table's width and by the mean over groups: a wide table over short prefixes, or one large
// group among many small ones, gets the slower kind.
constexpr int64_t kWidePairs = 64, kWidePairsShort = 512, kShortTable = 2048;

bool narrow_size(int32_t d) { return d == 80 || d == 96 || d == 112; }

}  // namespace

bool prefix_mfma_supported(int32_t head_dim, int32_t block_size, int q_dtype, int kv_dtype) {
    if (block_size < 16) return false;
    if (kv_dtype == KVFP8_E4M3FN) return head_dim == 64 || head_dim == 128 || narrow_size(head_dim);
    return (head_dim == 64 || head_dim == 128) && (kv_dtype == KVFP8_BF16 || kv_dtype == KVFP8_F16) && q_dtype == kv_dtype;
}

PrefixMfmaPlan prefix_mfma_plan(int64_t rows, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t groups,
                                int64_t bt_width, int32_t block_size, int q_dtype, bool prompt) {
    PrefixMfmaPlan p = {};
    const int64_t cus = device_cus(), heads = num_q_heads / num_kv_heads;
    const int64_t pairs = rows * heads, mean = groups > 0 ? pairs / groups : 0;
    p.rows = q_dtype == KVFP8_F32 || mean < (bt_width * block_size <= kShortTable ? kWidePairsShort : kWidePairs) ? 16 : 256;
    p.step_shift = p.rows == 16 ? 5 : 6;
    // Splits of 128 tokens or more: 540 rows x 1000 tokens of head size 80 in the prompt form 17.9 us against 21.7 with 256,
    // blocks of 16 on 1024 tokens 12.4 against 14.1 (whole call). Blocks of 256 rows beside own tokens of 256: 128 pairs x
    // 4096 tokens 19.8 us, with 128 24.0.
    const int64_t least = prompt || p.rows == 16 ? 128 : 256;
    const int64_t most = bt_width * block_size / least > 0 ? bt_width * block_size / least : 1;
    // Own tokens: 16 q heads of `own_heads` KV heads a workgroup, one wave or more a head, so that no more than half of the
    // CUs are taken where the heads allow it and the prefixes run beside them (24 x 8 KV heads behind 1024 tokens: 14.5 us
    // a call with 96 workgroups, 19.6 with 192); below that the waves of a workgroup serve one head and long contexts
    // are split.
    p.own_heads = 1;
    p.own_splits = 1;
    if (!prompt) {
        p.own_blocks = (int32_t)((heads + 15) / 16);
        const int64_t items = rows * p.own_blocks * num_kv_heads;
        while (p.own_heads < kWaves && num_kv_heads % (2 * p.own_heads) == 0 && items / p.own_heads > cus / 2) p.own_heads *= 2;
        const int64_t wanted = cus / 2 / (items / p.own_heads);
        p.own_splits = (int32_t)(wanted < 1 ? 1 : (wanted < most ? wanted : most));
        p.own_groups = (int32_t)(items / p.own_heads * p.own_splits);
    }
    // Prefixes: the workgroups that are left of one per CU; with more own tokens than fit beside them, all.
    p.blocks = (int32_t)((pairs + (int64_t)groups * (p.rows - 1)) / p.rows);                    // every group's last block may be unfilled
    const int64_t columns = (int64_t)p.blocks * num_kv_heads;
    const int64_t left = p.own_groups <= cus / 2 ? cus - p.own_groups : cus;
    int64_t splits = columns > 0 ? (left + columns / 2) / columns : 1;
    splits = splits < most ? splits : most;
    p.splits = (int32_t)(splits < 1 ? 1 : splits);
    // Prompt form, more row blocks than run at once: an XCD's last ones, which would leave CUs idle, are split into as
    // many parts as end soonest (a part costs its states, about 1/50 of a round).
    p.per_xcd = (int32_t)((columns * p.splits + kXcds - 1) / kXcds);
    p.tail_from = p.per_xcd;
    p.tail_splits = 1;
    const bool in_place = prompt && p.splits == 1 && p.rows > 16;
    const int64_t at_once = cus / kXcds;
    if (in_place && at_once > 0 && p.per_xcd > at_once) {
        const int64_t tail = p.per_xcd % at_once;
        float best = 1.0f;
        for (int parts = 2; tail > 0 && parts <= 8 && parts <= most; ++parts) {
            const float cost = (float)((tail * parts + at_once - 1) / at_once) / parts + 0.02f * parts;
            if (cost < best) {
                best = cost;
                p.tail_from = (int32_t)(p.per_xcd - tail);
                p.tail_splits = parts;
            }
        }
    }
    p.states = in_place ? (int64_t)kXcds * (p.per_xcd - p.tail_from) * p.rows * p.tail_splits : rows * num_q_heads * (p.splits + (prompt ? 0 : p.own_splits));
    p.part_l = (int64_t)align256((size_t)p.states * 4);
    p.part_acc = 2 * p.part_l;
    p.bytes = p.part_acc + (int64_t)align256((size_t)p.states * head_dim * 4);
    return p;
}

template <int QT>
hipError_t launch_prefix_mfma(PrefixArgs a, int kv_dtype, const PrefixMfmaPlan& p, void* workspace, hipStream_t s) {
    char* ws = reinterpret_cast<char*>(workspace);
    a.splits = p.splits;
    a.own_splits = p.own_splits;
    a.step_shift = p.step_shift;
    a.d.part_m = reinterpret_cast<float*>(ws);
    a.d.part_l = reinterpret_cast<float*>(ws + p.part_l);
    a.d.part_acc = reinterpret_cast<float*>(ws + p.part_acc);
    PrefixGrid g;
    const int64_t total = (int64_t)p.blocks * a.d.num_kv_heads * p.splits;
    g.blocks = p.blocks;
    g.total = (int32_t)total;
    g.per_xcd = p.per_xcd;
    g.tail_from = p.tail_from;
    g.tail_splits = p.tail_splits;
    g.prefix_groups = kXcds * (p.tail_from + (p.per_xcd - p.tail_from) * p.tail_splits);
    g.own_groups = p.own_groups;
    g.own_heads = p.own_heads;
    g.own_blocks = p.own_blocks;
    const int64_t q_size = QT == KVFP8_F32 ? 4 : 2;
    g.q_vec = (uintptr_t)a.d.q % 16 == 0 && a.d.q_stride_b * q_size % 16 == 0 && a.d.q_stride_h * q_size % 16 == 0;
    if (g.prefix_groups + g.own_groups > 0) {
        hipError_t err;
        if constexpr (QT == KVFP8_F32) err = launch_narrow_kv<QT>(a, kv_dtype, g, s);
        else err = p.rows > 16 ? launch_prefix_wide<QT>(a, kv_dtype, g, s) : launch_narrow_kv<QT>(a, kv_dtype, g, s);
        if (err != hipSuccess) return err;
    }
    if (a.cu == nullptr) return launch_join<QT, true>(a, s);
    if (p.states == 0) return hipSuccess;
    if (p.tail_splits > 1) {
        const dim3 grid((unsigned)(kXcds * (p.per_xcd - p.tail_from)) * (unsigned)(p.rows / 16));
        if (a.d.head_dim == 64) hipLaunchKernelGGL((prefix_tail_kernel<1, QT>), grid, dim3(256), 0, s, a, g, p.rows);
        else hipLaunchKernelGGL((prefix_tail_kernel<2, QT>), grid, dim3(256), 0, s, a, g, p.rows);
        return hipGetLastError();
    }
    return launch_join<QT, false>(a, s);
}

template hipError_t launch_prefix_mfma<KVFP8_F32>(PrefixArgs, int, const PrefixMfmaPlan&, void*, hipStream_t);
template hipError_t launch_prefix_mfma<KVFP8_F16>(PrefixArgs, int, const PrefixMfmaPlan&, void*, hipStream_t);
template hipError_t launch_prefix_mfma<KVFP8_BF16>(PrefixArgs, int, const PrefixMfmaPlan&, void*, hipStream_t);

}  // namespace kvfp8
