// FP8 paged decode attention on the gfx950 matrix cores: launches (the kernels and their description
// are in decode_mfma_kernels.h).
#include "decode_mfma_kernels.h"

namespace kvfp8 {

namespace {

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int ilog2(int64_t x) {
    int s = 0;
    while ((int64_t)1 << s < x) ++s;
    return s;
}

// Waves that serve distinct KV heads: one per head, up to kMaxWaves.
int waves_for(int32_t num_kv_heads) { return num_kv_heads < kMaxWaves ? num_kv_heads : kMaxWaves; }

// Fewer KV heads than kMaxWaves, dividing it: the plain decode runs kMaxWaves waves per
// workgroup, R = kMaxWaves / heads replicas of each head (kRep), when
//   - the replicas' merge buffer fits in LDS beside the batch-sized tables, and
//   - the batch can give every replica steps: its tile capacity (batch x table width)
//     is at least 2 R tiles per CU. Below that most replicas idle and the 8-wave
//     workgroups measured slower (cfg1: 8.5 against 6.5 us).
// The fused append + decode kernel keeps one wave per head: with the replicas' merge
// it spills registers and measured 1.3-2.7 us slower.
constexpr size_t kMaxGroupLds = 64 * 1024;
template <int C>
constexpr size_t replica_merge_bytes() { return (size_t)(kMaxWaves / 2) * (4 * (4 * C) + 2) * 64 * sizeof(float); }
template <int C>
bool replicated(const DecodeArgs& d, size_t table_lds) {
    if (d.num_kv_heads >= kMaxWaves || kMaxWaves % d.num_kv_heads != 0) return false;
    if (table_lds + replica_merge_bytes<C>() > kMaxGroupLds) return false;
    const int64_t tiles = (int64_t)d.batch * d.bt_width * (d.block_size / 16);
    return tiles >= (int64_t)device_cus() * 2 * (kMaxWaves / d.num_kv_heads);
}

int64_t max_groups(int32_t num_kv_heads) {
    const int per_cu = kWavesPerCu / waves_for(num_kv_heads);
    return (int64_t)device_cus() * (per_cu > 0 ? per_cu : 1);
}

template <int C, int QT, int ES, int kSets, bool kAppend, bool kF16, bool kRep, bool kNarrow, bool kState>
hipError_t launch_w(const MfmaArgs& a, int64_t cap, hipStream_t s, int phases) {
    const int threads = 64 * (kRep ? kMaxWaves : waves_for(a.d.num_kv_heads));
    const size_t lds = (size_t)(2 * a.d.batch + 1) * sizeof(int32_t) + (kRep ? replica_merge_bytes<C>() : 0);
    // Resident workgroups per CU: the register limit, queried once per (device,
    // workgroup size) without dynamic LDS, capped by what the dynamic LDS (batch-sized
    // tables, replica merge buffer; up to 64 KiB) leaves room for. Only a sizing
    // choice: the work split is correct for any grid.
    static int resident[64][kMaxWaves + 1] = {};     // per template instance
    static int lds_per_cu[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    int& per_cu = resident[dev][threads / 64];
    if (per_cu == 0) {
        const void* fn = reinterpret_cast<const void*>(&decode_mfma_kernel<C, QT, ES, kSets, kAppend, kF16, kRep, kNarrow, kState>);
        int n = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, threads, 0) != hipSuccess || n <= 0) n = 1;
        per_cu = n;
    }
    if (lds_per_cu[dev] == 0) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMaxSharedMemoryPerMultiprocessor, dev) != hipSuccess || n <= 0)
            n = 64 * 1024;
        lds_per_cu[dev] = n;
    }
    const int64_t by_lds = (int64_t)lds_per_cu[dev] / (int64_t)(lds + 4096);   // + static LDS
    const int64_t fit = by_lds < per_cu ? by_lds : per_cu;
    int64_t groups = (int64_t)device_cus() * (fit > 0 ? fit : 1);
    groups = groups < cap ? groups : cap;
    if (phases & kPhaseSplit) {
        const hipError_t err =
            launch_timed(decode_mfma_kernel<C, QT, ES, kSets, kAppend, kF16, kRep, kNarrow, kState>,
                         dim3((unsigned)groups), dim3(threads), lds, s, next_kernel_timing(), a);
        if (err != hipSuccess) return err;
    }
    if (kState || !(phases & kPhaseReduce)) return hipSuccess;
    const int64_t pairs = (int64_t)a.d.batch * a.d.num_q_heads;
    if constexpr (kNarrow) {
        const int64_t seq_tiles = a.d.bt_width * (a.d.block_size / 16);
        if (pairs < 4 * (int64_t)device_cus() && seq_tiles > kShareTiles) {
            hipLaunchKernelGGL((combine_mfma_kernel<C, QT, true, true>), dim3((unsigned)pairs), dim3(256), 0, s, a);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((combine_mfma_kernel<C, QT, kNarrow, false>), dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int C, int QT, int ES, int kSets, bool kAppend = false, bool kF16 = false, bool kNarrow = false>
hipError_t launch_c(const MfmaArgs& a, int64_t cap, hipStream_t s, int phases) {
    if constexpr (!kAppend) {
        if (replicated<C>(a.d, (size_t)(2 * a.d.batch + 1) * sizeof(int32_t)))
            return launch_w<C, QT, ES, kSets, kAppend, kF16, true, kNarrow, false>(a, cap, s, phases);
    }
    return launch_w<C, QT, ES, kSets, kAppend, kF16, false, kNarrow, false>(a, cap, s, phases);
}

template <int C, int QT, int ES, int kSets, bool kF16 = false, bool kNarrow = false>
hipError_t launch_states(const MfmaArgs& a, int64_t cap, hipStream_t s) {
    if (replicated<C>(a.d, (size_t)(2 * a.d.batch + 1) * sizeof(int32_t)))
        return launch_w<C, QT, ES, kSets, false, kF16, true, kNarrow, true>(a, cap, s, kPhaseSplit);
    return launch_w<C, QT, ES, kSets, false, kF16, false, kNarrow, true>(a, cap, s, kPhaseSplit);
}

}  // namespace

bool narrow_head(int32_t head_dim) { return head_dim == 80 || head_dim == 96 || head_dim == 112; }

bool mfma_decode_supported(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                           int64_t bt_width, int32_t block_size, int kv_dtype) {
    if (kv_dtype != KVFP8_E4M3FN && kv_dtype != KVFP8_BF16 && kv_dtype != KVFP8_F16) return false;
    if (head_dim != 64 && head_dim != 128 && !(narrow_head(head_dim) && kv_dtype == KVFP8_E4M3FN)) return false;
    if (block_size < 16 || block_size % 16 != 0) return false;
    if (num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 16) return false;
    if (num_kv_heads > kMaxWaves && num_kv_heads % kMaxWaves != 0) return false;
    if (batch <= 0 || batch > kMfmaMaxBatch) return false;
    // Tile indices are int32.
    if ((int64_t)batch * bt_width * (block_size / 16) >= ((int64_t)1 << 31)) return false;
    return true;
}

}  // namespace kvfp8

namespace kvfp8 {

// Workspace layout of the MFMA path: plan [batch + 2] int32, part_m, part_l
// [2 G_max Hq] float, part_acc [2 G_max Hq D] float (each 256-byte aligned).
int64_t mfma_workspace_layout(int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                              int64_t offsets[4]) {
    const int64_t states = 2 * max_groups(num_kv_heads) * num_q_heads;
    int64_t off = 0;
    offsets[0] = off;
    off += (int64_t)align256((size_t)(batch + 2) * sizeof(int32_t));
    offsets[1] = off;
    off += (int64_t)align256((size_t)states * sizeof(float));
    offsets[2] = off;
    off += (int64_t)align256((size_t)states * sizeof(float));
    offsets[3] = off;
    off += (int64_t)align256((size_t)states * head_dim * sizeof(float));
    return off;
}

// The kernel's arguments: the workspace's parts, and how q may be loaded.
MfmaArgs mfma_args(const DecodeArgs& d, int64_t q_size, void* workspace) {
    int64_t off[4];
    mfma_workspace_layout(d.batch, d.num_q_heads, d.num_kv_heads, d.head_dim, off);
    char* ws = reinterpret_cast<char*>(workspace);
    MfmaArgs a = {};
    a.d = d;
    a.tps_shift = ilog2(d.block_size / 16);
    a.plan = reinterpret_cast<int32_t*>(ws + off[0]);
    a.part_m = reinterpret_cast<float*>(ws + off[1]);
    a.part_l = reinterpret_cast<float*>(ws + off[2]);
    a.part_acc = reinterpret_cast<float*>(ws + off[3]);
    a.q_vec = ((uintptr_t)d.q % 16 == 0 && (d.q_stride_b * q_size) % 16 == 0 && (d.q_stride_h * q_size) % 16 == 0) ? 1 : 0;
    return a;
}

template <int QT>
hipError_t launch_mfma_decode(const DecodeArgs& d, int kv_dtype, void* workspace, hipStream_t stream, int phases) {
    const MfmaArgs a = mfma_args(d, QT == KVFP8_F32 ? 4 : 2, workspace);
    const int64_t cap = max_groups(d.num_kv_heads);
    if (narrow_head(d.head_dim)) return launch_c<2, QT, 1, 1, false, false, true>(a, cap, stream, phases);
    if (kv_dtype == KVFP8_BF16)
        return d.head_dim == 64 ? launch_c<1, QT, 2, 1>(a, cap, stream, phases)
                                : launch_c<2, QT, 2, 1>(a, cap, stream, phases);
    if (kv_dtype == KVFP8_F16) {
        // f16 cache with f16 q (the caller checked): f16 operands.
        if constexpr (QT == KVFP8_F16)
            return d.head_dim == 64 ? launch_c<1, QT, 2, 1, false, true>(a, cap, stream, phases)
                                    : launch_c<2, QT, 2, 1, false, true>(a, cap, stream, phases);
        else return hipErrorInvalidValue;
    }
    if (d.new_k != nullptr) {
        // Fused append + decode (e4m3fn only; the caller checked the shape).
        if (d.head_dim == 64) return launch_c<1, QT, 1, 1, true>(a, cap, stream, phases);
        return d.num_q_heads / d.num_kv_heads > 8 ? launch_c<2, QT, 1, 2, true>(a, cap, stream, phases)
                                                   : launch_c<2, QT, 1, 1, true>(a, cap, stream, phases);
    }
    if (d.head_dim == 64) return launch_c<1, QT, 1, 1>(a, cap, stream, phases);
    // Whole-row K layout: q heads 8..15 of a group need the second QK set.
    return d.num_q_heads / d.num_kv_heads > 8 ? launch_c<2, QT, 1, 2>(a, cap, stream, phases)
                                               : launch_c<2, QT, 1, 1>(a, cap, stream, phases);
}

template <int QT>
hipError_t launch_mfma_states(const DecodeArgs& d, int kv_dtype, void* workspace, const DecodeStates& out, hipStream_t stream) {
    MfmaArgs a = mfma_args(d, QT == KVFP8_F32 ? 4 : 2, workspace);
    a.seq_m = out.m;
    a.seq_l = out.l;
    a.seq_acc = out.acc;
    const int64_t cap = max_groups(d.num_kv_heads);
    if (narrow_head(d.head_dim)) return launch_states<2, QT, 1, 1, false, true>(a, cap, stream);
    if (kv_dtype == KVFP8_BF16) {
        if constexpr (QT == KVFP8_BF16)
            return d.head_dim == 64 ? launch_states<1, QT, 2, 1>(a, cap, stream) : launch_states<2, QT, 2, 1>(a, cap, stream);
        else return hipErrorInvalidValue;      // the caller checked: bf16 q
    }
    if (kv_dtype == KVFP8_F16) {
        if constexpr (QT == KVFP8_F16)
            return d.head_dim == 64 ? launch_states<1, QT, 2, 1, true>(a, cap, stream)
                                    : launch_states<2, QT, 2, 1, true>(a, cap, stream);
        else return hipErrorInvalidValue;      // f16 q
    }
    if (d.head_dim == 64) return launch_states<1, QT, 1, 1>(a, cap, stream);
    return d.num_q_heads / d.num_kv_heads > 8 ? launch_states<2, QT, 1, 2>(a, cap, stream)
                                               : launch_states<2, QT, 1, 1>(a, cap, stream);
}

template hipError_t launch_mfma_states<KVFP8_F32>(const DecodeArgs&, int, void*, const DecodeStates&, hipStream_t);
template hipError_t launch_mfma_states<KVFP8_F16>(const DecodeArgs&, int, void*, const DecodeStates&, hipStream_t);
template hipError_t launch_mfma_states<KVFP8_BF16>(const DecodeArgs&, int, void*, const DecodeStates&, hipStream_t);

template hipError_t launch_mfma_decode<KVFP8_F32>(const DecodeArgs&, int, void*, hipStream_t, int);
template hipError_t launch_mfma_decode<KVFP8_F16>(const DecodeArgs&, int, void*, hipStream_t, int);
template hipError_t launch_mfma_decode<KVFP8_BF16>(const DecodeArgs&, int, void*, hipStream_t, int);

}  // namespace kvfp8
