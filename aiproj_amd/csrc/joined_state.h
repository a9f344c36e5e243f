// Joining of softmax states (max, sum, weighted values) that several workgroups leave for a row.
#pragma once

#include "kvfp8_decode_common.h"
#include "paged_operands.h"

namespace kvfp8 {

namespace {

constexpr float kLn2 = 0.693147180559945309f;

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

}  // namespace

}  // namespace kvfp8
