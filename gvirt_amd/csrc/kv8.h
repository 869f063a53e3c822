// Dequantisation of 8-bit cache values, shared by the copy that serves the 16-bit kernels (kv_dequant.hip) and by the
// prefill kernel that reads quantised caches itself (prefill_mfma.hip): the same code, so the two give the same bits. Kernels
// that keep the scales apart (tree_stream.hip, attention_weights.hip) take the values alone.
#pragma once

#include <type_traits>

#include "common.h"

namespace xlite {

__device__ __forceinline__ float clamp_f16(float x) { return fminf(fmaxf(x, -65504.f), 65504.f); }
// the same for queries, whose NaNs stay NaNs
__device__ __forceinline__ float saturate_f16(float x)
{
    return __builtin_elementwise_minimum(__builtin_elementwise_maximum(x, -65504.f), 65504.f);
}

template <typename T, int KVF>
__device__ __forceinline__ uint4 dequant8(const uint2 &raw, float scale)
{
    float x[8];
    if constexpr (KVF == XLITE_HIP_KV_INT8) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int32_t b = static_cast<int8_t>(((j < 4 ? raw.x : raw.y) >> (8 * (j % 4))) & 0xffu);
            x[j] = static_cast<float>(b) * scale;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int w = static_cast<int>(j < 4 ? raw.x : raw.y);
            float f;
            switch (j % 4) {
            case 0: f = __builtin_amdgcn_cvt_f32_fp8(w, 0); break;
            case 1: f = __builtin_amdgcn_cvt_f32_fp8(w, 1); break;
            case 2: f = __builtin_amdgcn_cvt_f32_fp8(w, 2); break;
            default: f = __builtin_amdgcn_cvt_f32_fp8(w, 3); break;
            }
            x[j] = f * scale;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        x[j] = clamp_f16(x[j]);
    }
    return make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
}

// eight bytes as fp16, without their scale: exact (an e4m3 NaN becomes -65504, as above)
template <int KVF>
__device__ __forceinline__ uint4 widen8(const uint2 &raw)
{
    if constexpr (KVF == XLITE_HIP_KV_INT8) {
        // 0x6400 | u is 1024 + u, and u = b + 128
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 bias = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
        auto two = [&](uint32_t u, uint32_t select) {
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, select)) + bias);
        };
        const uint32_t x = raw.x ^ 0x80808080u, y = raw.y ^ 0x80808080u;
        return make_uint4(two(x, 0x04010400u), two(x, 0x04030402u), two(y, 0x04010400u), two(y, 0x04030402u));
    } else {
        return dequant8<FP16, KVF>(raw, 1.0f);
    }
}

// eight 16-bit values (of a query) of storage type FROM as type TO
template <typename FROM, typename TO>
__device__ __forceinline__ uint4 convert8(const uint4 &x)
{
    if constexpr (std::is_same<FROM, TO>::value) {
        return x;
    } else {
        auto one = [](uint32_t w) {
            return TO::pack(saturate_f16(FROM::lo(w)), saturate_f16(FROM::hi(w)));
        };
        return make_uint4(one(x.x), one(x.y), one(x.z), one(x.w));
    }
}

}  // namespace xlite
