// Codes of a cache in 8 bits as values: e4m3 times the power of two that a token's head has, a byte b that stands for 2^(b - 127)
// (255: not a number).  Four significant bits times a power are a value of bfloat16 exactly for b from 3 to 246, of half precision from
// 112 to 134; beyond, the conversion rounds to nearest even, to subnormal numbers and infinities too.
#pragma once

#include "fp8_device.h"
#include "layer_kernels.h"

namespace phyai {

constexpr uint32_t kNanCodes = 0x7F7F7F7Fu;

// Two codes times a power as two values in a word: one instruction, which takes the power from the exponent's bits alone: 0.0 is 2^-127.
template <int TYPE>
__device__ __forceinline__ uint32_t widen2(uint32_t codes, float power, bool upper) {
    if constexpr (TYPE == HEAD_BF16) {
        const auto v = upper ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, power, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, power, false);
        return __builtin_bit_cast(uint32_t, v);
    } else {
        const auto v = upper ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, power, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, power, false);
        return __builtin_bit_cast(uint32_t, v);
    }
}
// Sixteen codes, as two chunks of eight values; of a known power.
template <int TYPE>
__device__ __forceinline__ void widen16(const v4i& codes, uint32_t power, v4i* out) {
    const float by = __uint_as_float(power << 23);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const uint32_t a = (uint32_t)codes[2 * x], b = (uint32_t)codes[2 * x + 1];
        out[x] = v4i{(int)widen2<TYPE>(a, by, false), (int)widen2<TYPE>(a, by, true), (int)widen2<TYPE>(b, by, false), (int)widen2<TYPE>(b, by, true)};
    }
}

}  // namespace phyai
