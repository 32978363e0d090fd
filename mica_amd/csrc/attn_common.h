// What the attention kernels share: operand types, the bf16 MFMA, LDS-DMA descriptors and waits.
#pragma once

#include "common.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kBufferFlags = 0x00020000;   // raw buffer, 32-bit data format (gfx9)

MICA_DEVICE f32x16 mfma_bf16(const bf16x8 &a, const bf16x8 &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
template <int N>
MICA_DEVICE void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// This wave's LDS accesses have ended.
MICA_DEVICE void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(0xf | (3 << 14) | (7 << 4)); }

// Combine a value with the one held by lane l ^ 32 (v_permlane32_swap: no LDS round trip).  With the
// same register as both operands, the swap leaves (own, other) in lanes 0-31 and (other, own) in lanes
// 32-63, so max and sum come out bit-identical in every lane.
MICA_DEVICE float half_swap_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
MICA_DEVICE float half_swap_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
