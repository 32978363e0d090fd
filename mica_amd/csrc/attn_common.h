// What the attention kernels share: operand types, the bf16 MFMA, LDS-DMA descriptors and waits.
#pragma once

#include "common.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kBufferFlags = 0x00020000;   // raw buffer, 32-bit data format (gfx9)
constexpr float kLog2e = 1.44269504088896341f;

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

// A V value (bf16 code) that is not finite as the largest finite value of its sign, NaN with the given sign (0 or 0x8000);
// 0 for a finite one.  Times 2^127 and summed by the matrix cores these give +-inf, and, with both signs, NaN.
MICA_DEVICE uint32_t odd_value(uint32_t h, uint32_t nan_sign) {
    if ((h & 0x7f80u) != 0x7f80u) return 0u;
    return 0x7f7fu | ((h & 0x7fu) ? nan_sign : (h & 0x8000u));
}

// A workgroup barrier that waits for nothing else; no access to memory moves across it.
MICA_DEVICE void meet() {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
// A transposing read.  The compiler knows nothing of what the DMA in flight writes, and would let every one of these reads
// wait for all of it, the next tile's too.  `w`, which nothing is accessed through, says that the read meets no unknown
// store; the waits are the loop's own.  (16 x 64 nodes after 4000 keys 97.9 -> 94.5 us, 2 x 32 nodes after 10000 38.3 -> 36.)
MICA_DEVICE s16x4 tr_read(lds_s16x4 *p, lds_void *__restrict w) {
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
    __builtin_assume(w != nullptr);
    return x;
}
// 16 bytes of LDS at address a, likewise.
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
MICA_DEVICE u32x4 lds_read(uint32_t a, lds_void *__restrict w) {
    const u32x4 x = *(lds_u32x4 *)(uintptr_t)a;
    __builtin_assume(w != nullptr);
    return x;
}
