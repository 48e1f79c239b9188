// wf_kv.h -- one-byte K/V codes (OCP e4m3fn, int8) to bf16 or f16 in registers, for the attention kernels.
#pragma once
#include "wf_device.h"

namespace wf {

// FP8 (OCP e4m3fn) K/V caches: a fragment is 8 one-byte keys / dims (8 bytes per lane, 512
// contiguous bytes per wave-instruction), widened to bf16 in registers (exact: every e4m3 value is
// a bf16 value). The per-layer scales are folded into the score scale (K) and the partial records
// (V), so the arithmetic after the widening is the bf16 path's.
typedef __bf16 v2bf_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint4 fp8x8_to_bf16(uint2 r) {
    const v2bf_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x, 1.0f, false);
    const v2bf_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.x, 1.0f, true);
    const v2bf_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.y, 1.0f, false);
    const v2bf_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r.y, 1.0f, true);
    return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                      __builtin_bit_cast(uint32_t, d));
}
// int8 K/V caches (the reference's default KVCacheDtype.INT8, kv_cache/kv_cache.py:159-218, with a
// static per-layer scale): a fragment is 8 signed codes (8 bytes per lane), widened exactly -- each
// byte biased to unsigned (xor 0x80), v_cvt_f32_ubyteN, -128, then bf16 (|code| <= 127 is
// exact in bf16). Scales folded like FP8's.
#ifndef WF_I8_PK  // 0: the earlier form (hipcc folds the -128 into an integer subtract: SDWA + v_cvt_f32_i32)
#define WF_I8_PK 1
#endif
__device__ __forceinline__ uint32_t i8x2_to_bf16(uint32_t u, int sh) {
    const float lo = (float)((u >> sh) & 0xffu) - 128.0f, hi = (float)((u >> (sh + 8)) & 0xffu) - 128.0f;
    return pk_bf16(lo, hi);
}
// four biased bytes -> floats (v_cvt_f32_ubyte0..3), -128 on pairs (scalar adds in this build), packed to bf16
__device__ __forceinline__ uint2 i8x4_to_bf16_pk(uint32_t x) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    f2 a = {(float)(x & 0xffu), (float)((x >> 8) & 0xffu)};
    f2 b = {(float)((x >> 16) & 0xffu), (float)(x >> 24)};
    asm volatile("" : "+v"(a), "+v"(b));  // keep the conversions unsigned-byte (no integer -128 fold)
    const f2 m = {-128.f, -128.f};
    a += m;
    b += m;
    return make_uint2(pk_bf16(a.x, a.y), pk_bf16(b.x, b.y));
}
__device__ __forceinline__ uint4 i8x8_to_bf16(uint2 r) {
    const uint32_t x = r.x ^ 0x80808080u, y = r.y ^ 0x80808080u;
    if constexpr (WF_I8_PK) {
        const uint2 lo = i8x4_to_bf16_pk(x), hi = i8x4_to_bf16_pk(y);
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    return make_uint4(i8x2_to_bf16(x, 0), i8x2_to_bf16(x, 16), i8x2_to_bf16(y, 0), i8x2_to_bf16(y, 16));
}

// The same with the byte picked and sign-extended by the conversion itself (one instruction a code, 12 for 8 codes
// with the packing, against 22)
__device__ __forceinline__ uint32_t i8x2_to_bf16_sext(uint32_t u, int sh) {
    return pk_bf16((float)(int8_t)(u >> sh), (float)(int8_t)(u >> (sh + 8)));
}
__device__ __forceinline__ uint4 i8x8_to_bf16_sext(uint2 r) {
    return make_uint4(i8x2_to_bf16_sext(r.x, 0), i8x2_to_bf16_sext(r.x, 16), i8x2_to_bf16_sext(r.y, 0), i8x2_to_bf16_sext(r.y, 16));
}

// The same codes as f16 (exact too). int8: the byte, biased to unsigned, is the mantissa of 1024 + code + 128, a subtraction
// away from the code: 10 instructions for 8 codes.
typedef _Float16 v2h_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t i8x2_to_f16(uint32_t biased, uint32_t sel) {
    const v2h_t h = __builtin_bit_cast(v2h_t, __builtin_amdgcn_perm(0x64646464u, biased, sel));
    return __builtin_bit_cast(uint32_t, h - v2h_t{(_Float16)1152.f, (_Float16)1152.f});
}
__device__ __forceinline__ uint4 i8x8_to_f16(uint2 r) {
    const uint32_t x = r.x ^ 0x80808080u, y = r.y ^ 0x80808080u;
    return make_uint4(i8x2_to_f16(x, 0x04010400u), i8x2_to_f16(x, 0x04030402u), i8x2_to_f16(y, 0x04010400u), i8x2_to_f16(y, 0x04030402u));
}
__device__ __forceinline__ uint4 fp8x8_to_f16(uint2 r) {
    const v2h_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.x, 1.0f, false);
    const v2h_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.x, 1.0f, true);
    const v2h_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.y, 1.0f, false);
    const v2h_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(r.y, 1.0f, true);
    return make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, c),
                      __builtin_bit_cast(uint32_t, d));
}

}  // namespace wf
