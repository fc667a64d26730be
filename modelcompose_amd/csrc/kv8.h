// Numbers of the 8-bit KV cache (mc_kv8_cache): formats, conversions and the quantiser, shared by the kernels of kv8.hip.
#pragma once
#include "common.h"

// A cached vector x[0 .. D) of one (sequence, position, key head) is D codes and ONE fp32 scale:
//   amax = max(max |x|, 2^-100), scale = amax * (1 / T), code = rne(x * (T / amax)), value = code * scale     (T: 448 e4m3, 127 int8)
// in fp32, every operation rounded on its own (no contraction), so any IEEE program reproduces the codes bit for bit.  The floor 2^-100 gives zero
// vectors a scale and keeps T / amax finite.  A vector that holds an infinity or NaN is stored as zero codes with a NaN scale: it reads as
// NaN throughout and, because the codes themselves are finite, touches nothing else.
constexpr uint32_t kKv8AmaxFloor = 0x0d800000u;        // bits of 2^-100

template <int FMT>
__device__ __forceinline__ float kv8_top() { return FMT == MC_KV8_E4M3 ? 448.0f : 127.0f; }

struct Kv8Scale { float scale, inv; bool finite; };
// bits: the largest |x| of the vector as a bit pattern (sign bit clear): the order of the patterns is the order of the magnitudes, with NaN on top
template <int FMT>
__device__ __forceinline__ Kv8Scale kv8_scale(uint32_t bits) {
    Kv8Scale r;
    r.finite = bits < 0x7f800000u;
    const float amax = __uint_as_float(bits > kKv8AmaxFloor ? bits : kKv8AmaxFloor);
    r.inv = kv8_top<FMT>() / amax;                                  // IEEE division
    r.scale = r.finite ? amax * (FMT == MC_KV8_E4M3 ? (float)(1.0 / 448.0) : (float)(1.0 / 127.0)) : __uint_as_float(0x7fc00000u);
    return r;
}

// four codes, x0 in the low byte
template <int FMT>
__device__ __forceinline__ uint32_t kv8_pack4(float x0, float x1, float x2, float x3, const Kv8Scale& s) {
    if (!s.finite) return 0u;
    x0 *= s.inv; x1 *= s.inv; x2 *= s.inv; x3 *= s.inv;            // |x| <= T (1 + 2^-22): no code beyond T after rounding
    if constexpr (FMT == MC_KV8_E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, w, true);
    } else {
        const int a = (int)rintf(x0), b = (int)rintf(x1), c = (int)rintf(x2), d = (int)rintf(x3);
        return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
    }
}

// the four values of a word of codes, as exact floats
template <int FMT>
__device__ __forceinline__ void kv8_unpack4(uint32_t w, float (&f)[4]) {
    if constexpr (FMT == MC_KV8_E4M3) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        f[0] = lo[0]; f[1] = lo[1]; f[2] = hi[0]; f[3] = hi[1];
    } else {
        f[0] = (float)(int8_t)(w & 255); f[1] = (float)(int8_t)((w >> 8) & 255); f[2] = (float)(int8_t)((w >> 16) & 255); f[3] = (float)((int32_t)w >> 24);
    }
}

// ---- matrix-instruction operands from codes ------------------------------------------------------------------------------------------
typedef __bf16 kv8_b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 kv8_b16x8 __attribute__((ext_vector_type(8)));        // bfloat16 in both builds: the value operand (below)

// Codes b0, b1 of half HI of a word as one word of two 16-bit floats; every code is exact in bfloat16 and in IEEE half.
template <int FMT, bool F16, bool HI>
__device__ __forceinline__ uint32_t kv8_pair(uint32_t w) {
    if constexpr (FMT == MC_KV8_E4M3) {
        if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
        else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
    } else {
        float a, b;                                                  // the byte is picked and sign-extended by the conversion itself
        if constexpr (HI) {
            asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(a) : "v"(w));
            asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(b) : "v"(w));
        } else {
            asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(a) : "v"(w));
            asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(b) : "v"(w));
        }
        if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
        else return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);      // the high halves: integers below 2^8 end there
    }
}
// the largest / the sum of a value over the lanes lane ^ 16, lane ^ 32, lane ^ 48, in every lane (row swaps instead of LDS shuffles)
__device__ __forceinline__ float kv8_quarters_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float kv8_quarters_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}
// the value of lane ^ 8 (rotation by 8 within each row of 16)
__device__ __forceinline__ float kv8_other_half(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x128, 0xf, 0xf, true));
}
// eight consecutive codes as an operand of the storage element (keys against the queries)
template <int FMT>
__device__ __forceinline__ bf16x8 kv8_row8(uint32_t w0, uint32_t w1) {
    constexpr bool F16 = MC_STORAGE_IS_F16;
    const u32x4 o = {kv8_pair<FMT, F16, false>(w0), kv8_pair<FMT, F16, true>(w0), kv8_pair<FMT, F16, false>(w1), kv8_pair<FMT, F16, true>(w1)};
    return __builtin_bit_cast(bf16x8, o);
}
