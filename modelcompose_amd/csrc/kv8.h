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
