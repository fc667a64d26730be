// Linears with 4-bit weights: out[M, N] = x[M, K] W^T with W[n][k] = scale[n][k / group] * (code[n][k] - zero[n][k / group]), for the few rows of a
// decode step (the reference's load_4bit keeps the base linears in 4 bits: modelcompose/model/builder.py:30-39, through a third-party CUDA
// library; own layout and arithmetic here).  The codes are two to a byte, k even in the low half, row-major [N, K / 2]; scales 16-bit [N, K / group];
// zeros uint8 [N, K / group] or absent (8).
#include "common.h"

namespace {

struct Q4Params {
    const bf16_t* x; int64_t ldx;
    const uint8_t* codes; int64_t ldc; const bf16_t* scales; int64_t lds; const uint8_t* zeros; int64_t ldz;
    const bf16_t* bias; const bf16_t* residual; int64_t ldr;
    void* out; int64_t ldo; int out_f32;
    int M, N, K, gshift;                     // group = 1 << gshift
};

__device__ __forceinline__ void q4_store(const Q4Params& p, int m, int n, float y) {
    if (p.bias) y += (float)p.bias[n];
    if (p.residual) y += (float)p.residual[m * p.ldr + n];
    if (p.out_f32) ((float*)p.out)[m * p.ldo + n] = y;
    else ((bf16_t*)p.out)[m * p.ldo + n] = (bf16_t)y;
}

// a wave per output column; 8 codes (4 bytes) per lane and step
__global__ __launch_bounds__(256) void linear_q4_kernel(Q4Params p) {
    const int lane = threadIdx.x & 63, n = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= p.N) return;
    for (int m = 0; m < p.M; ++m) {
        float y = 0.f;
        for (int k = lane * 8; k < p.K; k += 512) {
            const uint32_t w = *(const uint32_t*)(p.codes + n * p.ldc + k / 2);
            const int g = k >> p.gshift;
            const float s = (float)p.scales[n * p.lds + g], z = p.zeros ? (float)p.zeros[n * p.ldz + g] : 8.f;
            const bf16x8 x8 = *(const bf16x8*)(p.x + m * p.ldx + k);
            float a = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) a = fmaf((float)((w >> (4 * j)) & 15u) - z, (float)x8[j], a);
            y = fmaf(a, s, y);
        }
        y = wave_sum(y);
        if (lane == 0) q4_store(p, m, n, y);
    }
}

// ---- weights ----------------------------------------------------------------------------------------------------------------------
// Codes, scales and zero points of a 16-bit weight: a group of g elements on g / 8 lanes.  Symmetric: scale = st(amax / 7), code = rne(w / scale) + 8;
// with zero points: scale = st((max - min) / 15) over the range widened to hold 0, zero = rne(-min / scale), code = rne(w / scale) + zero; codes
// clamped to 0..15.  Codes come from the scale as it is stored (st = rounded to 16 bits), so the products the kernels form are the nearest ones.
__global__ __launch_bounds__(256) void quantize_q4_kernel(const bf16_t* w, int64_t ldw, uint8_t* codes, bf16_t* scales, uint8_t* zeros, int N, int K, int gshift) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = K / 8;      // K / 8 lanes per row; groups never straddle waves (group <= 128: 16 lanes)
    const bool in = i < N * per;
    const int n = in ? (int)(i / per) : 0, k = in ? (int)(i % per) * 8 : 0;
    bf16x8 v = {};
    if (in) v = *(const bf16x8*)(w + n * ldw + k);
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) { lo = fminf(lo, (float)v[j]); hi = fmaxf(hi, (float)v[j]); }
    for (int o = (1 << gshift) / 16; o > 0; o >>= 1) { lo = fminf(lo, __shfl_xor(lo, o, 64)); hi = fmaxf(hi, __shfl_xor(hi, o, 64)); }
    const float s = (float)(bf16_t)(zeros ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.f);
    const float z = zeros ? fminf(fmaxf(s > 0.f ? rintf(-lo / s) : 0.f, 0.f), 15.f) : 8.f;
    uint32_t out = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float c = (s > 0.f ? rintf((float)v[j] / s) : 0.f) + z;
        out |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * j);
    }
    if (!in) return;
    *(uint32_t*)(codes + ((int64_t)n * K + k) / 2) = out;
    if ((k & ((1 << gshift) - 1)) == 0) {
        const int64_t g = (int64_t)n * (K >> gshift) + (k >> gshift);
        scales[g] = (bf16_t)s;
        if (zeros) zeros[g] = (uint8_t)z;
    }
}

// the 16-bit packed layout of gemm.hip ([ceil16(N) / 16][ceil64(K) / 32][64 lanes][8], zero padded) of scale * (code - zero), rounded once
__global__ __launch_bounds__(256) void dequantize_q4_kernel(Q4Params p, bf16_t* packed, int kblocks, int64_t total) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int lane = (int)(i & 63);
    const int64_t blk = i >> 6;
    const int n = (int)(blk / kblocks) * 16 + (lane & 15), k = (int)(blk % kblocks) * 32 + (lane >> 4) * 8;
    bf16x8 o = {};
    if (n < p.N && k < p.K) {
        const uint32_t w = *(const uint32_t*)(p.codes + n * p.ldc + k / 2);
        const int g = k >> p.gshift;
        const float s = (float)p.scales[n * p.lds + g], z = p.zeros ? (float)p.zeros[n * p.ldz + g] : 8.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (bf16_t)(((float)((w >> (4 * j)) & 15u) - z) * s);
    }
    *(bf16x8*)(packed + i * 8) = o;
}

int group_shift(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

int check_weight(const mc_q4_weight* w, const char* who) {
    MC_CHECK_ARG(w && w->codes && w->scales, "%s: null weight", who);
    MC_CHECK_ARG(group_shift(w->group) >= 0, "%s: group %d not supported (32, 64 or 128)", who, w->group);
    MC_CHECK_ARG(w->N > 0 && w->K > 0 && w->K % w->group == 0, "%s: N = %d, K = %d must be positive and K a multiple of the group %d", who, w->N, w->K, w->group);
    MC_CHECK_ARG((uintptr_t)w->codes % 16 == 0 && w->ldc % 16 == 0 && w->ldc >= w->K / 2, "%s: rows of codes must be 16-byte aligned", who);
    MC_CHECK_ARG((uintptr_t)w->scales % 2 == 0 && w->lds >= w->K / w->group && (!w->zeros || w->ldz >= w->K / w->group), "%s: bad scales or zeros", who);
    return 0;
}

}  // namespace

extern "C" int mc_linear_q4_bf16(const void* x, int64_t ldx, const mc_q4_weight* w, const void* bias, const void* residual, int64_t ldr, void* out, int64_t ldo,
                                 int M, int out_f32, void* stream) {
    if (int e = check_weight(w, "mc_linear_q4_bf16")) return e;
    MC_CHECK_ARG(M >= 0 && M <= 64, "mc_linear_q4_bf16: M = %d rows (at most 64: larger ones take the 16-bit form, mc_dequantize_q4_bf16)", M);
    MC_CHECK_ARG(x && out && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 && (M <= 1 || ldx >= w->K), "mc_linear_q4_bf16: rows of x must be 16-byte aligned");
    MC_CHECK_ARG((uintptr_t)out % (out_f32 ? 4 : 2) == 0 && (M <= 1 || (ldo >= w->N && (!residual || ldr >= w->N))), "mc_linear_q4_bf16: bad output or residual rows");
    if (M == 0) return 0;
    Q4Params p{(const bf16_t*)x, ldx, (const uint8_t*)w->codes, w->ldc, (const bf16_t*)w->scales, w->lds, (const uint8_t*)w->zeros, w->ldz, (const bf16_t*)bias,
               (const bf16_t*)residual, ldr, out, ldo, out_f32, M, w->N, w->K, group_shift(w->group)};
    linear_q4_kernel<<<(w->N + 3) / 4, 256, 0, (hipStream_t)stream>>>(p);
    MC_CHECK_LAUNCH();
    return 0;
}

extern "C" int mc_quantize_q4_bf16(const void* w, int64_t ldw, void* codes, void* scales, void* zeros, int N, int K, int group, void* stream) {
    MC_CHECK_ARG(w && codes && scales, "mc_quantize_q4_bf16: null pointer");
    MC_CHECK_ARG(group_shift(group) >= 0 && N > 0 && K > 0 && K % group == 0, "mc_quantize_q4_bf16: N = %d, K = %d, group %d (32, 64 or 128, dividing K)", N, K, group);
    MC_CHECK_ARG((uintptr_t)w % 16 == 0 && ldw % 8 == 0 && ldw >= K && (uintptr_t)codes % 16 == 0, "mc_quantize_q4_bf16: rows must be 16-byte aligned");
    const int64_t blocks = ((int64_t)N * (K / 8) + 255) / 256;
    MC_CHECK_ARG(blocks < (1LL << 23), "mc_quantize_q4_bf16: %d x %d is too large for one launch", N, K);
    quantize_q4_kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>((const bf16_t*)w, ldw, (uint8_t*)codes, (bf16_t*)scales, (uint8_t*)zeros, N, K, group_shift(group));
    MC_CHECK_LAUNCH();
    return 0;
}

extern "C" int mc_dequantize_q4_bf16(const mc_q4_weight* w, void* packed, void* stream) {
    if (int e = check_weight(w, "mc_dequantize_q4_bf16")) return e;
    MC_CHECK_ARG(packed && (uintptr_t)packed % 16 == 0, "mc_dequantize_q4_bf16: null or misaligned output");
    Q4Params p{};
    p.codes = (const uint8_t*)w->codes; p.ldc = w->ldc; p.scales = (const bf16_t*)w->scales; p.lds = w->lds; p.zeros = (const uint8_t*)w->zeros; p.ldz = w->ldz;
    p.N = w->N; p.K = w->K; p.gshift = group_shift(w->group);
    const int kblocks = (w->K + 63) / 64 * 2;
    const int64_t total = (int64_t)((w->N + 15) / 16) * kblocks * 64, blocks = (total + 255) / 256;
    MC_CHECK_ARG(blocks < (1LL << 23), "mc_dequantize_q4_bf16: %d x %d is too large for one launch", w->N, w->K);
    dequantize_q4_kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(p, (bf16_t*)packed, kblocks, total);
    MC_CHECK_LAUNCH();
    return 0;
}
