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
    const bf16_t* xp;                        // x in operand order (pack_x_kernel), for more than 16 rows
};

// y[m][n] from the definition, in 64 bits: for an output whose sums over the bare codes came out infinite or NaN.  sum q x and z sum x both pass the range where
// sum (q - z) x need not (an infinity in x has the sign of q - z, not inf - inf; 15 x overflows before s (q - z) x does).  Looking for such an output costs 0.1 us of
// 1 x 4096 x 4096 (4.4 -> 4.5) and 0.15 of 48 x 12288 x 4096 (16.8 -> 16.95).
// Computing one takes a lane 130 us at K = 4096 (all 12288 x 48, an infinity in every row: 2 ms); a sequence that has become NaN takes nothing (its first step ends it).
__device__ float q4_define(const Q4Params& p, int m, int n) {
    double y = 0;
    const uint8_t* row = p.codes + n * p.ldc;
    const bf16_t* x = p.x + m * p.ldx;
#pragma unroll 1
    for (int k = 0; k < p.K && y == y; k += 8) {
        const int g = k >> p.gshift;
        const uint32_t w = *(const uint32_t*)(row + k / 2);
        const bf16x8 v = *(const bf16x8*)(x + k);
        const double s = (double)(float)p.scales[n * p.lds + g];
        const int z = p.zeros ? p.zeros[n * p.ldz + g] : 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) y = fma(s * (double)((int)((w >> (4 * j)) & 15u) - z), (double)(float)v[j], y);
    }
    return (float)y;
}

__device__ __forceinline__ void q4_store(const Q4Params& p, int m, int n, float y) {
    if (p.bias) y += (float)p.bias[n];
    if (p.residual) y += (float)p.residual[m * p.ldr + n];
    if (p.out_f32) ((float*)p.out)[m * p.ldo + n] = y;
    else ((bf16_t*)p.out)[m * p.ldo + n] = (bf16_t)y;
}

typedef uint32_t u32_u2 __attribute__((aligned(2)));
typedef uint32_t u32x2_u2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_u2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32_u __attribute__((aligned(1)));
typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(1)));
typedef uint16_t u16_u __attribute__((aligned(1)));

constexpr int kQ4Block = 128;                    // columns of K that a wave takes at a time: 16 bytes of codes per lane

// 8 codes of a word as 16-bit floats in column order.  A byte 0 .. 15 read as OCP e4m3 is its 2^-9 th part, exactly (the subnormals and the first binade of the
// format have one spacing), and the conversion multiplies by its scale operand: 0.5 instructions per code, none for an offset.
__device__ __forceinline__ bf16x8 q4_codes(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    const uint32_t a = __builtin_amdgcn_perm(hi, lo, 0x05010400u), b = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
#if MC_STORAGE_IS_F16
    const u32x4 o = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 512.f, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 512.f, true))};
#else
    const u32x4 o = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.f, true)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.f, false)), __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.f, true))};
#endif
    return __builtin_bit_cast(bf16x8, o);
}

__device__ __forceinline__ float q4_scale(uint32_t bits) { return (float)__builtin_bit_cast(bf16_t, (uint16_t)bits); }

// y[m][n] = sum over the groups g of s[n][g] (sum_k q[n][k] x[m][k] - z[n][g] sum_k x[m][k]), the inner sums on the matrix cores with the codes as exact integers: the
// products are exact, the zero point is taken out of a sum of the same size (the codes reach 15, not 128 as with a biased exponent trick, so little is lost), the scale
// is applied once per group in fp32.  sum_k x comes from the same instruction against a column of ones.
//
// A workgroup owns R blocks of 16 output columns over the whole of K; its W waves split K into contiguous chunks of 128-column blocks (a function of K and N), each wave
// runs one chain in ascending k, the W chains are added in a fixed order: a row's bits depend neither on M nor on R.  Codes go from memory to registers once: 16 bytes
// per lane, rows of 64 bytes side by side (consecutive rows of a row-major weight are one stream), a 4 x 4 transpose of words over the lane quarters
// (v_permlane32_swap, v_permlane16_swap) turns them into the operands of four consecutive 32-column products.  x comes from the L2, once per workgroup (over 16 rows in operand order: q4_pack_x_kernel).
// Scales and zero points of 8 blocks are read at once, two blocks' per lane quarter, and handed round by ds_bpermute: a load of two bytes from each of 16 rows
// costs the memory pipeline as much as 1 KiB of codes (8 x 32000 x 4096, groups of 64: 36 us with a scale and a zero load per block, 31 so,
// the rest of the kernel being the same).
template <int W, int MB, int R, int U, int UX, int GS, bool ZP>
__global__ __launch_bounds__(W * 64) void linear_q4_kernel(Q4Params p) {
    constexpr int NG = 128 >> GS;                // groups per block
    constexpr int H = W / 2;
    __shared__ __attribute__((aligned(16))) float red[H][R * MB][64][4];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int blocks = (p.K + kQ4Block - 1) / kQ4Block, per = blocks / W, extra = blocks % W;
    const int first = wave * per + min(wave, extra), count = per + (wave < extra ? 1 : 0);
    const int tiles = (p.N + 15) >> 4;

    const uint8_t* wrow[R]; const uint8_t* zrow[R]; const bf16_t* srow[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t n = min(min((int)blockIdx.x * R + r, tiles - 1) * 16 + c, p.N - 1);
        wrow[r] = p.codes + n * p.ldc;
        srow[r] = p.scales + n * p.lds;
        zrow[r] = p.zeros + n * p.ldz;
    }
    const bf16_t* xrow = MB > 1 ? p.xp + lane * 8 : p.x + (int64_t)min(c, p.M - 1) * p.ldx + 8 * g;

    u32x4 wq[U][R];
    bf16x8 xq[UX][MB][4];
    // i: block of the chunk; past its end the last block is read again (and its scales are dropped).  The last block of K may be short (K % 128 = 32, 64 or 96): its
    // missing pieces are whole groups (K is a multiple of the group), are read from inside the row and have the scale 0.  No branches: they would cost the
    // loads their order.
    auto load_w = [&](int u, int i) {
        const int k = (first + min(i, count - 1)) * kQ4Block, last = ((p.K - k) >> 5) - 1;      // last: index of the last piece of 32 columns
#pragma unroll
        for (int r = 0; r < R; ++r) wq[u][r] = *(const u32x4*)(wrow[r] + (k >> 1) + 16 * min(g, last));      // (cached: half a line now, half with the next block)
    };
    // scales and zero points of blocks 8 t .. 8 t + 7 of the chunk: quarter g holds those of blocks 8 t + 2 g and the next, 2 NG of them
    constexpr int ZW = NG == 4 ? 2 : 1;
    struct Scales { uint32_t s[R][NG], z[R][ZW]; };
    const int groups = p.K >> GS;
    auto load_s = [&](Scales& o, int t) {
        const int q0 = (first + 8 * t + 2 * g) * NG;
        if ((first + 8 * t + 8) * NG <= groups) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const bf16_t* s = srow[r] + q0;
                const uint8_t* z = zrow[r] + q0;
                if constexpr (NG == 1) { o.s[r][0] = *(const u32_u2*)s; if (ZP) o.z[r][0] = *(const u16_u*)z; }
                else if constexpr (NG == 2) { const u32x2 v = *(const u32x2_u2*)s; o.s[r][0] = v[0]; o.s[r][1] = v[1]; if (ZP) o.z[r][0] = *(const u32_u*)z; }
                else {
                    const u32x4 v = *(const u32x4_u2*)s;
#pragma unroll
                    for (int q = 0; q < 4; ++q) o.s[r][q] = v[q];
                    if (ZP) { const u32x2 y = *(const u32x2_u*)z; o.z[r][0] = y[0]; o.z[r][1] = y[1]; }
                }
            }
        } else {                                     // the end of the row: what there is
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int q = 0; q < ZW; ++q) o.z[r][q] = 0;
#pragma unroll
                for (int q = 0; q < 2 * NG; ++q) {
                    const int at = min(q0 + q, groups - 1);
                    const uint32_t v = q0 + q < groups ? *(const uint16_t*)(srow[r] + at) : 0u;
                    if (q & 1) o.s[r][q >> 1] |= v << 16; else o.s[r][q >> 1] = v;
                    if (ZP) o.z[r][q >> 2] |= (uint32_t)zrow[r][at] << (8 * (q & 3));
                }
            }
        }
    };
    auto load_x = [&](int u, int i) {
        const int k = (first + min(i, count - 1)) * kQ4Block;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int kk = min(k + 32 * j, p.K - 32);
#pragma unroll
            for (int b = 0; b < MB; ++b) xq[u][b][j] = *(const bf16x8*)(xrow + (MB > 1 ? ((int64_t)(kk >> 5) * MB + b) * 512 : kk));
        }
    };

    f32x4 acc[R][MB];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[r][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
    bf16x8 ones;
#pragma unroll
    for (int j = 0; j < 8; ++j) ones[j] = (bf16_t)1.f;

    // odd: parity of block i (of the chunk)
    auto use = [&](const Scales& o, int u, int ux, int odd, int i) {
        const int from = 4 * c + 64 * ((i & 7) >> 1);
        uint32_t sv[R][(NG + 1) / 2], zv[R], w[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int q = 0; q < (NG + 1) / 2; ++q) {
                const uint32_t v = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)o.s[r][NG == 1 ? 0 : odd * (NG / 2) + q]);
                sv[r][q] = i < count ? (NG == 1 && odd ? v >> 16 : v) : 0u;
            }
            if (ZP) {
                zv[r] = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)o.z[r][NG == 4 ? odd : 0]);
                if constexpr (NG < 4) { if (odd) zv[r] >>= 8 * NG; }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const auto a = __builtin_amdgcn_permlane32_swap(wq[u][r][0], wq[u][r][2], false, false);
            const auto b = __builtin_amdgcn_permlane32_swap(wq[u][r][1], wq[u][r][3], false, false);
            const auto d = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
            const auto e = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
            w[r][0] = d[0]; w[r][1] = d[1]; w[r][2] = e[0]; w[r][3] = e[1];
        }
        constexpr int JG = 4 / NG;               // products per group
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            f32x4 sx[MB], pr[R][MB];
#pragma unroll
            for (int b = 0; b < MB; ++b) sx[b] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int b = 0; b < MB; ++b) pr[r][b] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = q * JG; j < (q + 1) * JG; ++j) {
#pragma unroll
                for (int b = 0; b < MB; ++b) sx[b] = mc_mfma_16x16x32(xq[ux][b][j], ones, sx[b]);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const bf16x8 wf = q4_codes(w[r][j]);
#pragma unroll
                    for (int b = 0; b < MB; ++b) pr[r][b] = mc_mfma_16x16x32(xq[ux][b][j], wf, pr[r][b]);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float s = q4_scale(q & 1 ? sv[r][q >> 1] >> 16 : sv[r][q >> 1]), z = ZP ? (float)((zv[r] >> (8 * q)) & 255u) : 8.f;
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[r][b][t] = fmaf(s, fmaf(-z, sx[b][t], pr[r][b][t]), acc[r][b][t]);
            }
            if constexpr (NG > 1) __builtin_amdgcn_sched_barrier(0);               // (groups interleaved by the scheduler spill)
        }
    };
    if (count > 0) {
        Scales cur, nxt;
        load_s(cur, 0);
#pragma unroll
        for (int u = 0; u < U; ++u) load_w(u, u);
#pragma unroll
        for (int u = 0; u < UX; ++u) load_x(u, u);
        if (8 < count) load_s(nxt, 1);
        int i = 0;
        auto turn = [&] {                        // every 8 blocks the next scales
            if (i && !(i & 7)) {
                cur = nxt;
                if (i + 8 < count) load_s(nxt, (i >> 3) + 1);
            }
        };
        for (; i + U < count; i += U) {          // (U divides 8)
            turn();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                use(cur, u, u % UX, u & 1, i + u);
                load_w(u, i + U + u);
                load_x(u % UX, i + u + UX);
            }
        }
        turn();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            use(cur, u, u % UX, u & 1, i + u);
            if (u + UX < U) load_x(u % UX, i + u + UX);
        }
    }

    // the W chains: (w + (w + W / 2)) for the lower half, then those in order
    if (wave >= H) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int b = 0; b < MB; ++b) *(f32x4*)&red[wave - H][r * MB + b][lane][0] = acc[r][b];
    }
    __syncthreads();
    if (wave < H) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int b = 0; b < MB; ++b) {       // (slot `wave` is read and rewritten by this wave only)
                acc[r][b] += *(f32x4*)&red[wave][r * MB + b][lane][0];
                *(f32x4*)&red[wave][r * MB + b][lane][0] = acc[r][b];
            }
    }
    __syncthreads();
    for (int q = wave; q < R * MB; q += W) {
        const int r = q / MB, b = q % MB;
        f32x4 v = *(f32x4*)&red[0][q][lane][0];
#pragma unroll
        for (int w = 1; w < H; ++w) v += *(f32x4*)&red[w][q][lane][0];
        const int n = (blockIdx.x * R + r) * 16 + c, m0 = b * 16 + 4 * g;
        if (n >= p.N) continue;
        if (!(fabsf(v[0]) < INFINITY && fabsf(v[1]) < INFINITY && fabsf(v[2]) < INFINITY && fabsf(v[3]) < INFINITY)) {
#pragma unroll 1
            for (int t = 0; t < 4; ++t) {
                float y = t == 0 ? v[0] : t == 1 ? v[1] : t == 2 ? v[2] : v[3];
                if (fabsf(y) < INFINITY || m0 + t >= p.M) continue;
                y = q4_define(p, m0 + t, n);
                v[0] = t == 0 ? y : v[0]; v[1] = t == 1 ? y : v[1]; v[2] = t == 2 ? y : v[2]; v[3] = t == 3 ? y : v[3];
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (m0 + t < p.M) q4_store(p, m0 + t, n, v[t]);
    }
}

// x [M, K] in operand order, [K / 32][MB][64 lanes][8], rows from M on zero: the rows of x lie a power of two apart as a rule, and the 16 rows of an operand, read by every
// workgroup at once, then come from few channels of the L2
__global__ __launch_bounds__(256) void q4_pack_x_kernel(const bf16_t* x, int64_t ldx, bf16_t* xp, int M, int K, int mb) {
    const int i = blockIdx.x * 256 + threadIdx.x, lane = i & 63, f = i >> 6, kb = f / mb, b = f % mb;
    if (kb * 32 >= K) return;
    const int m = b * 16 + (lane & 15);
    bf16x8 v = {};
    if (m < M) v = *(const bf16x8*)(x + (int64_t)m * ldx + kb * 32 + 8 * (lane >> 4));
    *(bf16x8*)(xp + (int64_t)i * 8) = v;
}

template <int W, int MB, int R, int U, int UX, int GS>
void q4_launch_z(const Q4Params& p, hipStream_t s) {
    const int grid = ((p.N + 15) / 16 + R - 1) / R;
    if (p.zeros) linear_q4_kernel<W, MB, R, U, UX, GS, true><<<grid, W * 64, 0, s>>>(p);
    else linear_q4_kernel<W, MB, R, U, UX, GS, false><<<grid, W * 64, 0, s>>>(p);
}

template <int W, int MB, int R, int U, int UX>
void q4_launch_g(const Q4Params& p, hipStream_t s) {
    if (p.gshift == 7) q4_launch_z<W, MB, R, U, UX, 7>(p, s);
    else if (p.gshift == 6) q4_launch_z<W, MB, R, U, UX, 6>(p, s);
    else q4_launch_z<W, MB, R, U, UX, 5>(p, s);
}

// Times with weights in turn, none found in the last-level cache, as a decode step meets them (a single 4096 x 4096 weight replayed from it takes 4.9 us instead of 6.6).
// R blocks of 16 columns per workgroup: enough to bring the workgroups down to one per CU, up to 3 (x is read once per workgroup: 48 x 12288 x 4096 takes 24.1 us with R = 1, 21.7
// with 2, 19.2 with 3, 48 x 22016 x 4096 40.8, 31.0 and 27.5; 1 x 4096 x 4096, whose 256 blocks just fill the chip, 6.6, 8.4 and 10.4).  Waves per workgroup, a function of N alone
// because it decides the order of the sums: 8 up to 512 blocks, where longer chains leave the chip idle (48 x 4096 x 11008: 23.7 against 25.8 us, 48 x 4096 x 4096 11.9 against
// 12.4, 1 x 4096 x 4096 either way 6.6), 4 above, where shorter ones spend their time starting and ending (8 x 32000 x 4096: 22.9 against 29.3 us, 48 x 22016 x 4096 27.5 against 31.8;
// 48 x 12288 x 4096, at the border, 19.2 against 18.5).
// Above 16 rows a SIMD has one wave, and its time is its own instructions' and what its loads leave open: of 17 us of 48 x 12288 x 4096 with the weight in the cache the packing of x
// takes 3, the sums over the waves and the stores 2, the loop 8 without any load and 13 with them.  One wave per row block instead (three a SIMD, codes converted three
// times): 22 us; x or codes requested two blocks ahead: 18.
template <int MB>
void q4_launch(const Q4Params& p, hipStream_t s) {
    const int tiles = (p.N + 15) / 16;
    if (tiles <= 256) q4_launch_g<8, MB, 1, 2, 1>(p, s);
    else if (tiles <= 512) q4_launch_g<8, MB, 2, 2, 1>(p, s);
    else q4_launch_g<4, MB, 3, 2, 1>(p, s);
}

// ---- weights ----------------------------------------------------------------------------------------------------------------------
// Codes, scales and zero points of a 16-bit weight: a group of g elements on g / 8 lanes.  Symmetric: scale = st(amax / 7), code = rne(w / scale) + 8;
// with zero points: scale = st((max - min) / 15) over the range widened to hold 0, zero = rne(-min / scale), code = rne(w / scale) + zero; codes
// clamped to 0..15.  Codes come from the scale as it is stored (st = rounded to 16 bits), so the products the kernels form are the nearest ones.  A group that holds
// an infinity or NaN gets the scale NaN: what it multiplies becomes NaN.
__global__ __launch_bounds__(256) void quantize_q4_kernel(const bf16_t* w, int64_t ldw, uint8_t* codes, bf16_t* scales, uint8_t* zeros, int N, int K, int gshift) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = K / 8;      // K / 8 lanes per row; groups never straddle waves (group <= 128: 16 lanes)
    const bool in = i < N * per;
    const int n = in ? (int)(i / per) : 0, k = in ? (int)(i % per) * 8 : 0;
    bf16x8 v = {};
    if (in) v = *(const bf16x8*)(w + n * ldw + k);
    float lo = 0.f, hi = 0.f;
    int odd = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { const float f = (float)v[j]; lo = fminf(lo, f); hi = fmaxf(hi, f); odd |= !(fabsf(f) < INFINITY); }
    for (int o = (1 << gshift) / 16; o > 0; o >>= 1) { lo = fminf(lo, __shfl_xor(lo, o, 64)); hi = fmaxf(hi, __shfl_xor(hi, o, 64)); odd |= __shfl_xor(odd, o, 64); }
    const float range = hi - lo < INFINITY ? (hi - lo) / 15.f : hi / 15.f - lo / 15.f;       // (the largest numbers of both signs: finite all the same)
    const float s = odd ? __uint_as_float(0x7fc00000u) : (float)(bf16_t)(zeros ? range : fmaxf(hi, -lo) / 7.f);
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
    MC_CHECK_ARG(w->N > 0 && w->N <= (1 << 30) && w->K > 0 && w->K <= (1 << 22) && w->K % w->group == 0, "%s: N = %d, K = %d must be positive, K a multiple of the group %d and at most 2^22", who, w->N, w->K, w->group);
    MC_CHECK_ARG((uintptr_t)w->codes % 16 == 0 && w->ldc % 16 == 0 && w->ldc >= w->K / 2, "%s: rows of codes must be 16-byte aligned", who);
    MC_CHECK_ARG((uintptr_t)w->scales % 2 == 0 && w->lds >= w->K / w->group && (!w->zeros || w->ldz >= w->K / w->group), "%s: bad scales or zeros", who);
    return 0;
}

}  // namespace

extern "C" int mc_linear_q4_bf16(const void* x, int64_t ldx, const mc_q4_weight* w, const void* bias, const void* residual, int64_t ldr, void* out, int64_t ldo,
                                 int M, int out_f32, void* workspace, void* stream) {
    if (int e = check_weight(w, "mc_linear_q4_bf16")) return e;
    MC_CHECK_ARG(M >= 0 && M <= 64, "mc_linear_q4_bf16: M = %d rows (at most 64: larger ones take the 16-bit form, mc_dequantize_q4_bf16)", M);
    MC_CHECK_ARG(x && out && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 && (M <= 1 || ldx >= w->K), "mc_linear_q4_bf16: rows of x must be 16-byte aligned");
    MC_CHECK_ARG((uintptr_t)out % (out_f32 ? 4 : 2) == 0 && (M <= 1 || (ldo >= w->N && (!residual || ldr >= w->N))), "mc_linear_q4_bf16: bad output or residual rows");
    if (M == 0) return 0;
    Q4Params p{(const bf16_t*)x, ldx, (const uint8_t*)w->codes, w->ldc, (const bf16_t*)w->scales, w->lds, (const uint8_t*)w->zeros, w->ldz, (const bf16_t*)bias,
               (const bf16_t*)residual, ldr, out, ldo, out_f32, M, w->N, w->K, group_shift(w->group), nullptr};
    hipStream_t s = (hipStream_t)stream;
    const int mb = (M + 15) / 16;
    if (mb > 1) {
        MC_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0, "mc_linear_q4_bf16: more than 16 rows need a workspace of mc_linear_q4_workspace_bytes, 16-byte aligned");
        p.xp = (const bf16_t*)workspace;
        q4_pack_x_kernel<<<(w->K / 32 * mb * 64 + 255) / 256, 256, 0, s>>>(p.x, ldx, (bf16_t*)workspace, M, w->K, mb);
    }
    switch (mb) {
        case 1: q4_launch<1>(p, s); break;
        case 2: q4_launch<2>(p, s); break;
        case 3: q4_launch<3>(p, s); break;
        default: q4_launch<4>(p, s); break;
    }
    MC_CHECK_LAUNCH();
    return 0;
}

extern "C" int mc_linear_q4_workspace_bytes(int M, int K, int64_t* bytes) {
    MC_CHECK_ARG(bytes && M >= 0 && M <= 64 && K > 0 && K <= (1 << 22), "mc_linear_q4_workspace_bytes: bad arguments");
    *bytes = M > 16 ? (int64_t)((M + 15) / 16) * 16 * K * 2 : 0;
    return 0;
}

extern "C" int mc_quantize_q4_bf16(const void* w, int64_t ldw, void* codes, void* scales, void* zeros, int N, int K, int group, void* stream) {
    MC_CHECK_ARG(w && codes && scales, "mc_quantize_q4_bf16: null pointer");
    MC_CHECK_ARG(group_shift(group) >= 0 && N > 0 && N <= (1 << 30) && K > 0 && K <= (1 << 22) && K % group == 0, "mc_quantize_q4_bf16: N = %d, K = %d, group %d (32, 64 or 128, dividing K)", N, K, group);
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
