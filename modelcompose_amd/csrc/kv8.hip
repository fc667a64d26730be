// 8-bit KV cache: the cache write of a projection's rows (rotation + quantisation), the read-back to 16 bits, and decode attention over the codes.
//
// Same places as the 16-bit forms (rope_kv_kernel, attn_decode_kernel; LlamaAttention.forward, modelcompose/model/language_model/
// multimodal_llama.py:281-312); the reference keeps its cache in 16 bits.  Half the bytes per cached key: a decode step at batch 48 spends most of its
// time reading them.
#include "kv8.h"

#include <type_traits>

namespace {

struct Cache {
    uint8_t* k; float* ks; uint8_t* v; float* vs;
    int64_t sb, sh, st, ssb, ssh;
    int B, Hkv, S;
};

// ---- cache write ------------------------------------------------------------------------------------------------------------------
struct RopeParams {
    const bf16_t* qkv; int64_t ld;
    const int32_t* row_b; const int32_t* row_pos; const int32_t* row_t;
    const float* cosT; const float* sinT; int max_pos;
    bf16_t* q_out; Cache c;
    int M, H, Lq, blocks_per_row;
};

// the 8 elements half a vector away: lane ^ 8 at D = 128 (a rotation of the row of 16 lanes), lane ^ 4 at D = 64
template <int D>
__device__ __forceinline__ bf16x8 kv8_partner(bf16x8 x) {
    u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (uint32_t)(D == 128 ? __builtin_amdgcn_update_dpp(0, (int)w[j], 0x128, 0xf, 0xf, true) : __shfl_xor((int)w[j], 4, 64));
    return __builtin_bit_cast(bf16x8, w);
}

// One vector (a head of q, k or v of one row) per D / 8 lanes, 8 elements in each; a thread takes kRopeVecs vectors, all requested before the first is used.
// HBM-bound: reads the row once, writes q (16 bits) and the codes once.  48 x 2793 rows of 96 heads (ragged, 4.1 GB): 1.02 ms, 1.24 with one vector a thread, 1.06 with three.
constexpr int kRopeVecs = 2;
template <int D, int FMT>
__global__ __launch_bounds__(256) void rope_kv8_kernel(RopeParams p) {
#pragma clang fp contract(off)
    constexpr int LPV = D / 8, VPB = 256 / LPV;
    const int row = blockIdx.x / p.blocks_per_row, nv = p.H + 2 * p.c.Hkv;
    const int vec0 = (blockIdx.x - row * p.blocks_per_row) * (VPB * kRopeVecs) + threadIdx.x / LPV, d = (threadIdx.x % LPV) * 8;
    const int b = p.row_b[row], pos = p.row_pos[row], t = p.row_t[row];
    // rows of no sequence (b < 0: padding), and rows that do not fit the cache, the tables or q_out: nothing is written
    if (b < 0 || b >= p.c.B || pos < 0 || pos >= p.c.S || pos >= p.max_pos || t < 0 || t >= p.Lq) return;
    const bf16_t* x = p.qkv + (int64_t)row * p.ld + d;
    bf16x8 in[kRopeVecs];
#pragma unroll
    for (int r = 0; r < kRopeVecs; ++r) in[r] = *(const bf16x8*)(x + (int64_t)min(vec0 + r * VPB, nv - 1) * D);
    const bool lo = d < D / 2;
    const float* cr = p.cosT + (int64_t)pos * (D / 2) + (lo ? d : d - D / 2);
    const float* sr = p.sinT + (int64_t)pos * (D / 2) + (lo ? d : d - D / 2);
    f32x4 cs[2], sn[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) { cs[h] = *(const f32x4*)(cr + 4 * h); sn[h] = *(const f32x4*)(sr + 4 * h); }
#pragma unroll
    for (int r = 0; r < kRopeVecs; ++r) {
        const int vec = vec0 + r * VPB;
        const bf16x8 other = kv8_partner<D>(in[r]);             // (before any lane leaves)
        if (vec >= nv) continue;                                // (whole groups of LPV lanes: the shuffles below stay inside a group)
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (float)in[r][j];
        if (vec < p.H) {                                        // the bits of the 16-bit path's queries (mc_rope_pair)
            bf16x8 o;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float z = (float)other[j];
                float o1, o2;
                mc_rope_pair(lo ? y[j] : z, lo ? z : y[j], cs[j >> 2][j & 3], sn[j >> 2][j & 3], o1, o2);
                o[j] = (bf16_t)(lo ? o1 : o2);
            }
            *(bf16x8*)(p.q_out + ((int64_t)b * p.Lq + t) * p.H * D + vec * D + d) = o;
            continue;
        }
        // keys go from fp32 straight to codes: one rounding, not a 16-bit one first; products and sum rounded on their own
        const bool is_k = vec < p.H + p.c.Hkv;
        if (is_k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float u = y[j] * cs[j >> 2][j & 3], w = (float)other[j] * sn[j >> 2][j & 3];
                y[j] = lo ? u - w : u + w;
            }
        }
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = LPV / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
        const Kv8Scale s = kv8_scale<FMT>(m);
        const int hk = vec - p.H - (is_k ? 0 : p.c.Hkv);
        const u32x2 codes = {kv8_pack4<FMT>(y[0], y[1], y[2], y[3], s), kv8_pack4<FMT>(y[4], y[5], y[6], y[7], s)};
        *(u32x2*)((is_k ? p.c.k : p.c.v) + b * p.c.sb + hk * p.c.sh + pos * p.c.st + d) = codes;
        if (d == 0) (is_k ? p.c.ks : p.c.vs)[b * p.c.ssb + hk * p.c.ssh + pos] = s.scale;
    }
}

// ---- read-back --------------------------------------------------------------------------------------------------------------------
// k_out / v_out [B, Hkv, n, D] = code * scale, zero rows from kv_lens[b] on.  A lane takes 8 codes (8 bytes in, 16 out).
template <int D, int FMT>
__global__ __launch_bounds__(256) void kv8_read_kernel(Cache c, const int32_t* kv_lens, int n, bf16_t* k_out, bf16_t* v_out) {
    const int64_t per = (int64_t)n * (D / 8);
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= per) return;
    const int pos = (int)(i / (D / 8)), d = (int)(i % (D / 8)) * 8;
    for (int bh = blockIdx.y; bh < c.B * c.Hkv; bh += gridDim.y) {
        const int b = bh / c.Hkv, hk = bh % c.Hkv;
        const bool in = !kv_lens || pos < kv_lens[b];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            bf16x8 o = {};
            if (in) {
                const u32x2 w = *(const u32x2*)((kv ? c.v : c.k) + b * c.sb + hk * c.sh + pos * c.st + d);
                const float s = (kv ? c.vs : c.ks)[b * c.ssb + hk * c.ssh + pos];
                float f[4];
                kv8_unpack4<FMT>(w[0], f);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = (bf16_t)fp32_first(f[j] * s);
                kv8_unpack4<FMT>(w[1], f);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[4 + j] = (bf16_t)fp32_first(f[j] * s);
            }
            *(bf16x8*)((kv ? v_out : k_out) + ((int64_t)bh * n + pos) * D + d) = o;
        }
    }
}

// ---- decode attention -------------------------------------------------------------------------------------------------------------
struct AttnParams8 {
    const bf16_t* q; int64_t q_sb, q_sh;           // query heads (rotated), or with `cosT` the pre-rotary rows q | k | v of the step's tokens (q_sb their stride)
    Cache c;
    bf16_t* o; int64_t o_sb;
    float* ws;                                     // [B][H][ws_chunks][D + 4] partials: acc[D], m, l, -, -
    const int32_t* kv_lens; const uint8_t* key_valid; int64_t kv_stride;
    const float* cosT; const float* sinT; int max_pos;
    int H, G, groups, ws_chunks, self_combine;     // G = H / Hkv query heads per key head, in `groups` groups of at most 8
    float scale_log2e;
};

// number of keys; with an append, lengths that could not be appended count as none
__device__ __forceinline__ int attn8_len(const AttnParams8& p, int b) {
    const int n = p.kv_lens ? p.kv_lens[b] : p.c.S;
    if (p.cosT && (n > p.c.S || n > p.max_pos)) return 0;
    return max(0, min(n, p.c.S));
}

// Keys of one partial: a function of the sequence's own length, so that short sequences still spread over many workgroups (1 x 2809 keys: 12.6 us with 512, 17.3 with 1024;
// 48 x 2809, where it does not matter, 146 and 144) and long ones are not ground into partials (8 x 32768 keys: 97 us with 512, 92 with 2048).
__host__ __device__ inline int attn8_chunk(int n) { return n <= 4096 ? 512 : n <= 16384 ? 1024 : 2048; }
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(1)));

// The partials (acc[D], m, l) of one head -> its output row, by a workgroup of 256.  In batches of up to 256: the batch's weights exp2(m - running maximum) are
// computed by one thread each and kept in LDS; thread (s, d) adds the partials s, s + 256 / D, .. of element d; the 256 / D sums are added in order.
template <int D>
__device__ __forceinline__ void attn8_join(const float* parts, int np, bf16_t* o, float* lds) {
#pragma clang fp contract(off)
    constexpr int SEG = 256 / D;
    const int tid = threadIdx.x, d = tid % D, sg = tid / D;
    float top = -INFINITY, ll = 0.f, aa = 0.f;         // ll: this thread's share of the sum
    for (int c0 = 0; c0 < np; c0 += 256) {
        const int cn = min(256, np - c0);
        const float* batch = parts + (int64_t)c0 * (D + 4);
        float m = -INFINITY, l = 0.f;
        if (tid < cn) { m = batch[(int64_t)tid * (D + 4) + D]; l = batch[(int64_t)tid * (D + 4) + D + 1]; }
        const float wm = wave_max(m);
        __syncthreads();
        if ((tid & 63) == 0) lds[256 + (tid >> 6)] = wm;
        __syncthreads();
        float mn = top;
#pragma unroll
        for (int w = 0; w < 4; ++w) mn = fmaxf(mn, lds[256 + w]);
        const float base = mn == -INFINITY ? 0.f : mn;      // nothing attended yet, or nothing but NaN
        const float a = __builtin_amdgcn_exp2f(m - base), old = __builtin_amdgcn_exp2f(top - base);
        top = mn;
        lds[tid] = a;
        ll = fmaf(l, a, ll * old);
        aa *= old;
        __syncthreads();
        int c = sg;
        for (; c + 7 * SEG < cn; c += 8 * SEG) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = batch[(int64_t)(c + j * SEG) * (D + 4) + d];
#pragma unroll
            for (int j = 0; j < 8; ++j) aa = fmaf(x[j], lds[c + j * SEG], aa);
        }
        for (; c < cn; c += SEG) aa = fmaf(batch[(int64_t)c * (D + 4) + d], lds[c], aa);
    }
    ll = wave_sum(ll);
    __syncthreads();
    if ((tid & 63) == 0) lds[256 + (tid >> 6)] = ll;
    lds[tid] = aa;
    __syncthreads();
    if (!sg) {
        ll = (lds[256] + lds[257]) + (lds[258] + lds[259]);
#pragma unroll
        for (int s = 1; s < SEG; ++s) aa += lds[s * D + d];
        o[d] = (bf16_t)(ll == 0.f ? 0.f : aa / ll);
    }
    __syncthreads();                                       // (the next head's join reuses lds)
}

// the step's token: its key rotated and its key and value quantised to position pos by the first 2 D / 8 lanes of a wave (rope_kv8_kernel's arithmetic)
template <int D, int FMT>
__device__ __forceinline__ void attn8_append(const AttnParams8& p, int b, int hk, int pos, int lane) {
#pragma clang fp contract(off)
    constexpr int LPV = D / 8;
    const bool is_v = lane >= LPV, on = lane < 2 * LPV;
    const int i4 = (lane % LPV) * 4;
    const bf16_t* x = p.q + (int64_t)b * p.q_sb + (int64_t)(p.H + hk + (is_v ? p.c.Hkv : 0)) * D + i4;
    float a[4] = {}, bb[4] = {};
    if (on) {
        const bf16x4 xa = *(const bf16x4*)x, xb = *(const bf16x4*)(x + D / 2);
        const f32x4 cs = *(const f32x4*)(p.cosT + (int64_t)pos * (D / 2) + i4), sn = *(const f32x4*)(p.sinT + (int64_t)pos * (D / 2) + i4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = (float)xa[j]; bb[j] = (float)xb[j];
            if (!is_v) {
                const float u = a[j] * cs[j], w = bb[j] * sn[j], y = bb[j] * cs[j], z = a[j] * sn[j];
                a[j] = u - w;
                bb[j] = y + z;
            }
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, max(__float_as_uint(a[j]) & 0x7fffffffu, __float_as_uint(bb[j]) & 0x7fffffffu));
#pragma unroll
    for (int o = LPV / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    if (!on) return;
    const Kv8Scale s = kv8_scale<FMT>(m);
    uint8_t* dst = (is_v ? p.c.v : p.c.k) + b * p.c.sb + hk * p.c.sh + pos * p.c.st + i4;
    *(uint32_t*)dst = kv8_pack4<FMT>(a[0], a[1], a[2], a[3], s);
    *(uint32_t*)(dst + D / 2) = kv8_pack4<FMT>(bb[0], bb[1], bb[2], bb[3], s);
    if (i4 == 0) (is_v ? p.c.vs : p.c.ks)[b * p.c.ssb + hk * p.c.ssh + pos] = s.scale;
}

// Decode attention on the matrix cores, for up to 8 query heads that share a key head.
//
// S^T = K Q^T: the keys are the rows (A operand, codes widened to 16 bits, exact), the heads the columns.  Of the 16 columns, column c and column c + 8 are
// the same head; with row r of half t standing for key 8 (r >> 2) + 4 t + (r & 3), lane (c, g) ends up with the scores of keys 8 g .. 8 g + 7 of head
// c & 7 - exactly the layout in which the next product O^T = V^T P^T wants its B operand, so the probabilities never leave the lane.  They
// enter that product as bfloat16, whose 8 significant bits are three parts of the fp32 weight w = p * v_scale = hi + mid + low, exactly: hi in columns 0 .. 7 and mid in columns
// 8 .. 15 of one operand, low in columns 0 .. 7 of a second (bfloat16 also in the half-precision build: w has a wide range).  Of
// the 16-bit outputs of 48 x 2809 keys 0.6 in a thousand are not the rounded exact value (the same in fp32 in torch: 1.3); with two parts, off by 2^-17, it was 2.5, in
// 144.0 us where three take 145.5 (1 x 2809: 12.4 against 12.6).
// V^T's operand needs 8 keys of one element per lane: the bytes of two keys' rows are paired by v_perm.
//
// A workgroup of 4 waves takes chunks (attn8_chunk keys) blockIdx.y, + gridDim.y, ..; wave w the 32-key tiles w, w + 4, .. of a chunk, from a fresh (m, l, acc); the
// waves are joined through LDS in wave order, the chunks by attn8_join in chunk order.  Which workgroup takes which chunk changes no bit.
//
// HBM-bound with many sequences: 48 x 2809 keys, 32 heads, D = 128 146 us = 5.7 TB/s (a kernel on the vector units, one head per workgroup: 157; the same loads
// without the arithmetic: 138); 8 x 32768 keys, 32 heads over 8 92 us = 4.3 TB/s (757).  Latency-bound with few: 1 x 2809 keys 13 us, 3.8 of them the join.
// Three waves per SIMD at D = 128 (168 registers): with two 162 us, with four the tile spills (229).
template <int D, int FMT, bool KM>
__global__ __launch_bounds__(256, D == 128 ? 3 : 4) void attn_decode8_kernel(AttnParams8 p) {
    // (a score and the maximum taken from it have to be the same number: fused into the difference, the score's product would not be rounded, and at 1e30 the
    // two no longer cancel)
#pragma clang fp contract(off)
    constexpr int NU = D / 64, NT = D / 16;
    __shared__ __attribute__((aligned(16))) float red[2][4][8][D + 4];          // two chunks' worth: one barrier per chunk
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int grp = blockIdx.x % p.groups, bk = blockIdx.x / p.groups, b = bk / p.c.Hkv, hk = bk % p.c.Hkv;
    const int h0 = hk * p.G + grp * 8, nh = min(8, p.G - grp * 8);
    const int n = attn8_len(p, b), chunk = attn8_chunk(n), nch = (n + chunk - 1) / chunk;
    const uint8_t* kb = p.c.k + b * p.c.sb + hk * p.c.sh;
    const uint8_t* vb = p.c.v + b * p.c.sb + hk * p.c.sh;
    const float* ksb = p.c.ks + b * p.c.ssb + hk * p.c.ssh;
    const float* vsb = p.c.vs + b * p.c.ssb + hk * p.c.ssh;

    if (p.cosT && n > 0 && (nch - 1) % gridDim.y == blockIdx.y) {       // this workgroup reads the new key: it appends it first
        if (wave == 0) attn8_append<D, FMT>(p, b, hk, n - 1, lane);
        __syncthreads();
    }

    // A wave's 32-key tile.  The operands want, in lane (c, g): of half h of K, key 8 (c >> 2) + 4 h + (c & 3), codes 64 u + 16 g .. + 15; of V, key 8 g + j, the
    // D / 16 codes from vd on; the scales of keys 8 g .. + 7.  With D = 128 rows are whole 128-byte lines, and a load that takes half lines of twice the
    // rows runs 8-10 % slower (48 x 2809 keys, the loads alone: 149 against 138 us): lane c reads 16-byte pieces of the rows c & 7 and (c & 7) + 8 of a half (V: of
    // an even or an odd key), eight lanes to a row, and swaps with lane c ^ 8 what belongs there (settle()).
    // Addresses are a uniform base plus one 32-bit lane offset each (32 rows span less than 2^31 bytes: host check).
    u32x4 kr[2][NU];
    uint32_t vr[8][NU];
    float ks[8], vs[8];
    const uint32_t st = (uint32_t)p.c.st, soff = 8 * g, vd = D == 128 ? 16 * (c & 7) + 8 * (c >> 3) : 4 * c;
    const uint32_t koff = D == 128 ? (uint32_t)(8 * ((c & 7) >> 2) + (c & 3)) * st + 64 * (c >> 3) + 16 * g : (uint32_t)(8 * (c >> 2) + (c & 3)) * st + 16 * g;
    const uint32_t voff = D == 128 ? (uint32_t)(8 * g + (c >> 3)) * st + 16 * (c & 7) : (uint32_t)(8 * g) * st + vd;
    auto load_k = [&](int key0) {
        const uint8_t* t = kb + (int64_t)key0 * p.c.st;
        const float* z = ksb + key0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < NU; ++u) kr[h][u] = __builtin_nontemporal_load((const u32x4*)(t + (4 * h + 16 * u) * p.c.st + koff));
        const f32x4 s0 = *(const f32x4_u*)(z + soff), s1 = *(const f32x4_u*)(z + 4 + soff);
#pragma unroll
        for (int j = 0; j < 4; ++j) { ks[j] = s0[j]; ks[4 + j] = s1[j]; }
    };
    auto load_v = [&](int key0) {
        const uint8_t* t = vb + (int64_t)key0 * p.c.st;
        const float* z = vsb + key0;
#pragma unroll
        for (int j = 0; j < 8; j += NU) {
            const uint8_t* r = t + j * p.c.st + voff;
            if constexpr (NU == 2) {
                const u32x4 w = __builtin_nontemporal_load((const u32x4*)r);
                vr[j][0] = w[0]; vr[j][1] = w[1]; vr[j + 1][0] = w[2]; vr[j + 1][1] = w[3];
            } else vr[j][0] = __builtin_nontemporal_load((const uint32_t*)r);
        }
        const f32x4 s0 = *(const f32x4_u*)(z + soff), s1 = *(const f32x4_u*)(z + 4 + soff);
#pragma unroll
        for (int j = 0; j < 4; ++j) { vs[j] = s0[j]; vs[4 + j] = s1[j]; }
    };
    // what the loads brought to where the operands want it: a takes the other's b in the upper 8 columns, b the other's a in the lower 8
    auto swap8 = [](uint32_t& a, uint32_t& b) {
        const uint32_t x = (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, 0x128, 0xf, 0xc, false);
        b = (uint32_t)__builtin_amdgcn_update_dpp((int)b, (int)a, 0x128, 0xf, 0x3, false);
        a = x;
    };
    auto settle_k = [&] {
        if constexpr (NU == 2)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int w = 0; w < 4; ++w) { uint32_t a = kr[h][0][w], b_ = kr[h][1][w]; swap8(a, b_); kr[h][0][w] = a; kr[h][1][w] = b_; }
    };
    auto settle_v = [&] {
        if constexpr (NU == 2)
#pragma unroll
            for (int j = 0; j < 8; j += 2) { swap8(vr[j][0], vr[j + 1][0]); swap8(vr[j][1], vr[j + 1][1]); }
    };
    // the last, partial tile: rows behind the end are read as the last row (and not attended)
    auto load_tail = [&](int key0) {
        const int last = n - 1 - key0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t r = key0 + min(8 * (c >> 2) + 4 * h + (c & 3), last);
#pragma unroll
            for (int u = 0; u < NU; ++u) kr[h][u] = *(const u32x4*)(kb + r * p.c.st + 64 * u + 16 * g);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t r = key0 + min(8 * g + j, last);
#pragma unroll
            for (int u = 0; u < NU; ++u) vr[j][u] = *(const uint32_t*)(vb + r * p.c.st + vd + 4 * u);
            ks[j] = ksb[r];
            vs[j] = vsb[r];
        }
    };

    int ch = blockIdx.y, key0 = ch * chunk + wave * 32;
    if (key0 + 32 <= n) { load_k(key0); load_v(key0); }

    // the queries, as B operands: column c is head c & 7, step 2 u + e holds elements 64 u + 16 g + 8 e .. + 7
    bf16x8 qf[2 * NU];
    {
        const bf16_t* x = p.q + (int64_t)b * p.q_sb + (int64_t)(h0 + min(c & 7, nh - 1)) * (p.cosT ? D : p.q_sh);
#pragma unroll
        for (int t = 0; t < 2 * NU; ++t) {
            const int d = 64 * (t >> 1) + 16 * g + 8 * (t & 1);
            qf[t] = *(const bf16x8*)(x + d);
            if (p.cosT && n > 0) {
                const bool lo = d < D / 2;
                const bf16x8 y = *(const bf16x8*)(x + (lo ? d + D / 2 : d - D / 2));
                const float* cr = p.cosT + (int64_t)(n - 1) * (D / 2) + (lo ? d : d - D / 2);
                const float* sr = p.sinT + (int64_t)(n - 1) * (D / 2) + (lo ? d : d - D / 2);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = (float)qf[t][i], z = (float)y[i];
                    float o1, o2;
                    mc_rope_pair(lo ? a : z, lo ? z : a, cr[i], sr[i], o1, o2);
                    qf[t][i] = (bf16_t)(lo ? o1 : o2);
                }
            }
        }
    }

    float m, l;
    f32x4 acc[NT];
    int flip = 0;
    // One tile: the scores from kr / ks, then the outputs from vr / vs.  next_k, next_v request the following tile's rows as soon as this one's are used.
    // ok: which of this lane's 8 keys are attended (MASKED; else all).  raw: the registers are as load_k / load_v left them.
    auto tile = [&](auto masked, auto raw, uint32_t ok, auto&& next_k, auto&& next_v) {
        constexpr bool MASKED = decltype(masked)::value, RAW = decltype(raw)::value;
        if constexpr (RAW) settle_k();
        f32x4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int h = 0; h < 2; ++h) s[h] = mc_mfma_16x16x32(kv8_row8<FMT>(kr[h][u][2 * e], kr[h][u][2 * e + 1]), qf[2 * u + e], s[h]);
        float sc[8], mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sc[j] = s[j >> 2][j & 3] * (ks[j] * p.scale_log2e);
            if (MASKED && !((ok >> j) & 1u)) sc[j] = -INFINITY;
            mx = fmaxf(mx, sc[j]);
        }
        next_k();
        mx = kv8_quarters_max(mx);
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx), a = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);      // (m = -inf: 0)
            m = mn;
            l *= a;
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[i] *= a;
        }
        const float base = m == -INFINITY ? 0.f : m;
        if constexpr (RAW) settle_v();
        u32x4 pf, pl;
        const uint32_t upper = c < 8 ? 0u : 0xffffffffu;
#pragma unroll
        for (int j2 = 0; j2 < 4; ++j2) {
            float w[2], rest[2], low[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = 2 * j2 + i;
                const float e = __builtin_amdgcn_exp2f(sc[j] - base);
                l += e;
                w[i] = e * vs[j];
                if (MASKED && !((ok >> j) & 1u)) {                  // nothing of a masked key: not its scale, not its codes (either may be no number)
                    w[i] = 0.f;
#pragma unroll
                    for (int u = 0; u < NU; ++u) vr[j][u] = 0u;
                }
            }
            const kv8_b16x2 hi = {(__bf16)w[0], (__bf16)w[1]};
#pragma unroll
            for (int i = 0; i < 2; ++i) rest[i] = w[i] - (float)hi[i];
            const kv8_b16x2 mid = {(__bf16)rest[0], (__bf16)rest[1]};
#pragma unroll
            for (int i = 0; i < 2; ++i) low[i] = rest[i] - (float)mid[i];
            const uint32_t h2 = __builtin_bit_cast(uint32_t, hi), m2 = __builtin_bit_cast(uint32_t, mid), l2 = __builtin_bit_cast(uint32_t, (kv8_b16x2){(__bf16)low[0], (__bf16)low[1]});
            pf[j2] = (m2 & upper) | (h2 & ~upper);
            pl[j2] = l2 & ~upper;
        }
        // V^T operands: row c of product i is element vd + i, of keys 8 g .. 8 g + 7
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            uint32_t pr[4][2];
#pragma unroll
            for (int k2 = 0; k2 < 4; ++k2) {
                pr[k2][0] = __builtin_amdgcn_perm(vr[2 * k2 + 1][u], vr[2 * k2][u], 0x05010400u);       // elements 0 and 1 of two keys
                pr[k2][1] = __builtin_amdgcn_perm(vr[2 * k2 + 1][u], vr[2 * k2][u], 0x07030602u);       // 2 and 3
            }
            if (u == NU - 1) next_v();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u32x4 o;
#pragma unroll
                for (int k2 = 0; k2 < 4; ++k2) o[k2] = i & 1 ? kv8_pair<FMT, false, true>(pr[k2][i >> 1]) : kv8_pair<FMT, false, false>(pr[k2][i >> 1]);
                acc[4 * u + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kv8_b16x8, o), __builtin_bit_cast(kv8_b16x8, pl), acc[4 * u + i], 0, 0, 0);
                acc[4 * u + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kv8_b16x8, o), __builtin_bit_cast(kv8_b16x8, pf), acc[4 * u + i], 0, 0, 0);
            }
        }
    };

    for (; ch < nch; ch += gridDim.y) {
        m = -INFINITY; l = 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
        const int end = (ch + 1) * chunk;
        const uint8_t* kv = p.key_valid + (int64_t)b * p.kv_stride;
        for (; key0 < end && key0 + 32 <= n; key0 += 128) {
            const int next = key0 + 128 < end ? key0 + 128 : (ch + (int)gridDim.y) * chunk + wave * 32;
            uint32_t ok = 0;
            if constexpr (KM) {
                const u32x2 w = *(const u32x2_u*)(kv + key0 + soff);
#pragma unroll
                for (int j = 0; j < 8; ++j) ok |= ((w[j >> 2] >> (8 * (j & 3))) & 255u) ? 1u << j : 0u;
            }
            tile(std::integral_constant<bool, KM>{}, std::true_type{}, ok, [&] { if (next + 32 <= n) load_k(next); }, [&] { if (next + 32 <= n) load_v(next); });
        }
        if (key0 < end && key0 < n) {
            load_tail(key0);
            uint32_t ok = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = key0 + 8 * g + j;
                bool in = key < n;
                if constexpr (KM) in = in && kv[min(key, n - 1)] != 0;
                ok |= in ? 1u << j : 0u;
            }
            tile(std::true_type{}, std::false_type{}, ok, [] {}, [] {});
        }
        key0 = (ch + (int)gridDim.y) * chunk + wave * 32;

        // this wave's partial: high and low columns together, then over the quarters for l.  acc[i][r] is row 4 g + r of product i, head c
        l = kv8_quarters_sum(l);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][r] += kv8_other_half(acc[i][r]);
        if (c < nh) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < NT; i += 4) *(f32x4*)&red[flip][wave][c][(D == 128 ? 64 * (g & 1) + 16 * r + 8 * (g >> 1) : 16 * g + 4 * r) + i] = (f32x4){acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
            if (g == 0) { red[flip][wave][c][D] = m; red[flip][wave][c][D + 1] = l; }
        }
        __syncthreads();
        for (int e = tid; e < nh * D; e += 256) {
            const int h = e / D, d = e % D;
            const float (*r)[8][D + 4] = red[flip];
            float mm = -INFINITY;
#pragma unroll
            for (int w_ = 0; w_ < 4; ++w_) mm = fmaxf(mm, r[w_][h][D]);
            const float base = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f, aa = 0.f;
#pragma unroll
            for (int w_ = 0; w_ < 4; ++w_) {
                const float a = __builtin_amdgcn_exp2f(r[w_][h][D] - base);
                ll = fmaf(r[w_][h][D + 1], a, ll);
                aa = fmaf(r[w_][h][d], a, aa);
            }
            float* part = p.ws + ((int64_t)(b * p.H + h0 + h) * p.ws_chunks + ch) * (D + 4);
            part[d] = aa;
            if (d == 0) { part[D] = mm; part[D + 1] = ll; }
        }
        flip ^= 1;                                          // (a wave cannot write this half again before all have passed the next chunk's barrier)
    }
    if (!p.self_combine) return;
    __syncthreads();
    for (int h = h0; h < h0 + nh; ++h)
        attn8_join<D>(p.ws + (int64_t)(b * p.H + h) * p.ws_chunks * (D + 4), nch, p.o + (int64_t)b * p.o_sb + h * D, &red[0][0][0][0]);
}

template <int D>
__global__ __launch_bounds__(256) void attn_decode8_join_kernel(AttnParams8 p) {
    __shared__ float lds[260];
    const int b = blockIdx.x / p.H, h = blockIdx.x % p.H, n = attn8_len(p, b), chunk = attn8_chunk(n);
    attn8_join<D>(p.ws + (int64_t)blockIdx.x * p.ws_chunks * (D + 4), (n + chunk - 1) / chunk, p.o + (int64_t)b * p.o_sb + h * D, lds);
}

// the most partials any length up to S has (a length just below a change of the chunk has more than those above it)
int attn8_max_parts(int S) {
    int most = 0;
    for (int n : {S, S < 4096 ? S : 4096, S < 16384 ? S : 16384}) {
        const int c = attn8_chunk(n), parts = (n + c - 1) / c;
        most = parts > most ? parts : most;
    }
    return most;
}

int check_cache(const mc_kv8_cache* c, const char* who) {
    MC_CHECK_ARG(c && c->k && c->v && c->k_scale && c->v_scale, "%s: null cache pointer", who);
    MC_CHECK_ARG(c->format == MC_KV8_E4M3 || c->format == MC_KV8_INT8, "%s: cache format %d", who, c->format);
    MC_CHECK_ARG(c->D == 64 || c->D == 128, "%s: head_dim %d not supported (64 or 128)", who, c->D);
    MC_CHECK_ARG(c->B > 0 && c->Hkv > 0 && c->S > 0 && c->S <= (1 << 30), "%s: bad cache shape B=%d Hkv=%d S=%d", who, c->B, c->Hkv, c->S);
    MC_CHECK_ARG((int64_t)c->B * c->Hkv < (1LL << 24), "%s: B * Hkv = %lld is too large", who, (long long)c->B * c->Hkv);
    MC_CHECK_ARG(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0 && (c->sb | c->sh | c->st) % 16 == 0, "%s: the codes' rows must be 16-byte aligned", who);
    MC_CHECK_ARG(c->st > 0 && c->st < (1LL << 26), "%s: %lld bytes from one position to the next", who, (long long)c->st);
    MC_CHECK_ARG(((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 4 == 0, "%s: the scales must be 4-byte aligned", who);
    return 0;
}

Cache dev_cache(const mc_kv8_cache* c) {
    return Cache{(uint8_t*)c->k, c->k_scale, (uint8_t*)c->v, c->v_scale, c->sb, c->sh, c->st, c->scale_sb, c->scale_sh, c->B, c->Hkv, c->S};
}

#define KV8_MASKED(D, F) attn_decode8_kernel<D, F, true>
#define KV8_PLAIN(D, F) attn_decode8_kernel<D, F, false>
#define KV8_ROPE(D, F) rope_kv8_kernel<D, F>
#define KV8_READ(D, F) kv8_read_kernel<D, F>
#define KV8_DISPATCH(c, KERNEL, grid, block, lds, s, ...)                                                          \
    do {                                                                                                           \
        if ((c)->D == 128 && (c)->format == MC_KV8_E4M3) KERNEL(128, MC_KV8_E4M3)<<<grid, block, lds, s>>>(__VA_ARGS__); \
        else if ((c)->D == 128) KERNEL(128, MC_KV8_INT8)<<<grid, block, lds, s>>>(__VA_ARGS__);                     \
        else if ((c)->format == MC_KV8_E4M3) KERNEL(64, MC_KV8_E4M3)<<<grid, block, lds, s>>>(__VA_ARGS__);         \
        else KERNEL(64, MC_KV8_INT8)<<<grid, block, lds, s>>>(__VA_ARGS__);                                         \
    } while (0)

int rope_launch(const mc_kv8_cache* c, RopeParams& p, hipStream_t s, const char* who) {
    const int nv = p.H + 2 * c->Hkv, vpb = 256 / (c->D / 8) * kRopeVecs;
    p.blocks_per_row = (nv + vpb - 1) / vpb;
    MC_CHECK_ARG((int64_t)p.M * p.blocks_per_row < (1LL << 23), "%s: too many rows (%d of %d heads) for one launch", who, p.M, nv);
    KV8_DISPATCH(c, KV8_ROPE, p.M * p.blocks_per_row, 256, 0, s, p);
    MC_CHECK_LAUNCH();
    return 0;
}

int check_rope(const void* qkv, int64_t ld, const float* cos_table, const float* sin_table, int max_pos, int H, const mc_kv8_cache* c, const char* who) {
    if (int e = check_cache(c, who)) return e;
    MC_CHECK_ARG(qkv && cos_table && sin_table, "%s: null pointer", who);
    MC_CHECK_ARG(H > 0 && H % c->Hkv == 0, "%s: %d query heads over %d key heads", who, H, c->Hkv);
    MC_CHECK_ARG((uintptr_t)qkv % 16 == 0 && ld % 8 == 0 && ld >= (int64_t)(H + 2 * c->Hkv) * c->D, "%s: qkv rows must be 16-byte aligned and hold %d heads", who,
                 H + 2 * c->Hkv);
    MC_CHECK_ARG(((uintptr_t)cos_table | (uintptr_t)sin_table) % 16 == 0 && max_pos > 0, "%s: the tables must be 16-byte aligned", who);
    return 0;
}

// 4096 workgroups fill the chip five times over, while there are chunks to hand out (48 x 2809 keys: 146 us with 4608 workgroups, 152 with 1536, 157 with 9216)
int attn8_launch(AttnParams8& p, const mc_kv8_cache* c, hipStream_t s, const char* who) {
    const int chunks = attn8_max_parts(c->S);
    p.G = p.H / c->Hkv;
    p.groups = (p.G + 7) / 8;
    p.ws_chunks = chunks;
    const int64_t wgs = (int64_t)c->B * c->Hkv * p.groups;
    MC_CHECK_ARG(c->B == 1 || p.o_sb >= (int64_t)p.H * c->D, "%s: output rows overlap", who);
    MC_CHECK_ARG(wgs < (1LL << 23) && (int64_t)c->B * p.H < (1LL << 23), "%s: B * H = %lld is too large for one launch", who, (long long)c->B * p.H);
    // up to two chunks: one workgroup takes both and joins them itself.  Launched one call at a time the second launch costs more than it saves (5 x 517 keys: 14.8
    // against 17.4 us a call); replayed from a graph it would pay (12.4 against 10.3)
    const int want = (int)((4096 + wgs - 1) / wgs), split = chunks <= 2 ? 1 : want < chunks ? want : chunks;
    p.self_combine = split == 1;
    const dim3 grid((unsigned)wgs, split);
    if (p.key_valid) KV8_DISPATCH(c, KV8_MASKED, grid, 256, 0, s, p);
    else KV8_DISPATCH(c, KV8_PLAIN, grid, 256, 0, s, p);
    if (!p.self_combine) {
        if (c->D == 128) attn_decode8_join_kernel<128><<<c->B * p.H, 256, 0, s>>>(p);
        else attn_decode8_join_kernel<64><<<c->B * p.H, 256, 0, s>>>(p);
    }
    MC_CHECK_LAUNCH();
    return 0;
}

}  // namespace

extern "C" int mc_rope_kv8(const void* qkv, int64_t ld, const int32_t* row_b, const int32_t* row_pos, const int32_t* row_t, const float* cos_table,
                           const float* sin_table, int max_pos, void* q_out, const mc_kv8_cache* cache, int M, int H, int Lq, void* stream) {
    if (int e = check_rope(qkv, ld, cos_table, sin_table, max_pos, H, cache, "mc_rope_kv8")) return e;
    MC_CHECK_ARG(row_b && row_pos && row_t && q_out && (uintptr_t)q_out % 16 == 0, "mc_rope_kv8: null or misaligned pointer");
    MC_CHECK_ARG(M >= 0 && Lq > 0, "mc_rope_kv8: bad shape M=%d Lq=%d", M, Lq);
    if (M == 0) return 0;
    RopeParams p{(const bf16_t*)qkv, ld, row_b, row_pos, row_t, cos_table, sin_table, max_pos, (bf16_t*)q_out, dev_cache(cache), M, H, Lq, 0};
    return rope_launch(cache, p, (hipStream_t)stream, "mc_rope_kv8");
}

extern "C" int mc_kv8_read(const mc_kv8_cache* cache, const int32_t* kv_lens, int n, void* k_out, void* v_out, void* stream) {
    if (int e = check_cache(cache, "mc_kv8_read")) return e;
    MC_CHECK_ARG(k_out && v_out && ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0, "mc_kv8_read: null or misaligned output");
    MC_CHECK_ARG(n >= 0 && n <= cache->S, "mc_kv8_read: %d positions of a cache of %d", n, cache->S);
    if (n == 0) return 0;
    const int64_t blocks = ((int64_t)n * (cache->D / 8) + 255) / 256;
    MC_CHECK_ARG(blocks < (1LL << 23), "mc_kv8_read: %d positions are too many for one launch", n);
    const int bh = cache->B * cache->Hkv;
    const dim3 grid((unsigned)blocks, bh < 4096 ? bh : 4096);
    KV8_DISPATCH(cache, KV8_READ, grid, 256, 0, (hipStream_t)stream, dev_cache(cache), kv_lens, n, (bf16_t*)k_out, (bf16_t*)v_out);
    MC_CHECK_LAUNCH();
    return 0;
}

extern "C" int mc_attn_decode8_workspace_bytes(int B, int H, int D, int S, int64_t* bytes) {
    MC_CHECK_ARG(bytes && B > 0 && H > 0 && D > 0 && S > 0, "mc_attn_decode8_workspace_bytes: bad arguments");
    *bytes = (int64_t)B * H * attn8_max_parts(S) * (D + 4) * 4;
    return 0;
}

extern "C" int mc_attn_decode8(const void* q, int64_t q_sb, int64_t q_sh, const mc_kv8_cache* cache, const int32_t* kv_lens, const void* key_valid,
                               int64_t key_valid_stride, void* o, int64_t o_sb, void* workspace, int H, float scale, void* stream) {
    if (int e = check_cache(cache, "mc_attn_decode8")) return e;
    MC_CHECK_ARG(q && o && workspace, "mc_attn_decode8: null pointer");
    MC_CHECK_ARG(H > 0 && H % cache->Hkv == 0, "mc_attn_decode8: %d query heads over %d key heads", H, cache->Hkv);
    MC_CHECK_ARG((uintptr_t)q % 16 == 0 && (q_sb | q_sh) % 8 == 0, "mc_attn_decode8: query rows must be 16-byte aligned");
    AttnParams8 p{(const bf16_t*)q, q_sb, q_sh, dev_cache(cache), (bf16_t*)o, o_sb, (float*)workspace, kv_lens, (const uint8_t*)key_valid, key_valid_stride,
                  nullptr, nullptr, 0, H, 0, 0, 0, 0, scale * 1.4426950408889634f};
    return attn8_launch(p, cache, (hipStream_t)stream, "mc_attn_decode8");
}

extern "C" int mc_attn_decode8_rope(const void* qkv, int64_t qkv_ld, const float* cos_table, const float* sin_table, int max_pos, const mc_kv8_cache* cache,
                                    const int32_t* kv_lens, const void* key_valid, int64_t key_valid_stride, void* o, int64_t o_sb, void* workspace, int H,
                                    float scale, void* stream) {
    if (int e = check_rope(qkv, qkv_ld, cos_table, sin_table, max_pos, H, cache, "mc_attn_decode8_rope")) return e;
    MC_CHECK_ARG(kv_lens && o && workspace, "mc_attn_decode8_rope: null pointer");
    AttnParams8 p{(const bf16_t*)qkv, qkv_ld, cache->D, dev_cache(cache), (bf16_t*)o, o_sb, (float*)workspace, kv_lens, (const uint8_t*)key_valid, key_valid_stride,
                  cos_table, sin_table, max_pos, H, 0, 0, 0, 0, scale * 1.4426950408889634f};
    return attn8_launch(p, cache, (hipStream_t)stream, "mc_attn_decode8_rope");
}
