// 8-bit KV cache: the cache write of a projection's rows (rotation + quantisation), the read-back to 16 bits, and decode attention over the codes.
//
// Same places as the 16-bit forms (rope_kv_kernel, attn_decode_kernel; LlamaAttention.forward, modelcompose/model/language_model/
// multimodal_llama.py:281-312); the reference keeps its cache in 16 bits.  Half the bytes per cached key: a decode step at batch 48 spends most of its
// time reading them.
#include "kv8.h"

namespace {

struct Cache {
    uint8_t* k; float* ks; uint8_t* v; float* vs;
    int64_t sb, sh, st, ssb, ssh;
    int B, Hkv, S;
};

// ---- cache write ------------------------------------------------------------------------------------------------------------------
struct RopeParams {
    const bf16_t* qkv; int64_t ld;
    const int32_t* row_b; const int32_t* row_pos; const int32_t* row_t;      // row_b null: row r is sequence r, position kv_lens[r] - 1, query row 0
    const int32_t* kv_lens;
    const float* cosT; const float* sinT; int max_pos;
    bf16_t* q_out; Cache c;
    int M, H, Lq, blocks_per_row;
};

// One vector (a head of q, k or v of one row) per D / 8 lanes: a lane holds elements 4 i .. 4 i + 3 of both halves, i.e. whole rotation pairs.
// HBM-bound: reads the row once, writes q (16 bits) and the codes once.
template <int D, int FMT>
__global__ __launch_bounds__(256) void rope_kv8_kernel(RopeParams p) {
#pragma clang fp contract(off)
    constexpr int LPV = D / 8, VPB = 256 / LPV;
    const int row = blockIdx.x / p.blocks_per_row;
    const int vec = (blockIdx.x - row * p.blocks_per_row) * VPB + threadIdx.x / LPV, i4 = (threadIdx.x % LPV) * 4;
    if (vec >= p.H + 2 * p.c.Hkv) return;                       // (whole groups of LPV lanes leave: the shuffles below stay inside a group)
    int b, pos, t;
    if (p.row_b) { b = p.row_b[row]; pos = p.row_pos[row]; t = p.row_t[row]; }
    else { b = row; pos = p.kv_lens[row] - 1; t = 0; }
    // rows of no sequence (b < 0: padding), and rows that do not fit the cache, the tables or q_out: nothing is written
    if (b < 0 || b >= p.c.B || pos < 0 || pos >= p.c.S || pos >= p.max_pos || t < 0 || t >= p.Lq) return;
    const bf16_t* x = p.qkv + (int64_t)row * p.ld + (int64_t)vec * D + i4;
    const bf16x4 xa = *(const bf16x4*)x, xb = *(const bf16x4*)(x + D / 2);
    float a[4], bb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) { a[j] = (float)xa[j]; bb[j] = (float)xb[j]; }
    if (vec < p.H + p.c.Hkv) {
        const f32x4 cs = *(const f32x4*)(p.cosT + (int64_t)pos * (D / 2) + i4), sn = *(const f32x4*)(p.sinT + (int64_t)pos * (D / 2) + i4);
        if (vec < p.H) {                                          // the bits of the 16-bit path's queries (mc_rope_pair)
            bf16x4 oa, ob;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float o1, o2;
                mc_rope_pair(a[j], bb[j], cs[j], sn[j], o1, o2);
                oa[j] = (bf16_t)o1; ob[j] = (bf16_t)o2;
            }
            bf16_t* o = p.q_out + ((int64_t)b * p.Lq + t) * p.H * D + vec * D + i4;
            *(bf16x4*)o = oa;
            *(bf16x4*)(o + D / 2) = ob;
            return;
        }
        // keys go from fp32 straight to codes: one rounding, not a 16-bit one first; products and sum rounded on their own
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float u = a[j] * cs[j], w = bb[j] * sn[j], y = bb[j] * cs[j], z = a[j] * sn[j];
            a[j] = u - w;
            bb[j] = y + z;
        }
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, max(__float_as_uint(a[j]) & 0x7fffffffu, __float_as_uint(bb[j]) & 0x7fffffffu));
#pragma unroll
    for (int o = LPV / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    const Kv8Scale s = kv8_scale<FMT>(m);
    const bool is_k = vec < p.H + p.c.Hkv;
    const int hk = vec - p.H - (is_k ? 0 : p.c.Hkv);
    uint8_t* dst = (is_k ? p.c.k : p.c.v) + b * p.c.sb + hk * p.c.sh + pos * p.c.st + i4;
    *(uint32_t*)dst = kv8_pack4<FMT>(a[0], a[1], a[2], a[3], s);
    *(uint32_t*)(dst + D / 2) = kv8_pack4<FMT>(bb[0], bb[1], bb[2], bb[3], s);
    if (i4 == 0) (is_k ? p.c.ks : p.c.vs)[b * p.c.ssb + hk * p.c.ssh + pos] = s.scale;
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
                for (int j = 0; j < 4; ++j) o[j] = (bf16_t)(f[j] * s);
                kv8_unpack4<FMT>(w[1], f);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[4 + j] = (bf16_t)(f[j] * s);
            }
            *(bf16x8*)((kv ? v_out : k_out) + ((int64_t)bh * n + pos) * D + d) = o;
        }
    }
}

// ---- decode attention -------------------------------------------------------------------------------------------------------------
struct AttnParams8 {
    const bf16_t* q; int64_t q_sb, q_sh;
    Cache c;
    bf16_t* o; int64_t o_sb;
    const int32_t* kv_lens; const uint8_t* key_valid; int64_t kv_stride;
    int H, appended, max_pos;          // appended: the last key is this step's token; lengths that could not be appended give a zero row
    float scale_log2e;
};

__device__ __forceinline__ int attn8_len(const AttnParams8& p, int b) {
    const int n = p.kv_lens ? p.kv_lens[b] : p.c.S;
    if (p.appended && (n > p.c.S || n > p.max_pos)) return 0;
    return min(n, p.c.S);
}

// One workgroup per query head; a key is held by D / 16 lanes; every group of lanes runs the online softmax over its keys.
template <int D, int FMT>
__global__ __launch_bounds__(256) void attn_decode8_kernel(AttnParams8 p) {
    // a score and the maximum taken from it have to be the same number: fused into the difference, the score's product is not rounded, and at 1e30 what
    // it differs by is no longer small
#pragma clang fp contract(off)
    constexpr int LPK = D / 16, KPW = 64 / LPK;
    __shared__ float red[4][D + 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = blockIdx.x / p.H, h = blockIdx.x % p.H, hk = h / (p.H / p.c.Hkv);
    const int n = attn8_len(p, b);
    const int slot = lane / LPK, dl = (lane % LPK) * 16;
    float q[16], acc[16], m = -1e30f, l = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) { q[i] = n > 0 ? (float)p.q[b * p.q_sb + h * p.q_sh + dl + i] : 0.f; acc[i] = 0.f; }
    const uint8_t* kb = p.c.k + b * p.c.sb + hk * p.c.sh + dl;
    const uint8_t* vb = p.c.v + b * p.c.sb + hk * p.c.sh + dl;
    for (int j0 = wave * KPW; j0 < n; j0 += 4 * KPW) {
        const int j = j0 + slot;
        const bool ok = j < n && (!p.key_valid || p.key_valid[b * p.kv_stride + j]);
        u32x4 kw = {}, vw = {};
        float ks = 0.f, vs = 0.f;
        if (ok) {
            kw = *(const u32x4*)(kb + j * p.c.st);
            vw = *(const u32x4*)(vb + j * p.c.st);
            ks = p.c.ks[b * p.c.ssb + hk * p.c.ssh + j];
            vs = p.c.vs[b * p.c.ssb + hk * p.c.ssh + j];
        }
        float s = 0.f, f[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            kv8_unpack4<FMT>(kw[w], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) s = fmaf(q[4 * w + i], f[i], s);
        }
#pragma unroll
        for (int o = 1; o < LPK; o <<= 1) s += __shfl_xor(s, o, 64);
        s *= ks * p.scale_log2e;
        const float mn = ok ? fmaxf(m, s) : m, a = __builtin_amdgcn_exp2f(m - mn), e = ok ? __builtin_amdgcn_exp2f(s - mn) : 0.f;
        m = mn;
        l = fmaf(l, a, e);
        const float ev = ok ? e * vs : 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            kv8_unpack4<FMT>(vw[w], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[4 * w + i] = fmaf(ev, f[i], acc[4 * w + i] * a);
        }
    }
#pragma unroll
    for (int o = LPK; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(m, o, 64), l2 = __shfl_xor(l, o, 64), mn = fmaxf(m, m2);
        const float a1 = __builtin_amdgcn_exp2f(m - mn), a2 = __builtin_amdgcn_exp2f(m2 - mn);
        l = l * a1 + l2 * a2;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = acc[i] * a1 + __shfl_xor(acc[i], o, 64) * a2;
        m = mn;
    }
    if (slot == 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) red[wave][dl + i] = acc[i];
        if (dl == 0) { red[wave][D] = m; red[wave][D + 1] = l; }
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    float mm = -1e30f, ll = 0.f, aa = 0.f;
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, red[w][D]);
    for (int w = 0; w < 4; ++w) {
        const float a = __builtin_amdgcn_exp2f(red[w][D] - mm);
        ll = fmaf(red[w][D + 1], a, ll);
        aa = fmaf(red[w][d], a, aa);
    }
    p.o[b * p.o_sb + h * D + d] = (bf16_t)(ll == 0.f ? 0.f : aa / ll);
}

int check_cache(const mc_kv8_cache* c, const char* who) {
    MC_CHECK_ARG(c && c->k && c->v && c->k_scale && c->v_scale, "%s: null cache pointer", who);
    MC_CHECK_ARG(c->format == MC_KV8_E4M3 || c->format == MC_KV8_INT8, "%s: cache format %d", who, c->format);
    MC_CHECK_ARG(c->D == 64 || c->D == 128, "%s: head_dim %d not supported (64 or 128)", who, c->D);
    MC_CHECK_ARG(c->B > 0 && c->Hkv > 0 && c->S > 0, "%s: bad cache shape B=%d Hkv=%d S=%d", who, c->B, c->Hkv, c->S);
    MC_CHECK_ARG((int64_t)c->B * c->Hkv < (1LL << 24), "%s: B * Hkv = %lld is too large", who, (long long)c->B * c->Hkv);
    MC_CHECK_ARG(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0 && (c->sb | c->sh | c->st) % 16 == 0, "%s: the codes' rows must be 16-byte aligned", who);
    MC_CHECK_ARG(((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 4 == 0, "%s: the scales must be 4-byte aligned", who);
    return 0;
}

Cache dev_cache(const mc_kv8_cache* c) {
    return Cache{(uint8_t*)c->k, c->k_scale, (uint8_t*)c->v, c->v_scale, c->sb, c->sh, c->st, c->scale_sb, c->scale_sh, c->B, c->Hkv, c->S};
}

#define KV8_DISPATCH(c, KERNEL, grid, block, lds, s, ...)                                                          \
    do {                                                                                                           \
        if ((c)->D == 128 && (c)->format == MC_KV8_E4M3) KERNEL<128, MC_KV8_E4M3><<<grid, block, lds, s>>>(__VA_ARGS__); \
        else if ((c)->D == 128) KERNEL<128, MC_KV8_INT8><<<grid, block, lds, s>>>(__VA_ARGS__);                     \
        else if ((c)->format == MC_KV8_E4M3) KERNEL<64, MC_KV8_E4M3><<<grid, block, lds, s>>>(__VA_ARGS__);         \
        else KERNEL<64, MC_KV8_INT8><<<grid, block, lds, s>>>(__VA_ARGS__);                                         \
    } while (0)

int rope_launch(const mc_kv8_cache* c, RopeParams& p, hipStream_t s, const char* who) {
    const int nv = p.H + 2 * c->Hkv, vpb = 256 / (c->D / 8);
    p.blocks_per_row = (nv + vpb - 1) / vpb;
    MC_CHECK_ARG((int64_t)p.M * p.blocks_per_row < (1LL << 23), "%s: too many rows (%d of %d heads) for one launch", who, p.M, nv);
    KV8_DISPATCH(c, rope_kv8_kernel, p.M * p.blocks_per_row, 256, 0, s, p);
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

int attn8_launch(const void* q, int64_t q_sb, int64_t q_sh, const mc_kv8_cache* c, const int32_t* kv_lens, const void* key_valid, int64_t kv_stride,
                 void* o, int64_t o_sb, int H, int appended, int max_pos, float scale, hipStream_t s) {
    AttnParams8 p{(const bf16_t*)q, q_sb, q_sh, dev_cache(c), (bf16_t*)o, o_sb, kv_lens, (const uint8_t*)key_valid, kv_stride, H, appended, max_pos,
                  scale * 1.4426950408889634f};
    KV8_DISPATCH(c, attn_decode8_kernel, c->B * H, 256, 0, s, p);
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
    RopeParams p{(const bf16_t*)qkv, ld, row_b, row_pos, row_t, nullptr, cos_table, sin_table, max_pos, (bf16_t*)q_out, dev_cache(cache), M, H, Lq, 0};
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
    KV8_DISPATCH(cache, kv8_read_kernel, grid, 256, 0, (hipStream_t)stream, dev_cache(cache), kv_lens, n, (bf16_t*)k_out, (bf16_t*)v_out);
    MC_CHECK_LAUNCH();
    return 0;
}

extern "C" int mc_attn_decode8_workspace_bytes(int B, int H, int D, int S, int64_t* bytes) {
    (void)S;
    MC_CHECK_ARG(bytes && B > 0 && H > 0 && D > 0, "mc_attn_decode8_workspace_bytes: bad arguments");
    *bytes = (int64_t)B * H * D * 2;
    return 0;
}

extern "C" int mc_attn_decode8(const void* q, int64_t q_sb, int64_t q_sh, const mc_kv8_cache* cache, const int32_t* kv_lens, const void* key_valid,
                               int64_t key_valid_stride, void* o, int64_t o_sb, void* workspace, int H, float scale, void* stream) {
    if (int e = check_cache(cache, "mc_attn_decode8")) return e;
    MC_CHECK_ARG(q && o && workspace, "mc_attn_decode8: null pointer");
    MC_CHECK_ARG(H > 0 && H % cache->Hkv == 0, "mc_attn_decode8: %d query heads over %d key heads", H, cache->Hkv);
    MC_CHECK_ARG((uintptr_t)q % 16 == 0 && (q_sb | q_sh) % 8 == 0, "mc_attn_decode8: query rows must be 16-byte aligned");
    return attn8_launch(q, q_sb, q_sh, cache, kv_lens, key_valid, key_valid_stride, o, o_sb, H, 0, 0, scale, (hipStream_t)stream);
}

extern "C" int mc_attn_decode8_rope(const void* qkv, int64_t qkv_ld, const float* cos_table, const float* sin_table, int max_pos, const mc_kv8_cache* cache,
                                    const int32_t* kv_lens, const void* key_valid, int64_t key_valid_stride, void* o, int64_t o_sb, void* workspace, int H,
                                    float scale, void* stream) {
    if (int e = check_rope(qkv, qkv_ld, cos_table, sin_table, max_pos, H, cache, "mc_attn_decode8_rope")) return e;
    MC_CHECK_ARG(kv_lens && o && workspace, "mc_attn_decode8_rope: null pointer");
    const int D = cache->D;
    RopeParams p{(const bf16_t*)qkv, qkv_ld, nullptr, nullptr, nullptr, kv_lens, cos_table, sin_table, max_pos, (bf16_t*)workspace, dev_cache(cache), cache->B, H, 1, 0};
    if (int e = rope_launch(cache, p, (hipStream_t)stream, "mc_attn_decode8_rope")) return e;
    return attn8_launch(workspace, (int64_t)H * D, D, cache, kv_lens, key_valid, key_valid_stride, o, o_sb, H, 1, max_pos, scale, (hipStream_t)stream);
}
