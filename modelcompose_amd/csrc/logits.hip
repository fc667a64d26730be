// Logits processor: repetition / presence / frequency penalties, additive biases and a token mask on fp32 logits, in one pass before the arg-max or the
// sampler (generate(repetition_penalty = ..): RepetitionPenaltyLogitsProcessor of transformers 4.31 generation/logits_process.py, reached through
// modelcompose/eval/model_multimodal_qa_loader.py:94-102; the other members are what serving APIs add to it).
//
// For a row with prompt tokens P and generated tokens G, per token t:
//   seen = t in P or G, c = number of t in G
//   l = seen ? (l > 0 ? l / repetition : l * repetition) : l
//   l = l - (frequency * c + presence * (c > 0))
//   l = l + sum of the row's biases for t
//   l = -inf unless bit t of the row's mask is set
// HBM-bound at batch, latency-bound for one row.  A workgroup owns a slice of the vocabulary: it requests its logits and the first ids of the row, counts the tokens
// that fall into the slice in LDS (integer atomics: the order cannot change the result), and finishes the logits from registers.  Every slice reads the whole
// history, from the L2 after the first; in exchange there is no workspace, no second launch and no atomic on memory.  What a workgroup takes is latency - one round of
// loads, two barriers - so everything it will need is requested before the first wait, and LDS is kept small enough for 4 workgroups per CU (64 x 131072 with
// histories of 5120: 45 us with 2048 tokens a workgroup and the loads one after another, 25 with 44 KiB of LDS, 21 so).
#include "common.h"

namespace {

constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u;     // prompt tokens set the first, biases the second, generated tokens count below
constexpr int kMaxBias = 1024;

// A workgroup of THREADS takes a slice of SLICE tokens of one row.  VEC: rows are 16-byte aligned and a thread takes 4 logits side by side
template <int THREADS, int SLICE, bool VEC>
__global__ __launch_bounds__(THREADS) void logits_process_kernel(mc_logits_args a) {
    constexpr int PER = SLICE / THREADS, BP = kMaxBias / THREADS;
    static_assert(SLICE % THREADS == 0 && (!VEC || PER % 4 == 0) && kMaxBias % THREADS == 0, "a thread's logits and biases");
    __shared__ __attribute__((aligned(16))) uint32_t cnt[SLICE];
    __shared__ uint32_t b_at[kMaxBias];                         // biases of this slice: offset in the slice << 10 | place in the row's list, sorted below,
    __shared__ float b_val[kMaxBias];                           // and value
    __shared__ int n_listed;
    const int64_t row = blockIdx.y;
    const int t0 = blockIdx.x * SLICE, n = min(SLICE, a.V - t0), tid = threadIdx.x;
    const float* in = a.logits + row * a.ld + t0;
    float* out = a.out + row * a.ld_out + t0;
    // element j of this thread
    auto at = [&](int j) { return VEC ? (j >> 2) * 4 * THREADS + tid * 4 + (j & 3) : j * THREADS + tid; };

    // one history: U ids per thread in flight.  The first are requested whatever the length is (inside the array), before it is known
    const int64_t* p_ids = a.prompt_ids + row * a.ld_prompt;
    const int64_t* o_ids = a.output_ids + row * a.ld_output;
    const int32_t* b_ids = a.bias_ids + row * a.ld_bias;
    const float* b_in = a.bias + row * a.ld_bias;
    constexpr int U = 8;
    int64_t pt[U], ot[U / 2];
    int32_t bt[BP];
    float bv[BP];
    if (a.prompt_cols > 0)
#pragma unroll
        for (int u = 0; u < U; ++u) pt[u] = p_ids[min(tid + u * THREADS, a.prompt_cols - 1)];
    if (a.output_cols > 0)
#pragma unroll
        for (int u = 0; u < U / 2; ++u) ot[u] = o_ids[min(tid + u * THREADS, a.output_cols - 1)];
    if (a.n_bias > 0)
#pragma unroll
        for (int u = 0; u < BP; ++u) { bt[u] = b_ids[min(tid + u * THREADS, a.n_bias - 1)]; bv[u] = b_in[min(tid + u * THREADS, a.n_bias - 1)]; }
    const int p_len = a.prompt_lens ? min(a.prompt_lens[row], a.prompt_cols) : a.prompt_cols;
    const int o_len = a.output_lens ? min(a.output_lens[row], a.output_cols) : a.output_cols;
    float l[PER];
#pragma unroll
    for (int j = 0; j < PER; j += VEC ? 4 : 1) {
        if constexpr (VEC) {
            if (at(j) + 4 <= n) {
                const f32x4 v = *(const f32x4*)(in + at(j));
                l[j] = v[0]; l[j + 1] = v[1]; l[j + 2] = v[2]; l[j + 3] = v[3];
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) l[j + q] = at(j + q) < n ? in[at(j + q)] : 0.f;
            }
        } else l[j] = at(j) < n ? in[at(j)] : 0.f;
    }
    for (int i = tid; i < SLICE; i += THREADS) cnt[i] = 0;
    if (tid == 0) n_listed = 0;
    __syncthreads();

    auto inside = [&](int64_t id, int& o) { const int64_t d = id - t0; o = (int)d; return d >= 0 && d < n; };
    int o;
    if (a.prompt_cols > 0) {
        for (int i0 = tid; i0 < p_len; i0 += U * THREADS) {
            if (i0 != tid)
#pragma unroll
                for (int u = 0; u < U; ++u) pt[u] = p_ids[min(i0 + u * THREADS, p_len - 1)];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * THREADS < p_len && inside(pt[u], o)) atomicOr(&cnt[o], kSeen);
        }
    }
    if (a.output_cols > 0) {
        for (int i0 = tid; i0 < o_len; i0 += U / 2 * THREADS) {
            if (i0 != tid)
#pragma unroll
                for (int u = 0; u < U / 2; ++u) ot[u] = o_ids[min(i0 + u * THREADS, o_len - 1)];
#pragma unroll
            for (int u = 0; u < U / 2; ++u)
                if (i0 + u * THREADS < o_len && inside(ot[u], o)) atomicAdd(&cnt[o], 1u);
        }
    }
    if (a.n_bias > 0) {
#pragma unroll
        for (int u = 0; u < BP; ++u)
            if (tid + u * THREADS < a.n_bias && inside(bt[u], o)) {
                const int e = atomicAdd(&n_listed, 1);
                b_at[e] = (uint32_t)o << 10 | (uint32_t)(tid + u * THREADS);
                b_val[e] = bv[u];
                atomicOr(&cnt[o], kBiased);
            }
    }
    __syncthreads();

    const float rep = a.repetition ? a.repetition[row] : 1.f, pres = a.presence ? a.presence[row] : 0.f, freq = a.frequency ? a.frequency[row] : 0.f;
    const uint32_t* bits = a.allowed ? (const uint32_t*)a.allowed + row * a.ld_allowed : nullptr;
    const int k = a.n_bias > 0 ? n_listed : 0;
    // The biases of a token side by side and in the order of the row's list: a bitonic sort of the slice's entries (up to 1024: 55 exchanges), so that a list costs its
    // length and not its square (1 x 2048: 1024 entries of one token 27 us, of different ones 13; walking the list for every entry took 75 ms and 40 us).
    if (k > 1) {
        int P = 2;
        while (P < k) P *= 2;
        for (int e = k + tid; e < P; e += THREADS) b_at[e] = 0xffffffffu;
        for (int size = 2; size <= P; size *= 2)
            for (int half = size / 2; half > 0; half /= 2) {
                __syncthreads();
                for (int t = tid; t < P / 2; t += THREADS) {
                    const int x = 2 * t - (t & (half - 1)), y = x + half;
                    const uint32_t wx = b_at[x], wy = b_at[y];
                    if ((wx > wy) == !(x & size)) {
                        const float vx = b_val[x], vy = b_val[y];
                        b_at[x] = wy; b_at[y] = wx;
                        b_val[x] = vy; b_val[y] = vx;
                    }
                }
            }
        __syncthreads();
    }
    // the first entry at or behind this offset
    auto entry = [&](int offset) {
        int lo = 0, hi = k;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (b_at[mid] >> 10 < (uint32_t)offset) lo = mid + 1; else hi = mid;
        }
        return lo;
    };
    auto finish = [&](float x, uint32_t c, int i) {
        const uint32_t g = c & ~(kSeen | kBiased);
        if ((c & ~kBiased) && rep != 1.f) x = x > 0.f ? x / rep : x * rep;
        if (g) x -= freq * (float)g + pres;
        if (c & kBiased) {                                      // a token listed more than once gets the sum, in the order of the row's list
            const int end = entry(i + 1);
            float sum = 0.f;
#pragma unroll 8
            for (int e = entry(i); e < end; ++e) sum += b_val[e];
            x += sum;
        }
        return x;
    };
#pragma unroll
    for (int j = 0; j < PER; j += VEC ? 4 : 1) {
        const int i = at(j);
        if (i >= n) continue;
        if constexpr (VEC) {
            const u32x4 c = *(const u32x4*)(cnt + i);
            const uint32_t w = bits ? bits[(t0 + i) >> 5] >> ((t0 + i) & 31) : 15u;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (c[q]) l[j + q] = finish(l[j + q], c[q], i + q);
                if (!((w >> q) & 1u)) l[j + q] = -INFINITY;
            }
            if (i + 4 <= n) *(f32x4*)(out + i) = (f32x4){l[j], l[j + 1], l[j + 2], l[j + 3]};
            else {
#pragma unroll
                for (int q = 0; q < 4; ++q) if (i + q < n) out[i + q] = l[j + q];
            }
        } else {
            if (cnt[i]) l[j] = finish(l[j], cnt[i], i);
            out[i] = !bits || ((bits[(t0 + i) >> 5] >> ((t0 + i) & 31)) & 1u) ? l[j] : -INFINITY;
        }
    }
}

}  // namespace

extern "C" int mc_logits_process_f32(const mc_logits_args* a, void* stream) {
    MC_CHECK_ARG(a && a->logits && a->out, "mc_logits_process_f32: null pointer");
    MC_CHECK_ARG(a->M >= 0 && a->M < 65536 && a->V > 0 && a->V <= (1 << 30), "mc_logits_process_f32: bad shape M=%d V=%d", a->M, a->V);
    MC_CHECK_ARG(a->M <= 1 || (a->ld >= a->V && a->ld_out >= a->V), "mc_logits_process_f32: rows overlap");
    MC_CHECK_ARG((!a->prompt_ids || (a->prompt_cols >= 0 && a->prompt_cols <= (1 << 30))) && (!a->output_ids || (a->output_cols >= 0 && a->output_cols <= (1 << 30))),
                 "mc_logits_process_f32: negative or overlong history");
    MC_CHECK_ARG(!a->bias_ids || (a->bias && a->n_bias >= 0 && a->n_bias <= kMaxBias), "mc_logits_process_f32: %d biases per row (at most 1024)", a->n_bias);
    if (a->M == 0) return 0;
    mc_logits_args b = *a;
    if (!b.bias_ids) b.n_bias = 0;
    if (!b.prompt_ids) b.prompt_cols = 0;
    if (!b.output_ids) b.output_cols = 0;
    hipStream_t s = (hipStream_t)stream;
    const bool vec = ((uintptr_t)b.logits | (uintptr_t)b.out) % 16 == 0 && (b.M == 1 || (b.ld | b.ld_out) % 4 == 0);
    // large slices as soon as they fill the chip (each reads the whole history; 64 x 131072: 21 us, with 8192 tokens 26, with 1024 threads 29), small ones for few rows
    // (1 x 32000: 4.2 us, with 256 threads 4.6)
    const int large = (b.V + 4095) / 4096, small = (b.V + 511) / 512;
    if ((int64_t)b.M * large < 256) logits_process_kernel<512, 512, false><<<dim3(small, b.M), 512, 0, s>>>(b);
    else if (vec) logits_process_kernel<512, 4096, true><<<dim3(large, b.M), 512, 0, s>>>(b);
    else logits_process_kernel<512, 4096, false><<<dim3(large, b.M), 512, 0, s>>>(b);
    MC_CHECK_LAUNCH();
    return 0;
}
