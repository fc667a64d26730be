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
// HBM-bound at batch, latency-bound for one row.  A workgroup owns a slice of the vocabulary: it counts the row's tokens that fall into the slice in LDS
// (integer atomics: the order cannot change the result), then streams the slice once.  Every slice reads the whole history, from the L2 after
// the first; in exchange there is no workspace, no second launch and no atomic on memory.
#include "common.h"

namespace {

constexpr int kSlice = 2048;
constexpr uint32_t kSeen = 0x80000000u;                        // prompt tokens set this bit, generated ones count below it

__global__ __launch_bounds__(256) void logits_process_kernel(mc_logits_args a) {
    __shared__ uint32_t cnt[kSlice];
    __shared__ float bias[kSlice];
    const int row = blockIdx.y, t0 = blockIdx.x * kSlice, n = min(kSlice, a.V - t0), tid = threadIdx.x;
    for (int i = tid; i < n; i += 256) { cnt[i] = 0; bias[i] = 0.f; }
    __syncthreads();
    if (a.prompt_ids) {
        const int len = a.prompt_lens ? min(a.prompt_lens[row], a.prompt_cols) : a.prompt_cols;
        const int64_t* ids = a.prompt_ids + row * a.ld_prompt;
        for (int i = tid; i < len; i += 256) {
            const int64_t t = ids[i] - t0;
            if (t >= 0 && t < n) atomicOr(&cnt[t], kSeen);
        }
    }
    if (a.output_ids) {
        const int len = a.output_lens ? min(a.output_lens[row], a.output_cols) : a.output_cols;
        const int64_t* ids = a.output_ids + row * a.ld_output;
        for (int i = tid; i < len; i += 256) {
            const int64_t t = ids[i] - t0;
            if (t >= 0 && t < n) atomicAdd(&cnt[t], 1u);
        }
    }
    if (a.bias_ids) {
        // a token listed twice gets the sum, added by its first entry in list order: no float atomics
        const int32_t* ids = a.bias_ids + row * a.ld_bias;
        const float* val = a.bias + row * a.ld_bias;
        for (int i = tid; i < a.n_bias; i += 256) {
            const int id = ids[i];
            if (id < t0 || id >= t0 + n) continue;
            float s = 0.f;
            bool first = true;
            for (int j = 0; j < a.n_bias; ++j) {
                if (ids[j] != id) continue;
                if (j < i) { first = false; break; }
                s += val[j];
            }
            if (first) bias[id - t0] = s;
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.f, pres = a.presence ? a.presence[row] : 0.f, freq = a.frequency ? a.frequency[row] : 0.f;
    const float* in = a.logits + row * a.ld + t0;
    float* out = a.out + row * a.ld_out + t0;
    const uint32_t* bits = a.allowed ? (const uint32_t*)a.allowed + row * a.ld_allowed : nullptr;
    for (int i = tid; i < n; i += 256) {
        float l = in[i];
        const uint32_t c = cnt[i];
        if (c) {
            if (rep != 1.f) l = l > 0.f ? l / rep : l * rep;
            const uint32_t g = c & ~kSeen;
            if (g) l -= freq * (float)g + pres;
        }
        if (a.bias_ids) l += bias[i];
        if (bits && !((bits[(t0 + i) >> 5] >> ((t0 + i) & 31)) & 1u)) l = -INFINITY;
        out[i] = l;
    }
}

}  // namespace

extern "C" int mc_logits_process_f32(const mc_logits_args* a, void* stream) {
    MC_CHECK_ARG(a && a->logits && a->out, "mc_logits_process_f32: null pointer");
    MC_CHECK_ARG(a->M >= 0 && a->V > 0 && a->M < 65536, "mc_logits_process_f32: bad shape M=%d V=%d", a->M, a->V);
    MC_CHECK_ARG(a->M <= 1 || (a->ld >= a->V && a->ld_out >= a->V), "mc_logits_process_f32: rows overlap");
    MC_CHECK_ARG((!a->prompt_ids || a->prompt_cols >= 0) && (!a->output_ids || a->output_cols >= 0), "mc_logits_process_f32: negative history length");
    MC_CHECK_ARG(!a->bias_ids || (a->bias && a->n_bias >= 0 && a->n_bias <= 4096), "mc_logits_process_f32: %d biases per row (at most 4096)", a->n_bias);
    if (a->M == 0) return 0;
    logits_process_kernel<<<dim3((a->V + kSlice - 1) / kSlice, a->M), 256, 0, (hipStream_t)stream>>>(*a);
    MC_CHECK_LAUNCH();
    return 0;
}
