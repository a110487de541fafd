// Settings on logits in front of the draw: penalties for tokens that a request has in its text, biases, and the tokens that a grammar allows.
#include "lanes.h"

namespace {

constexpr int THREADS = 512, SPAN = THREADS * 8;           // tokens of the vocabulary that a workgroup takes
constexpr uint32_t PROMPT = 1u << 31;                      // in a count: the token is in the prompt

struct adjust_args {
    const half_t *logits;
    half_t *out;
    int64_t ld, ld_out;
    const int32_t *requests, *history, *history_lengths, *prompt_lengths;
    const float *repetition, *frequency, *presence;
    const int32_t *drafted, *bias_tokens;
    const float *bias;
    const uint8_t *allowed;
    const int32_t *allowed_rows;
    int first, V, B, most, path, biases, masks, spans;       // (first: the launch's first row)
    int64_t mask_bytes;
};

// A workgroup counts the request's tokens of its span in LDS, and walks its logits once.
template <bool PENALTIES, bool BIAS>
__global__ __launch_bounds__(THREADS) void logits_adjust_kernel(const adjust_args a) {
    __shared__ uint32_t counts[PENALTIES ? SPAN : 1], entry[BIAS ? SPAN : 1];
    const int local = (int)(blockIdx.x / a.spans), from = (int)(blockIdx.x - (unsigned)local * a.spans) * SPAN, row = a.first + local, tid = threadIdx.x;
    int b = a.requests ? a.requests[row] : row;
    const bool known = b >= 0 && b < a.B;
    b = known ? b : 0;
    float repetition = 1.f, frequency = 0.f, presence = 0.f;
    bool counted = false, biased = false;
    if (PENALTIES && known) {
        if (a.repetition) repetition = a.repetition[b];
        if (!(repetition > 0.f)) repetition = 1.f;
        if (a.frequency) frequency = a.frequency[b];
        if (a.presence) presence = a.presence[b];
        counted = repetition != 1.f || frequency != 0.f || presence != 0.f;
        if (counted) {
#pragma unroll
            for (int i = 0; i < 8; i++) counts[tid + i * THREADS] = 0;
        }
    }
    if (BIAS && known) {
        biased = true;
#pragma unroll
        for (int i = 0; i < 8; i++) entry[tid + i * THREADS] = 0;
    }
    if (counted || biased) __syncthreads();
    if (counted) {
        const int n = min(max(a.history_lengths ? a.history_lengths[b] : a.most, 0), a.most), prompt = a.prompt_lengths ? a.prompt_lengths[b] : 0;
        const int32_t *text = a.history + (int64_t)b * a.most;
        for (int i = tid; i < n; i += THREADS) {
            const uint32_t t = (uint32_t)text[i] - (uint32_t)from;
            if (t < (uint32_t)SPAN) {
                if (i < prompt) atomicOr(&counts[t], PROMPT);
                else atomicAdd(&counts[t], 1u);
            }
        }
        const int32_t *path = a.drafted + (int64_t)row * a.path;
        for (int i = tid; i < a.path; i += THREADS) {
            const uint32_t t = (uint32_t)path[i] - (uint32_t)from;
            if (t < (uint32_t)SPAN) atomicAdd(&counts[t], 1u);
        }
    }
    if (biased) {
        const int32_t *tokens = a.bias_tokens + (int64_t)b * a.biases;
        for (int i = tid; i < a.biases; i += THREADS) {
            const uint32_t t = (uint32_t)tokens[i] - (uint32_t)from;
            if (t < (uint32_t)SPAN) atomicMax(&entry[t], (uint32_t)i + 1);       // (the last entry of a token counts)
        }
    }
    if (counted || biased) __syncthreads();
    const int state = a.allowed ? (a.allowed_rows ? a.allowed_rows[row] : row) : -1;
    const uint8_t *allowed = state >= 0 && state < a.masks ? a.allowed + (int64_t)state * a.mask_bytes : nullptr;
    const half_t *x = a.logits + row * a.ld;
    half_t *y = a.out + row * a.ld_out;
    auto one = [&](half_t in, int t, bool fits) {          // the logit of token from + t
        float v = (float)in;
        bool finite = __builtin_isfinite(v);
        if (counted) {
            const uint32_t c = counts[t], said = c & ~PROMPT;
            if (c != 0) v = v > 0.f ? v / repetition : v * repetition;
            if (said != 0) v = v - frequency * (float)said - presence;
        }
        if (biased) {
            const uint32_t e = entry[t];
            if (e != 0) {
                const float w = a.bias[(int64_t)b * a.biases + e - 1];
                v += w;
                finite = finite && __builtin_isfinite(w);
            }
        }
        if (finite) v = fminf(fmaxf(v, -65504.f), 65504.f);
        return fits ? (half_t)v : (half_t)-INFINITY;
    };
    const int t0 = 8 * tid, i0 = from + t0;
    if (i0 >= a.V) return;
    const uint32_t bits = allowed ? allowed[i0 >> 3] : 0xffu;
    if (((uintptr_t)x | (uintptr_t)y) % 16 == 0 && i0 + 8 <= a.V) {
        const half8_t in = *reinterpret_cast<const half8_t *>(x + i0);
        half8_t o;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = one(in[e], t0 + e, bits >> e & 1);
        *reinterpret_cast<half8_t *>(y + i0) = o;
    } else {
        for (int e = 0; e < 8 && i0 + e < a.V; e++) y[i0 + e] = one(x[i0 + e], t0 + e, bits >> e & 1);
    }
}

}  // namespace

int bs_launch_logits_adjust(const half_t *logits, int64_t ld, half_t *out, int64_t ld_out, const int32_t *requests, const int32_t *history, const int32_t *history_lengths,
                            const int32_t *prompt_lengths, const float *repetition, const float *frequency, const float *presence, const int32_t *drafted,
                            const int32_t *bias_tokens, const float *bias, const int32_t *allowed, const int32_t *allowed_rows, int rows, int V, int B, int most, int path,
                            int biases, int masks, hipStream_t s) {
    const int spans = (int)bs_cdiv(V, SPAN), per = (1 << 23) / spans;     // rows of a launch: a grid holds 2^32 threads
    const bool penalties = (history || drafted) && (repetition || frequency || presence), biased = bias_tokens && biases > 0;
    auto *kernel = penalties ? (biased ? logits_adjust_kernel<true, true> : logits_adjust_kernel<true, false>)
                             : (biased ? logits_adjust_kernel<false, true> : logits_adjust_kernel<false, false>);
    for (int r = 0; r < rows; r += per) {
        const int n = rows - r < per ? rows - r : per;
        const adjust_args a = {logits, out, ld, ld_out, requests, history, history_lengths, prompt_lengths, repetition, frequency, presence, drafted, bias_tokens, bias,
                               (const uint8_t *)allowed, allowed_rows, r, V, B, history ? most : 0, drafted ? path : 0, biases, masks, spans, 4 * bs_cdiv(V, 32)};
        kernel<<<(unsigned)((int64_t)n * spans), THREADS, 0, s>>>(a);
        BS_LAUNCH_CHECK();
    }
    return BS_OK;
}
