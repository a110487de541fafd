// Settings on logits in front of the draw: penalties for tokens that a request has in its text, biases, and the tokens that a grammar allows.
#include "lanes.h"

namespace {

constexpr int THREADS = 512, RUN = THREADS * 8, RUNS = 2, SPAN = RUN * RUNS;          // tokens of the vocabulary that a workgroup takes: eight in a row to a thread, twice
constexpr int BATCH = 8;                                   // tokens of the text that a thread requests at once
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
    int V, B, most, path, biases, masks, spans;
    int64_t mask_bytes;
};

// A workgroup counts the request's tokens of its span in LDS, and walks its logits once, which it requests before all else.  Tokens with a bias are a few of many: they are marked in a bit array, and a wave
// that meets one looks it up in the request's list, 64 entries at a time.
// What bounds it is the chain of a workgroup (row -> request -> text -> counts), hidden by the others of a CU, and the bytes: 384 rows of 128256 with texts of 3000, 197 MB and the texts from the L2,
// 60 us (a copy of as much 40); one row 5.8 (a launch).  One eight per thread 76, four 65, 256 threads 69, 1024 77: more workgroups read the text more often, larger ones leave a CU fewer to hide it.
template <bool PENALTIES, bool BIAS>
__global__ __launch_bounds__(THREADS) void logits_adjust_kernel(const adjust_args a) {
    __shared__ __attribute__((aligned(16))) uint32_t counts[PENALTIES ? SPAN : 4];
    __shared__ uint32_t marked[BIAS ? SPAN / 32 : 1];
    const int row = (int)(blockIdx.x / a.spans), from = (int)(blockIdx.x - (unsigned)row * a.spans) * SPAN, tid = threadIdx.x, lane = tid & 63;
    const half_t *x = a.logits + row * a.ld;
    half_t *y = a.out + row * a.ld_out;
    const bool whole = ((uintptr_t)x | (uintptr_t)y) % 16 == 0;
    half8_t in[RUNS];
#pragma unroll
    for (int n = 0; n < RUNS; n++) {
        const int i = from + n * RUN + 8 * tid;
        in[n] = (half8_t)(half_t)0;
        if (whole && i + 8 <= a.V) in[n] = *reinterpret_cast<const half8_t *>(x + i);
        else
            for (int e = 0; e < 8; e++)
                if (i + e < a.V) in[n][e] = x[i + e];
    }
    const int state = a.allowed ? (a.allowed_rows ? a.allowed_rows[row] : row) : -1;
    const uint8_t *allowed = state >= 0 && state < a.masks ? a.allowed + (int64_t)state * a.mask_bytes : nullptr;
    uint32_t bits[RUNS];
#pragma unroll
    for (int n = 0; n < RUNS; n++) {
        const int i = from + n * RUN + 8 * tid;
        bits[n] = allowed && i < a.V ? allowed[i >> 3] : 0xffu;
    }
    int b = a.requests ? a.requests[row] : row;
    const bool known = b >= 0 && b < a.B;
    b = known ? b : 0;
    float repetition = 1.f, frequency = 0.f, presence = 0.f;
    bool counted = false;
    if (PENALTIES && known) {
        const int length = a.history_lengths ? a.history_lengths[b] : a.most, prompt = a.prompt_lengths ? a.prompt_lengths[b] : 0;
        if (a.repetition) repetition = a.repetition[b];
        if (a.frequency) frequency = a.frequency[b];
        if (a.presence) presence = a.presence[b];
        if (!(repetition > 0.f)) repetition = 1.f;
        counted = repetition != 1.f || frequency != 0.f || presence != 0.f;
        if (counted) {
#pragma unroll
            for (int i = 0; i < SPAN / 4 / THREADS; i++) *reinterpret_cast<uint4_t *>(&counts[4 * (tid + i * THREADS)]) = (uint4_t)0u;
            if (BIAS && tid < SPAN / 32) marked[tid] = 0;
            __syncthreads();
            const int n = min(max(length, 0), a.most);
            const int32_t *text = a.history + (int64_t)b * a.most;
            for (int i0 = 0; i0 < n; i0 += BATCH * THREADS) {
                int32_t t[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; k++) {
                    const int i = i0 + k * THREADS + tid;
                    t[k] = i < n ? text[i] : -1;
                }
#pragma unroll
                for (int k = 0; k < BATCH; k++) {
                    const int i = i0 + k * THREADS + tid;
                    const uint32_t at = (uint32_t)t[k] - (uint32_t)from;
                    if (i >= n || at >= (uint32_t)SPAN) continue;
                    if (i < prompt) atomicOr(&counts[at], PROMPT);
                    else atomicAdd(&counts[at], 1u);
                }
            }
            const int32_t *path = a.drafted + (int64_t)row * a.path;
            for (int i = tid; i < a.path; i += THREADS) {
                const uint32_t at = (uint32_t)path[i] - (uint32_t)from;
                if (at < (uint32_t)SPAN) atomicAdd(&counts[at], 1u);
            }
        }
    }
    const bool biased = BIAS && known;
    const int32_t *tokens = a.bias_tokens + (int64_t)b * a.biases;
    if (biased) {
        if (!counted) {
            if (tid < SPAN / 32) marked[tid] = 0;
            __syncthreads();
        }
        for (int i = tid; i < a.biases; i += THREADS) {
            const uint32_t at = (uint32_t)tokens[i] - (uint32_t)from;
            if (at < (uint32_t)SPAN) atomicOr(&marked[at >> 5], 1u << (at & 31));
        }
    }
    if (counted || biased) __syncthreads();
#pragma unroll
    for (int n = 0; n < RUNS; n++) {
        const int t0 = n * RUN + 8 * tid, i0 = from + t0;
        float v[8];
        uint32_t finite = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = (float)in[n][e];
            finite |= (uint32_t)__builtin_isfinite(v[e]) << e;
        }
        if (counted) {
            uint32_t c[8];
            *reinterpret_cast<uint4_t *>(c) = *reinterpret_cast<const uint4_t *>(&counts[t0]);
            *reinterpret_cast<uint4_t *>(c + 4) = *reinterpret_cast<const uint4_t *>(&counts[t0 + 4]);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t said = c[e] & ~PROMPT;
                if (c[e] != 0) v[e] = v[e] > 0.f ? v[e] / repetition : v[e] * repetition;
                if (said != 0) v[e] = v[e] - frequency * (float)said - presence;
            }
        }
        if (biased) {
            uint32_t mine = marked[t0 >> 5] >> (t0 & 31) & 0xff;
            for (uint64_t who = __ballot(mine != 0); who != 0; who = __ballot(mine != 0)) {
                const int leader = __builtin_ctzll(who), e_of = __builtin_ctz((uint32_t)__builtin_amdgcn_readlane((int)mine, leader));
                const int32_t token = __builtin_amdgcn_readlane(i0, leader) + e_of;
                int last = -1;                   // (of several entries for a token the last counts)
                for (int j0 = 0; j0 < a.biases; j0 += 64) {
                    const uint64_t here = __ballot(j0 + lane < a.biases && tokens[j0 + lane] == token);
                    if (here != 0) last = j0 + 63 - __builtin_clzll(here);
                }
                const float w = a.bias[(int64_t)b * a.biases + last];
                const bool fine = __builtin_isfinite(w);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (lane == leader && e == e_of) {
                        v[e] += w;
                        finite &= fine ? 0xffu : ~(1u << e);
                    }
                if (lane == leader) mine &= mine - 1;
            }
        }
        half8_t o;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (finite >> e & 1) v[e] = fminf(fmaxf(v[e], -65504.f), 65504.f);
            o[e] = bits[n] >> e & 1 ? (half_t)v[e] : (half_t)-INFINITY;
        }
        if (whole && i0 + 8 <= a.V) *reinterpret_cast<half8_t *>(y + i0) = o;
        else
            for (int e = 0; e < 8; e++)
                if (i0 + e < a.V) y[i0 + e] = o[e];
    }
}

}  // namespace

int bs_launch_logits_adjust(const half_t *logits, int64_t ld, half_t *out, int64_t ld_out, const int32_t *requests, const int32_t *history, const int32_t *history_lengths,
                            const int32_t *prompt_lengths, const float *repetition, const float *frequency, const float *presence, const int32_t *drafted,
                            const int32_t *bias_tokens, const float *bias, const int32_t *allowed, const int32_t *allowed_rows, int rows, int V, int B, int most, int path,
                            int biases, int masks, hipStream_t s) {
    const int spans = (int)bs_cdiv(V, SPAN);               // (R V <= 2^33 and R <= 2^20: at most 2^21 workgroups)
    const bool penalties = (history || drafted) && (repetition || frequency || presence), biased = bias_tokens && biases > 0;
    auto *kernel = penalties ? (biased ? logits_adjust_kernel<true, true> : logits_adjust_kernel<true, false>)
                             : (biased ? logits_adjust_kernel<false, true> : logits_adjust_kernel<false, false>);
    const adjust_args a = {logits, out, ld, ld_out, requests, history, history_lengths, prompt_lengths, repetition, frequency, presence, drafted, bias_tokens, bias,
                           (const uint8_t *)allowed, allowed_rows, V, B, history ? most : 0, drafted ? path : 0, biases, masks, spans, 4 * bs_cdiv(V, 32)};
    kernel<<<(unsigned)((int64_t)rows * spans), THREADS, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
