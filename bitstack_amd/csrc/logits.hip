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

// A workgroup counts the request's tokens of its span in LDS.  Its logits, which it requests before all else, go out as they came (bits, not values) but for those that are not allowed and those with a
// count or a bias, which are a few of many: a lane takes one of its eight after the other.  Tokens with a bias are marked in a bit array, and the whole wave looks one up in the request's list, 64
// entries at a time.
// What bounds it is the chain of a workgroup (row -> request -> text -> counts -> out), which the others of a CU hide in part: 384 rows of 128256 with texts of 3000, 197 MB of logits and the texts from the
// L2, 61 us (with texts of 500 49; a copy of as much 40), 200 rows of 50000 17, one row 5.9 (a launch).  Every logit computed, as if it had a count, takes 90 % of the vector units: 54 and 19 where this takes
// 49 and 17, but 10 instead of 13 for 32 rows of 32000 with texts of 20000.  In spans of half as many logits 80, of twice as many 67; 256 threads 71, 1024 58, but 200 rows then 20 (fewer at once).
// Rows one after another in a workgroup, the next one's logits requested ahead and a request's counts kept: 91, on registers for half as many workgroups.
template <bool PENALTIES, bool BIAS>
__global__ __launch_bounds__(THREADS) void logits_adjust_kernel(const adjust_args a) {
    __shared__ __attribute__((aligned(16))) uint32_t counts[PENALTIES ? SPAN : 4];
    __shared__ uint32_t marked[BIAS ? SPAN / 32 : 1];
    const int row = (int)(blockIdx.x / a.spans), from = (int)(blockIdx.x - (unsigned)row * a.spans) * SPAN, tid = threadIdx.x, lane = tid & 63;
    const half_t *x = a.logits + row * a.ld;
    half_t *y = a.out + row * a.ld_out;
    const bool whole = ((uintptr_t)x | (uintptr_t)y) % 16 == 0;
    uint4_t in[RUNS];                            // eight halves
#pragma unroll
    for (int n = 0; n < RUNS; n++) {
        const int i = from + n * RUN + 8 * tid;
        if (whole && i + 8 <= a.V) in[n] = *reinterpret_cast<const uint4_t *>(x + i);
        else {
            half8_t v = (half8_t)(half_t)0;
            for (int e = 0; e < 8; e++)
                if (i + e < a.V) v[e] = x[i + e];
            in[n] = __builtin_bit_cast(uint4_t, v);
        }
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
    const bool biased = BIAS && known;
    if (PENALTIES && known) {
        const int length = a.history_lengths ? a.history_lengths[b] : a.most, prompt = a.prompt_lengths ? a.prompt_lengths[b] : 0;
        if (a.repetition) repetition = a.repetition[b];
        if (a.frequency) frequency = a.frequency[b];
        if (a.presence) presence = a.presence[b];
        if (!(repetition > 0.f)) repetition = 1.f;
        counted = repetition != 1.f || frequency != 0.f || presence != 0.f;
        if (counted) {
            if (BIAS && tid < SPAN / 32) marked[tid] = 0;
#pragma unroll
            for (int i = 0; i < SPAN / 4 / THREADS; i++) *reinterpret_cast<uint4_t *>(&counts[4 * (tid + i * THREADS)]) = (uint4_t)0u;
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
        uint4_t o = in[n];
        if (counted || biased) {
            const uint32_t with_bias = biased ? marked[t0 >> 5] >> (t0 & 31) & 0xff : 0;
            uint32_t todo = with_bias;
            if (counted) {
                const uint4_t lo = *reinterpret_cast<const uint4_t *>(&counts[t0]), hi = *reinterpret_cast<const uint4_t *>(&counts[t0 + 4]);
#pragma unroll
                for (int e = 0; e < 4; e++) todo |= (lo[e] != 0 ? 1u << e : 0) | (hi[e] != 0 ? 16u << e : 0);
            }
            while (__any(todo != 0)) {           // (all lanes: some may have none left)
                const int e = todo != 0 ? __builtin_ctz(todo) : 0;
                const uint32_t pair = e < 4 ? (e < 2 ? o[0] : o[1]) : (e < 6 ? o[2] : o[3]);
                float v = (float)__builtin_bit_cast(half_t, (uint16_t)(pair >> 16 * (e & 1)));
                bool finite = __builtin_isfinite(v);
                if (counted) {
                    const uint32_t c = counts[t0 + e], said = c & ~PROMPT;
                    if (c != 0) v = v > 0.f ? v / repetition : v * repetition;
                    if (said != 0) v = v - frequency * (float)said - presence;
                }
                if (biased) {
                    const bool mine = todo != 0 && (with_bias >> e & 1);
                    for (uint64_t who = __ballot(mine); who != 0; who &= who - 1) {
                        const int leader = __builtin_ctzll(who);
                        const int32_t token = __builtin_amdgcn_readlane(i0 + e, leader);
                        int last = -1;           // (of several entries for a token the last counts)
                        for (int j0 = 0; j0 < a.biases; j0 += 64) {
                            const uint64_t here = __ballot(j0 + lane < a.biases && tokens[j0 + lane] == token);
                            if (here != 0) last = j0 + 63 - __builtin_clzll(here);
                        }
                        const float w = a.bias[(int64_t)b * a.biases + last];
                        if (lane == leader) {
                            v += w;
                            finite = finite && __builtin_isfinite(w);
                        }
                    }
                }
                if (finite) v = fminf(fmaxf(v, -65504.f), 65504.f);
                const uint32_t half = __builtin_bit_cast(uint16_t, (half_t)v), keep = e & 1 ? 0xffffu : 0xffff0000u, put = half << 16 * (e & 1);
                if (todo != 0) {
                    o[0] = e >> 1 == 0 ? (o[0] & keep) | put : o[0];
                    o[1] = e >> 1 == 1 ? (o[1] & keep) | put : o[1];
                    o[2] = e >> 1 == 2 ? (o[2] & keep) | put : o[2];
                    o[3] = e >> 1 == 3 ? (o[3] & keep) | put : o[3];
                }
                todo &= todo - 1;
            }
        }
        if (allowed) {
            constexpr uint32_t LOW = 0xfc00u;    // -inf
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const uint32_t lo = bits[n] >> 2 * d & 1 ? o[d] : LOW, hi = bits[n] >> (2 * d + 1) & 1 ? o[d] : LOW << 16;
                o[d] = (lo & 0xffffu) | (hi & 0xffff0000u);
            }
        }
        if (whole && i0 + 8 <= a.V) *reinterpret_cast<uint4_t *>(y + i0) = o;
        else {
            const half8_t h = __builtin_bit_cast(half8_t, o);
            for (int e = 0; e < 8; e++)
                if (i0 + e < a.V) y[i0 + e] = h[e];
        }
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
