// The next token of every row from its logits, with temperature, top-k, top-p and min-p, from a random number that is given.
//
//   w_i = exp((x_i - max) / T)                     in 64 bits: a random number next to a border of a large vocabulary is decided by 1e-9 of the sum
//   top-k   the k largest; among equals the lowest indexes
//   top-p   of those, in the same order, the ones whose larger ones sum to less than p times the sum
//   min-p   of those, the ones with w_i >= min-p (the largest weight is 1)
//   token   the lowest index whose sum of kept weights up to it is more than u times the sum of all kept
//
// Weights are summed as whole numbers in units of 2^-44: the order of the parts then changes nothing (2^18 weights of up to one fit 63 bits, and what the
// unit cuts off is 2^-45 per weight).  fp16 values are compared by their bits in the order of the numbers (a key of 16 bits): a border is found by counting, the
// upper 12 bits of all keys first, then the lower four of the keys that share the border's, and it is a key and the number of tokens with
// that key that stay.  No sorting, and a sum over tokens with one key is a product.
#include "common.h"

namespace {

constexpr int SP_THREADS = 1024, SP_WAVES = SP_THREADS / 64, SP_BINS = 4096, SP_MAX_V = 1 << 18;
constexpr int SP_SPANS = SP_MAX_V / 512 + 1;     // spans of 64 pieces of eight values
constexpr int SP_UNIT = 44;
constexpr double SP_ONE = (double)(1ull << SP_UNIT);
typedef unsigned long long u64;
typedef uint16_t ushort8_t __attribute__((ext_vector_type(8)));

// 2^(y / 32) in units of 2^-44, y <= 0: the table's 2^(j / 32) times a polynomial of degree five for the rest (relative error below 1e-14)
__device__ __forceinline__ double sp_exp2(const double *table, double y) {
    const double n = __builtin_rint(y), r = (y - n) * 0.021660849392498290;       // ln(2) / 32
    const int k = (int)n;
    double p = 1.0 / 120;
    p = __builtin_fma(p, r, 1.0 / 24);
    p = __builtin_fma(p, r, 1.0 / 6);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return ldexp(table[k & 31] * p, (k >> 5) + SP_UNIT);
}
__device__ __forceinline__ u64 sp_whole(double v) {       // the nearest whole number of 0 <= v <= 2^44
    return __builtin_bit_cast(u64, v + 4503599627370496.0) & ((1ull << 52) - 1);
}

// exclusive sum over the workgroup, and the whole one; `to` is free again behind the next barrier
template <typename T>
__device__ __forceinline__ T sp_before(T v, T *to, T &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T below = __shfl_up(s, o, 64);
        if (lane >= o) s += below;
    }
    if (lane == 63) to[wave] = s;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < SP_WAVES; w++) {
        if (w == wave) before = total;
        total += to[w];
    }
    return before + s - v;
}

// The row's values as keys, eight at a time: 0 what has no weight (-inf, NaN, in front of the row or behind it), otherwise the bits in the order of
// the numbers, +0 and -0 alike.  Pieces lie on 16 bytes, so the first and the last may be partial.
struct sp_row {
    const half_t *x;
    int V, ahead;                                // values of the first piece in front of the row
    __device__ __forceinline__ int pieces() const { return (V + ahead + 7) / 8; }
    __device__ __forceinline__ int index(int piece, int e) const { return 8 * piece + e - ahead; }
    __device__ __forceinline__ ushort8_t keys(int piece) const {
        half8_t v;
        const int at = 8 * piece - ahead;
        if (at >= 0 && at + 8 <= V) {
            v = *reinterpret_cast<const half8_t *>(x + at);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = at + e >= 0 && at + e < V ? x[at + e] : (half_t)-INFINITY;
        }
        const ushort8_t raw = __builtin_bit_cast(ushort8_t, v);
        ushort8_t k;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint16_t bits = raw[e], size = bits & 0x7fff;
            const uint16_t key = bits & 0x8000 ? 0x8000 - size : 0x8000 + size;
            k[e] = size > 0x7c00 || bits == 0xfc00 ? 0 : key;
        }
        return k;
    }
};
__device__ __forceinline__ double sp_value(int key) {
    const uint16_t bits = key >= 0x8000 ? key - 0x8000 : 0x8000 | (0x8000 - key);
    return (double)(float)__builtin_bit_cast(half_t, bits);
}

__global__ __launch_bounds__(SP_THREADS) void sample_kernel(const half_t *__restrict__ logits, int64_t ld, const float *__restrict__ uniform,
                                                            const float *__restrict__ temperature, const int32_t *__restrict__ top_k,
                                                            const float *__restrict__ top_p, const float *__restrict__ min_p, int64_t *__restrict__ out, int V) {
    __shared__ uint32_t count[SP_BINS];
    __shared__ u64 mass[SP_BINS], span[SP_SPANS], part[SP_WAVES], weight16[16], found_sum[2], found_mass[2];
    __shared__ uint32_t part32[SP_WAVES], count16[16];
    __shared__ double table[32];
    __shared__ int found[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
    sp_row row;
    row.x = logits + b * ld;
    row.V = V;
    row.ahead = (int)((reinterpret_cast<uintptr_t>(row.x) & 15) / 2);
    const int pieces = row.pieces(), spans = (pieces + 63) / 64;
    if (tid < 32) table[tid] = exp2((double)tid / 32.0);

    // ---- the largest
    uint32_t best = 0;
    for (int c = tid; c < pieces; c += SP_THREADS) {
        const ushort8_t k = row.keys(c);
#pragma unroll
        for (int e = 0; e < 8; e++) best = max(best, (uint32_t)k[e]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) best = max(best, (uint32_t)__shfl_xor(best, o, 64));
    if (lane == 0) part32[wave] = best;
    __syncthreads();
    for (int w = 0; w < SP_WAVES; w++) best = max(best, part32[w]);
    const int top = (int)best;
    if (top == 0) {                              // nothing but -inf and NaN
        if (tid == 0) out[b] = 0;
        return;
    }
    const float T = temperature ? temperature[b] : 1.f;
    const bool greedy = !(T > 0.f);
    const double largest = sp_value(top), scale = 32.0 * 1.4426950408889634074 / (double)T;
    auto weight = [&](int key) -> double {       // in units of 2^-44
        if (key == top) return SP_ONE;
        const double y = (sp_value(key) - largest) * scale;
        return y > -32.0 * (SP_UNIT + 2) ? sp_exp2(table, y) : 0.0;
    };
    // The lowest index whose sum of value(key, index) up to it is more than `share` of (whole sum - less); every thread gets it (-1: all are zero).
    // A span of 512 values is one wave's: spans are summed, then the one in which it lies is gone through.
    auto nth = [&](auto value, auto target) -> int {
        __syncthreads();
        for (int s = wave; s < spans; s += SP_WAVES) {
            const int c = s * 64 + lane;
            u64 sum = 0;
            if (c < pieces) {
                const ushort8_t k = row.keys(c);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (k[e]) sum += value((int)k[e], row.index(c, e));
            }
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
            if (lane == 0) span[s] = sum;
        }
        if (tid == 0) { found[0] = -1; found[1] = -1; }
        __syncthreads();
        const u64 mine = tid < spans ? span[tid] : 0;
        static_assert(SP_SPANS <= SP_THREADS, "one span per thread");
        u64 total;
        const u64 before = sp_before(mine, part, total);
        const double goal = target(total);
        if (mine && (double)before <= goal && (double)(before + mine) > goal) {
            found[0] = tid;
            found_sum[0] = before;
        }
        __syncthreads();
        if (found[0] >= 0 && wave == 0) {
            const int c = found[0] * 64 + lane;
            u64 w[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = 0;
            if (c < pieces) {
                const ushort8_t k = row.keys(c);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (k[e]) w[e] = value((int)k[e], row.index(c, e));
                    sum += w[e];
                }
            }
            u64 s = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 below = __shfl_up(s, o, 64);
                if (lane >= o) s += below;
            }
            u64 at = found_sum[0] + s - sum;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (w[e] && (double)at <= goal && (double)(at + w[e]) > goal) found[1] = row.index(c, e);
                at += w[e];
            }
        }
        __syncthreads();
        return found[1];
    };
    if (greedy) {
        const int at = nth([&](int key, int) -> u64 { return key == top; }, [](u64) { return 0.0; });
        if (tid == 0) out[b] = at;
        return;
    }

    // ---- top-k and top-p: the key at the border, and how many tokens with that key stay
    const int k = top_k ? top_k[b] : 0;
    const double p = top_p ? (double)top_p[b] : 1.0;
    const bool by_count = k > 0 && k < V, by_sum = p < 1.0;
    int least = 1, last_index = V - 1;           // the border, and the last index with that key that stays
    if (by_count || by_sum) {
        for (int i = tid; i < SP_BINS; i += SP_THREADS) {
            count[i] = 0;
            mass[i] = 0;
        }
        if (tid == 0) { found[2] = found[3] = -1; }
        __syncthreads();
        for (int c = tid; c < pieces; c += SP_THREADS) {
            const ushort8_t key = row.keys(c);
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (key[e]) {
                    atomicAdd(&count[key[e] >> 4], 1u);
                    if (by_sum) atomicAdd(&mass[key[e] >> 4], sp_whole(weight(key[e])));
                }
        }
        __syncthreads();
        // bins from the top, four per thread
        uint32_t n4 = 0;
        u64 m4 = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            n4 += count[SP_BINS - 1 - 4 * tid - i];
            m4 += mass[SP_BINS - 1 - 4 * tid - i];
        }
        uint32_t all_count;
        u64 all_mass;
        const uint32_t n_before = sp_before(n4, part32, all_count);
        const u64 m_before = sp_before(m4, part, all_mass);
        int bin_k = -1;
        u64 limit = all_mass;                    // the sum that top-k leaves
        uint32_t stay = 0;                       // tokens with the border's key that stay, of `those`
        uint32_t those = 0;
        // the 16 keys of a bin: how many tokens each, and their weight
        auto look_into = [&](int bin) {
            __syncthreads();
            if (tid < 16) {
                count16[tid] = 0;
                weight16[tid] = bin * 16 + tid <= top && bin * 16 + tid >= 1 ? sp_whole(weight(bin * 16 + tid)) : 0;
            }
            __syncthreads();
            for (int c = tid; c < pieces; c += SP_THREADS) {
                const ushort8_t key = row.keys(c);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (key[e] && key[e] >> 4 == bin) atomicAdd(&count16[key[e] & 15], 1u);
            }
            __syncthreads();
        };
        if (by_count && all_count > (uint32_t)k) {
            uint32_t n = n_before;
            u64 m = m_before;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int bin = SP_BINS - 1 - 4 * tid - i;
                if (n < (uint32_t)k && n + count[bin] >= (uint32_t)k) {
                    found[2] = bin;
                    found_sum[0] = n;
                    found_mass[0] = m;
                }
                n += count[bin];
                m += mass[bin];
            }
            __syncthreads();
            bin_k = found[2];
            look_into(bin_k);
            uint32_t at = (uint32_t)found_sum[0];
            limit = found_mass[0];
            for (int j = 15; j >= 0; j--) {      // (every thread the same)
                const uint32_t c = count16[j], take = min(c, (uint32_t)k - at);
                if (c) {
                    limit += take * weight16[j];
                    at += take;
                    least = bin_k * 16 + j;
                    stay = take;
                    those = c;
                }
                if (at == (uint32_t)k) break;
            }
        }
        if (by_sum) {
            const double goal = fmax(p * (double)limit, 0.5);       // (the largest always stays)
            u64 m = m_before;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int bin = SP_BINS - 1 - 4 * tid - i;
                if ((double)m < goal && (double)(m + mass[bin]) >= goal) {
                    found[3] = bin;
                    found_mass[1] = m;
                }
                m += mass[bin];
            }
            __syncthreads();
            const int bin_p = found[3];
            if (bin_p >= 0) {
                if (bin_p != bin_k) look_into(bin_p);
                u64 at = found_mass[1];
                for (int j = 15; j >= 0; j--) {
                    const uint32_t c = count16[j];
                    const u64 w = weight16[j];
                    if (c == 0 || w == 0) continue;
                    if (bin_p * 16 + j < least) break;              // (top-k's border comes first)
                    if ((double)(at + c * w) >= goal) {
                        const double need = ceil((goal - (double)at) / (double)w);
                        const uint32_t take = need < 1.0 ? 1 : need > (double)c ? c : (uint32_t)need;
                        stay = bin_p * 16 + j == least ? min(stay, take) : take;
                        least = bin_p * 16 + j;
                        those = c;
                        break;
                    }
                    at += c * w;
                }
            }
        }
        if (stay < those) {                      // some of the tokens with the border's key go: those with the highest indexes
            const int at = least;
            last_index = nth([&](int key, int) -> u64 { return key == at; }, [&](u64) { return (double)stay - 1.0; });
        }
    }

    // ---- min-p and the draw
    const double floor_w = min_p && min_p[b] > 0.f ? (double)fminf(min_p[b], 1.f) * SP_ONE : 0.0;       // (the largest always stays)
    float u = uniform[b];
    u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
    const int token = nth([&](int key, int index) -> u64 {
        if (key < least || (key == least && index > last_index)) return 0;
        const double w = weight(key);
        return w >= floor_w ? sp_whole(w) : 0;
    }, [&](u64 total) { return (double)u * (double)total; });
    if (tid == 0) out[b] = token;
}

}  // namespace

int bs_launch_sample(const half_t *logits, int64_t ld, const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                     int64_t *out, int B, int V, hipStream_t s) {
    if (V > SP_MAX_V) return BS_ERR_SHAPE;
    sample_kernel<<<B, SP_THREADS, 0, s>>>(logits, ld, uniform, temperature, top_k, top_p, min_p, out, V);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
