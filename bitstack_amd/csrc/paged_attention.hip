// One new token per request over the paged cache: out = softmax(q k^T / sqrt(D)) v over the request's positions, the last of them this
// step's own, which is rotated and appended here.
//
// A unit is the up to 16 query heads of one KV head that share its rows: they are the columns of both products, so K and V are read once.
//   scores  S[position, head] = K q     16x16x32, K rows as loaded (a lane: position l % 16, dimensions 32 c + 8 (l / 16) ..); the rotated query
//                                       in two fp16 terms too, x / 2 = hi + lo / 2^11: half of it, as a rotation goes up to sqrt(2) times the largest fp16 number, and the rest
//                                       enlarged, so that it is one of fp16's full numbers whatever x is (2^-22 of x).  Up to eight heads leave columns free: those are the second
//                                       terms', and a score is the sum of two lanes; with more heads it is a product of its own.  (Rounded to fp16 the query alone put
//                                       the result's error against 64 bits from 2.0e-4, the rounding of the result, to 3.4e-4.)
//   output  O[dim, head] += V^T P       16x16x32, four positions twice: P is split into two fp16 terms and the eight k slots of a lane hold {hi, lo}
//                                       against {v, v}.  The largest weight goes in as 2^15, as far up as fp16 lets it: p = hi + lo to 2^-22 of itself down to weights
//                                       of 2^-18 of the largest, below that to 2^-40 of the largest (as 1 it would be 2^-25: a weight of e^-16 was off by 6 %)
// A lane of the scores holds positions 4 (l / 16) + i of head l % 16, which is what the second product wants of P; V needs no transposition
// either: a lane loads dimensions W r .. W r + W - 1 (r = l % 16, W = D / 16) of its four positions, and product j takes element j of each, so that its
// row r is dimension W r + j.  Maximum, sum and output are fp32, in base 2; K of the next tile of 16 positions is requested behind the scores, V behind the
// output product, the tile's page one tile further ahead.
//
// The split: the lengths are known on the device alone, so every workgroup works out from them what it is to do.  The first B workgroups of a unit take
// one request each, or the first part of it; if requests are longer than C = (all tiles) / (parts that fill the chip), the next ones take
// the further parts, in order.  (The further parts first: 172 us instead of 105 for two requests of 80000, the numbers that no part has leave gaps.)  Parts leave (max, sum, weighted v)
// in the workspace, and a second launch puts them together, in order: the result does not depend on which came first.
//
// What bounds it is the cache's bytes, at up to 6.4 TB/s (a kernel that only reads): 2 requests of 60001 and 99991, 64 heads on 8 of 128, 655 MB, 105 us and 4.7 for the parts = 6.2 TB/s; 48 of 1 to 4096, 32 on 8, 404 MB, 74 and
// 4.7 (5.5: unequal lengths, 51 % of the waves' time is waiting for memory, 32 % for the turn to issue); 200 of 100 to 1500, 16 on 16 of 64, 658 MB, 119 (5.5: for one head in use the vector units are busy 48 % with
// rotating, splitting and folding).  Short requests wait for their chain: one of 385, 32 heads on 8, 8.1 us and one of 20 5.1 in a table that is not cut; in a longer one, as a server's is, the second launch is
// there too, and heads stay together: 10.7 and 7.4.
#include "common.h"

namespace {

constexpr int PA_TILE = 16, PA_HEADS = 16;       // positions of a tile; query heads of a unit
constexpr float PA_UP = 32768.f, PA_REST = 2048.f;         // what the weights, and the second terms of the queries, are multiplied by on their way into fp16
// (us with 4 waves / 8: 48 requests of 1 to 4096, 32 heads on 8, 83.9 / 72.6; 2 of 80000, 128 on 8, 128.8 / 112.0; 16 of 100 to 8000, 32 on 2, 24.0 / 23.7; 1 of 700 11.2 / 11.7)
constexpr int WAVES = 8, THREADS = WAVES * 64;

struct pa_args {
    const half_t *qkv, *cosv, *sinv;
    half_t *kpages, *vpages;
    const int32_t *lengths;
    const int64_t *slots;
    half_t *out;
    int32_t *heads_of;                           // workspace: {first further part, further parts} of every request
    float *part;                                 // ... and what the parts leave
    int ldqkv, B, heads, kv_heads, groups, per_unit, max_pos, shift, max_pages, pool, parts, least;
};

// positions that the cache holds of a request (without its own): 0 for a length that is none
__device__ __forceinline__ int pa_cached(const pa_args &a, int len) {
    return len > 0 && len <= a.max_pos && (int64_t)len <= (int64_t)a.max_pages << a.shift ? len - 1 : 0;
}
__device__ __forceinline__ int pa_tiles(int cached) { return (cached + PA_TILE - 1) / PA_TILE; }
__device__ __forceinline__ int pa_further(int tiles, int most) { return tiles > most ? (tiles + most - 1) / most - 1 : 0; }

__device__ __forceinline__ int pa_sum(int v, int *to) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) to[threadIdx.x >> 6] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) s += to[w];
    return s;
}

// the value of the lane eight on (or back) in the row of 16
__device__ __forceinline__ float eight_on(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));    // row_ror:8
}

template <int D, int HP, bool STREAM>
__global__ __launch_bounds__(THREADS) void attention_paged_kernel(const pa_args a, const int32_t *__restrict__ table) {
    constexpr int W = D / 16, NC = D / 32, D2 = D / 2;
    typedef half_t vec_t __attribute__((ext_vector_type(W)));
    __shared__ __attribute__((aligned(16))) half_t qrot[2][HP][D];             // rotated queries, first and second terms
    __shared__ __attribute__((aligned(16))) half_t knew[D], vnew[D];           // this position's rotated k and v
    __shared__ float wm[HP][WAVES], wl[HP][WAVES];                             // per wave: running max, sum of exp
    __shared__ __attribute__((aligned(16))) float wacc[HP][WAVES][D];
    __shared__ int sums[WAVES], found[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int units = a.kv_heads * a.groups, unit = blockIdx.x % units, work = blockIdx.x / units;
    const int hk = unit % a.kv_heads, hg = unit / a.kv_heads, rep = a.heads / a.kv_heads;
    const int head0 = hk * rep + hg * a.per_unit, nh = min(a.per_unit, rep - hg * a.per_unit);

    int b = work, part = 0;
    const bool first_part = work < a.B;
    // ---- which request, which part of it
    int64_t slot = first_part ? a.slots[work] : 0;
    int most = 0, further = 0, place = 0;        // tiles of a part at most; further parts of this request, and the first one's number
    if (a.parts > 0) {
        int all = 0;
        for (int i = tid; i < a.B; i += THREADS) all += pa_tiles(pa_cached(a, a.lengths[i]));
        all = pa_sum(all, sums);
        most = max(a.least, (all + a.parts - 1) / a.parts);
        if (first_part) further = pa_further(pa_tiles(pa_cached(a, a.lengths[b])), most);
    }
    if (!first_part || further > 0) {            // numbers of the further parts: a running sum over the requests
        if (tid == 0) found[0] = -1;
        int before = 0;
        const int wanted = work - a.B;
        for (int i0 = 0; i0 < a.B; i0 += THREADS) {
            const int i = i0 + tid, mine = i < a.B ? pa_further(pa_tiles(pa_cached(a, a.lengths[i])), most) : 0;
            int s = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int below = __shfl_up(s, o, 64);
                if (lane >= o) s += below;
            }
            __syncthreads();
            if (lane == 63) sums[wave] = s;
            __syncthreads();
            int ahead = before;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                if (w < wave) ahead += sums[w];
                before += sums[w];
            }
            const int first = ahead + s - mine;
            if (first_part ? i == b : wanted >= first && wanted < first + mine) {
                found[0] = i;
                found[1] = first;
                found[2] = mine;
            }
        }
        __syncthreads();
        if (found[0] < 0) return;                // no such part
        b = __builtin_amdgcn_readfirstlane(found[0]);
        place = __builtin_amdgcn_readfirstlane(found[1]);
        further = __builtin_amdgcn_readfirstlane(found[2]);
        if (!first_part) {
            part = wanted - place + 1;
            slot = a.slots[b];
        }
    }
    const int len = a.lengths[b];
    const bool live = slot >= 0 && slot < (int64_t)a.pool << a.shift && len > 0 && len <= a.max_pos && (int64_t)len <= (int64_t)a.max_pages << a.shift;
    half_t *orow = a.out + ((int64_t)b * a.heads + head0) * D;
    if (part == 0 && unit == 0 && a.parts > 0 && tid == 0) {
        a.heads_of[2 * b] = place;
        a.heads_of[2 * b + 1] = live ? further : 0;
    }
    if (!live) {                                 // an idle row: zeros, and nothing is stored
        if (part == 0)
            for (int it = tid; it < nh * D; it += THREADS) orow[it] = (half_t)0;
        return;
    }
    const int pos = len - 1, tiles = pa_tiles(pos), parts = further + 1;
    const int t_first = (int)((int64_t)tiles * part / parts), t_end = (int)((int64_t)tiles * (part + 1) / parts);

    // ---- the rows of the cache
    const int64_t page_step = (int64_t)a.kv_heads * D << a.shift, head_at = (int64_t)hk * D << a.shift;
    half8_t k8[NC];
    vec_t v8[4];
    const int32_t *row = table + (int64_t)b * a.max_pages;
    auto page_of = [&](int t) { return row[__builtin_amdgcn_readfirstlane((t * PA_TILE) >> a.shift)]; };
    auto good = [&](int id) { return id >= 0 && id < a.pool; };       // (positions of a page that does not exist are left out)
    auto at_row = [&](int id, int t, int r) {    // rows past the last are the last again; their scores are masked
        return (int64_t)(good(id) ? id : 0) * page_step + head_at + (int64_t)(min(t * PA_TILE + r, pos - 1) & ((1 << a.shift) - 1)) * D;
    };
    auto fetch = [](const auto *p) {
        if constexpr (STREAM) return __builtin_nontemporal_load(p);
        else return *p;
    };
    auto fetch_k = [&](int id, int t) {
        const half_t *p = a.kpages + at_row(id, t, r16) + 8 * g;
#pragma unroll
        for (int c = 0; c < NC; c++) k8[c] = fetch(reinterpret_cast<const half8_t *>(p + 32 * c));
    };
    auto fetch_v = [&](int id, int t) {
#pragma unroll
        for (int i = 0; i < 4; i++) v8[i] = fetch(reinterpret_cast<const vec_t *>(a.vpages + at_row(id, t, 4 * g + i) + W * r16));
    };
    int t = t_first + wave;
    int id = 0, next_id = 0;
    if (t < t_end) id = page_of(t);
    if (t + WAVES < t_end) next_id = page_of(t + WAVES);
    // this position's own: pairs (i, i + D / 2) of the unit's queries, of k and of v
    constexpr int PAIRS = (HP + 2) * D2, EACH = (PAIRS + THREADS - 1) / THREADS;
    half_t pa[EACH], pb[EACH];
    const half_t *qh = a.qkv + (int64_t)b * a.ldqkv;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int it = tid + e * THREADS, h = it / D2, i = it % D2;
        pa[e] = pb[e] = (half_t)0;
        const int at = h < HP ? (head0 + h) * D : (a.heads + (h - HP) * a.kv_heads + hk) * D;
        if (h < HP + 2 && (h >= HP || h < nh)) {
            pa[e] = qh[at + i];
            pb[e] = qh[at + i + D2];
        }
    }
    if (t < t_end) {
        fetch_k(id, t);
        fetch_v(id, t);
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int it = tid + e * THREADS, h = it / D2, i = it % D2;
        if (h < HP + 1) {
            const float c = (float)a.cosv[(int64_t)pos * D2 + i], sn = (float)a.sinv[(int64_t)pos * D2 + i];
            const float x = (float)pa[e] * c - (float)pb[e] * sn, y = (float)pb[e] * c + (float)pa[e] * sn;
            if (h < HP) {
                const half_t x0 = (half_t)(0.5f * x), y0 = (half_t)(0.5f * y);
                qrot[0][h][i] = x0;
                qrot[0][h][i + D2] = y0;
                qrot[1][h][i] = (half_t)((0.5f * x - (float)x0) * PA_REST);
                qrot[1][h][i + D2] = (half_t)((0.5f * y - (float)y0) * PA_REST);
            } else {
                knew[i] = (half_t)x;
                knew[i + D2] = (half_t)y;
            }
        } else if (h < HP + 2) {
            vnew[i] = pa[e];
            vnew[i + D2] = pb[e];
        }
    }
    __syncthreads();
    if (part == 0 && hg == 0 && tid < D) {       // one workgroup of the KV head appends this position to the cache
        const int64_t at = (slot >> a.shift) * page_step + head_at + (slot & ((1 << a.shift) - 1)) * D + tid;
        a.kpages[at] = knew[tid];
        a.vpages[at] = vnew[tid];
    }

    // column r: first terms of head r; up to eight heads: column 8 + r the second terms
    constexpr int TERMS = HP > 8 ? 2 : 1;
    half8_t q8[TERMS][NC];
    const int column = HP > 8 ? r16 : r16 & 7;
#pragma unroll
    for (int e = 0; e < TERMS; e++)
#pragma unroll
        for (int c = 0; c < NC; c++)
            q8[e][c] = column < HP ? *reinterpret_cast<const half8_t *>(&qrot[HP > 8 ? e : r16 >> 3][column < HP ? column : 0][32 * c + 8 * g]) : (half8_t)(half_t)0;
    const float scale2 = (D == 128 ? 0.17677669529663689f : 0.25f) * 1.4426950408889634f;     // 2 log2(e) / sqrt(D): the queries' terms are of half of them
    const float term = TERMS == 1 && r16 >= 8 ? scale2 / PA_REST : scale2;     // (of this lane's column)
    float m = -INFINITY, l = 0.f;                // of head l % 16; the sum over this lane's positions only
    float4_t acc[W];
#pragma unroll
    for (int j = 0; j < W; j++) acc[j] = (float4_t)0.f;
    auto scores = [&]() {                        // log2(e) / sqrt(D) q k
        float4_t s = (float4_t)0.f, rest = (float4_t)0.f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[c], q8[0][c], s, 0, 0, 0);
            if (TERMS == 2) rest = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[c], q8[TERMS - 1][c], rest, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float one = s[i] * term;
            s[i] = TERMS == 1 ? one + eight_on(one) : __builtin_fmaf(rest[i], scale2 / PA_REST, one);
        }
        return s;
    };
    auto fold = [&](const float4_t s, int valid) {                      // the tile's first `valid` positions (at least one)
        float p[4], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            p[i] = 4 * g + i < valid ? s[i] : -INFINITY;
            mx = fmaxf(mx, p[i]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m, mx), r = __builtin_amdgcn_exp2f(m - mn);      // exp2(-inf) = 0 on the first tile
        m = mn;
        half8_t p8;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            p[i] = __builtin_amdgcn_exp2f(p[i] - mn);
            sum += p[i];
            p8[i] = (half_t)(p[i] * PA_UP);
            p8[i + 4] = (half_t)__builtin_fmaf(p[i], PA_UP, -(float)p8[i]);
        }
        l = l * r + sum;
        if (__any(r != 1.f)) {
#pragma unroll
            for (int j = 0; j < W; j++) acc[j] *= r;
        }
#pragma unroll
        for (int j = 0; j < W; j++) {
            const half8_t v = {v8[0][j], v8[1][j], v8[2][j], v8[3][j], v8[0][j], v8[1][j], v8[2][j], v8[3][j]};
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p8, acc[j], 0, 0, 0);
        }
    };
    while (t < t_end) {
        const int next = t + WAVES, now = id;
        const float4_t s = scores();
        id = next_id;
        if (next < t_end) fetch_k(id, next);
        if (next + WAVES < t_end) next_id = page_of(next + WAVES);
        if (good(now)) fold(s, pos - t * PA_TILE);
        if (next < t_end) fetch_v(id, next);
        t = next;
    }
    // its own k and v, from LDS, by the wave whose turn is next: a tile with one position
    const bool own = part == 0 && wave == (t_end - t_first) % WAVES;
    auto take_own = [&]() {
#pragma unroll
        for (int c = 0; c < NC; c++) k8[c] = *reinterpret_cast<const half8_t *>(&knew[32 * c + 8 * g]);
#pragma unroll
        for (int i = 0; i < 4; i++) v8[i] = *reinterpret_cast<const vec_t *>(&vnew[W * r16]);
    };
    if (own) {
        take_own();
        fold(scores(), 1);
    }

    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (r16 < HP && g == 0) { wm[r16][wave] = m; wl[r16][wave] = l; }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < W; j++) sum += (acc[j][0] + acc[j][1]) + (acc[j][2] + acc[j][3]);
    if (__builtin_expect(__any(sum != sum), 0)) {
        // An infinite k or v: times a second term of zero or of the other sign, or a masked weight, it is NaN in the products, and so is the weight of a score of -inf next to
        // a maximum of -inf.  The wave's positions twice more (maximum, then sums), head by head, query and weights as one fp32 number each: a lane has the score of position
        // r16, dimensions 32 c + 8 g .., and owns dimensions W r16 .. W r16 + W - 1 of the output.  A score of -inf weighs nothing, one of +inf or NaN makes its head NaN.
#pragma unroll 1
        for (int h = 0; h < nh; h++) {
            auto each_tile = [&](auto f) {
#pragma unroll 1
                for (t = t_first + wave; t < t_end; t += WAVES) {
                    id = page_of(t);
                    if (!good(id)) continue;
                    fetch_k(id, t);
                    fetch_v(id, t);
                    f(pos - t * PA_TILE);
                }
                if (own) {
                    take_own();
                    f(1);
                }
            };
            auto score = [&]() {
                float d = 0.f;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const half8_t q0 = *reinterpret_cast<const half8_t *>(&qrot[0][h][32 * c + 8 * g]), q1 = *reinterpret_cast<const half8_t *>(&qrot[1][h][32 * c + 8 * g]);
#pragma unroll
                    for (int e = 0; e < 8; e++) d = __builtin_fmaf(__builtin_fmaf((float)q1[e], 1.f / PA_REST, (float)q0[e]), (float)k8[c][e], d);
                    __builtin_amdgcn_sched_barrier(0);       // (all pieces side by side take registers, and with heads of 64 a workgroup per CU: 85 instead of 78)
                }
                d += __shfl_xor(d, 16, 64);
                d += __shfl_xor(d, 32, 64);
                return d * scale2;
            };
            float top = -INFINITY, sum_w = 0.f, o[W];
            each_tile([&](int valid) {
                const float s = score();
                if (r16 < valid) top = fmaxf(top, s);
            });
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
            const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int e = 0; e < W; e++) o[e] = 0.f;
            each_tile([&](int valid) {
                const float w = r16 < valid ? __builtin_amdgcn_exp2f(score() - from) : 0.f;
                sum_w += w;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float wi = __shfl(w, 4 * g + i, 64);
#pragma unroll
                    for (int e = 0; e < W; e++)
                        if (4 * g + i < valid) o[e] += wi * (float)v8[i][e];
                }
            });
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) sum_w += __shfl_xor(sum_w, x, 64);
            if (lane == 0) { wm[h][wave] = top; wl[h][wave] = sum_w; }
#pragma unroll
            for (int e = 0; e < W; e++) {
                o[e] += __shfl_xor(o[e], 16, 64);
                o[e] += __shfl_xor(o[e], 32, 64);
                if (g == 0) wacc[h][wave][W * r16 + e] = o[e];
            }
        }
    } else if (r16 < HP) {
#pragma unroll
        for (int i = 0; i < 4; i++)              // row 4 g + i of product j is dimension W (4 g + i) + j
#pragma unroll
            for (int j = 0; j < W; j += 4)
                *reinterpret_cast<float4_t *>(&wacc[r16][wave][W * (4 * g + i) + j]) = (float4_t){acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]} * (1.f / PA_UP);
    }
    __syncthreads();
    const int64_t mine = ((int64_t)(part == 0 ? b : a.B + place + part - 1) * a.kv_heads + hk) * rep + hg * a.per_unit;
    for (int it = tid; it < nh * D; it += THREADS) {
        const int h = it / D, dim = it % D;
        float mx = wm[h][0];
#pragma unroll
        for (int w = 1; w < WAVES; w++) mx = fmaxf(mx, wm[h][w]);
        float o = 0.f, den = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float r = wl[h][w] != 0.f ? __builtin_amdgcn_exp2f(wm[h][w] - mx) : 0.f;    // 0: a wave that saw no position
            o += wl[h][w] != 0.f ? r * wacc[h][w][dim] : 0.f;
            den += r * wl[h][w];
        }
        if (further > 0) {                       // part[request or further part][head][max, sum, pad, pad, weighted v]
            float *to = a.part + (mine + h) * (D + 4);
            to[4 + dim] = o;
            if (dim == 0) { to[0] = mx; to[1] = den; }
        } else {
            orow[it] = (half_t)(o / den);
        }
    }
}

// The parts of a head put together, in order: G threads per dimension take G runs of them, eight parts requested at once, and one puts the runs together; H heads to a workgroup.
template <int D, int G, int H>
__global__ __launch_bounds__(D * G * H) void attention_paged_merge_kernel(const float *__restrict__ part, const int32_t *__restrict__ heads_of, half_t *__restrict__ out,
                                                                          int B, int heads, int groups) {
    __shared__ float sm[H][G][D], sd[H][G][D], so[H][G][D];
    const int dim = threadIdx.x % D, g = threadIdx.x / D % G, h = threadIdx.x / (D * G), b = blockIdx.x / groups, head = blockIdx.x % groups * H + h;
    const int place = heads_of[2 * b], parts = heads_of[2 * b + 1] + 1;
    if (parts == 1) return;                      // written by the first launch
    auto from = [&](int i) { return part + ((int64_t)(i == 0 ? b : B + place + i - 1) * heads + min(head, heads - 1)) * (D + 4); };
    const int each = (parts + G - 1) / G, i_end = min((g + 1) * each, parts);
    float mx = -INFINITY, o = 0.f, den = 0.f;
    for (int i0 = g * each; i0 < i_end; i0 += 8) {
        float m[8], l[8], v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float *p = from(min(i0 + j, i_end - 1));
            m[j] = p[0];
            l[j] = i0 + j < i_end ? p[1] : 0.f;  // (0: a part that saw no position, or none)
            v[j] = p[4 + dim];
        }
        float top = mx;
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, l[j] != 0.f ? m[j] : -INFINITY);
        const float r0 = den != 0.f ? __builtin_amdgcn_exp2f(mx - top) : 0.f;
        o = den != 0.f ? o * r0 : 0.f;
        den *= r0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float r = l[j] != 0.f ? __builtin_amdgcn_exp2f(m[j] - top) : 0.f;
            o += l[j] != 0.f ? r * v[j] : 0.f;
            den += r * l[j];
        }
        mx = top;
    }
    if (G > 1) {
        sm[h][g][dim] = mx;
        sd[h][g][dim] = den;
        so[h][g][dim] = o;
        __syncthreads();
        if (g > 0) return;
#pragma unroll
        for (int j = 1; j < G; j++) mx = fmaxf(mx, sd[h][j][dim] != 0.f ? sm[h][j][dim] : -INFINITY);
        const float r0 = den != 0.f ? __builtin_amdgcn_exp2f(sm[h][0][dim] - mx) : 0.f;
        o = den != 0.f ? o * r0 : 0.f;
        den *= r0;
#pragma unroll
        for (int j = 1; j < G; j++) {
            const float d = sd[h][j][dim], r = d != 0.f ? __builtin_amdgcn_exp2f(sm[h][j][dim] - mx) : 0.f;
            o += d != 0.f ? r * so[h][j][dim] : 0.f;
            den += r * d;
        }
    }
    if (head < heads) out[((int64_t)b * heads + head) * D + dim] = (half_t)(o / den);
}

struct pa_shape {
    int rep, groups, per_unit, units, parts, least;        // (least: tiles of a part)
};
pa_shape shape_of(int B, int heads, int kv_heads, int64_t positions) {
    pa_shape p;
    p.rep = heads / kv_heads;
    // Tables that are not cut: a few workgroups' to 768 positions, more ones' to 1024.  (us, cut / whole: 1 request of 700, 32 heads on 8, 11.8 / 10.9, of 900 11.8 / 12.7; 16 of up to 800 15.0 / 12.6, 16 of up to
    // 1500 18.3 / 20.0; 48 of up to 1000 29.2 / 23.5, one of 1000 among 47 of 100 15.3 / 14.7, up to 1500 38.6 / 39.0; 256 of up to 1000 101.7 / 97.1.)
    const int64_t together = (int64_t)B * kv_heads * bs_cdiv(p.rep, PA_HEADS);
    const bool whole = positions <= (together <= 64 ? 768 : 1024);
    // One head to a unit where that leaves at most a workgroup per CU and nothing is cut: heads that share rows then read them again from the L2, side by side.  (us, heads together / one by
    // one: 1 request of 385, 32 heads on 8, 8.7 / 8.3, 64 on 8 9.8 / 8.2; 8 of 300 to 500, 32 on 8, 9.7 / 9.5; but 32 of 10 to 500 12.3 / 24.0.)
    // The rules go by the table's width, as the host does not know the lengths: requests of up to 1000 positions in tables of 8192 pay the second launch (48 of them 28.5 us instead of 21.0).
    p.groups = whole && (int64_t)B * heads <= 256 ? p.rep : (int)bs_cdiv(p.rep, PA_HEADS);
    p.per_unit = (int)bs_cdiv(p.rep, p.groups);
    p.units = kv_heads * p.groups;
    // Workgroups that further parts add: with few first ones all together are one per CU, with more two (as many as fit beside each other), beyond that enough of them
    // to even out unequal lengths.  (us at 256 in all / 512 in all / 768 more: 1 request of 40000, 32 heads on 8 KV heads, 35.3 / 36.7 / 41.3; 2 of 80000, 64 on 8, 107 / 112 / 112; 16 of 100 to
    // 8000 63.1 / 57.6 / 60.8; with 256 more / 768 more 48 of 1 to 4096 89 / 75.7.)
    const int64_t first = (int64_t)B * p.units, further = first <= 64 ? 256 - first : first <= 256 ? 512 - first : 768;
    p.parts = whole ? 0 : (int)(further / p.units);        // (0 for more than 768 units, which are enough by themselves: nothing is cut, and the grid holds 2^22 of them)
    // Shorter parts where few workgroups leave room: 4 tiles instead of 8 12.0 us -> 11.3 for 1 request of 1000; but 47 of 100 and one of 1000 15.3 -> 21.5.
    p.least = first <= 64 ? 4 : 8;
    return p;
}

// A cache that the last-level cache cannot hold is read past it.  (us without / with: 48 requests of 1 to 4096, 404 MB, 82.3 / 76.2; 2 of 80000, 655 MB, 132.8 / 115.6; but 8 of 2000,
// 67 MB, over and over 22.4 / 25.5, and 48 of up to 1000, 96 MB of a pool of 1 GiB, 21.0 / 25.3.  The rule goes by the pool, as the host does not know the lengths: a step's layers together read more than
// the pages of one, which are gone from the cache when the next step comes to them.)
constexpr int64_t PA_STREAM = 256ll << 20;

template <int D, int HP>
int launch(const pa_args &a, const int32_t *table, int64_t workgroups, hipStream_t s) {
    const bool stream = ((int64_t)a.pool << a.shift) * a.kv_heads * D * 4 >= PA_STREAM;
    (stream ? attention_paged_kernel<D, HP, true> : attention_paged_kernel<D, HP, false>)<<<(unsigned)workgroups, THREADS, 0, s>>>(a, table);
    BS_LAUNCH_CHECK();
    if (a.parts == 0) return BS_OK;
    // Few heads: the parts of each in four runs; many: several heads to a workgroup, most of which have one part.  (us, runs / heads: 1 request of 8000, 32 heads, 14.7 / 16.6; 2 of
    // 80000, 64 heads, 107.9 / 108.4; 8 of up to 8000, 32 heads, 33.5 / 33.1; 48 of up to 4096 88.0 / 85.5.)
    const bool few = (int64_t)a.B * a.heads < 256;
    const int groups = few ? a.heads : (a.heads + 3) / 4;
    (few ? attention_paged_merge_kernel<D, 4, 1> : attention_paged_merge_kernel<D, 1, 4>)<<<(unsigned)((int64_t)a.B * groups), D * 4, 0, s>>>(a.part, a.heads_of, a.out, a.B, a.heads, groups);
    BS_LAUNCH_CHECK();
    return BS_OK;
}

}  // namespace

int64_t bs_attention_paged_scratch(int B, int heads, int kv_heads, int head_dim, int max_pages, int page) {
    const pa_shape p = shape_of(B, heads, kv_heads, (int64_t)max_pages * page);
    return p.parts ? bs_cdiv(8ll * B, 16) * 16 + (int64_t)(B + p.parts) * heads * (head_dim + 4) * 4 : 0;
}

int bs_launch_attention_paged(const half_t *qkv, int ldqkv, half_t *kpages, half_t *vpages, const half_t *cos, const half_t *sin, const int32_t *table,
                              const int32_t *lengths, const int64_t *slots, half_t *out, int B, int heads, int kv_heads, int head_dim, int max_pos,
                              int shift, int max_pages, int pool, void *workspace, hipStream_t s) {
    const pa_shape p = shape_of(B, heads, kv_heads, (int64_t)max_pages << shift);
    const int64_t workgroups = (int64_t)(B + p.parts) * p.units;          // (at most 2^22 and 768: 2^32 threads hold them)
    pa_args a = {qkv, cos, sin, kpages, vpages, lengths, slots, out, (int32_t *)workspace, (float *)((char *)workspace + bs_cdiv(8ll * B, 16) * 16),
                 ldqkv, B, heads, kv_heads, p.groups, p.per_unit, max_pos, shift, max_pages, pool, p.parts, p.least};
    if (head_dim == 128)
        return p.per_unit > 8 ? launch<128, 16>(a, table, workgroups, s) : p.per_unit > 4 ? launch<128, 8>(a, table, workgroups, s) : p.per_unit > 2 ? launch<128, 4>(a, table, workgroups, s)
             : p.per_unit > 1 ? launch<128, 2>(a, table, workgroups, s) : launch<128, 1>(a, table, workgroups, s);
    return p.per_unit > 8 ? launch<64, 16>(a, table, workgroups, s) : p.per_unit > 4 ? launch<64, 8>(a, table, workgroups, s) : p.per_unit > 2 ? launch<64, 4>(a, table, workgroups, s)
         : p.per_unit > 1 ? launch<64, 2>(a, table, workgroups, s) : launch<64, 1>(a, table, workgroups, s);
}
