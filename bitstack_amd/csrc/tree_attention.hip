// Attention of drafted tokens over the paged cache: out[t] = softmax(q[t] k^T / sqrt(D)) v over the positions that the request held and those nodes of its tree, stored
// behind them, that masks[t] names.
//
// The rows of a KV head of a request are its nodes' queries of that head's group, the head fastest: nodes * group of them, which all read the same K and V.  A workgroup takes 16, 32, 64 or 128 of them, the
// columns of both products, and walks the positions in stages of 32.
//   scores  S[position, row] = K q      16x16x32
//   output  O[dim, row] += V^T P        16x16x32; a lane of the scores holds four positions of a row in each of two tiles of 16, which are the eight k slots of this product
// Up to 32 rows a wave takes every fourth stage with K and V in registers; beyond, every wave has 16 or 32 rows, and the stages come to LDS straight from the pages (no registers).
// Maximum, sum and output are fp32, in base 2.  The weights enter the second product as two fp16 terms, p = hi + lo, the largest as 2^15: held to 2^-22 of themselves down to 2^-18 of the
// largest, below that to 2^-40 of the largest.  (hi alone: an error against 64 bits of 2.2 to 2.7e-4 where the result's rounding is 2.1e-4, and where many weights are rounded up values of 65504
// everywhere became infinities, as the sum below the line is that of the fp32 weights.  The second terms' products cost 0 to 2 % up to 32 rows
// of a KV head, 0 to 5 with 64, a sixth to a quarter with 128: 64 requests of 4000, 32 heads on 8, 16 nodes 174 -> 183 us, 32 nodes 226 -> 266; 2 documents of 80000 with trees of 64 441 -> 545.)
//
// What a row does not see has a weight of zero, but zero times an infinity is NaN: in the stages with nodes V is looked through, and infinities and NaN, if any, are taken out of the
// product.  Rows that see them, or whose result is not finite for another reason, are computed again, each by a wave, in fp32.
//
// The split: as the lengths are known on the device alone, every workgroup works out from them what it is to do (ta_deal).  What is not a whole request's leaves (max, sum, weighted v) in
// the workspace, and a second launch puts the parts together, in order: the result does not depend on which came first.
//
// What bounds it: up to 64 rows the cache's bytes (64 requests of 4000, 32 heads on 8: 4 nodes 169 us, 8 nodes 173, 16 nodes 183, 6.2 to 5.8 TB/s; 200 of 100 to 1500, 16 on 16 of 64, 123 us, 5.4 TB/s; 48 of
// up to 4096 with 1 to 16 nodes 88, 4.6 TB/s and the second launch's 7); with 128 what is issued (2 documents of 80000 with trees of 64, 64 heads on 8: 0.336 TFLOP in 545 us, 0.62 PFLOP/s where a large matrix
// product reaches 1.2: an exponential, a maximum and two roundings per 512 flops, and a third of the matrix instructions for the second terms); one short request is the chain of latencies (11.8 us).
#include "lanes.h"

#include <type_traits>

namespace {

constexpr int TA_P = 32;                         // positions of a stage; LDS holds four
constexpr float TA_LOW = -1e30f;                 // a maximum before the first score (finite scores are above it)
constexpr float TA_UP = 15.f;                    // log2 of the largest weight

struct ta_args {
    const half_t *q, *kpages, *vpages;
    const int32_t *table, *lengths, *granted, *starts;
    const int64_t *masks;
    half_t *out;
    int32_t *before;                             // workspace: stages of the requests before each one, (or parts); of all, shares, stages of a part
    float *part;                                 // ... and what parts leave: [share, first or last][node][head][max, sum, pad, pad, weighted v]
    float per_rep, part_cost;                    // 1 / (heads per KV head); what a part of all units costs, in stages
    int ldq, B, T, nodes, heads, kv_heads, row_tiles, shift, max_pages, pool, shares, more;      // (shares 0: a workgroup of a unit takes one request)
};

struct ta_request {
    int start, end, n, len;                      // token rows, nodes (0: idle), positions with the nodes
    __device__ __forceinline__ ta_request() {}
    __device__ __forceinline__ ta_request(const ta_args &a, int b) {
        start = min(max(a.starts[b], 0), a.T);
        end = min(max(a.starts[b + 1], start), a.T);
        n = a.granted[b];
        len = a.lengths[b];
        if (n < 1 || n > a.nodes || n > end - start || len < n || (int64_t)len > (int64_t)a.max_pages << a.shift) n = len = 0;
    }
    __device__ __forceinline__ int stages() const { return (len + TA_P - 1) / TA_P; }
};
// node of a row: row / rep, at most 64
__device__ __forceinline__ int ta_node(int row, int rep, float per_rep) {
    const int node = (int)((float)row * per_rep), rest = row - node * rep;
    return rest < 0 ? node - 1 : rest >= rep ? node + 1 : node;
}
// share g of `sum` stages dealt to `shares`: where it begins; and whose stage x is
__device__ __forceinline__ int ta_begins(int g, int sum, int shares) { return (int)((int64_t)g * sum / shares); }
__device__ __forceinline__ int ta_whose(int x, int sum, int shares) { return (int)((((int64_t)x + 1) * shares - 1) / sum); }
// parts of a request that has `stages`, none of more than `per`; where part i of n begins
__device__ __forceinline__ int ta_parts(int stages, int per) { return (int)((uint32_t)(stages + per - 1) / (uint32_t)per); }
__device__ __forceinline__ int ta_cut(int i, int stages, int n) { return (int)((int64_t)i * stages / n); }

// v, of which nothing is worked out ahead of here (registers are short in the loops over the stages)
__device__ __forceinline__ int ta_here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// weights i and i + 1 as sums of two fp16 terms each
__device__ __forceinline__ void ta_terms(const float (&p)[2], int i, half8_t &p8, half8_t &rest8) {
    float one = 1.f;
    half2_t h = {(half_t)p[0], (half_t)p[1]};
    asm("" : "+v"(h), "+s"(one));                // (two are rounded by one instruction, and each one's rest is another)
#pragma unroll
    for (int e = 0; e < 2; e++) {
        p8[i + e] = h[e];
        rest8[i + e] = (half_t)__builtin_fmaf(p[e], one, -(float)h[e]);
    }
}

// the larger of v here and in the lane whose number differs by W (16 or 32), or (SUM) both together
template <int W, bool SUM = false>
__device__ __forceinline__ float across(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = W == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return SUM ? __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b) : fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// the largest of all lanes' v, or (SUM) their sum
template <bool SUM>
__device__ __forceinline__ float ta_all(float v) {
    auto both = [&](uint32_t other) { v = SUM ? v + __builtin_bit_cast(float, other) : fmaxf(v, __builtin_bit_cast(float, other)); };
    both(bs_lane<0xb1>(__builtin_bit_cast(uint32_t, v)));        // quad_perm 1, 0, 3, 2
    both(bs_lane<0x4e>(__builtin_bit_cast(uint32_t, v)));        // quad_perm 2, 3, 0, 1
    both(bs_lane<0x141>(__builtin_bit_cast(uint32_t, v)));       // 8 lanes mirrored, then 16
    both(bs_lane<0x140>(__builtin_bit_cast(uint32_t, v)));
    return across<32, SUM>(across<16, SUM>(v));
}

typedef __attribute__((address_space(3))) void *ta_lds;

// What a workgroup is at: stages st .. st_end - 1 of request b.
struct ta_work {
    int g, at, end;                              // its share, stages still to do
    int b, before, st, st_end, slot;             // before: stages (or parts) of the requests in front of b; slot: of a part; -1: the whole request
    ta_request rq;
    __device__ __forceinline__ void take(int first) {
        const int stages = rq.stages();
        st = at - before;
        st_end = min(stages, st + end - at);
        slot = st == 0 && st_end == stages ? -1 : 2 * g + (at != first);
        at += st_end - st;
    }
    __device__ __forceinline__ void take_part(int per) {
        const int stages = rq.stages(), n = ta_parts(stages, per);
        st = ta_cut(g - before, stages, n);
        st_end = ta_cut(g - before + 1, stages, n);
        slot = n == 1 ? -1 : 2 * g;
        at = end = 0;
    }
};
__device__ __forceinline__ ta_request ta_uniform(const ta_request &r, int lane) {
    ta_request u;
    u.start = (int)bs_read((uint32_t)r.start, lane);
    u.end = (int)bs_read((uint32_t)r.end, lane);
    u.n = (int)bs_read((uint32_t)r.n, lane);
    u.len = (int)bs_read((uint32_t)r.len, lane);
    return u;
}
// How the stages of all requests, `sum`, are dealt to a.shares workgroups of a unit.
// Equal shares keep the workgroups busy to the end whatever the lengths are, but one may hold the end of a request and the beginning of another: each costs its chain of latencies (lengths, pages, K, what it
// leaves), 4 us, and is a part.  Each request's own parts, one to a workgroup, have one chain, but may be unequal.  They are taken where they fit and none has `more` stages more than an equal share (16
// up to 32 rows, whose stages take 0.3 us, else 32).  us, equal shares / own parts: 5 requests of up to 1000 with 8 nodes 22.5 / 14.0, 16 of up to 250 22.0 / 13.6, 64 of up to 1000 with 32 nodes 77 / 71, and without
// the limit 32 requests of up to 4000 with 4 nodes 55 / 69.
// A part has at least 4 stages; more where the longest request would be in many, which the second launch takes eight at a time (8 nodes, one request of 4000: 8 stages 16.6, 4 stages 20.1); and more
// where all of them are many: what all units leave of one costs part_cost stages, so that parts of sqrt(part_cost sum) stages cost as much as they have (16 requests of 390: whole 15, in four 25).
struct ta_deal {
    int sum, shares, per;                        // per: stages of a part at most; 0: equal shares
    // live: requests that have stages; longest: the most of one; count(per): parts of all requests
    template <typename C>
    __device__ __forceinline__ ta_deal(const ta_args &a, int sum, int live, int longest, C count) : sum(sum) {
        const int even = (int)((uint32_t)(sum + a.shares - 1) / (uint32_t)a.shares), least = max(4, (int)__builtin_amdgcn_sqrtf(fmaxf(0.25f * (float)longest, a.part_cost * (float)sum)));
        per = 0;
        shares = a.shares;
        if (live <= a.shares) {
            const int room = a.shares - live;    // (a request has less than one part more than its stages / per)
            per = max(even, least);
            int n = count(per);
            if (n > a.shares) {
                per = room > 0 ? min(longest, max(least, (int)((uint32_t)(sum + room - 1) / (uint32_t)room))) : longest;
                if (per > even + a.more) per = 0;
                else n = count(per);
            }
            if (per) shares = n;
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            a.before[a.B] = sum;
            a.before[a.B + 1] = shares;
            a.before[a.B + 2] = per;
        }
    }
};
// The next request of the share (up to 64 requests: the first one too): false where there is none.  Up to 64 requests every wave finds it by itself, a lane a request.
template <bool FIRST>
__device__ __forceinline__ bool ta_next_of_few(const ta_args &a, ta_work &w, int &first) {
    const int lane = ta_here(threadIdx.x & 63);
    const ta_request r(a, min(lane, a.B - 1));
    auto plus = [](uint32_t x, uint32_t y) { return x + y; };
    const int stages = lane < a.B ? r.stages() : 0;
    int upto = (int)bs_scan((uint32_t)stages, plus), mine = stages, x = w.at, per = 0;
    if (FIRST) {
        const int longest = (int)bs_read(bs_scan((uint32_t)stages, [](uint32_t x, uint32_t y) { return max(x, y); }), 63);
        int parts = 0, parts_upto = 0;
        const ta_deal d(a, (int)bs_read((uint32_t)upto, 63), __popcll(__ballot(stages > 0)), longest, [&](int per) {
            parts = ta_parts(stages, per);
            parts_upto = (int)bs_scan((uint32_t)parts, plus);
            return (int)bs_read((uint32_t)parts_upto, 63);
        });
        if (w.g >= d.shares) return false;
        per = d.per;
        if (per) {
            x = w.g;
            mine = parts;
            upto = parts_upto;
        } else {
            x = w.at = first = ta_begins(w.g, d.sum, d.shares);
            w.end = ta_begins(w.g + 1, d.sum, d.shares);
        }
    }
    if (per == 0 && w.at >= w.end) return false;
    w.b = __builtin_ctzll(__ballot(x >= upto - mine && x < upto));
    w.before = (int)bs_read((uint32_t)(upto - mine), w.b);
    w.rq = ta_uniform(r, w.b);
    if (per) w.take_part(per);
    else w.take(first);
    return true;
}
// More: the workgroup looks for the first one together, and goes on from there.
template <int WAVES>
__device__ __forceinline__ bool ta_first_of_many(const ta_args &a, ta_work &w, int &first) {
    __shared__ int sums[3][WAVES], found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), THREADS = WAVES * 64;
    auto plus = [](uint32_t x, uint32_t y) { return x + y; };
    auto larger = [](uint32_t x, uint32_t y) { return max(x, y); };
    const int stages0 = tid < a.B ? ta_request(a, tid).stages() : 0;
    auto each = [&](auto f) {
        f(stages0);
        for (int i = tid + THREADS; i < a.B; i += THREADS) f(ta_request(a, i).stages());
    };
    uint32_t sum_of = 0, live_of = 0, longest_of = 0;
    each([&](int n) {
        sum_of += n;
        live_of += n > 0;
        longest_of = max(longest_of, (uint32_t)n);
    });
    sum_of = bs_read(bs_scan(sum_of, plus), 63);
    live_of = bs_read(bs_scan(live_of, plus), 63);
    longest_of = bs_read(bs_scan(longest_of, larger), 63);
    if (lane == 0) {
        sums[0][wave] = (int)sum_of;
        sums[1][wave] = (int)live_of;
        sums[2][wave] = (int)longest_of;
    }
    __syncthreads();
    int sum = 0, live = 0, longest = 0;
#pragma unroll
    for (int v = 0; v < WAVES; v++) {
        sum += sums[0][v];
        live += sums[1][v];
        longest = max(longest, sums[2][v]);
    }
    const ta_deal d(a, sum, live, longest, [&](int per) {
        uint32_t parts = 0;
        each([&](int n) { parts += ta_parts(n, per); });
        parts = bs_read(bs_scan(parts, plus), 63);
        __syncthreads();
        if (lane == 0) sums[0][wave] = (int)parts;
        __syncthreads();
        int n = 0;
#pragma unroll
        for (int v = 0; v < WAVES; v++) n += sums[0][v];
        return n;
    });
    if (w.g >= d.shares) return false;
    const int x = d.per ? w.g : ta_begins(w.g, sum, d.shares);
    if (d.per == 0) {
        w.at = first = x;
        w.end = ta_begins(w.g + 1, sum, d.shares);
        if (w.at >= w.end) return false;
    }
    int before = 0;
    for (int i0 = 0; i0 < a.B && before <= x; i0 += THREADS) {
        const int i = i0 + tid, stages = i0 == 0 ? stages0 : i < a.B ? ta_request(a, i).stages() : 0, mine = d.per ? ta_parts(stages, d.per) : stages, upto = (int)bs_scan((uint32_t)mine, plus);
        __syncthreads();
        if (lane == 63) sums[0][wave] = upto;
        __syncthreads();
        int from = before + upto - mine;
#pragma unroll
        for (int v = 0; v < WAVES; v++) {
            if (v < wave) from += sums[0][v];
            before += sums[0][v];
        }
        if (x >= from && x < from + mine) {
            found[0] = i;
            found[1] = from;
        }
    }
    __syncthreads();
    w.b = __builtin_amdgcn_readfirstlane(found[0]);
    w.before = __builtin_amdgcn_readfirstlane(found[1]);
    w.rq = ta_uniform(ta_request(a, w.b), 0);
    if (d.per) w.take_part(d.per);
    else w.take(first);
    return true;
}
template <int WAVES>
__device__ __forceinline__ bool ta_first(const ta_args &a, int g, ta_work &w, int &first) {
    w.g = g;
    if (a.shares == 0) {                         // one request
        w.b = g;
        w.rq = ta_uniform(ta_request(a, g), 0);
        w.before = w.at = first = 0;
        w.end = w.rq.stages();
        if (w.end == 0) return false;
        w.take(first);
        return true;
    }
    return a.B <= 64 ? ta_next_of_few<true>(a, w, first) : ta_first_of_many<WAVES>(a, w, first);
}
__device__ __forceinline__ bool ta_next(const ta_args &a, ta_work &w, int &first) {
    if (w.at >= w.end) return false;
    if (a.B <= 64) return ta_next_of_few<false>(a, w, first);
    do {
        w.before += w.rq.stages();
        w.rq = ta_uniform(ta_request(a, ++w.b), 0);
    } while (w.rq.n == 0);
    w.take(first);
    return true;
}
// rows that are no node are zeros: those of every request that is this workgroup's to see to, and some of those of no request
template <int THREADS>
__device__ __forceinline__ void ta_idle(const ta_args &a, int g, int of, int D) {
    const int64_t orow = (int64_t)a.heads * D;
    auto idle = [&](int t) {
        for (int64_t i = threadIdx.x; i < orow; i += THREADS) a.out[t * orow + i] = (half_t)0;
    };
    const int last = min(max(a.starts[a.B], 0), a.T), first = min(max(a.starts[0], 0), a.T);
    for (int b = g; b < a.B; b += of) {
        const ta_request r(a, b);
        for (int t = r.start + r.n; t < r.end; t++) idle(t);
    }
    for (int t = last + g; t < a.T; t += of) idle(t);
    for (int t = g; t < first; t += of) idle(t);
}
// what a part leaves of a node's head
__device__ __forceinline__ float *ta_part_row(const ta_args &a, int slot, int node, int head, int D) {
    return a.part + (((int64_t)slot * a.nodes + node) * a.heads + head) * (D + 4);
}
// One row by one wave, in fp32, over positions p_first .. p_end - 1: the largest score first, then the sums.  A lane has a position's score, and owns dimensions D / 64 * lane .. of the output.
template <int D>
struct ta_again {
    float top, sum, o[D / 64];
    __device__ __forceinline__ ta_again(const ta_args &a, const ta_request &rq, const int32_t *ids, int node, int head, int hk, int p_first, int p_end, float scale2) {
        constexpr int PER = D / 64;
        const int lane = ta_here(threadIdx.x & 63), held = rq.len - rq.n;
        const half_t *qr = a.q + (int64_t)(rq.start + node) * a.ldq + head * D;
        const uint64_t sees = (uint64_t)a.masks[rq.start + node];
        auto where = [&](int p) {                // halves in front of position p; -1: not seen, or not there
            if (p >= p_end || (p >= held && !(sees >> (p - held) & 1))) return (int64_t)-1;
            const int id = ids[p >> a.shift];
            return id >= 0 && id < a.pool ? ((((int64_t)id * a.kv_heads + hk) << a.shift) + (p & ((1 << a.shift) - 1))) * D : (int64_t)-1;
        };
        auto score = [&](int64_t at) {
            if (at < 0) return -INFINITY;
            float d = 0.f;
#pragma unroll 1
            for (int c = 0; c < D; c += 8) {
                const half8_t k = *reinterpret_cast<const half8_t *>(a.kpages + at + c);
#pragma unroll
                for (int e = 0; e < 8; e++) d = __builtin_fmaf((float)qr[c + e], (float)k[e], d);
            }
            return d * scale2;
        };
        top = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < PER; e++) o[e] = 0.f;
        for (int p0 = p_first; p0 < p_end; p0 += 64) top = fmaxf(top, score(where(p0 + lane)));
        top = ta_all<false>(top);
        const float from = top == -INFINITY ? 0.f : top;
        for (int p0 = p_first; p0 < p_end; p0 += 64) {
            const int64_t at = where(p0 + lane);
            const float weight = __builtin_amdgcn_exp2f(score(at) - from + TA_UP);       // (a score of -inf weighs nothing; one of +inf, or NaN, is NaN)
            sum += weight;
#pragma unroll 1
            for (int i = 0; i < 64; i++) {
                const int64_t ai = (int64_t)((uint64_t)bs_read((uint32_t)((uint64_t)at >> 32), i) << 32 | bs_read((uint32_t)at, i));
                const float wi = __builtin_bit_cast(float, bs_read(__builtin_bit_cast(uint32_t, weight), i));
                if (ai < 0 || wi == 0.f) continue;
#pragma unroll
                for (int e = 0; e < PER; e++) o[e] = __builtin_fmaf(wi, (float)a.vpages[ai + PER * lane + e], o[e]);
            }
        }
        sum = ta_all<true>(sum);
        top = top == -INFINITY ? TA_LOW : top;
    }
};
constexpr __device__ float ta_scale(int D) { return (D == 128 ? 0.08838834764831845f : 0.125f) * 1.4426950408889634f; }       // log2(e) / sqrt(D)

// The pages of 64 tiles of 16 positions at a time, a lane a tile: two of each of 32 stages, which are `step` apart (tiles behind the last one are the last again).  A page that does not exist is
// read as the other of its stage; `gone`: tiles of such.
struct ta_pages {
    const int32_t *ids;
    int last_tile, shift, pool, step, raw, id;
    uint64_t gone;
    __device__ __forceinline__ bool good(int i) const { return i >= 0 && i < pool; }
    __device__ __forceinline__ void load(int st) {
        const int lane = threadIdx.x & 63;
        raw = ids[(min(2 * st + 2 * step * (lane >> 1) + (lane & 1), last_tile) * 16) >> shift];
    }
    __device__ __forceinline__ void take() {
        gone = ~__ballot(good(raw));
        const int beside = __builtin_amdgcn_update_dpp(0, raw, 0xb1, 0xf, 0xf, true);      // quad_perm 1, 0, 3, 2
        id = good(raw) ? raw : good(beside) ? beside : 0;
    }
};

// whether a row sees the nodes of four positions, the first of them `node` (below 0: a position that the request held); bits
__device__ __forceinline__ uint32_t ta_seen(uint64_t mask, int node) {
    return node >= 64 ? 0 : node >= 0 ? (uint32_t)(mask >> node) : node <= -4 ? 15 : (uint32_t)mask << -node | ((1u << -node) - 1);
}

// ---- few rows: what counts is the cache's bytes on their way.  A wave has all 16 QT rows and every fourth stage, K and V in registers: K of its next stage is requested behind the
// scores, V behind the output product, so that eight waves of a CU have 128 KB on their way.  What the waves have is put together in LDS.
template <int D, int QT, bool STREAM>
__global__ __launch_bounds__(256, 2) void attention_tree_few_kernel(const ta_args a) {
    constexpr int W = D / 16, NC = D / 32, WAVES = 4, THREADS = WAVES * 64, ROWS = 16 * QT;
    typedef half_t vec_t __attribute__((ext_vector_type(W)));
    __shared__ __attribute__((aligned(16))) float wo[WAVES][ROWS][D + 4];              // (rows a sixteenth of the banks' turn apart)
    __shared__ float wm[WAVES][ROWS], wl[WAVES][ROWS];
    __shared__ uint64_t odd_of[WAVES];           // nodes at which something in v is infinite or NaN
    __shared__ uint32_t bad[WAVES][ROWS];        // rows whose sums are not finite, or all, where a held position has such
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hk = blockIdx.x % a.kv_heads, g_of = blockIdx.x / a.kv_heads, rep = a.heads / a.kv_heads;
    const int64_t page_step = (int64_t)a.kv_heads * D << a.shift, head_at = (int64_t)hk * D << a.shift;
    ta_work w;
    int first;
    for (bool more = ta_first<WAVES>(a, g_of, w, first); more; more = ta_next(a, w, first)) {
        const int r16 = ta_here(lane) & 15, g = ta_here(lane) >> 4;
        const ta_request &rq = w.rq;
        const int rows = rq.n * rep, held = rq.len - rq.n, st_end = w.st_end;
        if (hk == 0 && w.st == 0 && tid == 0 && a.shares > 0) a.before[w.b] = w.before;
        ta_pages pg = {a.table + (int64_t)w.b * a.max_pages, (rq.len - 1) / 16, a.shift, a.pool, WAVES, 0, 0, 0};

        half8_t k8[2][NC];
        vec_t v8[8];
        int st = w.st + wave, rel = 0;        // (rel: lane of the stage's first tile in the pages)
        auto tile_at = [&](const half_t *of, int st, int lane_of, int i, int &rows_there) {
            const int pos = min(2 * st + i, pg.last_tile) * 16;
            rows_there = rq.len - pos;               // (the last one again behind them)
            return __builtin_amdgcn_make_buffer_rsrc((void *)(of + head_at + (int64_t)(int)bs_read((uint32_t)pg.id, lane_of + i) * page_step + (pos & ((1 << a.shift) - 1)) * D), 0, -1, 0x00020000);
        };
        auto fetch_k = [&](int st, int lane_of) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                int there;
                const __amdgpu_buffer_rsrc_t rsrc = tile_at(a.kpages, st, lane_of, i, there);
                const int at = (there < 16 ? min(r16, there - 1) : r16) * (2 * D) + 16 * g;
#pragma unroll
                for (int c = 0; c < NC; c++) k8[i][c] = __builtin_bit_cast(half8_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at + 64 * c, 0, STREAM ? 2 : 0));
            }
        };
        auto fetch_v = [&](int st, int lane_of) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                int there;
                const __amdgpu_buffer_rsrc_t rsrc = tile_at(a.vpages, st, lane_of, i, there);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int at = (there < 16 ? min(4 * g + e, there - 1) : 4 * g + e) * (2 * D) + 2 * W * r16;
                    if constexpr (D == 128) v8[4 * i + e] = __builtin_bit_cast(vec_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, 0, STREAM ? 2 : 0));
                    else v8[4 * i + e] = __builtin_bit_cast(vec_t, __builtin_amdgcn_raw_buffer_load_b64(rsrc, at, 0, STREAM ? 2 : 0));
                }
            }
        };
        if (st < st_end) {
            pg.load(st);
            pg.take();
            fetch_k(st, 0);
            fetch_v(st, 0);
            pg.load(st + 32 * WAVES);
        }

        half8_t q8[QT][NC];
        uint64_t mask[QT];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int row = min(16 * t + r16, rows - 1), node = ta_node(row, rep, a.per_rep);
            const half_t *p = a.q + (int64_t)(rq.start + node) * a.ldq + (hk * rep + row - node * rep) * D + 8 * g;
            if (((uintptr_t)a.q | (uintptr_t)(2 * a.ldq)) % 16 == 0) {
#pragma unroll
                for (int c = 0; c < NC; c++) q8[t][c] = *reinterpret_cast<const half8_t *>(p + 32 * c);
            } else {
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int e = 0; e < 8; e++) q8[t][c][e] = p[32 * c + e];
            }
            mask[t] = (uint64_t)a.masks[rq.start + node] & (rq.n < 64 ? (1ull << rq.n) - 1 : ~0ull);
        }
        const float scale2 = ta_scale(D);
        float m[QT], l[QT];                          // of row r16 of a tile; l over this lane's positions only
        float4_t acc[QT][W];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            m[t] = TA_LOW;
            l[t] = 0.f;
#pragma unroll
            for (int j = 0; j < W; j++) acc[t][j] = (float4_t)0.f;
        }
        bool odd_held = false;                       // (of this lane) v at a held position, or at these nodes, has an infinity or NaN
        uint64_t odd_nodes = 0;
        while (st < st_end) {
            const int next = st + WAVES;
            const int bits = (int)(pg.gone >> rel & 3);        // tiles of pages that do not exist
            float4_t s[QT][2];
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int i = 0; i < 2; i++) s[t][i] = (float4_t)0.f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int t = 0; t < QT; t++) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[i][c], q8[t][c], s[t][i], 0, 0, 0);
            rel += 2;
            if (rel == 64) {
                rel = 0;
                pg.take();
                pg.load(next + 32 * WAVES);
            }
            if (next < st_end) fetch_k(next, rel);
            const bool masked = TA_P * (st + 1) > held || bits != 0;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int t = 0; t < QT; t++) {
                        const uint32_t seen = bits >> i & 1 ? 0 : ta_seen(mask[t], TA_P * st + 16 * i + 4 * g - held);
#pragma unroll
                        for (int e = 0; e < 4; e++) s[t][i][e] = seen >> e & 1 ? s[t][i][e] : -INFINITY;
                    }
            }
            half8_t p8[QT], rest8[QT];
            float r[QT];
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float mx = s[t][0][0];
#pragma unroll
                for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[t][i >> 2][i & 3]);
                mx = across<32>(across<16>(mx));
                const float mn = fmaxf(m[t], mx * scale2), from = mn - TA_UP;
                r[t] = __builtin_amdgcn_exp2f(m[t] - mn);
                m[t] = mn;
                float sum[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float p[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][(i + e) >> 2][(i + e) & 3], scale2, -from));
                        sum[e] += p[e];
                    }
                    ta_terms(p, i, p8[t], rest8[t]);
                }
                l[t] = l[t] * r[t] + (sum[0] + sum[1]);
            }
            if (masked) {                            // infinities and NaN (times zero: NaN) become zeros, and their positions are noted
                vec_t check = (vec_t)(half_t)0;
#pragma unroll
                for (int i = 0; i < 8; i++) check += v8[i] * (vec_t)(half_t)0;
                bool odd = false;
#pragma unroll
                for (int j = 0; j < W; j++) odd = odd || check[j] != check[j];
                if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        bool here = false;
#pragma unroll
                        for (int j = 0; j < W; j++) {
                            const bool fine = (__builtin_bit_cast(uint16_t, (half_t)v8[i][j]) & 0x7c00u) != 0x7c00u;
                            here = here || !fine;
                            v8[i][j] = fine ? v8[i][j] : (half_t)0;
                        }
                        const int node = TA_P * st + 16 * (i >> 2) + 4 * g + (i & 3) - held;
                        if (here && node < 0) odd_held = true;
                        if (here && node >= 0 && node < rq.n) odd_nodes |= 1ull << node;
                    }
                }
            }
            if (__any(r[0] != 1.f || r[QT - 1] != 1.f)) {
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int j = 0; j < W; j++) acc[t][j] *= r[t];
            }
#pragma unroll
            for (int j = 0; j < W; j++) {
                const half8_t v = {v8[0][j], v8[1][j], v8[2][j], v8[3][j], v8[4][j], v8[5][j], v8[6][j], v8[7][j]};
#pragma unroll
                for (int t = 0; t < QT; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p8[t], acc[t][j], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < QT; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, rest8[t], acc[t][j], 0, 0, 0);
            }
            if (next < st_end) fetch_v(next, rel);
            st = next;
        }

#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int row = 16 * t + r16;
            l[t] = across<32, true>(across<16, true>(l[t]));
            if (g == 0) {
                wm[wave][row] = m[t];
                wl[wave][row] = l[t];
            }
            float sum = l[t];                        // (not finite: NaN, or an infinity)
#pragma unroll
            for (int j = 0; j < W; j++) sum += (acc[t][j][0] - acc[t][j][0]) + (acc[t][j][1] - acc[t][j][1]) + (acc[t][j][2] - acc[t][j][2]) + (acc[t][j][3] - acc[t][j][3]);
            const uint64_t not_finite = __ballot(sum != sum);
            if (g == 0) bad[wave][row] = (not_finite >> r16 | not_finite >> (r16 + 16) | not_finite >> (r16 + 32) | not_finite >> (r16 + 48)) & 1;
#pragma unroll
            for (int i = 0; i < 4; i++)              // row 4 g + i of product j is dimension W (4 g + i) + j
#pragma unroll
                for (int j = 0; j < W; j += 4)
                    *reinterpret_cast<float4_t *>(&wo[wave][row][W * (4 * g + i) + j]) = (float4_t){acc[t][j][i], acc[t][j + 1][i], acc[t][j + 2][i], acc[t][j + 3][i]};
        }
        if (__builtin_expect(__any(odd_held || odd_nodes != 0), 0)) {
            const bool held_too = __any(odd_held);
#pragma unroll
            for (int x = 1; x < 64; x <<= 1)
                odd_nodes |= (uint64_t)__shfl_xor((uint32_t)(odd_nodes >> 32), x, 64) << 32 | __shfl_xor((uint32_t)odd_nodes, x, 64);
            if (held_too) odd_nodes = ~0ull;
            if (held_too && lane < ROWS) bad[wave][lane] = 1;
        }
        if (lane == 0) odd_of[wave] = odd_nodes;
        __syncthreads();
        // rows that are computed again: not finite in one of the waves, or with such a node in sight
        uint32_t any = 0;
        uint64_t odd = 0;
#pragma unroll
        for (int v = 0; v < WAVES; v++) {
            any |= bad[v][lane % ROWS];
            odd |= odd_of[v];
        }
        uint64_t again = __ballot(lane < rows && any != 0);
        if (__builtin_expect(odd != 0, 0)) again |= __ballot(lane < rows && ((uint64_t)a.masks[rq.start + ta_node(min(lane, rows - 1), rep, a.per_rep)] & odd) != 0);
        if (__builtin_expect(again != 0, 0)) {             // (the same for all waves)
            int turn = 0;
            for (uint64_t left = again; left != 0; left &= left - 1, turn = turn + 1 == WAVES ? 0 : turn + 1) {
                if (turn != wave) continue;
                const int row = __builtin_ctzll(left), node = ta_node(row, rep, a.per_rep);
                const ta_again<D> x(a, rq, pg.ids, node, hk * rep + row - node * rep, hk, w.st * TA_P, min(st_end * TA_P, rq.len), scale2);
                if (lane < WAVES) {
                    wm[lane][row] = lane == 0 ? x.top : TA_LOW;
                    wl[lane][row] = lane == 0 ? x.sum : 0.f;
                }
#pragma unroll
                for (int e = 0; e < D / 64; e++) wo[0][row][D / 64 * lane + e] = x.o[e];
            }
            __syncthreads();
        }
        // the waves' put together: THREADS / ROWS threads for a row
        constexpr int SHARE = THREADS / ROWS, PER = D / SHARE / 4;       // ... and four dimensions, PER times
        const int row = tid / SHARE, node = ta_node(row, rep, a.per_rep), head = hk * rep + row - node * rep;
        if (row < rows) {
            // (all of it is read at once, and nothing behind a branch: a wait for each took 1.5 us)
            float4_t x[PER][WAVES];
            float tops[WAVES], sums[WAVES], r[WAVES], den = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; v++) {
                tops[v] = wm[v][row];
                sums[v] = wl[v][row];
            }
#pragma unroll
            for (int i = 0; i < PER; i++)
#pragma unroll
                for (int v = 0; v < WAVES; v++) x[i][v] = *reinterpret_cast<const float4_t *>(&wo[v][row][4 * (tid % SHARE) + 4 * SHARE * i]);
#pragma unroll
            for (int v = 0; v < WAVES; v++) asm volatile("" : "+v"(tops[v]), "+v"(sums[v]));
#pragma unroll
            for (int i = 0; i < PER; i++)
#pragma unroll
                for (int v = 0; v < WAVES; v++) asm volatile("" : "+v"(x[i][v]));
            float mx = tops[0];
#pragma unroll
            for (int v = 1; v < WAVES; v++) mx = fmaxf(mx, tops[v]);
#pragma unroll
            for (int v = 0; v < WAVES; v++) {
                float less = __builtin_amdgcn_exp2f(tops[v] - mx);
                asm volatile("" : "+v"(less));
                r[v] = sums[v] == 0.f ? 0.f : tops[v] == mx ? 1.f : less;           // (0: nothing was seen)
                den += sums[v] == 0.f ? 0.f : r[v] * sums[v];
            }
            const float inv = den != 0.f ? 1.f / den : 0.f;
            float *const part_row = ta_part_row(a, max(w.slot, 0), node, head, D);
            if (w.slot >= 0 && tid % SHARE == 0) {
                part_row[0] = mx;
                part_row[1] = den;
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int dim = 4 * (tid % SHARE) + 4 * SHARE * i;
                float4_t o = (float4_t)0.f;
#pragma unroll
                for (int v = 0; v < WAVES; v++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] += r[v] != 0.f ? r[v] * x[i][v][e] : 0.f;
                if (w.slot >= 0) *reinterpret_cast<float4_t *>(part_row + 4 + dim) = o;
                else {
                    half4_t h;
#pragma unroll
                    for (int e = 0; e < 4; e++) h[e] = (half_t)(den != 0.f ? o[e] * inv : 0.f);
                    half_t *to = a.out + ((int64_t)(rq.start + node) * a.heads + head) * D + dim;
                    if (((uintptr_t)a.out & 7) == 0) *reinterpret_cast<half4_t *>(to) = h;
                    else
#pragma unroll
                        for (int e = 0; e < 4; e++) to[e] = h[e];
                }
            }
        }
        if (w.at < w.end) __syncthreads();       // (the next request's go to the same places)
    }
    if (hk == 0) ta_idle<THREADS>(a, g_of, a.shares ? a.shares : a.B, D);
}

// ---- more rows: K and V come to LDS, for the WR waves of 16 QT rows each.  Many rows: what counts are the products and the softmax, and the scores of a stage are computed one stage ahead (AHEAD).
// Fewer: what counts are the bytes on their way, a stage more without that.  STREAM: past the last-level cache.
template <int D, int QT, int WR, bool AHEAD, bool STREAM>
__global__ __launch_bounds__(WR * 64, 2) void attention_tree_kernel(const ta_args a) {
    constexpr int W = D / 16, NC = D / 32, THREADS = WR * 64, ROWS = 16 * QT * WR;
    constexpr int PIECES = D / 32;               // requests of 1 KB (four lines of 256 bytes) for a tile of 16 rows
    constexpr int SHARE = 4 / WR;                // of a stage's four tiles (two of K, two of V) that a wave requests
    constexpr int EACH = SHARE * PIECES;
    // (an array per stage, K and then V: the compiler then knows that a request for one does not touch the others)
    __shared__ __attribute__((aligned(1024))) half_t s0[2 * TA_P * D], s1[2 * TA_P * D], s2[2 * TA_P * D], s3[2 * TA_P * D];
    __shared__ uint32_t odd_nodes[2];            // positions where something in v is infinite or NaN
    __shared__ int odd_held;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int units = a.kv_heads * a.row_tiles, unit = blockIdx.x % units, work = blockIdx.x / units;
    const int hk = unit % a.kv_heads, row0 = unit / a.kv_heads * ROWS, rep = a.heads / a.kv_heads;

    const int64_t page_step = (int64_t)a.kv_heads * D << a.shift, head_at = (int64_t)hk * D << a.shift;
    ta_work w;
    int first;
    for (bool more = ta_first<WR>(a, work, w, first); more; more = ta_next(a, w, first)) {
        const int r16 = ta_here(lane) & 15, g = ta_here(lane) >> 4;
        const ta_request &rq = w.rq;
        if (unit == 0 && w.st == 0 && tid == 0 && a.shares > 0) a.before[w.b] = w.before;
        const int all_rows = rq.n * rep;
        if (row0 >= all_rows) continue;
        const int held = rq.len - rq.n, st_first = w.st, st_end = w.st_end;
        ta_pages pg = {a.table + (int64_t)w.b * a.max_pages, (rq.len - 1) / 16, a.shift, a.pool, 1, 0, 0, 0};

        // ---- the rows of the cache
        // lane -> row and piece of it, for the requests of 1 KB, and where they lie (D == 64: two rows to a line): pieces XOR-ed with the line, V's by pairs
        auto stage_at = [&](auto ring) -> half_t * { return decltype(ring)::value == 0 ? s0 : decltype(ring)::value == 1 ? s1 : decltype(ring)::value == 2 ? s2 : s3; };
        const half_t *from[SHARE];                   // K or V of this head
#pragma unroll
        for (int u = 0; u < SHARE; u++) {
            const int v = (wave * SHARE + u) >> 1;
            from[u] = (v ? a.vpages : a.kpages) + head_at;
        }
        int gone_of = 0;                             // two bits for each of the last stages requested, the latest lowest
        auto request = [&](auto ring, int st) __attribute__((always_inline)) {
            half_t *const to = stage_at(ring);
            const int rel = 2 * (st - st_first);
            if (rel > 0 && (rel & 63) == 0) {
                pg.take();
                pg.load(st + 32);
            }
            gone_of = gone_of << 2 | (int)(pg.gone >> (rel & 63) & 3);
#pragma unroll
            for (int u = 0; u < SHARE; u++) {
                const int which = wave * SHARE + u, v = which >> 1, tile = which & 1;
                const int id = (int)bs_read((uint32_t)pg.id, (rel & 63) + tile), pos = min(2 * st + tile, pg.last_tile) * 16;
                const half_t *p = from[u] + (int64_t)id * page_step + (pos & ((1 << a.shift) - 1)) * D;
                const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, -1, 0x00020000);
                auto all = [&](auto whole) __attribute__((always_inline)) {
                    const int rows = rq.len - pos;   // rows of the tile that are there (the last one again behind them)
#pragma unroll
                    for (int j = 0; j < PIECES; j++) {
                        const int line = 4 * j + g;
                        int row, piece;
                        if (D == 128) {
                            row = line;
                            piece = r16 ^ (v ? 2 * (line & 7) : line);
                        } else {
                            row = 2 * line + (r16 >> 3);
                            piece = (r16 & 7) ^ (v ? 2 * (line & 3) : line & 7);
                        }
                        if (!decltype(whole)::value) row = min(row, rows - 1);
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (ta_lds)(to + (which * PIECES + j) * 512), 16, row * (D * 2) + 16 * piece, 0, 0, STREAM ? 2 : 0);
                    }
                };
                if (pos + 16 <= rq.len) all(std::true_type{});
                else all(std::false_type{});
            }
        };
        auto k_at = [](int row, int piece) { return D == 128 ? row * D + 8 * (piece ^ (row & 15)) : (row >> 1) * 128 + 64 * (row & 1) + 8 * (piece ^ (row >> 1 & 7)); };
        // 16 lanes read four rows of 16 dimensions of V, four in each lane, and get them turned: a lane a dimension.  Dimensions 16 j ..: XOR-ed with 16 j
        const int v_row = 4 * g + (r16 >> 2), v_from = TA_P * D + (D == 128 ? v_row * D + 16 * (v_row & 7) : (v_row >> 1) * 128 + 64 * (v_row & 1) + 16 * (v_row >> 1 & 3)) + 4 * (r16 & 3);

        __syncthreads();                             // (nobody is at the request before this one any more)
        if (tid < 2) odd_nodes[tid] = 0;             // (behind a barrier of the first stage when it is next written)
        if (tid == 2) odd_held = 0;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");    // (the loop's barriers alone wait for no LDS write)
        pg.load(st_first);
        pg.take();
        pg.load(st_first + 32);
        request(std::integral_constant<int, 0>{}, st_first);
        if (st_first + 1 < st_end) request(std::integral_constant<int, 1>{}, st_first + 1);
        else gone_of <<= 2;
        if (!AHEAD) {
            if (st_first + 2 < st_end) request(std::integral_constant<int, 2>{}, st_first + 2);
            else gone_of <<= 2;
        }

        // ---- the rows of q
        const bool mine = row0 + 16 * QT * wave < all_rows;
        half8_t q8[QT][NC];
        auto sees = [&](int node) { return (uint64_t)a.masks[rq.start + node] & (rq.n < 64 ? (1ull << rq.n) - 1 : ~0ull); };
        uint64_t mask[QT];                           // (AHEAD: read again where they are needed, registers are short)
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int row = min(row0 + 16 * (QT * wave + t) + r16, all_rows - 1), node = ta_node(row, rep, a.per_rep), head = hk * rep + row - node * rep;
            const half_t *p = a.q + (int64_t)(rq.start + node) * a.ldq + head * D + 8 * g;
            if (((uintptr_t)a.q | (uintptr_t)(2 * a.ldq)) % 16 == 0) {
#pragma unroll
                for (int c = 0; c < NC; c++) q8[t][c] = *reinterpret_cast<const half8_t *>(p + 32 * c);
            } else {
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int e = 0; e < 8; e++) q8[t][c][e] = p[32 * c + e];
            }
            if (!AHEAD) mask[t] = sees(node);
        }

        const float scale2 = ta_scale(D);
        float m[QT], l[QT];                          // of row r16 of a tile; l over this lane's positions only
        float4_t acc[QT][W];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            m[t] = TA_LOW;
            l[t] = 0.f;
#pragma unroll
            for (int j = 0; j < W; j++) acc[t][j] = (float4_t)0.f;
        }
        // infinities and NaN in a stage's v become zeros, and their positions are noted
        auto clean = [&](half_t *sv, int st) {
#pragma unroll 1
            for (int i = ta_here(tid); i < TA_P * D / 8; i += THREADS) {
                half8_t v = *reinterpret_cast<const half8_t *>(sv + 8 * i);
                bool odd = false;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool fine = (__builtin_bit_cast(uint16_t, (half_t)v[e]) & 0x7c00u) != 0x7c00u;
                    odd = odd || !fine;
                    v[e] = fine ? v[e] : (half_t)0;
                }
                if (!odd) continue;
                *reinterpret_cast<half8_t *>(sv + 8 * i) = v;
                const int line = i / 16, row = D == 128 ? line : 2 * line + (i >> 3 & 1), node = TA_P * st + row - held;
                if (node < 0) odd_held = 1;
                else if (node < rq.n) atomicOr(&odd_nodes[node >> 5], 1u << (node & 31));
            }
            __syncthreads();
        };
        auto scores = [&](const half_t *sk, float4_t (&s)[QT][2]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                half8_t k8[NC];
#pragma unroll
                for (int c = 0; c < NC; c++) k8[c] = *reinterpret_cast<const half8_t *>(sk + k_at(16 * i + r16, 4 * c + g));
#pragma unroll
                for (int t = 0; t < QT; t++) s[t][i] = (float4_t)0.f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int t = 0; t < QT; t++) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[c], q8[t][c], s[t][i], 0, 0, 0);
            }
        };
        // some of a stage's positions are nodes, behind the last one, or of a page that does not exist (`bits`: of its tiles)
        auto masked = [&](int st, int bits) { return TA_P * (st + 1) > held || bits != 0; };
        auto hide = [&](int st, int bits, float4_t (&s)[QT][2]) __attribute__((always_inline)) {
            if (AHEAD) {
#pragma unroll
                for (int t = 0; t < QT; t++) mask[t] = sees(ta_node(min(row0 + 16 * (QT * wave + t) + (ta_here(lane) & 15), all_rows - 1), rep, a.per_rep));
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    const uint32_t seen = bits >> i & 1 ? 0 : ta_seen(mask[t], TA_P * st + 16 * i + 4 * g - held);
#pragma unroll
                    for (int e = 0; e < 4; e++) s[t][i][e] = seen >> e & 1 ? s[t][i][e] : -INFINITY;
                }
            }
        };
        // the requests of this wave but for the last `later` stages have landed; behind the barrier everybody's have
        auto landed = [&](auto later) {
            constexpr int N = decltype(later)::value * EACH;
            static_assert(N < 64, "what the counter holds");
            __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | (N >> 4 << 14));
        };
        auto together = [&]() {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        float4_t sa[QT][2], sb[QT][2];
        half8_t p8[QT], rest8[QT];              // a weight is the sum of two
        half8_t vt[W];
        float r[QT];
        auto values = [&](const half_t *stage) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < W; j++) {
                typedef short short4_t __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) short4_t *from_t;
                const half_t *const p = stage + (v_from ^ 16 * j);
                const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((from_t)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((from_t)(p + 16 * D));
                vt[j] = __builtin_bit_cast(half8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        };
        // the running maximum and sum, the weights, and what the older sums are to be multiplied by
        auto softmax = [&](const float4_t (&s)[QT][2]) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < QT; t++) {
                float mx = s[t][0][0];
#pragma unroll
                for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[t][i >> 2][i & 3]);
                mx = across<32>(across<16>(mx));
                const float mn = fmaxf(m[t], mx * scale2), from = mn - TA_UP;
                r[t] = __builtin_amdgcn_exp2f(m[t] - mn);
                m[t] = mn;
                float sum[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float p[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][(i + e) >> 2][(i + e) & 3], scale2, -from));
                        sum[e] += p[e];
                    }
                    ta_terms(p, i, p8[t], rest8[t]);
                }
                l[t] = l[t] * r[t] + (sum[0] + sum[1]);
            }
#pragma unroll
            for (int t = 0; t < QT; t++) asm volatile("" : "+v"(p8[t]), "+v"(rest8[t]));   // (computed here, beside the products, and not behind the branch)
        };
        auto output = [&]() __attribute__((always_inline)) {
            if (__any(r[0] != 1.f || r[QT - 1] != 1.f)) {
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int j = 0; j < W; j++) acc[t][j] *= r[t];
            }
#pragma unroll
            for (int j = 0; j < W; j++) {
#pragma unroll
                for (int t = 0; t < QT; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[j], p8[t], acc[t][j], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < QT; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[j], rest8[t], acc[t][j], 0, 0, 0);
            }
        };
        // a stage
        auto walk = [&](auto ring, int st) __attribute__((always_inline)) {
            constexpr int R = decltype(ring)::value;
            // behind the barrier this stage is there, and nobody reads the one before this any more
            if (st + 2 < st_end) landed(std::integral_constant<int, 2>{});
            else if (st + 1 < st_end) landed(std::integral_constant<int, 1>{});
            else landed(std::integral_constant<int, 0>{});
            together();
            if (st + 3 < st_end) request(std::integral_constant<int, (R + 3) % 4>{}, st + 3);
            else gone_of <<= 2;
            const int bits = gone_of >> 6 & 3;
            half_t *const at = stage_at(ring);
            if (masked(st, bits)) clean(at + TA_P * D, st);
            if (!mine) return;
            values(at);
            scores(at, sa);
            if (masked(st, bits)) hide(st, bits, sa);
            softmax(sa);
            output();
        };
        // two stages: the second one's scores beside the first one's softmax
        auto walk_two = [&](auto ring, int st) __attribute__((always_inline)) {
            constexpr int R = decltype(ring)::value;
            landed(std::integral_constant<int, 0>{});
            together();
#pragma unroll
            for (int i = 2; i < 4; i++) {
                if (st + i >= st_end) gone_of <<= 2;
                else if (i == 2) request(std::integral_constant<int, (R + 2) % 4>{}, st + 2);
                else request(std::integral_constant<int, (R + 3) % 4>{}, st + 3);
            }
            const int bits = gone_of >> 6 & 3, bits_next = gone_of >> 4 & 3;
            half_t *const at = stage_at(ring), *const at_next = stage_at(std::integral_constant<int, R + 1>{});
            const bool two = st + 1 < st_end;
            if (masked(st, bits)) clean(at + TA_P * D, st);
            if (two && masked(st + 1, bits_next)) clean(at_next + TA_P * D, st + 1);
            if (!mine) return;
            scores(at, sa);
            if (masked(st, bits)) hide(st, bits, sa);
            scores(at_next, sb);                 // (behind the last stage: of whatever is there, for nobody)
            values(at);
            softmax(sa);
#pragma unroll
            for (int i = 0; i < 8 * QT; i++) {
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);           // a matrix instruction, then what fills its time
                __builtin_amdgcn_sched_group_barrier(0x402, 6, 0);
            }
            output();
            if (!two) return;
            values(at_next);
            if (masked(st + 1, bits_next)) hide(st + 1, bits_next, sb);
            softmax(sb);
            output();
        };
        for (int st = st_first; st < st_end; st += 4) {
            if (AHEAD) {
                walk_two(std::integral_constant<int, 0>{}, st);
                if (st + 2 < st_end) walk_two(std::integral_constant<int, 2>{}, st + 2);
            } else {
                walk(std::integral_constant<int, 0>{}, st);
                if (st + 1 < st_end) walk(std::integral_constant<int, 1>{}, st + 1);
                if (st + 2 < st_end) walk(std::integral_constant<int, 2>{}, st + 2);
                if (st + 3 < st_end) walk(std::integral_constant<int, 3>{}, st + 3);
            }
        }
        if (!mine) continue;

        // ---- what the wave has: [max, sum, pad, pad, weighted v] where other workgroups have parts, else the result
        const bool cut = w.slot >= 0;
        uint32_t again[QT];                          // (bit r: row r of the tile is computed again)
#pragma unroll
        for (int t = 0; t < QT; t++) {
            l[t] = across<32, true>(across<16, true>(l[t]));
            const int at = row0 + 16 * (QT * wave + t) + (ta_here(lane) & 15), row = min(at, all_rows - 1), node = ta_node(row, rep, a.per_rep), head = hk * rep + row - node * rep;
            const bool there = at < all_rows;
            const uint64_t seen = AHEAD ? sees(node) : mask[t];
            // NaN, or an infinity; a position that it sees had one
            float sum = l[t];
#pragma unroll
            for (int j = 0; j < W; j++) sum += (acc[t][j][0] - acc[t][j][0]) + (acc[t][j][1] - acc[t][j][1]) + (acc[t][j][2] - acc[t][j][2]) + (acc[t][j][3] - acc[t][j][3]);
            const uint64_t bad = __ballot(there && (sum != sum || odd_held != 0 || (seen & ((uint64_t)odd_nodes[1] << 32 | odd_nodes[0])) != 0));
            again[t] = (uint32_t)((bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffff);
            if (!there) continue;
            const float inv = l[t] != 0.f ? 1.f / l[t] : 0.f;              // (0: nothing was seen)
            if (cut) {
                float *to = ta_part_row(a, w.slot, node, head, D);
                if (g == 0) {
                    to[0] = m[t];
                    to[1] = l[t];
                }
#pragma unroll
                for (int j = 0; j < W; j++) *reinterpret_cast<float4_t *>(to + 4 + 16 * j + 4 * g) = acc[t][j];
            } else {
                half_t *to = a.out + ((int64_t)(rq.start + node) * a.heads + head) * D;
                const bool whole = ((uintptr_t)a.out & 7) == 0;
#pragma unroll
                for (int j = 0; j < W; j++) {        // row 4 g + i of product j is dimension 16 j + 4 g + i
                    half4_t o;
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] = (half_t)(acc[t][j][i] * inv);
                    if (whole) *reinterpret_cast<half4_t *>(to + 16 * j + 4 * g) = o;
                    else
#pragma unroll
                        for (int i = 0; i < 4; i++) to[16 * j + 4 * g + i] = o[i];
                }
            }
        }
        uint32_t all_again = 0;
#pragma unroll
        for (int t = 0; t < QT; t++) all_again |= again[t] << 16 * t;
        all_again = __builtin_amdgcn_readfirstlane(all_again);
#pragma unroll 1
        while (__builtin_expect(all_again != 0, 0)) {
            constexpr int PER = D / 64;
            const int which = __builtin_ctz(all_again), row = row0 + 16 * QT * wave + which, node = ta_node(row, rep, a.per_rep), head = hk * rep + row - node * rep;
            all_again &= all_again - 1;
            const ta_again<D> x(a, rq, pg.ids, node, head, hk, st_first * TA_P, min(st_end * TA_P, rq.len), scale2);
            const int64_t token_head = (int64_t)(rq.start + node) * a.heads + head;
            if (cut) {
                float *to = ta_part_row(a, w.slot, node, head, D);
                if (lane == 0) {
                    to[0] = x.top;
                    to[1] = x.sum;
                }
#pragma unroll
                for (int e = 0; e < PER; e++) to[4 + PER * ta_here(lane) + e] = x.o[e];
            } else {
                const float inv = x.sum != 0.f ? 1.f / x.sum : 0.f;
#pragma unroll
                for (int e = 0; e < PER; e++) a.out[token_head * D + PER * ta_here(lane) + e] = (half_t)(x.sum != 0.f ? x.o[e] * inv : 0.f);
            }
        }
    }
    if (unit == 0) ta_idle<THREADS>(a, work, a.shares ? a.shares : a.B, D);
}

// The parts of a row of a head put together, in order: D / 4 threads each, a workgroup a token's row.  What it takes is a chain of latencies: the request, looked for by 64 lanes at once, its lengths, the parts.
template <int D>
__global__ __launch_bounds__(256) void attention_tree_merge_kernel(const ta_args a) {
    constexpr int PER = D / 4, HEADS = 256 / PER, BATCH = 8;             // parts that are requested at once
    const int groups = (a.heads + HEADS - 1) / HEADS, t = blockIdx.x / groups, head = (blockIdx.x - t * groups) * HEADS + threadIdx.x / PER, dim = threadIdx.x % PER * 4, lane = threadIdx.x & 63;
    int lo = 0, hi = a.B;                        // the request: the first whose rows end behind t
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64, at = min(lo + step * (lane + 1), hi) - 1;        // the last request of the lane's part
        const int behind = __builtin_popcountll(__ballot(a.starts[at + 1] <= t)), first = min(lo + step * behind, hi);
        if (first < hi) hi = min(first + step, hi) - 1;
        lo = first;
    }
    if (lo >= a.B || head >= a.heads) return;
    const ta_request rq(a, lo);
    const int node = t - rq.start, stages = rq.stages();
    if (node < 0 || node >= rq.n) return;        // (zeros already)
    const int sum = a.before[a.B], shares = a.before[a.B + 1], per = a.before[a.B + 2], from = a.before[lo];
    const int g0 = per ? from : ta_whose(from, sum, shares), g1 = per ? from + ta_parts(stages, per) - 1 : ta_whose(from + stages - 1, sum, shares);
    if (g0 == g1) return;                        // written by the first launch
    const int slot0 = 2 * g0 + (per == 0 && from != ta_begins(g0, sum, shares));
    float mx = TA_LOW, den = 0.f;
    float4_t o = (float4_t)0.f;
    for (int j0 = g0; j0 <= g1; j0 += BATCH) {
        float m[BATCH], l[BATCH];
        float4_t v[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            const int g = min(j0 + j, g1);
            const float *p = ta_part_row(a, g == g0 ? slot0 : 2 * g, node, head, D);
            m[j] = p[0];
            l[j] = j0 + j <= g1 ? p[1] : 0.f;
            v[j] = *reinterpret_cast<const float4_t *>(p + 4 + dim);
        }
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
            if (l[j] == 0.f) continue;           // (nothing was seen, or no part)
            const float top = fmaxf(mx, m[j]), r0 = mx == top ? 1.f : __builtin_amdgcn_exp2f(mx - top), r = m[j] == top ? 1.f : __builtin_amdgcn_exp2f(m[j] - top);
            den = den * r0 + r * l[j];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (r0 != 0.f ? o[e] * r0 : 0.f) + (r != 0.f ? r * v[j][e] : 0.f);
            mx = top;
        }
    }
    half_t *to = a.out + ((int64_t)t * a.heads + head) * D + dim;
    const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) to[e] = (half_t)(den != 0.f ? o[e] * inv : 0.f);
}

__global__ __launch_bounds__(256) void attention_tree_zero_kernel(half_t *__restrict__ out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = (half_t)0;
}

struct ta_shape {
    int rows, units, shares;                     // rows of a workgroup
};
ta_shape shape_of(int B, int nodes, int heads, int kv_heads, int64_t positions) {
    ta_shape p;
    const int64_t rows = (int64_t)(heads / kv_heads) * nodes;
    // As many rows as there are, up to 128: K and V are read once for each tile of them.  (33 to 64 rows with K and V in registers, four tiles of columns to a wave: a quarter slower for 48 requests of up to
    // 4096 with 16 nodes; 64 rows to a wave, 256 to a workgroup: half slower for 2 of 80000 with trees of 64, the sums no longer fit the registers.)
    p.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    p.units = kv_heads * (int)bs_cdiv(rows, p.rows);
    // Two workgroups to a CU (768 of them in all: 233 us, 1024 208, 512 183 for 64 requests of 4000 with 16 nodes).  Tables of up to 512 positions, 16 stages, are not cut: the second launch costs 2.5 us and parts their
    // traffic (us, uncut / cut: one of 390 with 8 nodes 11.8 / 11.9, 16 of 390 12.7 / 16.2, 64 of 390 23 / 27; with 32 nodes 24 / 16, 26 / 29, 40 / 48).
    p.shares = positions <= 512 ? 0 : 512 / p.units > 1 ? 512 / p.units : 1;
    return p;
}
int64_t before_bytes(int B) { return bs_cdiv(4ll * (B + 3), 16) * 16; }

// A cache that the last-level cache cannot hold is read past it, where a workgroup of the unit has all of its rows (64 requests of 4000, 4 nodes 186 -> 169 us, 8 nodes 189 -> 173, 16 nodes 199 -> 183).  Where several read the
// same positions the second one finds them there (256 rows: a quarter slower past it).
constexpr int64_t TA_STREAM = 256ll << 20;

template <int D>
int launch(const ta_args &a, const ta_shape &p, hipStream_t s) {
    const unsigned grid = (unsigned)((int64_t)(p.shares ? p.shares : a.B) * p.units);
    const bool stream = ((int64_t)a.pool << a.shift) * a.kv_heads * D * 4 >= TA_STREAM;
    if (p.rows == 16) (stream ? attention_tree_few_kernel<D, 1, true> : attention_tree_few_kernel<D, 1, false>)<<<grid, 256, 0, s>>>(a);
    else if (p.rows == 32) (stream ? attention_tree_few_kernel<D, 2, true> : attention_tree_few_kernel<D, 2, false>)<<<grid, 256, 0, s>>>(a);
    else if (p.rows == 64) (stream ? attention_tree_kernel<D, 1, 4, false, true> : attention_tree_kernel<D, 1, 4, false, false>)<<<grid, 256, 0, s>>>(a);
    else attention_tree_kernel<D, 2, 4, true, false><<<grid, 256, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    if (p.shares == 0) return BS_OK;
    attention_tree_merge_kernel<D><<<(unsigned)((int64_t)a.T * bs_cdiv(a.heads, 256 / (D / 4))), 256, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    return BS_OK;
}

}  // namespace

int64_t bs_attention_tree_scratch(int B, int T, int nodes, int heads, int kv_heads, int head_dim, int max_pages, int page) {
    const ta_shape p = shape_of(B, nodes, heads, kv_heads, (int64_t)max_pages * page);
    return p.shares ? before_bytes(B) + 2ll * p.shares * nodes * heads * (head_dim + 4) * 4 : 0;
}

int bs_launch_attention_tree(const half_t *q, int ldq, const half_t *kpages, const half_t *vpages, const int32_t *table, const int32_t *lengths, const int32_t *granted,
                             const int32_t *starts, const int64_t *masks, half_t *out, int B, int T, int nodes, int heads, int kv_heads, int head_dim, int shift, int max_pages,
                             int pool, void *workspace, hipStream_t s) {
    if (B == 0) {
        attention_tree_zero_kernel<<<256, 256, 0, s>>>(out, (int64_t)T * heads * head_dim);
        BS_LAUNCH_CHECK();
        return BS_OK;
    }
    const ta_shape p = shape_of(B, nodes, heads, kv_heads, (int64_t)max_pages << shift);
    const ta_args a = {q, kpages, vpages, table, lengths, granted, starts, masks, out, (int32_t *)workspace, (float *)((char *)workspace + before_bytes(B)), 1.f / (float)(heads / kv_heads), (float)p.units / (p.rows == 16 ? 32.f : 16.f), ldq, B, T, nodes,
                       heads, kv_heads, p.units / kv_heads, shift, max_pages, pool, p.shares, p.rows <= 32 ? 16 : 32};
    return head_dim == 128 ? launch<128>(a, p, s) : launch<64>(a, p, s);
}
