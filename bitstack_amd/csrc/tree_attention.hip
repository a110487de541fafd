// Attention of drafted tokens over the paged cache: out[t] = softmax(q[t] k^T / sqrt(D)) v over the positions that the request held and those nodes of its tree, stored
// behind them, that masks[t] names.
//
// The rows of a KV head of a request are its nodes' queries of that head's group, the head fastest: nodes * group of them, which all read the same K and V.  A workgroup takes up to 16 QT WR of
// them, the columns of both products, and walks the positions in stages of 64, which come to LDS straight from the pages (no registers), one stage ahead, one barrier per stage.
// WR waves take 16 QT rows each, WP waves share the positions of a stage; what these leave is put together in LDS at the end.
//   scores  S[position, row] = K q      16x16x32; the 16-byte pieces of K's rows are XOR-ed with the row's number, so that 16 rows of one piece lie in different banks
//   output  O[dim, row] += V^T P        16x16x32; a lane of the scores holds four positions of a row in each of two tiles of 16, which are the eight k slots of this product, and V
//                                       is used as it lies: product j takes element j of the W = D / 16 dimensions that a lane reads
// Maximum, sum and output are fp32, in base 2.  The weights are rounded to fp16 for the second product (the queries are given in fp16), the largest as 2^15, so that one of
// 2^-40 of the largest is still held; their sum is that of the fp32 weights.
//
// What a row does not see has a weight of zero, but zero times an infinity is NaN: in the stages with nodes V is looked through, and infinities and NaN, if any, are taken out of the
// product.  Rows that see them, or whose result is not finite for another reason, are computed again, each by a wave, in fp32.
//
// The split: as the lengths are known on the device alone, every workgroup works out from them what it is to do.  The first B workgroups of a unit (row tile, KV head) take one request each, or the
// first part of it; requests longer than C = (all stages) / (further parts) are cut, and the next workgroups take the further parts, in order.  Parts leave
// (max, sum, weighted v) in the workspace, and a second launch puts them together, in order: the result does not depend on which came first.
#include "common.h"

#include <type_traits>

namespace {

constexpr int TA_P = 64;                         // positions of a stage
constexpr float TA_LOW = -1e30f;                 // a maximum before the first score (finite scores are above it)
constexpr float TA_UP = 15.f;                    // log2 of the largest weight

struct ta_args {
    const half_t *q, *kpages, *vpages;
    const int32_t *table, *lengths, *granted, *starts;
    const int64_t *masks;
    half_t *out;
    int32_t *parts_of;                           // workspace: {first further part, further parts} of every token row
    float *part;                                 // ... and what the parts leave: [token row or (further part, node)][head][max, sum, pad, pad, weighted v]
    int ldq, B, T, nodes, heads, kv_heads, row_tiles, shift, max_pages, pool, parts, least;
};

struct ta_request {
    int start, end, n, len;                      // token rows, nodes (0: idle), positions with the nodes
    __device__ __forceinline__ ta_request(const ta_args &a, int b) {
        start = min(max(a.starts[b], 0), a.T);
        end = min(max(a.starts[b + 1], start), a.T);
        n = a.granted[b];
        len = a.lengths[b];
        if (n < 1 || n > a.nodes || n > end - start || len < n || (int64_t)len > (int64_t)a.max_pages << a.shift) n = len = 0;
    }
    __device__ __forceinline__ int stages() const { return (len + TA_P - 1) / TA_P; }
};
__device__ __forceinline__ int ta_further(int stages, int most) { return stages > most ? (stages + most - 1) / most - 1 : 0; }

// the larger of v here and in the lane whose number differs by W (16 or 32), or (SUM) both together
template <int W, bool SUM = false>
__device__ __forceinline__ float across(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = W == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];
    return SUM ? __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b) : fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

typedef __attribute__((address_space(3))) void *ta_lds;

template <int D, int QT, int WR, int WP>
__global__ __launch_bounds__(WR *WP * 64, WR *WP == 2 ? 1 : 2) void attention_tree_kernel(const ta_args a) {
    constexpr int W = D / 16, NC = D / 32, WAVES = WR * WP, THREADS = WAVES * 64, ROWS = 16 * QT * WR;
    constexpr int A = TA_P / 16 / WP;            // tiles of 16 positions that a wave takes of a stage
    constexpr int LINES = D / 32;                // requests of 1 KB for a tile of 16 rows
    constexpr int TILES = TA_P / 16 / WAVES;     // tiles that a wave requests of a stage: 1 or 2, of K and of V
    typedef half_t vec_t __attribute__((ext_vector_type(W)));
    // (an array per operand and stage: the compiler then knows that a request for one does not touch the others)
    __shared__ __attribute__((aligned(1024))) half_t sk0[TA_P * D], sk1[TA_P * D], sv0[TA_P * D], sv1[TA_P * D];
    __shared__ float wm[WP][ROWS], wl[WP][ROWS];
    __shared__ int sums[WAVES], found[4], again[ROWS], odd_held;
    __shared__ uint32_t odd_nodes[2];            // positions where something in v is infinite or NaN
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int wr = wave / WP, wp = wave % WP;
    const int units = a.kv_heads * a.row_tiles, unit = blockIdx.x % units, work = blockIdx.x / units;
    const int hk = unit % a.kv_heads, row0 = unit / a.kv_heads * ROWS, rep = a.heads / a.kv_heads;

    // ---- which request, which part of it
    int b = work, part = 0, most = 0, further = 0, place = 0;          // stages of a part at most; further parts of this request, and the first one's number
    const bool first_part = work < a.B;
    if (a.parts > 0) {
        int all = 0;
        for (int i = tid; i < a.B; i += THREADS) all += ta_request(a, i).stages();
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) all += __shfl_xor(all, o, 64);
        if (lane == 0) sums[wave] = all;
        __syncthreads();
        all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) all += sums[w];
        most = max(a.least, (all + a.parts - 1) / a.parts);
        if (first_part) further = ta_further(ta_request(a, b).stages(), most);
    }
    if (!first_part || further > 0) {            // numbers of the further parts: a running sum over the requests
        if (tid == 0) found[0] = -1;
        int before = 0;
        const int wanted = work - a.B;
        for (int i0 = 0; i0 < a.B; i0 += THREADS) {
            const int i = i0 + tid, mine = i < a.B ? ta_further(ta_request(a, i).stages(), most) : 0;
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
        if (!first_part) part = wanted - place + 1;
    }
    const ta_request rq(a, b);
    const int64_t orow = (int64_t)a.heads * D;
    if (part == 0 && unit == 0) {                // rows that are no node: zeros; this request's, and some of those behind the last request's
        auto idle = [&](int t) {
            for (int i = tid; i < orow; i += THREADS) a.out[t * orow + i] = (half_t)0;
            if (a.parts > 0 && tid < 2) a.parts_of[2 * t + tid] = 0;
        };
        for (int t = rq.start + rq.n; t < rq.end; t++) idle(t);
        const int last = min(max(a.starts[a.B], 0), a.T), first = min(max(a.starts[0], 0), a.T);
        for (int t = last + b; t < a.T; t += a.B) idle(t);
        for (int t = b; t < first; t += a.B) idle(t);
        if (a.parts > 0)
            for (int j = tid; j < rq.n; j += THREADS) {
                a.parts_of[2 * (rq.start + j)] = place;
                a.parts_of[2 * (rq.start + j) + 1] = further;
            }
    }
    const int all_rows = rq.n * rep;
    if (row0 >= all_rows) return;
    const int held = rq.len - rq.n, stages = rq.stages(), parts = further + 1;
    const int st_first = (int)((int64_t)stages * part / parts), st_end = (int)((int64_t)stages * (part + 1) / parts);

    // ---- the rows of the cache
    const int64_t page_step = (int64_t)a.kv_heads * D << a.shift, head_at = (int64_t)hk * D << a.shift;
    const int32_t *ids = a.table + (int64_t)b * a.max_pages;
    const int last_tile = (rq.len - 1) / 16;
    // the pages of a stage's tiles (those behind the last tile are the last again), and which of them exist; ones that do not are read as another of the stage
    struct stage_pages { int id[4]; };
    auto pages_of = [&](int st) {
        stage_pages p;
#pragma unroll
        for (int i = 0; i < 4; i++) p.id[i] = ids[(min(4 * st + i, last_tile) * 16) >> a.shift];
        return p;
    };
    auto good = [&](int id) { return id >= 0 && id < a.pool; };
    // lane -> row of a tile and piece of it, for the requests of 1 KB, and where they lie: K's pieces XOR-ed with the row (D == 64: two rows to a line of 256 bytes; V's rows change places in it by turns)
    auto request = [&](auto stage, int st, const stage_pages &p) {
        half_t *const k_to = decltype(stage)::value ? sk1 : sk0, *const v_to = decltype(stage)::value ? sv1 : sv0;
        int other = 0;
#pragma unroll
        for (int i = 3; i >= 0; i--) other = good(p.id[i]) ? p.id[i] : other;
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            const int tile = wave * TILES + i;
            int id = p.id[0];
#pragma unroll
            for (int e = 1; e < 4; e++) id = tile == e ? p.id[e] : id;
            id = good(id) ? id : other;
            const int pos = min(4 * st + tile, last_tile) * 16, rows = rq.len - pos;       // rows of the tile that are there (the last one again behind them)
            const int64_t at = (int64_t)id * page_step + head_at + (int64_t)(pos & ((1 << a.shift) - 1)) * D;
            const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((void *)(a.kpages + at), 0, -1, 0x00020000);
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((void *)(a.vpages + at), 0, -1, 0x00020000);
#pragma unroll
            for (int j = 0; j < LINES; j++) {
                const int line = 4 * j + g;
                const int krow = D == 128 ? line : 2 * line + (r16 >> 3), piece = D == 128 ? r16 ^ line : (r16 & 7) ^ (line & 7);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (ta_lds)(k_to + tile * 16 * D + j * 512), 16, min(krow, rows - 1) * (D * 2) + 16 * piece, 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < LINES; j++) {
                const int line = 4 * j + g;
                const int vrow = D == 128 ? line : 2 * line + ((r16 >> 3) ^ (line >> 1 & 1)), piece = D == 128 ? r16 : r16 & 7;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (ta_lds)(v_to + tile * 16 * D + j * 512), 16, min(vrow, rows - 1) * (D * 2) + 16 * piece, 0, 0, 0);
            }
        }
    };
    auto k_at = [](int row, int piece) { return D == 128 ? row * D + 8 * (piece ^ (row & 15)) : (row >> 1) * 128 + 64 * (row & 1) + 8 * (piece ^ (row >> 1 & 7)); };
    auto v_at = [](int row) { return D == 128 ? row * D : (row >> 1) * 128 + 64 * ((row ^ row >> 2) & 1); };

    if (tid < 2) odd_nodes[tid] = 0;             // (behind a barrier of the first stage when it is next written)
    if (tid == 2) odd_held = 0;
    stage_pages now = pages_of(st_first), next = pages_of(min(st_first + 1, st_end - 1));
    request(std::integral_constant<int, 0>{}, st_first, now);

    // ---- the rows of q
    const bool mine = row0 + 16 * QT * wr < all_rows;
    half8_t q8[QT][NC];
    uint64_t mask[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int row = min(row0 + 16 * (QT * wr + t) + r16, all_rows - 1), node = row / rep;
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

    const float scale2 = (D == 128 ? 0.08838834764831845f : 0.125f) * 1.4426950408889634f;    // log2(e) / sqrt(D)
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
        for (int i = tid; i < TA_P * D / 8; i += THREADS) {
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
            const int line = i / 16, row = D == 128 ? line : 2 * line + ((i >> 3 & 1) ^ (line >> 1 & 1)), node = TA_P * st + row - held;
            if (node < 0) odd_held = 1;
            else if (node < rq.n) atomicOr(&odd_nodes[node >> 5], 1u << (node & 31));
        }
        __syncthreads();
    };
    // a stage, from LDS: scores, weights, output.  masked: some of its positions are nodes, behind the last one, or of pages that do not exist (bits of `there`: tiles that do)
    auto step = [&](bool masked, const half_t *sk, const half_t *sv, int st, int there) __attribute__((always_inline)) {
        float4_t s[QT][A];
#pragma unroll
        for (int i = 0; i < A; i++) {
            half8_t k8[NC];
#pragma unroll
            for (int c = 0; c < NC; c++) k8[c] = *reinterpret_cast<const half8_t *>(sk + k_at(16 * (A * wp + i) + r16, 4 * c + g));
#pragma unroll
            for (int t = 0; t < QT; t++) s[t][i] = (float4_t)0.f;
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int t = 0; t < QT; t++) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8[c], q8[t][c], s[t][i], 0, 0, 0);
        }
        vec_t v8[8];
        auto fetch_v = [&](int h) {
#pragma unroll
            for (int i = 0; i < 8; i++) v8[i] = *reinterpret_cast<const vec_t *>(sv + v_at(16 * (A * wp + 2 * h + (i >> 2)) + 4 * g + (i & 3)) + W * r16);
        };
        fetch_v(0);                              // (arrives during the softmax)
        __builtin_amdgcn_sched_barrier(0);
        if (masked) {
#pragma unroll
            for (int i = 0; i < A; i++) {
                const int node = TA_P * st + 16 * (A * wp + i) + 4 * g - held;             // (below 0: a position that the request held)
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    uint32_t seen = node >= 64 ? 0 : node >= 0 ? (uint32_t)(mask[t] >> node) : node <= -4 ? 15 : (uint32_t)mask[t] << -node | ((1u << -node) - 1);
                    if (!(there >> (A * wp + i) & 1)) seen = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) s[t][i][e] = seen >> e & 1 ? s[t][i][e] : -INFINITY;
                }
            }
        }
        float r[QT];
        half8_t p8[A / 2][QT];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            float mx = s[t][0][0];
#pragma unroll
            for (int i = 1; i < 4 * A; i++) mx = fmaxf(mx, s[t][i >> 2][i & 3]);
            mx = across<32>(across<16>(mx));
            const float mn = fmaxf(m[t], mx * scale2), from = mn - TA_UP;
            r[t] = __builtin_amdgcn_exp2f(m[t] - mn);
            m[t] = mn;
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4 * A; i++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i >> 2][i & 3], scale2, -from));
                sum[i & 1] += p;
                p8[i >> 3][t][i & 7] = (half_t)p;
            }
            l[t] = l[t] * r[t] + (sum[0] + sum[1]);
        }
        if (__any(r[0] != 1.f || r[QT - 1] != 1.f)) {
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
                for (int j = 0; j < W; j++) acc[t][j] *= r[t];
        }
#pragma unroll
        for (int h = 0; h < A / 2; h++) {
#pragma unroll
            for (int j = 0; j < W; j++) {
                const half8_t v = {v8[0][j], v8[1][j], v8[2][j], v8[3][j], v8[4][j], v8[5][j], v8[6][j], v8[7][j]};
#pragma unroll
                for (int t = 0; t < QT; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p8[h][t], acc[t][j], 0, 0, 0);
            }
            if (h + 1 < A / 2) fetch_v(h + 1);
        }
    };
    auto walk = [&](auto stage, int st) __attribute__((always_inline)) {
        // this wave's requests for the stage have landed; behind the barrier everybody's have, and nobody reads the other stage any more
        __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        int there = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) there |= (int)good(now.id[i]) << i;
        if (st + 1 < st_end) {
            request(std::integral_constant<int, 1 - decltype(stage)::value>{}, st + 1, next);
            now = next;
            next = pages_of(min(st + 2, st_end - 1));
        }
        half_t *const sk = decltype(stage)::value ? sk1 : sk0, *const sv = decltype(stage)::value ? sv1 : sv0;
        const bool masked = TA_P * (st + 1) > held || there != 15;
        if (masked) clean(sv, st);
        if (mine) step(masked, sk, sv, st, there);
    };
    for (int st = st_first; st < st_end; st += 2) {
        walk(std::integral_constant<int, 0>{}, st);
        if (st + 1 < st_end) walk(std::integral_constant<int, 1>{}, st + 1);
    }

    // ---- what the waves have: rows that are NaN are computed again, the others put together
    for (int i = tid; i < ROWS; i += THREADS) again[i] = 0;
    __syncthreads();                             // (nobody reads a stage any more: the weighted v take their place)
    auto wo_at = [&](int w, int row) -> float * {                          // [WP][ROWS][D] over the four arrays
        constexpr int PER = TA_P / 2;            // rows of an array
        const int i = w * ROWS + row, array = i / PER;
        return reinterpret_cast<float *>(array == 0 ? sk0 : array == 1 ? sk1 : array == 2 ? sv0 : sv1) + (i - array * PER) * D;
    };
    static_assert(WP * ROWS <= 4 * (TA_P / 2), "what the waves leave must fit the stages");
    if (mine) {
#pragma unroll
        for (int t = 0; t < QT; t++) {
            const int row = 16 * (QT * wr + t) + r16;
            l[t] = across<32, true>(across<16, true>(l[t]));
            if (g == 0) {
                wm[wp][row] = m[t];
                wl[wp][row] = l[t];
            }
            float sum = l[t];
#pragma unroll
            for (int j = 0; j < W; j++) sum += (acc[t][j][0] - acc[t][j][0]) + (acc[t][j][1] - acc[t][j][1]) + (acc[t][j][2] - acc[t][j][2]) + (acc[t][j][3] - acc[t][j][3]);
            // NaN, or an infinity; a position that it sees had one
            if (sum != sum || odd_held != 0 || (mask[t] & ((uint64_t)odd_nodes[1] << 32 | odd_nodes[0])) != 0) again[row] = 1;
#pragma unroll
            for (int i = 0; i < 4; i++)          // row 4 g + i of product j is dimension W (4 g + i) + j
#pragma unroll
                for (int j = 0; j < W; j += 4)
                    *reinterpret_cast<float4_t *>(wo_at(wp, row) + W * (4 * g + i) + j) = (float4_t){acc[t][j][i], acc[t][j + 1][i], acc[t][j + 2][i], acc[t][j + 3][i]};
        }
    }
    __syncthreads();
    const int rows = min(ROWS, all_rows - row0);
    for (int row = wave; row < rows; row += WAVES) {
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(again[row]) == 0, 1)) continue;
        // One row by one wave: the largest score first, then the sums.  A lane has a position's score, and owns dimensions EACH lane .. of the output.
        constexpr int EACH = D / 64;
        const int node = (row0 + row) / rep, p_end = min(st_end * TA_P, rq.len);
        const half_t *qr = a.q + (int64_t)(rq.start + node) * a.ldq + (hk * rep + row0 + row - node * rep) * D;
        const uint64_t sees = (uint64_t)a.masks[rq.start + node];
        auto where = [&](int p) {                // halves in front of position p; -1: not seen, or not there
            if (p >= p_end || (p >= held && !(sees >> (p - held) & 1))) return (int64_t)-1;
            const int id = ids[p >> a.shift];
            return good(id) ? (int64_t)id * page_step + head_at + (int64_t)(p & ((1 << a.shift) - 1)) * D : (int64_t)-1;
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
        float top = -INFINITY, sum = 0.f, o[EACH] = {};
        for (int p0 = st_first * TA_P; p0 < p_end; p0 += 64) top = fmaxf(top, score(where(p0 + lane)));
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        const float from = top == -INFINITY ? 0.f : top;
        for (int p0 = st_first * TA_P; p0 < p_end; p0 += 64) {
            const int64_t at = where(p0 + lane);
            const float w = __builtin_amdgcn_exp2f(score(at) - from + TA_UP);      // (a score of -inf weighs nothing; one of +inf, or NaN, is NaN)
            sum += w;
#pragma unroll 1
            for (int i = 0; i < 64; i++) {
                const int64_t ai = __shfl(at, i, 64);
                const float wi = __shfl(w, i, 64);
                if (ai < 0 || wi == 0.f) continue;
#pragma unroll
                for (int e = 0; e < EACH; e++) o[e] = __builtin_fmaf(wi, (float)a.vpages[ai + EACH * lane + e], o[e]);
            }
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x, 64);
        if (lane == 0) {
#pragma unroll
            for (int w = 0; w < WP; w++) {
                wm[w][row] = w == 0 ? (top == -INFINITY ? TA_LOW : top) : TA_LOW;
                wl[w][row] = w == 0 ? sum : 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < EACH; e++) wo_at(0, row)[EACH * lane + e] = o[e];
    }
    __syncthreads();
    for (int it = tid; it < rows * (D / 4); it += THREADS) {
        const int row = it / (D / 4), dim = it % (D / 4) * 4, all_row = row0 + row, node = all_row / rep, head = hk * rep + all_row - node * rep;
        float mx = wm[0][row];
#pragma unroll
        for (int w = 1; w < WP; w++) mx = fmaxf(mx, wm[w][row]);
        float den = 0.f;
        float4_t o = (float4_t)0.f;
#pragma unroll
        for (int w = 0; w < WP; w++) {
            if (wl[w][row] != 0.f) {             // (0: nothing was seen)
                const float r = wm[w][row] == mx ? 1.f : __builtin_amdgcn_exp2f(wm[w][row] - mx);
                den += r * wl[w][row];
                o += r * *reinterpret_cast<const float4_t *>(wo_at(w, row) + dim);
            }
        }
        if (further > 0) {
            const int64_t at = part == 0 ? (int64_t)(rq.start + node) * a.heads + head : ((int64_t)a.T + (int64_t)(place + part - 1) * a.nodes + node) * a.heads + head;
            float *to = a.part + at * (D + 4);
            *reinterpret_cast<float4_t *>(to + 4 + dim) = o;
            if (dim == 0) {
                to[0] = mx;
                to[1] = den;
            }
        } else {
            half_t *to = a.out + (int64_t)(rq.start + node) * orow + (int64_t)head * D + dim;
            const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) to[e] = (half_t)(den != 0.f ? o[e] * inv : 0.f);
        }
    }
}

// The parts of a row of a head put together, in order: D / 4 threads each.
template <int D>
__global__ __launch_bounds__(256) void attention_tree_merge_kernel(const float *__restrict__ part, const int32_t *__restrict__ parts_of, const int32_t *__restrict__ starts,
                                                                  half_t *__restrict__ out, int B, int T, int nodes, int heads) {
    constexpr int PER = D / 4;
    const int64_t i = (int64_t)blockIdx.x * (256 / PER) + threadIdx.x / PER;
    const int dim = threadIdx.x % PER * 4, t = (int)(i / heads), head = (int)(i % heads);
    if (t >= T) return;
    const int place = parts_of[2 * t], further = parts_of[2 * t + 1];
    if (further == 0) return;                    // written by the first launch
    int lo = 0, hi = B;                          // the request: the first whose rows end behind t
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (starts[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    const int node = t - max(starts[min(lo, B - 1)], 0);
    auto from = [&](int j) { return part + (j == 0 ? (int64_t)t * heads + head : ((int64_t)T + (int64_t)(place + j - 1) * nodes + node) * heads + head) * (D + 4); };
    float mx = TA_LOW, den = 0.f;
    float4_t o = (float4_t)0.f;
    for (int j0 = 0; j0 <= further; j0 += 4) {
        float m[4], l[4];
        float4_t v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float *p = from(min(j0 + j, further));
            m[j] = p[0];
            l[j] = j0 + j <= further ? p[1] : 0.f;
            v[j] = *reinterpret_cast<const float4_t *>(p + 4 + dim);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (l[j] == 0.f) continue;           // (nothing was seen, or no part)
            const float top = fmaxf(mx, m[j]), r0 = mx == top ? 1.f : __builtin_amdgcn_exp2f(mx - top), r = m[j] == top ? 1.f : __builtin_amdgcn_exp2f(m[j] - top);
            den = den * r0 + r * l[j];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (r0 != 0.f ? o[e] * r0 : 0.f) + (r != 0.f ? r * v[j][e] : 0.f);
            mx = top;
        }
    }
    half_t *to = out + ((int64_t)t * heads + head) * D + dim;
    const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) to[e] = (half_t)(den != 0.f ? o[e] * inv : 0.f);
}

__global__ __launch_bounds__(256) void attention_tree_zero_kernel(half_t *__restrict__ out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = (half_t)0;
}

struct ta_shape {
    int qt, wr, wp, row_tiles, units, parts, least;
};
ta_shape shape_of(int B, int nodes, int heads, int kv_heads, int64_t positions) {
    ta_shape p;
    const int rows = heads / kv_heads * nodes;
    p.qt = rows <= 16 ? 1 : 2;
    p.wr = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
    p.wp = rows <= 64 ? 2 : 1;
    p.row_tiles = (int)bs_cdiv(rows, 16 * p.qt * p.wr);
    p.units = kv_heads * p.row_tiles;
    const int64_t first = (int64_t)B * p.units, further = first <= 256 ? 512 - first : 768;
    p.least = 4;
    p.parts = positions <= p.least * TA_P ? 0 : (int)(further / p.units);
    return p;
}

template <int D>
int launch(const ta_args &a, const ta_shape &p, hipStream_t s) {
    const unsigned grid = (unsigned)((int64_t)(a.B + p.parts) * p.units);
    if (p.qt == 1) attention_tree_kernel<D, 1, 1, 2><<<grid, 128, 0, s>>>(a);
    else if (p.wr == 1) attention_tree_kernel<D, 2, 1, 2><<<grid, 128, 0, s>>>(a);
    else if (p.wr == 2) attention_tree_kernel<D, 2, 2, 2><<<grid, 256, 0, s>>>(a);
    else attention_tree_kernel<D, 2, 4, 1><<<grid, 256, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    if (p.parts == 0) return BS_OK;
    attention_tree_merge_kernel<D><<<(unsigned)bs_cdiv((int64_t)a.T * a.heads, 256 / (D / 4)), 256, 0, s>>>(a.part, a.parts_of, a.starts, a.out, a.B, a.T, a.nodes, a.heads);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
int64_t parts_of_bytes(int T) { return bs_cdiv(8ll * T, 16) * 16; }

}  // namespace

int64_t bs_attention_tree_scratch(int B, int T, int nodes, int heads, int kv_heads, int head_dim, int max_pages, int page) {
    const ta_shape p = shape_of(B, nodes, heads, kv_heads, (int64_t)max_pages * page);
    return p.parts ? parts_of_bytes(T) + ((int64_t)T + (int64_t)p.parts * nodes) * heads * (head_dim + 4) * 4 : 0;
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
    const ta_args a = {q, kpages, vpages, table, lengths, granted, starts, masks, out, (int32_t *)workspace, (float *)((char *)workspace + parts_of_bytes(T)), ldq, B, T, nodes,
                       heads, kv_heads, p.row_tiles, shift, max_pages, pool, p.parts, p.least};
    return head_dim == 128 ? launch<128>(a, p, s) : launch<64>(a, p, s);
}
