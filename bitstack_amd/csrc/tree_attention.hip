// Attention of drafted tokens over the paged cache: out[t] = softmax(q[t] k^T / sqrt(D)) v over the positions that the request held and those nodes of its tree, stored
// behind them, that masks[t] names.  The plain form: a workgroup per token row and head, a wave a position at a time, a lane D / 64 dimensions.
#include "common.h"

namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;

struct ta_args {
    const half_t *q, *kpages, *vpages;
    const int32_t *table, *lengths, *granted, *starts;
    const int64_t *masks;
    half_t *out;
    int ldq, B, T, nodes, heads, kv_heads, shift, max_pages, pool;
};

template <int D>
__global__ __launch_bounds__(THREADS) void attention_tree_kernel(const ta_args a) {
    constexpr int W = D / 64;
    __shared__ float wm[WAVES], wl[WAVES], wo[WAVES][D];
    const int head = blockIdx.x % a.heads, t = blockIdx.x / a.heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hk = head / (a.heads / a.kv_heads);
    int lo = 0, hi = a.B;                        // the last request that starts at t or before, and has rows
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.starts[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    const int b = lo;
    half_t *to = a.out + ((int64_t)t * a.heads + head) * D;
    int n = 0, len = 0;
    if (b < a.B) {
        const int start = a.starts[b], rows = min(a.starts[b + 1], a.T) - start;
        n = a.granted[b];
        len = a.lengths[b];
        if (n < 1 || n > a.nodes || n > rows || t - start >= n || len < n || (int64_t)len > (int64_t)a.max_pages << a.shift) n = 0;
    }
    float m = -INFINITY, l = 0.f, o[W] = {};
    if (n > 0) {
        float q[W];
        for (int w = 0; w < W; w++) q[w] = (float)a.q[(int64_t)t * a.ldq + head * D + W * lane + w];
        const uint64_t mask = (uint64_t)a.masks[t];
        for (int p = wave; p < len; p += WAVES) {
            if (p >= len - n && !(mask >> (p - len + n) & 1)) continue;
            const int id = a.table[(int64_t)b * a.max_pages + (p >> a.shift)];
            if (id < 0 || id >= a.pool) continue;
            const int64_t at = ((((int64_t)id * a.kv_heads + hk) << a.shift) + (p & ((1 << a.shift) - 1))) * D + W * lane;
            float s = 0.f;
            for (int w = 0; w < W; w++) s += q[w] * (float)a.kpages[at + w];
            for (int x = 32; x >= 1; x >>= 1) s += __shfl_xor(s, x, 64);
            s *= (D == 128 ? 0.08838834764831845f : 0.125f) * 1.4426950408889634f;
            if (s == -INFINITY) continue;
            const float mn = fmaxf(m, s), r = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn), e = __builtin_amdgcn_exp2f(s - mn);
            m = mn;
            l = l * r + e;
            for (int w = 0; w < W; w++) o[w] = o[w] * r + e * (float)a.vpages[at + w];
        }
    }
    if (lane == 0) { wm[wave] = m; wl[wave] = l; }
    for (int w = 0; w < W; w++) wo[wave][W * lane + w] = o[w];
    __syncthreads();
    for (int dim = threadIdx.x; dim < D; dim += THREADS) {
        float top = -INFINITY, den = 0.f, sum = 0.f;
        for (int w = 0; w < WAVES; w++) top = fmaxf(top, wl[w] != 0.f ? wm[w] : -INFINITY);
        for (int w = 0; w < WAVES; w++)
            if (wl[w] != 0.f) {
                const float r = wm[w] == top ? 1.f : __builtin_amdgcn_exp2f(wm[w] - top);
                den += r * wl[w];
                sum += r * wo[w][dim];
            }
        to[dim] = (half_t)(den != 0.f ? sum / den : 0.f);
    }
}

}  // namespace

int64_t bs_attention_tree_scratch(int, int, int, int, int, int, int, int) { return 0; }

int bs_launch_attention_tree(const half_t *q, int ldq, const half_t *kpages, const half_t *vpages, const int32_t *table, const int32_t *lengths, const int32_t *granted,
                             const int32_t *starts, const int64_t *masks, half_t *out, int B, int T, int nodes, int heads, int kv_heads, int head_dim, int shift, int max_pages,
                             int pool, void *workspace, hipStream_t s) {
    const ta_args a = {q, kpages, vpages, table, lengths, granted, starts, masks, out, ldq, B, T, nodes, heads, kv_heads, shift, max_pages, pool};
    if (head_dim == 128) attention_tree_kernel<128><<<(unsigned)((int64_t)T * heads), THREADS, 0, s>>>(a);
    else attention_tree_kernel<64><<<(unsigned)((int64_t)T * heads), THREADS, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
