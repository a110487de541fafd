// A key-value cache in pages, for requests of unequal lengths: which pages a step's tokens take (page_plan_kernel), and the prompts'
// keys and values on their way into them (rope_store_paged_kernel).
#include "common.h"

namespace {

// ---- plan ------------------------------------------------------------------------------------------------------------
// Per row b (a request): len positions held, `fresh` tokens to come, released (its pages go back first, len := 0).  With
// pages(n) = ceil(n / page): need = pages(len + fresh) - pages(len).  Free pages are a ring; a row's first new page is the one behind those
// of the rows before it, and a row is granted if the pages of all rows up to it are there.  Three sums over the rows (tokens, pages that
// come back, pages that are needed - this one last, for a row whose tokens lie behind the output takes none), then every row writes its
// part of the table, of the ring and of the slots.  Pages come from the front of the ring and go back behind its end, so that nothing
// written in a call is read in it.
// All sums are capped (tokens behind the last row, pages beyond what is there): a capped sum of non-negative numbers does not depend on
// the order of its parts, and 32 bits hold it whatever a caller's numbers are.
constexpr int PLAN_THREADS = 1024;

struct plan_args {
    const int32_t *lengths, *fresh;
    const uint8_t *released;
    int32_t *table, *ring;
    const int32_t *state;
    int32_t *lengths_out, *state_out, *granted, *starts, *positions;
    int64_t *slots;
    int B, T, shift, max_pages, pool;
};
// what a row has to write
struct plan_row {
    int32_t held;                                // positions, after a release
    int32_t fresh, granted;                      // tokens asked for, tokens that get slots (fresh or 0)
    int32_t start;                               // first token row
    int32_t need, first;                         // new pages, the first one's place behind the ring's front
    int32_t back, back_first;                    // pages that go back, the first one's place behind the ring's end
};

__device__ __forceinline__ uint32_t capped(uint32_t a, uint32_t b, uint32_t cap) { return min(a + b, cap); }    // (a, b <= cap < 2^31)

// exclusive capped sum over the workgroup, and the whole one; `to` is free again behind the next barrier
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t cap, uint32_t *to, uint32_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t below = __shfl_up(s, o, 64);
        if (lane >= o) s = capped(s, below, cap);
    }
    uint32_t mine = __shfl_up(s, 1, 64);
    if (lane == 0) mine = 0;
    if (lane == 63) to[wave] = s;
    __syncthreads();
    total = 0;
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 64; w++) {
        if (w == wave) before = total;
        total = capped(total, to[w], cap);
    }
    return capped(before, mine, cap);
}

__device__ __forceinline__ int plan_pages(int n, int shift) { return n > 0 ? ((n - 1) >> shift) + 1 : 0; }
__device__ __forceinline__ int plan_wrap(uint32_t i, int pool) { return i >= (uint32_t)pool ? (int)(i - pool) : (int)i; }   // i < 2 * pool

struct plan_state {
    int head, count, tail;                       // (a state that no ring can have is an empty ring)
    __device__ __forceinline__ plan_state(const int32_t *p, int pool) {
        head = p[0];
        count = p[1];
        if (head < 0 || head >= pool || count < 0 || count > pool) head = count = 0;
        tail = plan_wrap((uint32_t)head + count, pool);
    }
};

// entries [j0, j1) of a row by steps: pages that go back are read before the new ones take their place, by the same thread
__device__ __forceinline__ int plan_entries(const plan_row &r, int shift) {
    return max(r.back, plan_pages(r.held, shift) + r.need);
}
__device__ __forceinline__ int plan_first_entry(const plan_row &r, int shift) { return r.back ? 0 : plan_pages(r.held, shift); }
__device__ __forceinline__ void plan_entry(const plan_args &a, const plan_state &st, const plan_row &r, int b, int j) {
    int32_t *at = a.table + (int64_t)b * a.max_pages + j;
    const int own = j - plan_pages(r.held, a.shift);
    const bool taken = own >= 0 && own < r.need;
    const int32_t fresh = taken ? a.ring[plan_wrap((uint32_t)st.head + r.first + own, a.pool)] : 0;
    // (a ring that is full already takes no more: the pages of a table that does not belong to it)
    if (j < r.back && r.back_first + j < a.pool - st.count) a.ring[plan_wrap((uint32_t)st.tail + r.back_first + j, a.pool)] = *at;
    if (taken) *at = fresh;
}
__device__ __forceinline__ void plan_token(const plan_args &a, const plan_state &st, const plan_row &r, int b, int i) {
    if (r.start + i >= a.T) return;
    int64_t slot = -1;
    int pos = -1;
    if (i < r.granted) {
        pos = r.held + i;
        const int p = pos >> a.shift, own = p - plan_pages(r.held, a.shift);
        const int32_t id = own >= 0 ? a.ring[plan_wrap((uint32_t)st.head + r.first + own, a.pool)] : a.table[(int64_t)b * a.max_pages + p];
        slot = id < 0 ? -1 : ((int64_t)id << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    a.slots[r.start + i] = slot;
    a.positions[r.start + i] = pos;
}
__device__ __forceinline__ void plan_behind(const plan_args &a, int from, int step, int total) {
    for (int t = min(total, a.T) + from; t < a.T; t += step) {
        a.slots[t] = -1;
        a.positions[t] = -1;
    }
}

// The sums, by one workgroup.  ALL: it writes everything; otherwise it leaves what rows have to write in `rows` for plan_write_kernel.
// A thread writes the first two entries and tokens of its row itself, and a wave the rest of its rows one by one: with one token per row nobody waits
// for anybody, and a long row is written by 64 lanes.
// What bounds it: the chain launch -> lengths -> sums -> ring -> slots.
template <bool ALL>
__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(const plan_args a, plan_row *__restrict__ rows) {
    __shared__ uint32_t sums[3][PLAN_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63;
    const plan_state st(a.state, a.pool);
    const uint32_t token_cap = (uint32_t)a.T + 1, back_cap = (uint32_t)a.pool + 1, need_cap = (uint32_t)st.count + 1;
    uint32_t tokens = 0, back = 0, need = 0, taken = 0;
    const int most = (int)min((int64_t)a.max_pages << a.shift, (int64_t)INT32_MAX);
    for (int b0 = 0; b0 < a.B; b0 += PLAN_THREADS) {
        const int b = b0 + tid;
        const bool in = b < a.B;
        plan_row r = {};
        if (in) {
            const int len = min(max(a.lengths[b], 0), most);
            const bool gone = a.released && a.released[b];
            r.fresh = max(a.fresh[b], 0);
            r.held = gone ? 0 : len;
            r.back = gone ? plan_pages(len, a.shift) : 0;
        }
        uint32_t all_tokens, all_back, all_need;
        const uint32_t fresh = min((uint32_t)r.fresh, token_cap);
        const uint32_t start = capped(tokens, sum_before(fresh, token_cap, sums[0], all_tokens), token_cap);
        const uint32_t back_first = capped(back, sum_before(min((uint32_t)r.back, back_cap), back_cap, sums[1], all_back), back_cap);
        const bool possible = in && capped(start, fresh, token_cap) <= (uint32_t)a.T && r.fresh <= most - r.held;
        r.need = possible ? plan_pages(r.held + r.fresh, a.shift) - plan_pages(r.held, a.shift) : 0;
        const uint32_t want = min((uint32_t)r.need, need_cap);
        const uint32_t first = capped(need, sum_before(want, need_cap, sums[2], all_need), need_cap);
        const bool ok = possible && (r.need == 0 || capped(first, want, need_cap) <= (uint32_t)st.count);
        if (!ok) r.need = 0;
        r.granted = ok ? r.fresh : 0;
        r.start = (int)start;
        r.first = (int)first;
        r.back_first = (int)back_first;
        if (in) {
            a.lengths_out[b] = r.held + r.granted;
            a.granted[b] = r.granted;
            a.starts[b] = r.start;
            if (!ALL) rows[b] = r;
        }
        tokens = capped(tokens, all_tokens, token_cap);
        back = capped(back, all_back, back_cap);
        need = capped(need, all_need, need_cap);
        // the pages of the rows that were granted: the largest sum that ends with one of them (rows behind a refused one need none)
        const uint32_t end = ok && r.need ? first + (uint32_t)r.need : 0;
        taken = max(taken, end);
        if (ALL) {
            const int e0 = plan_first_entry(r, a.shift), e1 = plan_entries(r, a.shift);
            const int t1 = in ? min(r.fresh, max(a.T - r.start, 0)) : 0;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                if (j < t1) plan_token(a, st, r, b, j);
                if (e0 + j < e1) plan_entry(a, st, r, b, e0 + j);
            }
            for (uint64_t more = __ballot(t1 > 2 || e1 - e0 > 2); more; more &= more - 1) {
                const int w = __ffsll((unsigned long long)more) - 1;
                plan_row q;
                q.held = __shfl(r.held, w, 64);
                q.granted = __shfl(r.granted, w, 64);
                q.start = __shfl(r.start, w, 64);
                q.need = __shfl(r.need, w, 64);
                q.first = __shfl(r.first, w, 64);
                q.back = __shfl(r.back, w, 64);
                q.back_first = __shfl(r.back_first, w, 64);
                const int row = b - lane + w, f0 = __shfl(e0, w, 64), f1 = __shfl(e1, w, 64), u1 = __shfl(t1, w, 64);
                for (int i = 2 + lane; i < u1; i += 64) plan_token(a, st, q, row, i);
                for (int j = f0 + 2 + lane; j < f1; j += 64) plan_entry(a, st, q, row, j);
            }
        }
        __syncthreads();                         // (the sums' places are written again)
    }
    if (ALL) plan_behind(a, tid, PLAN_THREADS, (int)tokens);
    // the largest `taken` of all threads
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) taken = max(taken, (uint32_t)__shfl_xor(taken, o, 64));
    if (lane == 0) sums[0][tid >> 6] = taken;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < PLAN_THREADS / 64; w++) taken = max(taken, sums[0][w]);
        const int kept = min((int)back, a.pool - st.count);
        a.starts[a.B] = (int)tokens;
        a.state_out[0] = plan_wrap((uint32_t)st.head + taken, a.pool);
        a.state_out[1] = st.count - (int)taken + kept;
        if (!ALL) {                              // for plan_write_kernel: the state may have been overwritten
            plan_row r = {};
            r.held = st.head;
            r.fresh = st.count;
            r.start = (int)tokens;
            rows[a.B] = r;
        }
    }
}

// Everything that page_plan_kernel<false> has left: workgroup (b, y) takes every gridDim.y-th strip of row b, the row behind the last one the
// tokens behind the last one.
constexpr int PLAN_STRIP = 512;

__global__ __launch_bounds__(PLAN_STRIP) void plan_write_kernel(const plan_args a, const plan_row *__restrict__ rows) {
    const int b = blockIdx.x, from = blockIdx.y * PLAN_STRIP + threadIdx.x, step = gridDim.y * PLAN_STRIP;
    const plan_row s = rows[a.B], r = rows[b];
    const int32_t state[2] = {s.held, s.fresh};
    const plan_state st(state, a.pool);
    if (b == a.B) {
        plan_behind(a, from, step, s.start);
        return;
    }
    const int t1 = min(r.fresh, max(a.T - r.start, 0)), e1 = plan_entries(r, a.shift);
    for (int i = from; i < t1; i += step) plan_token(a, st, r, b, i);
    for (int j = plan_first_entry(r, a.shift) + from; j < e1; j += step) plan_entry(a, st, r, b, j);
}

// Up to so many rows and tokens one workgroup writes everything.
constexpr int PLAN_FEW_TOKENS = 4096, PLAN_FEW_ROWS = 1024;
bool plan_few(int B, int T) { return B <= PLAN_FEW_ROWS && T <= PLAN_FEW_TOKENS; }

// ---- store -----------------------------------------------------------------------------------------------------------
constexpr int THREADS = 256;

// One workgroup per token; an item is V dimensions of a head (for q and k together with the V that rotate against them).  The rotation is computed
// in fp32 and rounded once, as the decode step's.  A token without a slot (or with one, or a position, that does not exist) is not rotated
// and not stored.
template <int V>
__global__ __launch_bounds__(THREADS) void rope_store_paged_kernel(const half_t *q, half_t *qout, const half_t *__restrict__ k, const half_t *__restrict__ v,
                                                                   const half_t *__restrict__ cosv, const half_t *__restrict__ sinv,
                                                                   const int32_t *__restrict__ positions, const int64_t *__restrict__ slots,
                                                                   half_t *__restrict__ kpages, half_t *__restrict__ vpages, int ldq, int ldqo, int ldkv,
                                                                   int heads, int kv_heads, int d, int max_pos, int shift, int64_t places) {
    typedef half_t vec_t __attribute__((ext_vector_type(V)));
    const int64_t token = blockIdx.x;
    const int d2 = d / 2, per = d2 / V, qi = heads * per, ki = kv_heads * per;      // items of q and of k; v has 2 * ki
    const int64_t slot = slots[token];
    const int pos = positions[token];
    q += token * ldq;
    qout += token * ldqo;
    k += token * ldkv;
    v += token * ldkv;
    if (slot < 0 || slot >= places || pos < 0 || pos >= max_pos) {
        if (qout != q)
            for (int it = threadIdx.x; it < 2 * qi; it += THREADS) *reinterpret_cast<vec_t *>(qout + it * V) = *reinterpret_cast<const vec_t *>(q + it * V);
        return;
    }
    cosv += (int64_t)pos * d2;
    sinv += (int64_t)pos * d2;
    const int64_t head_stride = (int64_t)d << shift, at = (slot >> shift) * kv_heads * head_stride + (slot & ((1 << shift) - 1)) * d;
    for (int it = threadIdx.x; it < qi + 3 * ki; it += THREADS) {
        if (it >= qi + ki) {
            const int j = it - qi - ki, h = j / (2 * per), c = (j % (2 * per)) * V;
            *reinterpret_cast<vec_t *>(vpages + at + h * head_stride + c) = *reinterpret_cast<const vec_t *>(v + h * d + c);
            continue;
        }
        const bool is_q = it < qi;
        const int j = is_q ? it : it - qi, h = j / per, c = (j % per) * V;
        const half_t *from = (is_q ? q : k) + h * d + c;
        half_t *to = is_q ? qout + h * d + c : kpages + at + h * head_stride + c;
        const vec_t a = *reinterpret_cast<const vec_t *>(from), e = *reinterpret_cast<const vec_t *>(from + d2);
        const vec_t cs = *reinterpret_cast<const vec_t *>(cosv + c), sn = *reinterpret_cast<const vec_t *>(sinv + c);
        vec_t lo, hi;
#pragma unroll
        for (int i = 0; i < V; i++) {
            lo[i] = (half_t)((float)a[i] * (float)cs[i] - (float)e[i] * (float)sn[i]);
            hi[i] = (half_t)((float)e[i] * (float)cs[i] + (float)a[i] * (float)sn[i]);
        }
        *reinterpret_cast<vec_t *>(to) = lo;
        *reinterpret_cast<vec_t *>(to + d2) = hi;
    }
}

}  // namespace

int64_t bs_page_plan_scratch(int B, int T) { return plan_few(B, T) ? 0 : (int64_t)(B + 1) * sizeof(plan_row); }

int bs_launch_page_plan(const int32_t *lengths, const int32_t *fresh, const uint8_t *released, int32_t *table, int32_t *ring, const int32_t *state,
                        int32_t *lengths_out, int32_t *state_out, int32_t *granted, int32_t *starts, int32_t *positions, int64_t *slots, int B,
                        int T, int shift, int max_pages, int pool, void *workspace, hipStream_t s) {
    const plan_args a = {lengths, fresh, released, table, ring, state, lengths_out, state_out, granted, starts, positions, slots, B, T, shift, max_pages, pool};
    if (plan_few(B, T)) {
        page_plan_kernel<true><<<1, PLAN_THREADS, 0, s>>>(a, nullptr);
    } else {
        page_plan_kernel<false><<<1, PLAN_THREADS, 0, s>>>(a, (plan_row *)workspace);
        BS_LAUNCH_CHECK();
        // strips enough for one long row, few for many rows
        const int64_t strips = bs_cdiv(T, (int64_t)PLAN_STRIP * (B < 64 ? 1 : 16));
        plan_write_kernel<<<dim3(B + 1, (unsigned)(strips < 1 ? 1 : strips > 64 ? 64 : strips)), PLAN_STRIP, 0, s>>>(a, (const plan_row *)workspace);
    }
    BS_LAUNCH_CHECK();
    return BS_OK;
}

int bs_launch_rope_store_paged(const half_t *q, half_t *qout, const half_t *k, const half_t *v, const half_t *cos, const half_t *sin,
                               const int32_t *positions, const int64_t *slots, half_t *kpages, half_t *vpages, int ldq, int ldqo, int ldkv, int T,
                               int heads, int kv_heads, int d, int max_pos, int shift, int pool, hipStream_t s) {
    // 16-byte pieces where everything starts on 16 bytes
    bool wide = ldq % 8 == 0 && ldqo % 8 == 0 && ldkv % 8 == 0;
    for (const void *p : {(const void *)q, (const void *)qout, (const void *)k, (const void *)v, (const void *)cos, (const void *)sin, (const void *)kpages, (const void *)vpages})
        wide = wide && bs_aligned(p, 16);
    auto *kernel = wide ? rope_store_paged_kernel<8> : rope_store_paged_kernel<1>;
    kernel<<<T, THREADS, 0, s>>>(q, qout, k, v, cos, sin, positions, slots, kpages, vpages, ldq, ldqo, ldkv, heads, kv_heads, d, max_pos, shift,
                                 (int64_t)pool << shift);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
