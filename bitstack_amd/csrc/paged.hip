// A key-value cache in pages, for requests of unequal lengths: which pages a step's tokens take (page_plan_kernel), and the prompts'
// keys and values on their way into them (rope_store_paged_kernel).
#include "lanes.h"

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
    int64_t *slots, *row_slots;
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

// the capped sums of the waves before this one, of all, and of what is in front of this thread
struct plan_sum {
    uint32_t before, total;
    __device__ __forceinline__ plan_sum(uint32_t scanned, uint32_t cap, const uint32_t *waves) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        auto f = [cap](uint32_t a, uint32_t b) { return capped(a, b, cap); };
        const uint32_t upto = bs_row_scan(waves[lane & 15], f);
        total = bs_read(upto, 15);
        before = bs_lane_before(scanned);
        if (wave > 0) before = capped(bs_read(upto, wave - 1), before, cap);
    }
};
// a wave's capped sums up to each lane; the whole one goes to waves[wave]
__device__ __forceinline__ uint32_t plan_scan(uint32_t v, uint32_t cap, uint32_t *waves) {
    const uint32_t s = bs_scan(v, [cap](uint32_t a, uint32_t b) { return capped(a, b, cap); });
    if ((threadIdx.x & 63) == 63) waves[threadIdx.x >> 6] = s;
    return s;
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

// The entries of a row that change, first <= j < end: pages that go back are read before new ones take their place, by the same thread.  Several at a time: a
// load that stands behind another entry's store waits for nothing but it.
__device__ __forceinline__ int plan_entries(const plan_row &r, int shift) { return max(r.back, plan_pages(r.held, shift) + r.need); }
__device__ __forceinline__ int plan_first_entry(const plan_row &r, int shift) { return r.back ? 0 : plan_pages(r.held, shift); }
template <int N>
__device__ __forceinline__ void plan_write_entries(const plan_args &a, const plan_state &st, const plan_row &r, int b, int from, int step, int end) {
    int32_t *row = a.table + (int64_t)b * a.max_pages;
    const int have = plan_pages(r.held, a.shift);
    for (int j0 = from; j0 < end; j0 += N * step) {
        int32_t fresh[N], old[N];
        bool taken[N], back[N];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int j = j0 + n * step, own = j - have;
            taken[n] = j < end && own >= 0 && own < r.need;
            back[n] = j < end && j < r.back && r.back_first + j < a.pool - st.count;       // (a full ring takes no more: pages of a table that is not its own)
            fresh[n] = taken[n] ? a.ring[plan_wrap((uint32_t)st.head + r.first + own, a.pool)] : 0;
            old[n] = back[n] ? row[j] : 0;
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int j = j0 + n * step;
            if (back[n]) a.ring[plan_wrap((uint32_t)st.tail + r.back_first + j, a.pool)] = old[n];
            if (taken[n]) row[j] = fresh[n];
        }
    }
}
// a request's first token (if its row is one of the output's), and its slot for the request
__device__ __forceinline__ void plan_write_first(const plan_args &a, const plan_state &st, const plan_row &r, int b) {
    int64_t slot = -1;
    if (r.granted > 0) {
        const int p = r.held >> a.shift, own = p - plan_pages(r.held, a.shift);
        const int32_t id = own >= 0 ? a.ring[plan_wrap((uint32_t)st.head + r.first + own, a.pool)] : a.table[(int64_t)b * a.max_pages + p];
        if (id >= 0) slot = ((int64_t)id << a.shift) + (r.held & ((1 << a.shift) - 1));
    }
    if (r.fresh > 0 && r.start < a.T) {
        a.slots[r.start] = slot;
        a.positions[r.start] = r.granted > 0 ? r.held : -1;
    }
    if (a.row_slots) a.row_slots[b] = slot;
}
template <int N>
__device__ __forceinline__ void plan_write_tokens(const plan_args &a, const plan_state &st, const plan_row &r, int b, int from, int step, int end) {
    const int32_t *row = a.table + (int64_t)b * a.max_pages;
    const int have = plan_pages(r.held, a.shift);
    for (int i0 = from; i0 < end; i0 += N * step) {
        int32_t id[N];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int i = i0 + n * step, p = (r.held + i) >> a.shift, own = p - have;
            id[n] = -1;
            if (i < end && i < r.granted) id[n] = own >= 0 ? a.ring[plan_wrap((uint32_t)st.head + r.first + own, a.pool)] : row[p];
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int i = i0 + n * step, pos = r.held + i;
            if (i < end) {
                a.slots[r.start + i] = id[n] < 0 ? -1 : ((int64_t)id[n] << a.shift) + (pos & ((1 << a.shift) - 1));
                a.positions[r.start + i] = i < r.granted ? pos : -1;
            }
        }
    }
}
__device__ __forceinline__ void plan_behind(const plan_args &a, int from, int step, int total) {
    for (int t = min(total, a.T) + from; t < a.T; t += step) {
        a.slots[t] = -1;
        a.positions[t] = -1;
    }
}

// The sums, by one workgroup.  ALL: it writes everything; otherwise it leaves what rows have to write in `rows` for plan_write_kernel.
// A thread writes the first entry and token of its row itself, as nearly all rows of a decode step want no more; longer rows are dealt to the waves.
// What bounds it: the chain launch -> lengths -> sums -> ring -> slots.   48 rows of a token each: 5.5 us in a stream of
// calls (1.6 KB move); with rows of up to 500 pages that go back 6.9.
template <bool ALL>
__global__ __launch_bounds__(PLAN_THREADS) void page_plan_kernel(const plan_args a, plan_row *__restrict__ rows) {
    __shared__ uint32_t sums[3][PLAN_THREADS / 64];
    __shared__ plan_row longer[ALL ? PLAN_THREADS : 1];
    __shared__ int longer_row[ALL ? PLAN_THREADS : 1], n_longer;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    static_assert(PLAN_THREADS == 1024, "16 waves");
    if (tid == 0) n_longer = 0;
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
        const uint32_t fresh = min((uint32_t)r.fresh, token_cap);
        const uint32_t fresh_upto = plan_scan(fresh, token_cap, sums[0]), back_upto = plan_scan(min((uint32_t)r.back, back_cap), back_cap, sums[1]);
        __syncthreads();
        const plan_sum all_fresh(fresh_upto, token_cap, sums[0]), all_back(back_upto, back_cap, sums[1]);
        const uint32_t start = capped(tokens, all_fresh.before, token_cap), back_first = capped(back, all_back.before, back_cap);
        const bool possible = in && capped(start, fresh, token_cap) <= (uint32_t)a.T && r.fresh <= most - r.held;
        r.need = possible ? plan_pages(r.held + r.fresh, a.shift) - plan_pages(r.held, a.shift) : 0;
        const uint32_t want = min((uint32_t)r.need, need_cap), need_upto = plan_scan(want, need_cap, sums[2]);
        __syncthreads();
        const plan_sum all_need(need_upto, need_cap, sums[2]);
        const uint32_t first = capped(need, all_need.before, need_cap);
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
        tokens = capped(tokens, all_fresh.total, token_cap);
        back = capped(back, all_back.total, back_cap);
        need = capped(need, all_need.total, need_cap);
        // the pages of the rows that were granted: the largest sum that ends with one of them (rows behind a refused one need none)
        const uint32_t end = ok && r.need ? first + (uint32_t)r.need : 0;
        taken = max(taken, end);
        if (ALL) {
            const int e0 = plan_first_entry(r, a.shift), e1 = plan_entries(r, a.shift);
            const int t1 = in ? min(r.fresh, max(a.T - r.start, 0)) : 0;
            if (t1 > 1 || e1 - e0 > 1) {
                const int at = atomicAdd(&n_longer, 1);                  // (they write to places of their own: their order does not matter)
                longer[at] = r;
                longer_row[at] = b;
            }
            if (in) plan_write_first(a, st, r, b);
            plan_write_entries<1>(a, st, r, b, e0, 1, min(e1, e0 + 1));
            __syncthreads();
            // a wave per row, or several if there are fewer rows than waves
            const int rows_left = n_longer, share = max(1, PLAN_THREADS / 64 / max(rows_left, 1)), step = 64 * share;
            for (int i = wave / share; i < rows_left && wave / share * share + share <= PLAN_THREADS / 64; i += PLAN_THREADS / 64 / share) {
                const plan_row q = longer[i];
                const int row = longer_row[i], f0 = plan_first_entry(q, a.shift), from = 1 + wave % share * 64 + lane;
                plan_write_tokens<8>(a, st, q, row, from, step, min(q.fresh, max(a.T - q.start, 0)));
                plan_write_entries<8>(a, st, q, row, f0 + from, step, plan_entries(q, a.shift));
            }
        }
        __syncthreads();                         // (the sums' places and the list are written again)
        if (tid == 0) n_longer = 0;
    }
    if (ALL) plan_behind(a, tid, PLAN_THREADS, (int)tokens);
    // the largest `taken` of all threads
    taken = bs_read(bs_scan(taken, [](uint32_t a, uint32_t b) { return max(a, b); }), 63);
    if (lane == 0) sums[0][wave] = taken;
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

// (100 rows of up to 2000 tokens, 1.2 MB written: 3.0 us for the sums, 3.4 for this, each a launch with two dependent loads.)
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
    if (from == 0) plan_write_first(a, st, r, b);
    plan_write_tokens<4>(a, st, r, b, from > 0 ? from : step, step, t1);
    plan_write_entries<4>(a, st, r, b, plan_first_entry(r, a.shift) + from, step, e1);
}

// One workgroup writes everything in a decode step (a token per row, and a few rows more), and where a wave is left for every row of few tokens.
// (us, one launch / two: a token each for 48 rows 5.5 / 8.3, for 1024 5.6 / 8.3, for 4096 15.1 / 16.1; 1 row of 1024 tokens 6.4 / 8.3, 8 of 128 8.2 / 8.4; but
// 32 of 64 11.5 / 8.2, 500 of 8 45 / 8.3, 1 of 16384 11.7 / 8.3.)
bool plan_few(int B, int T) { return (B <= 4096 && T <= B + 64) || (B <= PLAN_THREADS / 64 && T <= 1024); }

// ---- store -----------------------------------------------------------------------------------------------------------
constexpr int THREADS = 256;

// One workgroup per token; an item is V dimensions of a head (for q and k together with the V that rotate against them).  The rotation is computed
// in fp32 and rounded once, as the decode step's.  What bounds it is the bytes: 9 prompts of up to 2048 tokens, 64 heads on 8 of 128,
// 567 MB read and written in 106 us = 5.4 TB/s (a copy of 4 GiB: 4.8; 79 % of the waves' time is waiting for memory).  Pieces of one value, for rows that do not
// start on 16 bytes: 28.5 us where 16 bytes take 16.5 (4096 tokens, 32 heads on 8), 5.9 / 5.3 (48 tokens).  A token without a slot (or with one, or a position, that does not exist) is not rotated
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
                        int32_t *lengths_out, int32_t *state_out, int32_t *granted, int32_t *starts, int32_t *positions, int64_t *slots, int64_t *row_slots,
                        int B, int T, int shift, int max_pages, int pool, void *workspace, hipStream_t s) {
    const plan_args a = {lengths, fresh, released, table, ring, state, lengths_out, state_out, granted, starts, positions, slots, row_slots, B, T, shift, max_pages, pool};
    if (plan_few(B, T)) {
        page_plan_kernel<true><<<1, PLAN_THREADS, 0, s>>>(a, nullptr);
    } else {
        page_plan_kernel<false><<<1, PLAN_THREADS, 0, s>>>(a, (plan_row *)workspace);
        BS_LAUNCH_CHECK();
        // (16 strips of a row to a workgroup, were all tokens one row's.  One: 500 rows of 60 tokens 33.6 us instead of 8.4; a row of 16384 takes 8.3 to 8.4 with both.)
        const int64_t strips = bs_cdiv(T, (int64_t)PLAN_STRIP * 16);
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
    for (int64_t t = 0; t < T; t += 1 << 23) {   // (a grid holds 2^32 threads along x)
        kernel<<<(unsigned)(T - t < 1 << 23 ? T - t : 1 << 23), THREADS, 0, s>>>(q + t * ldq, qout + t * ldqo, k + t * ldkv, v + t * ldkv, cos, sin, positions + t, slots + t, kpages,
                                                                                vpages, ldq, ldqo, ldkv, heads, kv_heads, d, max_pos, shift, (int64_t)pool << shift);
        BS_LAUNCH_CHECK();
    }
    return BS_OK;
}
