// Rows of a paged cache become copies of other rows (several continuations of one prompt, beams that change places), or empty.  Whole pages are shared: shares[p] is the number of rows that
// hold page p, less one.  The last page, when it is not full, will be written on: its positions are copied to a new page.  Pages whose last holder has left them go back.
#include "lanes.h"
#include "pages.h"

namespace {

constexpr int THREADS = 1024, WAVES = THREADS / 64;

// what becomes of a row (workspace)
struct fork_row {
    int32_t source;                              // itself: the row stays
    int32_t gives, whole, length;                // pages that it gives up; whole pages, and positions, that it holds afterwards
    int32_t fresh, of, rest, pad;                // its new page or -1, the page that this one is a copy of, positions of it
};

struct fork_args {
    const int32_t *source, *lengths;
    int32_t *table, *ring;
    const int32_t *state;
    int32_t *shares, *lengths_out, *state_out, *granted;
    half_t *kpages, *vpages;
    fork_row *rows;                              // workspace
    int32_t *needed, *freed, *owner, *stage;     // ... pages that new ones took (one number), pages that go back of every row, first giver of every page, the tables to come
    int64_t layer;
    int B, layers, kv_heads, pieces, shift, max_pages, pool, blocks;
};

__device__ __forceinline__ uint32_t fork_sum(uint32_t v, uint32_t *waves, uint32_t &total) {          // what is in front of this thread; the sum of all
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t upto = bs_scan(v, [](uint32_t x, uint32_t y) { return x + y; });
    __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    uint32_t before = upto - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        before += w < wave ? waves[w] : 0;
        total += waves[w];
    }
    return before;
}

// Who takes which new page, in order of the rows: the first one that finds none, and all later ones that need one, stay as they are.
__global__ __launch_bounds__(THREADS) void fork_plan_kernel(const fork_args a) {
    __shared__ uint32_t waves[WAVES];
    const plan_state st(a.state, a.pool);
    const int64_t most = min((int64_t)a.max_pages << a.shift, (int64_t)INT32_MAX);
    uint32_t used = 0, taken = 0;
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        fork_row r = {b, 0, 0, 0, -1, -1, 0, 0};
        bool need = false;
        if (b < a.B) {
            const int before = (int)min((int64_t)max(a.lengths[b], 0), most), s = a.source[b];
            r.length = before;
            if (s >= -1 && s < a.B && s != b) {
                r.source = s;
                r.gives = plan_pages(before, a.shift);
                r.length = s < 0 ? 0 : (int)min((int64_t)max(a.lengths[s], 0), most);
            }
            r.whole = r.length >> a.shift;
            r.rest = r.length & ((1 << a.shift) - 1);
            need = r.source >= 0 && r.source != b && r.rest > 0;
            if (need) r.of = a.table[(int64_t)s * a.max_pages + r.whole];
            else r.rest = 0;
        }
        uint32_t total;
        const uint32_t place = used + fork_sum(need, waves, total);
        const bool granted = !need || place < (uint32_t)st.count;
        if (need && granted) r.fresh = a.ring[plan_wrap((uint32_t)st.head + place, a.pool)];
        if (!granted) r = {b, 0, 0, (int)min((int64_t)max(a.lengths[b], 0), most), -1, -1, 0, 0};
        used += total;
        taken = min(used, (uint32_t)st.count);
        if (b < a.B) {
            a.rows[b] = r;
            a.granted[b] = granted;
        }
    }
    if (threadIdx.x == 0) *a.needed = (int32_t)taken;
}

__device__ __forceinline__ bool fork_page(int32_t p, int pool) { return p >= 0 && p < pool; }

// Tables, shares and the ring, by one workgroup: a wave per row, a lane per entry.  A page goes back when its shares fall below 0, and at the place of the first entry that gave it up: that is the
// smallest of its givers' numbers, whatever the order of the atomics.
// Few entries: N of a lane, which holds them from one pass to the next.  (4 rows of 19 pages: 19 us when every pass went through the tables again, with fences that write the L2 back, and 4.1 so.)
template <int N>
__device__ __forceinline__ void fork_few_tables(const fork_args &a) {
    __shared__ uint32_t counts[WAVES * N], upto[WAVES * N];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), chunks = (a.max_pages + 63) / 64;
    const plan_state st(a.state, a.pool);
    const int taken = *a.needed, room = a.pool - st.count;
    auto load = [](const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    fork_row r[N];
    int32_t gives[N], takes[N];                  // page that the entry gives up, and that it holds afterwards; -1: none
    int at[N];                                   // its number
#pragma unroll
    for (int n = 0; n < N; n++) {                // (the row's chunk n % chunks, of the row's turn n / chunks)
        const int b = wave + WAVES * (n / chunks);
        r[n].source = b;
        if (b < a.B) r[n] = a.rows[b];
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
        const int b = wave + WAVES * (n / chunks), j = 64 * (n % chunks) + lane;
        at[n] = b * a.max_pages + j;
        const bool moves = b < a.B && r[n].source != b;
        gives[n] = moves && j < r[n].gives ? a.table[(int64_t)at[n]] : -1;
        takes[n] = moves && j < r[n].whole ? a.table[(int64_t)r[n].source * a.max_pages + j] : -1;
    }
#pragma unroll
    for (int n = 0; n < N; n++)
        if (fork_page(gives[n], a.pool)) __hip_atomic_store(a.owner + gives[n], INT32_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) {
        if (fork_page(gives[n], a.pool)) {
            atomicMin(a.owner + gives[n], at[n]);
            atomicAdd(a.shares + gives[n], -1);
        }
        if (fork_page(takes[n], a.pool)) atomicAdd(a.shares + takes[n], 1);
    }
    __syncthreads();
    uint64_t back[N];
#pragma unroll
    for (int n = 0; n < N; n++) {
        const bool page = fork_page(gives[n], a.pool);
        const int32_t owner = page ? load(a.owner + gives[n]) : -1, left = page ? load(a.shares + gives[n]) : 0;
        back[n] = __ballot(page && owner == at[n] && left < 0);
        // in order of the rows, and of a row's chunks
        if (lane == 0 && n / chunks < N / chunks) counts[(wave + WAVES * (n / chunks)) * chunks + n % chunks] = __popcll(back[n]);
    }
    __syncthreads();
    const int entries = WAVES * (N / chunks) * chunks;
    if (wave == 0) {
        uint32_t sum = 0;
        for (int i0 = 0; i0 < entries; i0 += 64) {
            const uint32_t v = i0 + lane < entries ? counts[i0 + lane] : 0, s = bs_scan(v, [](uint32_t x, uint32_t y) { return x + y; });
            if (i0 + lane < entries) upto[i0 + lane] = sum + s - v;
            sum += bs_read(s, 63);
        }
        if (lane == 0) {
            a.state_out[0] = plan_wrap((uint32_t)st.head + taken, a.pool);
            a.state_out[1] = st.count - taken + min((int)sum, room);
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) {
        const int b = wave + WAVES * (n / chunks);
        if (b >= a.B || n / chunks >= N / chunks) continue;
        const int place = (int)upto[b * chunks + n % chunks] + __popcll(back[n] & ((1ull << lane) - 1));
        if (back[n] >> lane & 1) {
            __hip_atomic_store(a.shares + gives[n], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (place < room) a.ring[plan_wrap((uint32_t)st.tail + place, a.pool)] = gives[n];            // (a full ring takes no more)
        }
        if (r[n].source != b) {
            const int j = 64 * (n % chunks) + lane;
            if (j < r[n].whole) a.table[(int64_t)at[n]] = takes[n];
            else if (j == r[n].whole && r[n].rest > 0) a.table[(int64_t)at[n]] = r[n].fresh;
        }
        if (n % chunks == 0 && lane == 0) a.lengths_out[b] = r[n].length;
    }
}

// ... and as many as there are.  The choice goes by rows and the table's width, as lengths are known on the device alone.  us a call of a graph, 32 layers of 8 heads of 128: 4 rows of 300 positions 5.8 in tables of up to 64
// pages (an entry to a lane), 7.0 in one of 256 (four), 7.5 in one of 512 and 7.9 in one of 1024 (here); 17 rows of 300 9.3 in one of 128 (four), 11.1 in one of 129 (here); 48 rows 15.9 in one of 64, 25 in one of 65 (here);
// 4 rows of 8000, tables of 502 to 1024, 20 to 24.
__device__ __forceinline__ void fork_tables(const fork_args &a) {
    __shared__ uint32_t waves[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const plan_state st(a.state, a.pool);
    const int taken = *a.needed, room = a.pool - st.count;
    auto load = [](const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto entry = [&](int b, int j) { return b * a.max_pages + j; };       // (B * max_pages < 2^31)
    for (int b = wave; b < a.B; b += WAVES) {
        const fork_row r = a.rows[b];
        if (r.source == b) continue;
        for (int j = lane; j < r.gives; j += 64) {
            const int32_t p = a.table[(int64_t)entry(b, j)];
            if (fork_page(p, a.pool)) __hip_atomic_store(a.owner + p, INT32_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        for (int j = lane; j < r.whole; j += 64) a.stage[(int64_t)entry(b, j)] = a.table[(int64_t)entry(r.source, j)];
    }
    __syncthreads();
    for (int b = wave; b < a.B; b += WAVES) {
        const fork_row r = a.rows[b];
        if (r.source == b) continue;
        for (int j = lane; j < r.gives; j += 64) {
            const int32_t p = a.table[(int64_t)entry(b, j)];
            if (!fork_page(p, a.pool)) continue;
            atomicMin(a.owner + p, entry(b, j));
            atomicAdd(a.shares + p, -1);
        }
        for (int j = lane; j < r.whole; j += 64) {
            const int32_t p = a.stage[(int64_t)entry(b, j)];
            if (fork_page(p, a.pool)) atomicAdd(a.shares + p, 1);
        }
    }
    __syncthreads();
    auto goes = [&](int b, int j, const fork_row &r, int32_t &p) {
        p = j < r.gives ? a.table[(int64_t)entry(b, j)] : -1;
        return fork_page(p, a.pool) && load(a.owner + p) == entry(b, j) && load(a.shares + p) < 0;
    };
    for (int b = wave; b < a.B; b += WAVES) {
        const fork_row r = a.rows[b];
        int n = 0;
        int32_t p;
        if (r.source != b)
            for (int j0 = 0; j0 < r.gives; j0 += 64) n += __popcll(__ballot(goes(b, j0 + lane, r, p)));
        if (lane == 0) a.freed[b] = n;
    }
    __syncthreads();
    uint32_t all = 0;
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        uint32_t total;
        const uint32_t before = fork_sum(b < a.B ? (uint32_t)a.freed[b] : 0, waves, total);
        if (b < a.B) a.freed[b] = (int32_t)(all + before);
        all += total;
    }
    __syncthreads();
    for (int b = wave; b < a.B; b += WAVES) {
        const fork_row r = a.rows[b];
        if (lane == 0) a.lengths_out[b] = r.length;
        if (r.source == b) continue;
        int at = a.freed[b];
        for (int j0 = 0; j0 < r.gives; j0 += 64) {
            int32_t p;
            const bool back = goes(b, j0 + lane, r, p);
            const uint64_t who = __ballot(back);
            const int place = at + __popcll(who & ((1ull << lane) - 1));
            if (back) {
                __hip_atomic_store(a.shares + p, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (place < room) a.ring[plan_wrap((uint32_t)st.tail + place, a.pool)] = p;           // (a full ring takes no more)
            }
            at += __popcll(who);
        }
        for (int j = lane; j < r.whole; j += 64) a.table[(int64_t)entry(b, j)] = a.stage[(int64_t)entry(b, j)];
        if (lane == 0 && r.rest > 0) a.table[(int64_t)entry(b, r.whole)] = r.fresh;
    }
    if (threadIdx.x == 0) {
        a.state_out[0] = plan_wrap((uint32_t)st.head + taken, a.pool);
        a.state_out[1] = st.count - taken + min((int)all, room);
    }
}

// Workgroup 0 the tables, the others the positions of the last pages: a run (a head of a layer's keys or values) to a wave, four pieces of a lane on their way at once.  Bytes: 64 rows that become
// copies with half a page of 64 on average, 32 layers of 8 heads of 128, write 169 MB and read 75 (sources have several copies) in 54 us, what a copy takes for as many; 4 beams 4.1 us, the tables' chain.
__global__ __launch_bounds__(THREADS) void fork_apply_kernel(const fork_args a) {
    if (blockIdx.x == 0) {
        const int entries = (a.B + WAVES - 1) / WAVES * ((a.max_pages + 63) / 64);         // of a lane
        return entries <= 1 ? fork_few_tables<1>(a) : entries <= 4 ? fork_few_tables<4>(a) : fork_tables(a);
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = (blockIdx.x - 1) / a.blocks, block = (blockIdx.x - 1) - b * a.blocks;
    const fork_row r = a.rows[b];
    if (r.rest == 0 || !fork_page(r.fresh, a.pool) || !fork_page(r.of, a.pool)) return;
    const int runs = 2 * a.layers * a.kv_heads, pieces = r.rest * a.pieces;
    for (int run = block * WAVES + wave; run < runs; run += a.blocks * WAVES) {
        const int head = run % a.kv_heads, layer = run / a.kv_heads;
        half8_t *const base = reinterpret_cast<half8_t *>((layer & 1 ? a.vpages : a.kpages) + (layer >> 1) * a.layer);
        const half8_t *from = base + (((int64_t)r.of * a.kv_heads + head) << a.shift) * a.pieces;
        half8_t *to = base + (((int64_t)r.fresh * a.kv_heads + head) << a.shift) * a.pieces;
        for (int i = lane; i < pieces; i += 256) {
            half8_t v[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + 64 * e < pieces) v[e] = from[i + 64 * e];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (i + 64 * e < pieces) to[i + 64 * e] = v[e];
        }
    }
}

struct fork_space {
    int64_t rows, needed, freed, owner, stage, end;
};
fork_space space_of(int B, int max_pages, int pool) {
    fork_space s;
    s.rows = 0;
    s.needed = s.rows + (int64_t)B * (int64_t)sizeof(fork_row);
    s.freed = s.needed + 16;
    s.owner = s.freed + 4ll * B;
    s.stage = s.owner + 4ll * pool;
    s.end = bs_cdiv(s.stage + 4ll * B * max_pages, 16) * 16;
    return s;
}

}  // namespace

int64_t bs_page_fork_scratch(int B, int max_pages, int pool) { return space_of(B, max_pages, pool).end; }

int bs_launch_page_fork(const int32_t *source, const int32_t *lengths, int32_t *table, int32_t *ring, const int32_t *state, int32_t *shares, half_t *kpages, half_t *vpages,
                        int32_t *lengths_out, int32_t *state_out, int32_t *granted, int B, int layers, int kv_heads, int head_dim, int shift, int max_pages, int pool,
                        void *workspace, hipStream_t s) {
    const fork_space w = space_of(B, max_pages, pool);
    char *const p = (char *)workspace;
    const int64_t runs = bs_cdiv(2ll * layers * kv_heads, WAVES), fill = bs_cdiv(2048, B > 0 ? B : 1);
    fork_args a = {source, lengths, table, ring, state, shares, lengths_out, state_out, granted, kpages, vpages, (fork_row *)(p + w.rows), (int32_t *)(p + w.needed),
                   (int32_t *)(p + w.freed), (int32_t *)(p + w.owner), (int32_t *)(p + w.stage), ((int64_t)pool * kv_heads << shift) * head_dim, B, layers, kv_heads,
                   head_dim / 8, shift, max_pages, pool, (int)(runs < fill ? runs : fill)};
    fork_plan_kernel<<<1, THREADS, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    fork_apply_kernel<<<(unsigned)(1 + (int64_t)B * a.blocks), THREADS, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
