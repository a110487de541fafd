// Drafted tokens as a tree per request: which of them each one attends to (tree_plan_kernel), and what becomes of the tree when the model has answered
// (tree_accept_kernel).  Node j of a request is its token row starts[b] + j, parents[] < j.  A tree has up to 64 nodes: a wave is a request, a lane a node.
#include "lanes.h"
#include "pages.h"

namespace {

constexpr int NODES = 64, THREADS = 256, WAVES = THREADS / 64;

// request b's token rows start .. end - 1, the first `nodes` of them its tree: 0 without slots, or with more nodes than `most` or (lengths not null) than its length
struct tree_rows {
    int start, end, nodes;
    __device__ __forceinline__ tree_rows(const int32_t *starts, const int32_t *granted, const int32_t *lengths, int b, int T, int most) {
        start = min(max(starts[b], 0), T);
        end = min(max(starts[b + 1], start), T);
        const int n = granted[b];
        nodes = n > 0 && n <= most && n <= end - start && (!lengths || n <= lengths[b]) ? n : 0;
    }
};

// ---- masks and positions ----------------------------------------------------------------------------------------------
// A node's mask is its own bit and its parent's mask: six steps of pointer doubling, each of which takes over the mask of the node that the pointer is at and that node's pointer.  Its depth is
// the number of bits but one.  A chain of latencies: the request's rows, its parents, 18 lane
// shuffles.  One request of 24 nodes takes 1.6 us, 300 of up to 64 3.0.
__global__ __launch_bounds__(THREADS) void tree_plan_kernel(const int32_t *__restrict__ parents, const int32_t *__restrict__ lengths, const int32_t *__restrict__ granted,
                                                            const int32_t *__restrict__ starts, int32_t *__restrict__ positions, int64_t *__restrict__ masks, int B, int T,
                                                            int request_blocks) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x >= request_blocks) {     // rows of no request
        const int first = B > 0 ? min(max(starts[0], 0), T) : T, last = B > 0 ? min(max(starts[B], 0), T) : T;
        for (int64_t t = (int64_t)(blockIdx.x - request_blocks) * THREADS + threadIdx.x; t < T; t += (int64_t)(gridDim.x - request_blocks) * THREADS)
            if (t < first || t >= last || B == 0) {
                positions[t] = -1;
                masks[t] = 0;
            }
        return;
    }
    const int b = blockIdx.x * WAVES + wave;
    if (b >= B) return;
    const tree_rows r(starts, granted, lengths, b, T, NODES);
    const int held = max(lengths[b] - granted[b], 0);
    int p = lane < r.nodes ? parents[r.start + lane] : -1;
    if (p >= lane) p = -1;
    uint64_t mask = 1ull << lane;
#pragma unroll
    for (int s = 0; s < 6; s++) {
        const int from = p < 0 ? lane : p;
        const uint32_t lo = __shfl((uint32_t)mask, from, 64), hi = __shfl((uint32_t)(mask >> 32), from, 64);
        const int next = __shfl(p, from, 64);
        if (p >= 0) {
            mask |= (uint64_t)hi << 32 | lo;
            p = next;
        }
    }
    for (int t = r.start + lane; t < r.end; t += 64) {
        const bool node = t - r.start < r.nodes;           // (nodes <= 64: lane's own)
        positions[t] = node ? held + __popcll(mask) - 1 : -1;
        masks[t] = node ? (int64_t)mask : 0;
    }
}

// ---- acceptance ---------------------------------------------------------------------------------------------------------
// From node 0 on: the first child whose token is the target of the node that is reached, until there is none.  Node i of that path belongs to the i-th place behind the held
// positions, which is the slot of node i: its keys and values move there, in every layer.  path[i] >= i and both grow: whoever moves a piece of 16 bytes of a row for all
// nodes of the path in order, reads ahead of its writes as much as it likes.
struct accept_args {
    const int64_t *tokens, *targets, *slots;
    const int32_t *parents, *lengths, *granted, *starts;
    half_t *kpages, *vpages;
    int32_t *lengths_out, *accepted, *path;
    int64_t *token;
    int32_t *back;                               // workspace: {first page that goes back, pages} of every request
    int64_t layer;                               // halves of a layer's pages
    int B, T, nodes, blocks, layers, kv_heads, pieces, shift, max_pages, pool;
};

// One request by one wave, a lane a node.  `writes`: by the wave that writes what the caller gets, which looks at the length; the others, which move, cannot: that wave may have written on it.
struct accept_path {
    tree_rows r;
    int parent;
    int64_t drafted, target, slot;
    int at, count, mine;                         // the last node of the path, nodes on it, lane i: node i of it
    __device__ __forceinline__ accept_path(const accept_args &a, int b, bool writes) : r(a.starts, a.granted, writes ? a.lengths : nullptr, b, a.T, a.nodes) {
        const int lane = threadIdx.x & 63;
        const bool there = lane < r.nodes;
        parent = there ? a.parents[r.start + lane] : -1;
        drafted = there ? a.tokens[r.start + lane] : 0;
        target = there ? a.targets[r.start + lane] : 0;
        slot = there ? a.slots[r.start + lane] : -1;
    }
    __device__ __forceinline__ void walk() {
        const int lane = threadIdx.x & 63;
        at = count = 0;
        mine = -1;
        if (r.nodes == 0) return;
        mine = lane == 0 ? 0 : -1;
        count = 1;
        while (true) {
            const int64_t wanted = (int64_t)((uint64_t)bs_read((uint32_t)((uint64_t)target >> 32), at) << 32 | bs_read((uint32_t)target, at));
            const uint64_t fits = __ballot(lane > at && parent == at && drafted == wanted);
            if (fits == 0) break;
            at = __builtin_ctzll(fits);
            mine = lane == count ? at : mine;
            count++;
        }
    }
    // what the caller gets; {first page that goes back, pages}
    __device__ __forceinline__ int2 write(const accept_args &a, int b) const {
        const int lane = threadIdx.x & 63;
        const int most = (int)min((int64_t)a.max_pages << a.shift, (int64_t)INT32_MAX);
        const int before = min(max(a.lengths[b], 0), most), given = min(max(a.granted[b], 0), before), after = before - given + min(count, given), first = plan_pages(after, a.shift);
        if (lane < a.nodes) a.path[(int64_t)b * a.nodes + lane] = mine;
        if (lane == 0) {
            a.lengths_out[b] = after;
            a.accepted[b] = count;
        }
        if (count == 0 ? lane == 0 : lane == at) a.token[b] = count == 0 ? -1 : target;
        return {first, plan_pages(before, a.shift) - first};
    }
    // the moves, from the slot of node path[i] to that of node i: pieces `first`, `first` + step, ..
    __device__ __forceinline__ void move(const accept_args &a, int first, int step) const {
        const int lane = threadIdx.x & 63;
        const int32_t to = (int32_t)(slot >= 0 && slot < (int64_t)a.pool << a.shift ? slot : -1), from = __shfl(to, max(mine, 0), 64);
        const uint64_t left = __ballot(lane < count && mine != lane && to >= 0 && from >= 0);
        if (left == 0) return;
        const int units = 2 * a.layers * a.kv_heads * a.pieces, mask = (1 << a.shift) - 1;
        for (int u = first; u < units; u += step) {
            const int piece = u % a.pieces, head = u / a.pieces % a.kv_heads, layer = u / (a.pieces * a.kv_heads);
            half_t *const base = (layer & 1 ? a.vpages : a.kpages) + (layer >> 1) * a.layer + 8 * piece;
            auto where = [&](int32_t s) { return reinterpret_cast<half8_t *>(base + ((((int64_t)(s >> a.shift) * a.kv_heads + head) << a.shift) + (s & mask)) * (8 * a.pieces)); };
            for (uint64_t todo = left; todo != 0;) {
                half8_t v[8];
                uint64_t rest = todo;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (rest != 0) v[i] = *where((int32_t)bs_read((uint32_t)from, __builtin_ctzll(rest)));
                    rest &= rest - 1;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (todo != 0) *where((int32_t)bs_read((uint32_t)to, __builtin_ctzll(todo))) = v[i];
                    todo &= todo - 1;
                }
            }
        }
    }
};

// Many requests: workgroups of one request each; the ring in a launch of its own.  What bounds both is the chain row -> parents, tokens, targets -> path -> slots -> moves: 100 requests of up to 32 nodes, 32 layers
// of 8 heads of 128, 11.9 us and 3.9 for the ring (21 MB to and fro).
__global__ __launch_bounds__(THREADS) void tree_accept_kernel(const accept_args a) {
    const int b = blockIdx.x / a.blocks, block = blockIdx.x - b * a.blocks;
    const bool writes = block == 0 && threadIdx.x < 64;
    accept_path p(a, b, writes);
    p.walk();
    if (writes) {
        const int2 back = p.write(a, b);
        if (threadIdx.x == 0) {
            a.back[2 * b] = back.x;
            a.back[2 * b + 1] = back.y;
        }
    }
    p.move(a, block * THREADS + threadIdx.x, a.blocks * THREADS);
}

// Up to 64: one workgroup writes what the caller gets, and the ring; beside it, the others move.  (one request of 8 nodes, 32 layers of 8 heads of 128: 7.3 us a call, 4.8 on the device,
// with a second launch 10.3; 48 requests of up to 32 nodes, 10 MB to and fro, 8.0.)
constexpr int FEW = 64, FEW_THREADS = 1024, FEW_WAVES = FEW_THREADS / 64;
__global__ __launch_bounds__(FEW_THREADS) void tree_accept_few_kernel(const accept_args a, const int32_t *__restrict__ table, int32_t *ring, const int32_t *state, int32_t *state_out) {
    if (blockIdx.x > 0) {
        const int b = (blockIdx.x - 1) / a.blocks, block = (blockIdx.x - 1) - b * a.blocks;
        accept_path p(a, b, false);
        p.walk();
        return p.move(a, block * FEW_THREADS + threadIdx.x, a.blocks * FEW_THREADS);
    }
    __shared__ int first[FEW], pages[FEW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const plan_state st(state, a.pool);
    for (int b0 = 0; b0 < a.B; b0 += FEW_WAVES) {
        const int b = b0 + wave;
        if (b >= a.B) break;
        accept_path p(a, b, true);
        p.walk();
        const int2 back = p.write(a, b);
        if (lane == 0) {
            first[b] = back.x;
            pages[b] = back.y;
        }
    }
    __syncthreads();
    if (wave > 0) return;
    const int n = lane < a.B ? pages[lane] : 0, room = a.pool - st.count, upto = (int)bs_scan((uint32_t)n, [](uint32_t x, uint32_t y) { return x + y; }), sum = (int)bs_read((uint32_t)upto, 63);
    for (int j = 0; j < n && upto - n + j < room; j++) ring[plan_wrap((uint32_t)st.tail + upto - n + j, a.pool)] = table[(int64_t)lane * a.max_pages + first[lane] + j];
    if (lane == 0) {
        state_out[0] = st.head;
        state_out[1] = st.count + min(sum, room);
    }
}

// The pages behind what was accepted, in order of the requests, behind the ring's end.
constexpr int BACK_THREADS = 1024;
__global__ __launch_bounds__(BACK_THREADS) void tree_back_kernel(const int32_t *__restrict__ back, const int32_t *__restrict__ table, int32_t *ring, const int32_t *state,
                                                                 int32_t *state_out, int B, int max_pages, int pool) {
    __shared__ uint32_t waves[BACK_THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const plan_state st(state, pool);
    const int room = pool - st.count;
    int sum = 0;                                 // (B * max_pages < 2^31)
    for (int b0 = 0; b0 < B; b0 += BACK_THREADS) {
        const int b = b0 + threadIdx.x, n = b < B ? back[2 * b + 1] : 0, first = b < B ? back[2 * b] : 0;
        const uint32_t upto = bs_scan((uint32_t)n, [](uint32_t x, uint32_t y) { return x + y; });
        __syncthreads();
        if (lane == 63) waves[wave] = upto;
        __syncthreads();
        int at = sum + (int)upto - n;
        for (int w = 0; w < BACK_THREADS / 64; w++) {
            at += w < wave ? (int)waves[w] : 0;
            sum += (int)waves[w];
        }
        for (int j = 0; j < n && at + j < room; j++) ring[plan_wrap((uint32_t)st.tail + at + j, pool)] = table[(int64_t)b * max_pages + first + j];
    }
    if (threadIdx.x == 0) {
        state_out[0] = st.head;
        state_out[1] = st.count + min(sum, room);
    }
}

}  // namespace

int bs_launch_tree_plan(const int32_t *parents, const int32_t *lengths, const int32_t *granted, const int32_t *starts, int32_t *positions, int64_t *masks, int B, int T,
                        hipStream_t s) {
    const int requests = (int)bs_cdiv(B, WAVES);
    const int64_t rest = bs_cdiv(T, THREADS * 4);
    tree_plan_kernel<<<(unsigned)(requests + (rest < 1024 ? rest : 1024)), THREADS, 0, s>>>(parents, lengths, granted, starts, positions, masks, B, T, requests);
    BS_LAUNCH_CHECK();
    return BS_OK;
}

int64_t bs_tree_accept_scratch(int B) { return bs_cdiv(8ll * B, 16) * 16; }

int bs_launch_tree_accept(const int64_t *tokens, const int32_t *parents, const int64_t *targets, const int64_t *slots, const int32_t *lengths, const int32_t *granted,
                          const int32_t *starts, const int32_t *table, int32_t *ring, const int32_t *state, half_t *kpages, half_t *vpages, int32_t *lengths_out,
                          int32_t *state_out, int32_t *accepted, int32_t *path, int64_t *token, int B, int T, int nodes, int layers, int kv_heads, int head_dim, int shift,
                          int max_pages, int pool, void *workspace, hipStream_t s) {
    const int pieces = head_dim / 8, threads = B <= FEW ? FEW_THREADS : THREADS;
    const int64_t most = bs_cdiv(2ll * layers * kv_heads * pieces, threads), fill = bs_cdiv(1 << 20, (int64_t)(B > 0 ? B : 1) * threads);
    const int blocks = (int)(most < fill ? most : fill);
    const accept_args a = {tokens, targets, slots, parents, lengths, granted, starts, kpages, vpages, lengths_out, accepted, path, token, (int32_t *)workspace,
                           ((int64_t)pool * kv_heads << shift) * head_dim, B, T, nodes, blocks, layers, kv_heads, pieces, shift, max_pages, pool};
    if (B <= FEW) {
        tree_accept_few_kernel<<<(unsigned)(1 + B * blocks), FEW_THREADS, 0, s>>>(a, table, ring, state, state_out);
        BS_LAUNCH_CHECK();
        return BS_OK;
    }
    tree_accept_kernel<<<(unsigned)((int64_t)B * blocks), THREADS, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    tree_back_kernel<<<1, BACK_THREADS, 0, s>>>((const int32_t *)workspace, table, ring, state, state_out, B, max_pages, pool);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
