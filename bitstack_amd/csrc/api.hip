// C ABI glue: argument validation, path selection, status strings.
#include "common.h"

#include <algorithm>
#include <initializer_list>
#include <mutex>

extern "C" int bs_version(void) { return BS_VERSION_NUMBER; }

extern "C" const char *bs_error_string(int status) {
    switch (status) {
        case BS_OK: return "ok";
        case BS_ERR_NULL: return "a required pointer is NULL";
        case BS_ERR_SHAPE: return "non-positive or unsupported dimension";
        case BS_ERR_RANK: return "rank K must be in 1..16";
        case BS_ERR_ALIGN: return "pointer is not aligned as the entry point requires";
        case BS_ERR_WORKSPACE: return "workspace missing, misaligned or too small";
        case BS_ERR_NO_DEVICE: return "no usable HIP device";
        case BS_ERR_LIBRARY: return "the vendor GEMM library failed after it had accepted the call";
        default: break;
    }
    if (status <= BS_ERR_HIP_BASE) return hipGetErrorString((hipError_t)(BS_ERR_HIP_BASE - status));
    return "unknown status";
}

static int forward_dims(int I, int M, int N, int K, int T) {
    if (I < 0 || M <= 0 || N <= 0 || T < 0) return BS_ERR_SHAPE;
    if (N % 8 != 0) return BS_ERR_SHAPE;
    if (K < 1 || K > 16) return BS_ERR_RANK;
    return BS_OK;
}

static int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// Which kernel multiplies the rebuilt weight: this library's linear_f16_kernel unless the calling thread has asked
// for hipBLASLt with bs_set_dense_kernel(BS_DENSE_LIBRARY) (a comparator for tests and benchmarks: what the
// reference's F.linear runs on ROCm).  The setting belongs to the thread that made it, so a size query and the
// forward that follows it on the same thread always agree, whatever other threads do.
static thread_local int g_dense_kernel = 0;

static bool dense_wants_library(int M, int N) {
    return g_dense_kernel == BS_DENSE_LIBRARY && M % 8 == 0 && N % 8 == 0;
}

// Which kernel runs a forward of 49 tokens or more: by shape (0), or pinned for tests and benchmarks.  Per thread.
static thread_local int g_prefill_kernel = 0;
int bs_prefill_mode() { return g_prefill_kernel; }

extern "C" int bs_set_prefill_kernel(int mode) {
    if (mode < 0 || mode > 3) return BS_ERR_SHAPE;
    g_prefill_kernel = mode;
    return BS_OK;
}

extern "C" int bs_set_dense_kernel(int mode) {
    if (mode < 0 || mode > 2) return BS_ERR_SHAPE;
    g_dense_kernel = mode;
    return BS_OK;
}

// `library_ok`: the dense product may run on hipBLASLt (and then needs its scratch behind the weight)
static int64_t rebuild_need(int M, int N, int T, bool library_ok) {
    // the rebuilt weight, then the library GEMM's own scratch where that is the kernel, or the product's partial sums
    const bool library = library_ok && dense_wants_library(M, N);
    return round_up((int64_t)M * N * 2, 256) + round_up(std::max(library ? BS_DENSE_LIBRARY_WORKSPACE : 0, bs_linear_parts_bytes(T, M, N)), 256);
}
static int64_t workspace_need(int I, int M, int N, int K, int T, bool library_ok) {
    int st = forward_dims(I, M, N, K, T);
    if (st != BS_OK) return st;
    if (T == 0) return 0;
    const int64_t gemv = bs_gemv_group_workspace_bytes(&I, &M, 1, N, K, T);
    return gemv > 0 ? gemv : rebuild_need(M, N, T, library_ok);
}

extern "C" int64_t bs_workspace_bytes(int I, int M, int N, int K, int T) { return workspace_need(I, M, N, K, T, true); }

extern "C" int bs_decode_plan(int I, int M, int N, int K, int T, int *waves, int *row_tiles_per_wave,
                              int *workgroups, int *partials_per_row) {
    if (!waves || !row_tiles_per_wave || !workgroups || !partials_per_row) return BS_ERR_NULL;
    int st = forward_dims(I, M, N, K, T);
    if (st != BS_OK) return st;
    bs_gemv_plan_info(I, M, N, K, T, waves, row_tiles_per_wave, workgroups, partials_per_row);
    return BS_OK;
}

extern "C" int bs_decode_kernel(int I, int M, int N, int K, int T) {
    int st = forward_dims(I, M, N, K, T);
    if (st != BS_OK) return st;
    return bs_gemv_plan_kernel(I, M, N, K, T);
}

extern "C" int bs_set_decode_kernel(int mode) { return bs_gemv_set_kernel(mode); }

extern "C" int bs_forward_path(int I, int M, int N, int K, int T) {
    int st = forward_dims(I, M, N, K, T);
    if (st != BS_OK) return st;
    if (T == 0 || I == 0) return BS_PATH_REBUILD;      // (no blocks: the weight is zero; the forward still goes through the dense path)
    return bs_gemv_forward_path(I, M, N, K, T);
}

extern "C" int bs_sparse_kernel(const int *I, const int *M, int n, int N, int K, int T) {
    if (!I || !M) return BS_ERR_NULL;
    if (n < 1 || n > BS_MAX_GROUP) return BS_ERR_SHAPE;
    bool empty = T == 0;
    for (int j = 0; j < n; j++) {
        const int st = forward_dims(I[j], M[j], N, K, T);
        if (st != BS_OK) return st;
        empty = empty || I[j] == 0;
    }
    return empty ? 0 : bs_gemv_sparse_serves(I, M, n, N, K, T);
}

// `asked`: for the rank (16 or less) that the caller asks about
static int tile_kernel(const int *I, const int *M, int n, int N, int K, int T, int *columns, bool asked) {
    if (!I || !M || !columns) return BS_ERR_NULL;
    if (n < 1 || n > BS_MAX_GROUP) return BS_ERR_SHAPE;
    bool empty = T == 0;
    for (int j = 0; j < n; j++) {
        const int st = forward_dims(I[j], M[j], N, K, T);
        if (st != BS_OK) return st;
        empty = empty || I[j] == 0;
        columns[j] = 0;
    }
    return empty || !asked ? BS_TILE_NONE : bs_gemv_tile_kernel(I, M, n, N, K, T, columns);
}

extern "C" int bs_tile_kernel(const int *I, const int *M, int n, int N, int K, int T, int *columns) { return tile_kernel(I, M, n, N, K, T, columns, K == 16); }
extern "C" int bs_small_rank_kernel(const int *I, const int *M, int n, int N, int K, int T, int *columns) { return tile_kernel(I, M, n, N, K, T, columns, K < 16); }

static int forward_impl(const uint8_t *packed, const void *u, const void *vt, const void *x,
                        const void *bias, void *y, int I, int M, int N, int K, int T,
                        void *workspace, int64_t workspace_bytes, void *stream, bool library_ok) {
    int st = forward_dims(I, M, N, K, T);
    if (st != BS_OK) return st;
    if (T == 0) return BS_OK;
    if (!x || !y || (I > 0 && (!packed || !u || !vt))) return BS_ERR_NULL;
    if (!bs_aligned(packed, 16) || !bs_aligned(vt, 16) || !bs_aligned(x, 16) || !bs_aligned(u, 8) ||
        !bs_aligned(y, 2) || !bs_aligned(bias, 2))
        return BS_ERR_ALIGN;
    hipStream_t s = (hipStream_t)stream;

    bool taken;                                  // (asked once, with the plan: a decode call is over in some 8 us)
    st = bs_launch_gemv(packed, (const half_t *)u, (const half_t *)vt, (const half_t *)x, (const half_t *)bias, (half_t *)y, I, M, N, K, T,
                        workspace, workspace_bytes, &taken, s);
    if (taken) return st;
    if (!workspace || workspace_bytes < rebuild_need(M, N, T, library_ok) || !bs_aligned(workspace, 256)) return BS_ERR_WORKSPACE;
    half_t *w = (half_t *)workspace;
    st = bs_launch_reconstruct_packed(packed, (const half_t *)u, (const half_t *)vt, w, I, M, N, K, s);
    if (st != BS_OK) return st;
    if (library_ok && dense_wants_library(M, N)) {
        st = bs_launch_linear_library((const half_t *)x, w, (const half_t *)bias, (half_t *)y, T, M, N,
                                      (char *)workspace + round_up((int64_t)M * N * 2, 256), s);
        if (st != BS_ERR_SHAPE) return st;      // enqueued, or failed for good; BS_ERR_SHAPE: declined before anything was enqueued
    }
    return bs_launch_linear_parts((const half_t *)x, w, (const half_t *)bias, (half_t *)y, T, M, N,
                                  (float *)((char *)workspace + round_up((int64_t)M * N * 2, 256)), s);
}

extern "C" int bs_forward(const uint8_t *packed, const void *u, const void *vt, const void *x,
                          const void *bias, void *y, int I, int M, int N, int K, int T,
                          void *workspace, int64_t workspace_bytes, void *stream) {
    return forward_impl(packed, u, vt, x, bias, y, I, M, N, K, T, workspace, workspace_bytes, stream, true);
}

// ---- the forward for callers that cannot allocate ------------------------------------
// The scratch of the decode and strip kernels (partial row sums) lives in a file-scope device
// array instead of a caller-owned workspace.  Every GPU the library runs on holds its own copy
// of the array at its own address until the process ends; `scratch` itself is only the
// host-side handle of the symbol, so the address is looked up once per device (with that
// device current) and only the looked-up pointer is ever handed to a kernel.
static __device__ __align__(256) unsigned char scratch[BS_STATIC_SCRATCH_BYTES];
static void *g_scratch_ptr[BS_MAX_DEVICES];
static std::mutex g_scratch_mutex;

static int static_scratch(void **out) {
    int dev = -1;
    BS_HIP_TRY(hipGetDevice(&dev));
    if (dev < 0 || dev >= BS_MAX_DEVICES) return BS_ERR_NO_DEVICE;
    std::lock_guard<std::mutex> lock(g_scratch_mutex);
    if (!g_scratch_ptr[dev]) {
        void *p = nullptr;
        BS_HIP_TRY(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
        if (!p) return BS_ERR_NO_DEVICE;
        g_scratch_ptr[dev] = p;
    }
    *out = g_scratch_ptr[dev];
    return BS_OK;
}

extern "C" int bs_forward_static(const uint8_t *packed, const void *u, const void *vt, const void *x,
                                 const void *bias, void *y, int I, int M, int N, int K, int T, void *stream) {
    int st = forward_dims(I, M, N, K, T);
    if (st != BS_OK) return st;
    if (T == 0) return BS_OK;
    // sizes first: a call that would not fit is refused before any device is touched.  The dense product
    // always runs this library's own kernel here, whatever bs_set_dense_kernel says: the vendor GEMM wants
    // 64 MiB of scratch of its own, and setting it up allocates.
    const int64_t need = workspace_need(I, M, N, K, T, false);
    if (need < 0) return (int)need;
    if (need > (int64_t)BS_STATIC_SCRATCH_BYTES) return BS_ERR_WORKSPACE;
    void *ws = nullptr;
    st = static_scratch(&ws);
    if (st != BS_OK) return st;
    // nothing in the scratch has to start at zero: every partial sum a call reads it has written before
    return forward_impl(packed, u, vt, x, bias, y, I, M, N, K, T, ws, (int64_t)BS_STATIC_SCRATCH_BYTES, stream, false);
}

// ---- grouped decode forward ---------------------------------------------------
static int group_dims(const bs_matrix *mats, int n, int N, int K, int T) {
    if (!mats) return BS_ERR_NULL;
    if (n < 1 || n > BS_MAX_GROUP) return BS_ERR_SHAPE;
    for (int j = 0; j < n; j++) {
        int st = forward_dims(mats[j].I, mats[j].M, N, K, T);
        if (st != BS_OK) return st;
        if (mats[j].I < 1) return BS_ERR_SHAPE;
    }
    if (T < 1 || T > 48) return BS_ERR_SHAPE;
    return BS_OK;
}

extern "C" int64_t bs_forward_group_workspace_bytes(const bs_matrix *mats, int n, int N, int K, int T) {
    int st = group_dims(mats, n, N, K, T);
    if (st != BS_OK) return st;
    int I[BS_MAX_GROUP], M[BS_MAX_GROUP];
    for (int j = 0; j < n; j++) { I[j] = mats[j].I; M[j] = mats[j].M; }
    const int64_t b = bs_gemv_group_workspace_bytes(I, M, n, N, K, T);
    return b > 0 ? b : (int64_t)BS_ERR_SHAPE;
}

static int forward_group(const bs_matrix *mats, int n, int N, int K, const void *x, int T,
                         int epilogue, const void *residual, void *y, int input_rms, float eps,
                         void *workspace, int64_t workspace_bytes, void *stream) {
    int st = group_dims(mats, n, N, K, T);
    if (st != BS_OK) return st;
    if (epilogue != BS_EPI_NONE && epilogue != BS_EPI_RESIDUAL && epilogue != BS_EPI_SWIGLU) return BS_ERR_SHAPE;
    if (!x || !y || (epilogue == BS_EPI_RESIDUAL && !residual)) return BS_ERR_NULL;
    const uint8_t *packed[BS_MAX_GROUP];
    const half_t *u[BS_MAX_GROUP], *vt[BS_MAX_GROUP], *bias[BS_MAX_GROUP];
    int I[BS_MAX_GROUP], M[BS_MAX_GROUP];
    for (int j = 0; j < n; j++) {
        if (!mats[j].packed || !mats[j].u || !mats[j].vt) return BS_ERR_NULL;
        if (!bs_aligned(mats[j].packed, 16) || !bs_aligned(mats[j].vt, 16) || !bs_aligned(mats[j].u, 8) ||
            !bs_aligned(mats[j].bias, 2))
            return BS_ERR_ALIGN;
        packed[j] = mats[j].packed;
        u[j] = (const half_t *)mats[j].u;
        vt[j] = (const half_t *)mats[j].vt;
        bias[j] = (const half_t *)mats[j].bias;
        I[j] = mats[j].I;
        M[j] = mats[j].M;
    }
    if (!bs_aligned(x, 16) || !bs_aligned(y, 2) || !bs_aligned(residual, 2)) return BS_ERR_ALIGN;
    return bs_launch_gemv_group(n, packed, u, vt, bias, I, M, N, K, (const half_t *)x, T, epilogue,
                                (const half_t *)residual, (half_t *)y, input_rms, eps, workspace, workspace_bytes,
                                (hipStream_t)stream);
}

extern "C" int bs_forward_group(const bs_matrix *mats, int n, int N, int K, const void *x, int T,
                                int epilogue, const void *residual, void *y,
                                void *workspace, int64_t workspace_bytes, void *stream) {
    return forward_group(mats, n, N, K, x, T, epilogue, residual, y, 0, 0.f, workspace, workspace_bytes, stream);
}

extern "C" int bs_forward_group_rms(const bs_matrix *mats, int n, int N, int K, const void *x, int T, float eps,
                                    int epilogue, const void *residual, void *y,
                                    void *workspace, int64_t workspace_bytes, void *stream) {
    if (!(eps >= 0.f)) return BS_ERR_SHAPE;
    return forward_group(mats, n, N, K, x, T, epilogue, residual, y, 1, eps, workspace, workspace_bytes, stream);
}

extern "C" int bs_rmsnorm_f16(const void *x, const void *weight, void *y, int T, int H, float eps, void *stream) {
    if (T < 0 || H <= 0 || H % 8 != 0 || H > 16384) return BS_ERR_SHAPE;
    if (T == 0) return BS_OK;
    if (!x || !weight || !y) return BS_ERR_NULL;
    if (!bs_aligned(x, 16) || !bs_aligned(weight, 16) || !bs_aligned(y, 16)) return BS_ERR_ALIGN;
    return bs_launch_rmsnorm((const half_t *)x, (const half_t *)weight, (half_t *)y, T, H, eps, (hipStream_t)stream);
}

extern "C" int bs_add_rmsnorm_f16(const void *x, const void *add, void *sum, const void *weight, void *y, int T, int H, float eps,
                                  void *stream) {
    if (T < 0 || H <= 0 || H % 8 != 0 || H > 16384) return BS_ERR_SHAPE;
    if (T == 0) return BS_OK;
    if (!x || !add || !sum || !weight || !y) return BS_ERR_NULL;
    if (!bs_aligned(x, 16) || !bs_aligned(add, 16) || !bs_aligned(sum, 16) || !bs_aligned(weight, 16) || !bs_aligned(y, 16))
        return BS_ERR_ALIGN;
    return bs_launch_add_rmsnorm((const half_t *)x, (const half_t *)add, (half_t *)sum, (const half_t *)weight, (half_t *)y, T, H, eps,
                                 (hipStream_t)stream);
}

extern "C" int bs_rope_store_f16(void *q, int ldq, const void *k, const void *v, int ldkv, const void *cos, const void *sin,
                                 void *kcache, void *vcache, int B, int n, int heads, int kv_heads, int head_dim, int max_len, void *stream) {
    if (B < 0 || n < 0 || n > max_len || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || head_dim % 2 != 0 ||
        (int64_t)B * n > INT32_MAX || ((int64_t)heads + 3 * (int64_t)kv_heads) * head_dim > INT32_MAX ||
        ldq < (int64_t)heads * head_dim || ldkv < (int64_t)kv_heads * head_dim)
        return BS_ERR_SHAPE;
    if (B == 0 || n == 0) return BS_OK;
    if (!q || !k || !v || !cos || !sin || !kcache || !vcache) return BS_ERR_NULL;
    if (!bs_aligned(q, 16) || !bs_aligned(k, 16) || !bs_aligned(v, 16) || !bs_aligned(cos, 16) || !bs_aligned(sin, 16) ||
        !bs_aligned(kcache, 16) || !bs_aligned(vcache, 16))
        return BS_ERR_ALIGN;
    return bs_launch_rope_store((half_t *)q, (const half_t *)k, (const half_t *)v, (const half_t *)cos, (const half_t *)sin,
                                (half_t *)kcache, (half_t *)vcache, ldq, ldkv, B, n, heads, kv_heads, head_dim, max_len,
                                (hipStream_t)stream);
}

extern "C" int bs_attention_prefill_f16(const void *q, int ldq, const void *kcache, const void *vcache, void *out, int B, int n, int heads,
                                        int kv_heads, int head_dim, int max_len, void *stream) {
    if (B < 0 || n < 0 || n > max_len || n > 32 * 65535 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim != 128 ||
        (int64_t)B * heads > INT32_MAX || ldq < (int64_t)heads * head_dim || ldq % 8 != 0)
        return BS_ERR_SHAPE;
    if (B == 0 || n == 0) return BS_OK;
    if (!q || !kcache || !vcache || !out) return BS_ERR_NULL;
    if (!bs_aligned(q, 16) || !bs_aligned(kcache, 16) || !bs_aligned(vcache, 16) || !bs_aligned(out, 16)) return BS_ERR_ALIGN;
    return bs_launch_attention_prefill((const half_t *)q, (const half_t *)kcache, (const half_t *)vcache, (half_t *)out, ldq, B, n, heads,
                                       kv_heads, max_len, (hipStream_t)stream);
}

extern "C" int bs_silu_mul_f16(const void *gate, const void *up, void *y, int T, int width, int ld, void *stream) {
    if (T < 0 || width <= 0 || width > INT32_MAX - 4096 || ld < width) return BS_ERR_SHAPE;
    if (T == 0) return BS_OK;
    if (!gate || !up || !y) return BS_ERR_NULL;
    if (!bs_aligned(gate, 16) || !bs_aligned(up, 16) || !bs_aligned(y, 16)) return BS_ERR_ALIGN;
    if (T > 1 && (width % 8 != 0 || ld % 8 != 0)) return BS_ERR_ALIGN;
    return bs_launch_silu_mul((const half_t *)gate, (const half_t *)up, (half_t *)y, T, width, ld, (hipStream_t)stream);
}

// Several matrices on the same x as one product: rebuilt below each other, so that a narrow one (k, v) does not leave most of
// the chip idle by itself.  us one by one / as one, 4 blocks: 4096 + 1024 + 1024 rows of 4096 columns (48 MiB of weights) 84 / 63 at 130
// tokens, 104 / 75 at 700, 138 / 108 at 1400, 294 / 284 at 6000; 3 x 3072 of 3072 (54 MiB) 85 / 64, 128 / 82, 141 / 116, 375 / 339.
// The limits are where the rebuilt weights no longer stay in the cache between the two launches; 33 shapes from 10 to 384 MiB
// were timed at eight token counts.  Up to 96 MiB: 0.97 to 1.58 times as fast (3 x 4096 of 4096, on the limit: 1.34 at 700 tokens, 0.97
// at 1400, 1.02 to 1.09 from 2000; 2 x 8192 of 3072, too: 1.08, 1.00, 1.00 to 1.04).  Up to 128 MiB few tokens gain (5120 + 2 x 2560 of
// 5120, 100 MiB: 1.14 at 130, 1.05 at 2000; 2 x 10752 of 3072, 126 MiB: 1.30, 0.99) and many do not (0.98 at 6000).  Beyond, equally wide
// matrices lose (2 x 14336 of 4096, 224 MiB: 158 / 170 at 130, 399 / 401 at 1400; 2 x 10752, 168 MiB: 0.94 at 1400), narrow ones
// gain up to 160 MiB (8192 + 1024 + 1024 of 8192, on the limit: 166 / 124 at 130, 330 / 268 at 1400, 715 / 672 at 4500, 864 / 873 at 6000).
constexpr int64_t CAT_WEIGHT = 96ll << 20, CAT_WEIGHT_FEW = 128ll << 20, CAT_WEIGHT_NARROW = 160ll << 20;   // bytes
constexpr int CAT_FEW = 2048, CAT_NARROW_TOKENS = 4500;
static int64_t cat_rows(const bs_matrix *mats, int n, int N, int K, int T) {
    if (!mats || n < 2 || n > BS_MAX_GROUP) return 0;
    int64_t rows = 0;
    for (int j = 0; j < n; j++) {
        if (mats[j].bias || mats[j].I < 1 || forward_dims(mats[j].I, mats[j].M, N, K, T) != BS_OK ||
            bs_forward_path(mats[j].I, mats[j].M, N, K, T) != BS_PATH_REBUILD || dense_wants_library(mats[j].M, N))
            return 0;
        rows += mats[j].M;
    }
    int64_t narrowest = rows;
    for (int j = 0; j < n; j++)
        if (mats[j].M < narrowest) narrowest = mats[j].M;
    const int64_t limit = 8 * narrowest <= rows && T <= CAT_NARROW_TOKENS ? CAT_WEIGHT_NARROW : T <= CAT_FEW ? CAT_WEIGHT_FEW : CAT_WEIGHT;
    return N % 8 == 0 && rows * N * 2 <= limit ? rows : 0;
}

extern "C" int64_t bs_forward_cat_workspace_bytes(const bs_matrix *mats, int n, int N, int K, int T) {
    if (T <= 0 || N <= 0) return 0;
    const int64_t rows = cat_rows(mats, n, N, K, T);
    return rows ? round_up(rows * N * 2, 256) + round_up(bs_linear_parts_bytes(T, (int)rows, N), 256) : 0;
}

extern "C" int bs_forward_cat(const bs_matrix *mats, int n, int N, int K, const void *x, int T, void *y, void *workspace,
                              int64_t workspace_bytes, void *stream) {
    const int64_t need = bs_forward_cat_workspace_bytes(mats, n, N, K, T);
    if (need == 0) return BS_ERR_SHAPE;
    if (!x || !y) return BS_ERR_NULL;
    for (int j = 0; j < n; j++) {
        if (!mats[j].packed || !mats[j].u || !mats[j].vt) return BS_ERR_NULL;
        if (!bs_aligned(mats[j].packed, 16) || !bs_aligned(mats[j].vt, 16) || !bs_aligned(mats[j].u, 8)) return BS_ERR_ALIGN;
    }
    if (!bs_aligned(x, 16) || !bs_aligned(y, 2)) return BS_ERR_ALIGN;
    if (!workspace || workspace_bytes < need || !bs_aligned(workspace, 256)) return BS_ERR_WORKSPACE;
    half_t *w = (half_t *)workspace;
    int64_t rows = 0;
    const uint8_t *packed[BS_MAX_GROUP];
    const half_t *u[BS_MAX_GROUP], *vt[BS_MAX_GROUP];
    half_t *part[BS_MAX_GROUP];
    int I[BS_MAX_GROUP], M[BS_MAX_GROUP];
    for (int j = 0; j < n; j++) {
        packed[j] = (const uint8_t *)mats[j].packed;
        u[j] = (const half_t *)mats[j].u;
        vt[j] = (const half_t *)mats[j].vt;
        part[j] = w + rows * N;
        I[j] = mats[j].I;
        M[j] = mats[j].M;
        rows += M[j];
    }
    int st = bs_launch_tile_rebuild(n, packed, u, vt, I, M, part, N, K, (hipStream_t)stream);       // all in one launch, or one by one
    for (int j = 0; st == BS_ERR_SHAPE && j < n; j++) {
        const int one = bs_launch_reconstruct_packed(packed[j], u[j], vt[j], part[j], I[j], M[j], N, K, (hipStream_t)stream);
        if (one != BS_OK) return one;
        if (j + 1 == n) st = BS_OK;
    }
    if (st != BS_OK) return st;
    return bs_launch_linear_parts((const half_t *)x, w, nullptr, (half_t *)y, T, (int)rows, N,
                                  (float *)((char *)workspace + round_up(rows * N * 2, 256)), (hipStream_t)stream);
}

static int attention_shape(int B, int heads, int kv_heads, int head_dim, int max_len) {
    return B < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim != 128 || max_len < 1 || max_len > 8192 ? BS_ERR_SHAPE
                                                                                                                          : BS_OK;
}

extern "C" int64_t bs_attention_decode_workspace_bytes(int B, int heads, int kv_heads, int head_dim, int max_len) {
    const int st = attention_shape(B, heads, kv_heads, head_dim, max_len);
    return st != BS_OK ? st : bs_attention_parts_bytes(B, heads, kv_heads, max_len);
}

extern "C" int bs_attention_decode_ws_f16(const void *qkv, void *kcache, void *vcache, const void *cos, const void *sin,
                                          const int64_t *pos, void *out, int B, int heads, int kv_heads, int head_dim,
                                          int max_len, void *workspace, int64_t workspace_bytes, void *stream) {
    const int st = attention_shape(B, heads, kv_heads, head_dim, max_len);
    if (st != BS_OK) return st;
    if (B == 0) return BS_OK;
    if (!qkv || !kcache || !vcache || !cos || !sin || !pos || !out) return BS_ERR_NULL;
    if (!bs_aligned(qkv, 16) || !bs_aligned(kcache, 16) || !bs_aligned(vcache, 16) || !bs_aligned(cos, 16) ||
        !bs_aligned(sin, 16) || !bs_aligned(pos, 8) || !bs_aligned(out, 16))
        return BS_ERR_ALIGN;
    const bool room = workspace && bs_aligned(workspace, 16) &&
                      workspace_bytes >= bs_attention_parts_bytes(B, heads, kv_heads, max_len);
    return bs_launch_attention_decode((const half_t *)qkv, (half_t *)kcache, (half_t *)vcache, (const half_t *)cos,
                                      (const half_t *)sin, pos, (half_t *)out, B, heads, kv_heads, head_dim, max_len,
                                      room ? (float *)workspace : nullptr, (hipStream_t)stream);
}

extern "C" int bs_attention_decode_f16(const void *qkv, void *kcache, void *vcache, const void *cos, const void *sin,
                                       const int64_t *pos, void *out, int B, int heads, int kv_heads, int head_dim,
                                       int max_len, void *stream) {
    return bs_attention_decode_ws_f16(qkv, kcache, vcache, cos, sin, pos, out, B, heads, kv_heads, head_dim, max_len, nullptr, 0, stream);
}

extern "C" int bs_argmax_f16(const void *x, int64_t *out, int B, int V, void *stream) { return bs_argmax_advance_f16(x, out, nullptr, B, V, stream); }

extern "C" int bs_argmax_advance_f16(const void *x, int64_t *out, int64_t *pos, int B, int V, void *stream) {
    if (B < 0 || V <= 0) return BS_ERR_SHAPE;
    if (B == 0) return BS_OK;
    if (!x || !out) return BS_ERR_NULL;
    if (!bs_aligned(x, 16) || !bs_aligned(out, 8) || !bs_aligned(pos, 8) || (B > 1 && V % 8 != 0)) return BS_ERR_ALIGN;
    return bs_launch_argmax((const half_t *)x, out, pos, B, V, (hipStream_t)stream);
}

// ---- requests of unequal lengths -----------------------------------------------------------------
// log2 of a page's positions, or -1
static int page_shift(int page_size) {
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0) return -1;
    return __builtin_ctz((unsigned)page_size);
}
static bool pool_fits(int pool_pages, int page_size) { return pool_pages >= 1 && (int64_t)pool_pages * page_size <= INT32_MAX; }

static int plan_shape(int B, int T, int page_size, int max_pages, int pool_pages) {
    return B < 0 || B > 65536 || T < 0 || T > 1 << 30 || page_shift(page_size) < 0 || max_pages < 1 || max_pages > 1 << 24 || !pool_fits(pool_pages, page_size)
               ? BS_ERR_SHAPE
               : BS_OK;
}

extern "C" int64_t bs_page_plan_workspace_bytes(int B, int T) {
    return B < 0 || B > 65536 || T < 0 || T > 1 << 30 ? BS_ERR_SHAPE : bs_page_plan_scratch(B, T);
}

extern "C" int bs_page_plan(const int32_t *lengths, const int32_t *new_tokens, const uint8_t *released, int32_t *block_table, int32_t *free_pages,
                            const int32_t *free_state, int32_t *lengths_out, int32_t *free_state_out, int32_t *granted, int32_t *starts,
                            int32_t *positions, int64_t *slots, int64_t *row_slots, int B, int T, int page_size, int max_pages, int pool_pages,
                            void *workspace, int64_t workspace_bytes, void *stream) {
    const int st = plan_shape(B, T, page_size, max_pages, pool_pages);
    if (st != BS_OK) return st;
    if (!free_pages || !free_state || !free_state_out || !starts || (T > 0 && (!positions || !slots)) ||
        (B > 0 && (!lengths || !new_tokens || !block_table || !lengths_out || !granted)))
        return BS_ERR_NULL;
    for (const void *p : {(const void *)lengths, (const void *)new_tokens, (const void *)block_table, (const void *)free_pages, (const void *)free_state,
                          (const void *)lengths_out, (const void *)free_state_out, (const void *)granted, (const void *)starts, (const void *)positions})
        if (!bs_aligned(p, 4)) return BS_ERR_ALIGN;
    if (!bs_aligned(slots, 8) || !bs_aligned(row_slots, 8)) return BS_ERR_ALIGN;
    const int64_t need = bs_page_plan_scratch(B, T);
    if (need > 0 && (!workspace || workspace_bytes < need || !bs_aligned(workspace, 16))) return BS_ERR_WORKSPACE;
    return bs_launch_page_plan(lengths, new_tokens, released, block_table, free_pages, free_state, lengths_out, free_state_out, granted, starts, positions, slots,
                               row_slots, B, T, page_shift(page_size), max_pages, pool_pages, workspace, (hipStream_t)stream);
}

extern "C" int bs_rope_store_paged_f16(void *q, int ldq, void *q_out, int ldq_out, const void *k, const void *v, int ldkv, const void *cos, const void *sin,
                                       const int32_t *positions, const int64_t *slots, void *kpages, void *vpages, int T, int heads, int kv_heads,
                                       int head_dim, int max_pos, int page_size, int pool_pages, void *stream) {
    if (T < 0 || (head_dim != 64 && head_dim != 128) || kv_heads < 1 || max_pos < 1 || page_shift(page_size) < 0 || !pool_fits(pool_pages, page_size) ||
        (q && heads < 1) || ((q ? heads : 0) + 3 * (int64_t)kv_heads) * head_dim > INT32_MAX || ldkv < (int64_t)kv_heads * head_dim ||
        (q && ldq < (int64_t)heads * head_dim) || (q_out && ldq_out < (int64_t)heads * head_dim) || (q_out && !q) || (q && q_out == q && ldq_out != ldq))
        return BS_ERR_SHAPE;
    if (T == 0) return BS_OK;
    if (!k || !v || !cos || !sin || !positions || !slots || !kpages || !vpages) return BS_ERR_NULL;
    for (const void *p : {(const void *)q, (const void *)q_out, (const void *)k, (const void *)v, (const void *)cos, (const void *)sin, (const void *)kpages, (const void *)vpages})
        if (!bs_aligned(p, 2)) return BS_ERR_ALIGN;
    if (!bs_aligned(positions, 4) || !bs_aligned(slots, 8)) return BS_ERR_ALIGN;
    half_t *from = q ? (half_t *)q : (half_t *)k;          // (no heads: neither read nor written)
    return bs_launch_rope_store_paged(from, q_out ? (half_t *)q_out : from, (const half_t *)k, (const half_t *)v, (const half_t *)cos, (const half_t *)sin, positions,
                                      slots, (half_t *)kpages, (half_t *)vpages, q ? ldq : ldkv, q ? (q_out ? ldq_out : ldq) : ldkv, ldkv, T, q ? heads : 0,
                                      kv_heads, head_dim, max_pos, page_shift(page_size), pool_pages, (hipStream_t)stream);
}

static int attention_paged_shape(int B, int heads, int kv_heads, int head_dim, int page_size, int max_pages) {
    return B < 0 || B > 65536 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || (head_dim != 64 && head_dim != 128) || page_shift(page_size) < 0 ||
                   max_pages < 1 || (int64_t)max_pages * page_size > INT32_MAX || (int64_t)B * ((int64_t)max_pages * page_size / 16) > INT32_MAX ||
                   ((int64_t)heads + 2 * (int64_t)kv_heads) * head_dim > INT32_MAX || (int64_t)B * heads > 1 << 22
               ? BS_ERR_SHAPE
               : BS_OK;
}

extern "C" int64_t bs_attention_paged_workspace_bytes(int B, int heads, int kv_heads, int head_dim, int page_size, int max_pages) {
    const int st = attention_paged_shape(B, heads, kv_heads, head_dim, page_size, max_pages);
    return st != BS_OK ? st : B == 0 ? 0 : bs_attention_paged_scratch(B, heads, kv_heads, head_dim, max_pages, page_size);
}

extern "C" int bs_attention_paged_f16(const void *qkv, int ldqkv, void *kpages, void *vpages, const void *cos, const void *sin, const int32_t *block_table,
                                      const int32_t *lengths, const int64_t *slots, void *out, int B, int heads, int kv_heads, int head_dim, int max_pos,
                                      int page_size, int max_pages, int pool_pages, void *workspace, int64_t workspace_bytes, void *stream) {
    const int st = attention_paged_shape(B, heads, kv_heads, head_dim, page_size, max_pages);
    if (st != BS_OK) return st;
    if (max_pos < 1 || !pool_fits(pool_pages, page_size) || ldqkv < ((int64_t)heads + 2 * (int64_t)kv_heads) * head_dim) return BS_ERR_SHAPE;
    if (B == 0) return BS_OK;
    if (!qkv || !kpages || !vpages || !cos || !sin || !block_table || !lengths || !slots || !out) return BS_ERR_NULL;
    if (!bs_aligned(qkv, 2) || !bs_aligned(kpages, 16) || !bs_aligned(vpages, 16) || !bs_aligned(cos, 2) || !bs_aligned(sin, 2) || !bs_aligned(block_table, 4) ||
        !bs_aligned(lengths, 4) || !bs_aligned(slots, 8) || !bs_aligned(out, 2))
        return BS_ERR_ALIGN;
    const int64_t need = bs_attention_paged_scratch(B, heads, kv_heads, head_dim, max_pages, page_size);
    if (need > 0 && (!workspace || workspace_bytes < need || !bs_aligned(workspace, 16))) return BS_ERR_WORKSPACE;
    return bs_launch_attention_paged((const half_t *)qkv, ldqkv, (half_t *)kpages, (half_t *)vpages, (const half_t *)cos, (const half_t *)sin, block_table, lengths,
                                     slots, (half_t *)out, B, heads, kv_heads, head_dim, max_pos, page_shift(page_size), max_pages, pool_pages, workspace,
                                     (hipStream_t)stream);
}

static int sample_shape(int B, int V) {
    return B < 0 || B > 1 << 20 || V < 1 || V > 1 << 18 || (int64_t)B * V > 1ll << 33 ? BS_ERR_SHAPE : BS_OK;
}

extern "C" int64_t bs_sample_workspace_bytes(int B, int V) {
    const int st = sample_shape(B, V);
    return st != BS_OK ? st : B == 0 ? 0 : bs_sample_scratch(B, V);
}

extern "C" int bs_sample_f16(const void *logits, int64_t ld, const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p,
                             const float *min_p, int64_t *out, int B, int V, void *workspace, int64_t workspace_bytes, void *stream) {
    if (sample_shape(B, V) != BS_OK || (B > 1 && ld < V)) return BS_ERR_SHAPE;
    if (B == 0) return BS_OK;
    if (!logits || !uniform || !out) return BS_ERR_NULL;
    if (!bs_aligned(logits, 2) || !bs_aligned(uniform, 4) || !bs_aligned(temperature, 4) || !bs_aligned(top_k, 4) || !bs_aligned(top_p, 4) || !bs_aligned(min_p, 4) ||
        !bs_aligned(out, 8))
        return BS_ERR_ALIGN;
    if (!workspace || workspace_bytes < bs_sample_scratch(B, V) || !bs_aligned(workspace, 16)) return BS_ERR_WORKSPACE;
    return bs_launch_sample((const half_t *)logits, ld, uniform, temperature, top_k, top_p, min_p, out, B, V, workspace, (hipStream_t)stream);
}

// ---- drafted tokens, forked rows, settings on logits -----------------------------------------------
static bool all_aligned(std::initializer_list<const void *> pointers, uintptr_t to) {
    for (const void *p : pointers)
        if (!bs_aligned(p, to)) return false;
    return true;
}
static bool any_null(std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if (!p) return true;
    return false;
}

extern "C" int bs_tree_plan(const int32_t *parents, const int32_t *lengths, const int32_t *granted, const int32_t *starts, int32_t *positions, int64_t *masks, int B, int T,
                            void *stream) {
    if (B < 0 || B > 65536 || T < 0 || T > 1 << 30) return BS_ERR_SHAPE;
    if (T == 0) return BS_OK;
    if (any_null({parents, positions, masks}) || (B > 0 && any_null({lengths, granted, starts}))) return BS_ERR_NULL;
    if (!all_aligned({parents, lengths, granted, starts, positions}, 4) || !bs_aligned(masks, 8)) return BS_ERR_ALIGN;
    return bs_launch_tree_plan(parents, lengths, granted, starts, positions, masks, B, T, (hipStream_t)stream);
}

static int attention_tree_shape(int B, int T, int nodes, int heads, int kv_heads, int head_dim, int page_size, int max_pages) {
    return attention_paged_shape(B, heads, kv_heads, head_dim, page_size, max_pages) != BS_OK || T < 0 || (int64_t)T * heads > 1 << 22 || nodes < 1 || nodes > 64
               ? BS_ERR_SHAPE
               : BS_OK;
}

extern "C" int64_t bs_attention_tree_workspace_bytes(int B, int T, int nodes, int heads, int kv_heads, int head_dim, int page_size, int max_pages) {
    const int st = attention_tree_shape(B, T, nodes, heads, kv_heads, head_dim, page_size, max_pages);
    return st != BS_OK ? st : B == 0 || T == 0 ? 0 : bs_attention_tree_scratch(B, T, nodes, heads, kv_heads, head_dim, max_pages, page_size);
}

extern "C" int bs_attention_tree_f16(const void *q, int ldq, const void *kpages, const void *vpages, const int32_t *block_table, const int32_t *lengths,
                                     const int32_t *granted, const int32_t *starts, const int64_t *masks, void *out, int B, int T, int nodes, int heads, int kv_heads,
                                     int head_dim, int page_size, int max_pages, int pool_pages, void *workspace, int64_t workspace_bytes, void *stream) {
    const int st = attention_tree_shape(B, T, nodes, heads, kv_heads, head_dim, page_size, max_pages);
    if (st != BS_OK) return st;
    if (!pool_fits(pool_pages, page_size) || ldq < (int64_t)heads * head_dim) return BS_ERR_SHAPE;
    if (T == 0) return BS_OK;
    if (any_null({q, out, masks}) || (B > 0 && any_null({kpages, vpages, block_table, lengths, granted, starts}))) return BS_ERR_NULL;
    if (!all_aligned({q, out}, 2) || !all_aligned({kpages, vpages}, 16) || !all_aligned({block_table, lengths, granted, starts}, 4) || !bs_aligned(masks, 8))
        return BS_ERR_ALIGN;
    const int64_t need = B == 0 ? 0 : bs_attention_tree_scratch(B, T, nodes, heads, kv_heads, head_dim, max_pages, page_size);
    if (need > 0 && (!workspace || workspace_bytes < need || !bs_aligned(workspace, 16))) return BS_ERR_WORKSPACE;
    return bs_launch_attention_tree((const half_t *)q, ldq, (const half_t *)kpages, (const half_t *)vpages, block_table, lengths, granted, starts, masks, (half_t *)out, B,
                                    T, nodes, heads, kv_heads, head_dim, page_shift(page_size), max_pages, pool_pages, workspace, (hipStream_t)stream);
}

// a cache whose pieces of a row, in all layers, 32 bits count
static int layers_shape(int B, int layers, int kv_heads, int head_dim, int page_size, int max_pages, int pool_pages) {
    return B < 0 || B > 65536 || layers < 1 || kv_heads < 1 || head_dim < 8 || head_dim % 8 != 0 || kv_heads > 1 << 20 || head_dim > 1 << 20 ||
                   (int64_t)kv_heads * head_dim >= 1 << 28 || layers * ((int64_t)kv_heads * head_dim) >= 1 << 28 || page_shift(page_size) < 0 || max_pages < 1 ||
                   max_pages > 1 << 24 || (int64_t)B * max_pages > INT32_MAX || !pool_fits(pool_pages, page_size)
               ? BS_ERR_SHAPE
               : BS_OK;
}

extern "C" int64_t bs_tree_accept_workspace_bytes(int B) { return B < 0 || B > 65536 ? BS_ERR_SHAPE : bs_tree_accept_scratch(B); }

extern "C" int bs_tree_accept_f16(const int64_t *tokens, const int32_t *parents, const int64_t *targets, const int64_t *slots, const int32_t *lengths, const int32_t *granted,
                                  const int32_t *starts, const int32_t *block_table, int32_t *free_pages, const int32_t *free_state, void *kpages, void *vpages,
                                  int32_t *lengths_out, int32_t *free_state_out, int32_t *accepted, int32_t *path, int64_t *token, int B, int T, int nodes, int layers,
                                  int kv_heads, int head_dim, int page_size, int max_pages, int pool_pages, void *workspace, int64_t workspace_bytes, void *stream) {
    const int st = layers_shape(B, layers, kv_heads, head_dim, page_size, max_pages, pool_pages);
    if (st != BS_OK) return st;
    if (T < 0 || T > 1 << 30 || nodes < 1 || nodes > 64) return BS_ERR_SHAPE;
    if (any_null({free_pages, free_state, free_state_out}) || (T > 0 && any_null({tokens, parents, targets, slots})) ||
        (B > 0 && any_null({lengths, granted, starts, block_table, kpages, vpages, lengths_out, accepted, path, token})))
        return BS_ERR_NULL;
    if (!all_aligned({parents, lengths, granted, starts, block_table, free_pages, free_state, lengths_out, free_state_out, accepted, path}, 4) ||
        !all_aligned({tokens, targets, slots, token}, 8) || !all_aligned({kpages, vpages}, 16))
        return BS_ERR_ALIGN;
    if (B > 0 && (!workspace || workspace_bytes < bs_tree_accept_scratch(B) || !bs_aligned(workspace, 16))) return BS_ERR_WORKSPACE;
    return bs_launch_tree_accept(tokens, parents, targets, slots, lengths, granted, starts, block_table, free_pages, free_state, (half_t *)kpages, (half_t *)vpages,
                                 lengths_out, free_state_out, accepted, path, token, B, T, nodes, layers, kv_heads, head_dim, page_shift(page_size), max_pages, pool_pages,
                                 workspace, (hipStream_t)stream);
}

extern "C" int64_t bs_page_fork_workspace_bytes(int B, int max_pages, int pool_pages) {
    return B < 0 || B > 65536 || max_pages < 1 || max_pages > 1 << 24 || (int64_t)B * max_pages > INT32_MAX || pool_pages < 1 ? BS_ERR_SHAPE
                                                                                                                   : bs_page_fork_scratch(B, max_pages, pool_pages);
}

extern "C" int bs_page_fork_f16(const int32_t *source, const int32_t *lengths, int32_t *block_table, int32_t *free_pages, const int32_t *free_state, int32_t *shares,
                                void *kpages, void *vpages, int32_t *lengths_out, int32_t *free_state_out, int32_t *granted, int B, int layers, int kv_heads, int head_dim,
                                int page_size, int max_pages, int pool_pages, void *workspace, int64_t workspace_bytes, void *stream) {
    const int st = layers_shape(B, layers, kv_heads, head_dim, page_size, max_pages, pool_pages);
    if (st != BS_OK) return st;
    if (any_null({free_pages, free_state, free_state_out}) || (B > 0 && any_null({source, lengths, block_table, shares, kpages, vpages, lengths_out, granted})))
        return BS_ERR_NULL;
    if (!all_aligned({source, lengths, block_table, free_pages, free_state, shares, lengths_out, free_state_out, granted}, 4) || !all_aligned({kpages, vpages}, 16))
        return BS_ERR_ALIGN;
    if (!workspace || workspace_bytes < bs_page_fork_scratch(B, max_pages, pool_pages) || !bs_aligned(workspace, 16)) return BS_ERR_WORKSPACE;
    return bs_launch_page_fork(source, lengths, block_table, free_pages, free_state, shares, (half_t *)kpages, (half_t *)vpages, lengths_out, free_state_out, granted, B,
                               layers, kv_heads, head_dim, page_shift(page_size), max_pages, pool_pages, workspace, (hipStream_t)stream);
}

extern "C" int bs_logits_adjust_f16(const void *logits, int64_t ld, void *out, int64_t ld_out, const int32_t *requests, const int32_t *history, int history_width,
                                    const int32_t *history_lengths, const int32_t *prompt_lengths, const float *repetition, const float *frequency, const float *presence,
                                    const int32_t *drafted, int drafted_width, const int32_t *bias_tokens, const float *bias, int biases, const int32_t *allowed, int masks,
                                    const int32_t *allowed_rows, int R, int V, int B, void *stream) {
    if (sample_shape(R, V) != BS_OK || B < 0 || (R > 1 && (ld < V || ld_out < V)) || history_width < 0 || drafted_width < 0 || biases < 0 || masks < 0 ||
        history_width > 1 << 30 || drafted_width > 1 << 30 || (int64_t)history_width + drafted_width > INT32_MAX || biases > 1 << 30 ||   // (counts of 31 bits)
        ((history_lengths || prompt_lengths) && !history && history_width > 0) || (bias_tokens != nullptr) != (bias != nullptr) || (allowed_rows && !allowed && masks > 0) ||
        (allowed && !allowed_rows && masks < R) || (logits == out && ld != ld_out && R > 1) ||
        (!requests && B < R && (history || drafted || bias || repetition || frequency || presence)))
        return BS_ERR_SHAPE;
    if (R == 0) return BS_OK;
    if (!logits || !out) return BS_ERR_NULL;
    if (!all_aligned({logits, out}, 2) || !all_aligned({requests, history, history_lengths, prompt_lengths, repetition, frequency, presence, drafted, bias_tokens, bias, allowed,
                                                        allowed_rows}, 4))
        return BS_ERR_ALIGN;
    return bs_launch_logits_adjust((const half_t *)logits, ld, (half_t *)out, ld_out, requests, history, history_lengths, prompt_lengths, repetition, frequency, presence,
                                   drafted, bias_tokens, bias, allowed, allowed_rows, R, V, B, history_width, drafted_width, biases, masks, (hipStream_t)stream);
}
