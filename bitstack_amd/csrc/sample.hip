// The next token of every row from its logits, with temperature, top-k, top-p and min-p, from a random number that is given.
//
//   w_i = exp((x_i - max) / T)                     to 3e-13 of itself, summed in 64 bits: a random number next to a border of a large vocabulary is decided by 1e-9 of the sum.  (Four terms of
//                                                  a series, 1.4e-13, twice where a weight is a product of two; a fifth would cost every weight an operation more, for borders 1e-12 away)
//   top-k   the k largest; among equals the lowest indexes
//   top-p   of those, in the same order, the ones whose larger ones sum to less than p times the sum
//   min-p   of those, the ones with w_i >= min-p (the largest weight is 1)
//   token   the lowest index whose sum of kept weights up to it is more than u times the sum of all kept
//
// Nothing is sorted: fp16 values are compared by their bits in the order of the numbers (a key of 16 bits), and what stays is a border key and
// how many tokens with that key.  Borders are found by counting the tokens of every key in LDS; a sum over tokens with one key is then a
// product, so top-p needs a weight per key that occurs and not per token.  All sums are taken in one order: the result never varies.
//
// A row is cut into spans of 512 values, one wave's work.
//   sample_spans_kernel    every span's largest key and, where the row's sum is needed, its weights' sum next to its own largest
//   sample_rows_kernel     a row per workgroup: the largest; without top-k and top-p the span in which the random number falls, from the sums alone; otherwise the
//                          border, then the kept weights of the spans that reach it
//
// What bounds the first is its 64-bit operations where sums are wanted (200 rows of 50257: 12.3 us, 89 % of the vector units' cycles; 20 MB), otherwise the launch (2.5 us for a row of 32000).
// What bounds the second one is a chain of latencies (11 us for a row of 32000 with k 50 and top-p, 17 for top-p alone, 44 where it leaves most of 128256 tokens: counting 9,
// the keys' sums 10, the spans' 16), and instructions that come from memory the first time: they are the larger part of a short call, so
// loops over a piece's eight values stay loops there, and all kinds of rows draw in one place.
#include "lanes.h"

namespace {

constexpr int SP_THREADS = 1024, SP_MAX_V = 1 << 18;
constexpr int SP_SPANS = SP_MAX_V / 512;         // spans of 64 pieces of eight values
constexpr int SP_BINS = 36864;                   // keys that are counted at a time: all that 160 KB of LDS leave room for (from 12 down to -8 there are 37000)
typedef uint16_t ushort8_t __attribute__((ext_vector_type(8)));
typedef int16_t short8_t __attribute__((ext_vector_type(8)));

// 2^(j / 256)
constexpr int SP_POWER_COUNT = 256;
__constant__ const double SP_POWERS[SP_POWER_COUNT] = {
    1.0, 1.0027112750502025, 1.0054299011128027, 1.0081558981184175, 1.0108892860517005, 1.0136300849514894, 1.016378314910953, 1.019133996077738,
    1.0218971486541166, 1.0246677928971357, 1.0274459491187637, 1.030231637686041, 1.0330248790212284, 1.0358256936019572, 1.0386341019613787, 1.041450124688316,
    1.0442737824274138, 1.0471050958792898, 1.0499440858006872, 1.0527907730046264, 1.0556451783605572, 1.0585073227945128, 1.061377227289262, 1.0642549128844645,
    1.0671404006768237, 1.0700337118202419, 1.0729348675259756, 1.075843889062791, 1.0787607977571199, 1.0816856149932152, 1.0846183622133092, 1.0875590609177697,
    1.0905077326652577, 1.0934643990728858, 1.0964290818163769, 1.099401802630222, 1.102382583307841, 1.1053714457017412, 1.1083684117236787, 1.1113735033448175,
    1.1143867425958924, 1.1174081515673693, 1.1204377524096067, 1.12347556733302, 1.1265216186082418, 1.129575928566288, 1.1326385195987192, 1.1357094141578055,
    1.1387886347566916, 1.1418762039695616, 1.1449721444318042, 1.148076478840179, 1.1511892299529827, 1.154310420590216, 1.1574400736337511, 1.1605782120274988,
    1.1637248587775775, 1.1668800369524817, 1.1700437696832502, 1.1732160801636373, 1.1763969916502812, 1.1795865274628758, 1.182784710984341, 1.1859915656609938,
    1.189207115002721, 1.1924313825831512, 1.1956643920398273, 1.1989061670743806, 1.202156731452703, 1.2054161090051239, 1.2086843236265816, 1.2119613992768012,
    1.215247359980469, 1.2185422298274085, 1.2218460329727576, 1.2251587936371455, 1.22848053610687, 1.2318112847340759, 1.2351510639369334, 1.2384998981998165,
    1.241857812073484, 1.245224830175258, 1.2486009771892048, 1.2519862778663162, 1.255380757024691, 1.2587844395497165, 1.2621973503942507, 1.2656195145788063,
    1.2690509571917332, 1.2724917033894028, 1.275941778396392, 1.2794012075056693, 1.2828700160787783, 1.2863482295460256, 1.2898358734066657, 1.2933329732290895,
    1.2968395546510096, 1.3003556433796506, 1.3038812651919358, 1.3074164459346773, 1.3109612115247644, 1.3145155879493546, 1.318079601266064, 1.3216532776031575,
    1.3252366431597413, 1.3288297242059544, 1.3324325470831615, 1.3360451382041458, 1.339667524053303, 1.3432997311868353, 1.3469417862329458, 1.3505937158920345,
    1.3542555469368927, 1.3579273062129011, 1.3616090206382248, 1.365300717204012, 1.3690024229745905, 1.3727141650876684, 1.3764359707545302, 1.380167867260238,
    1.383909881963832, 1.387662042298529, 1.3914243757719262, 1.3951969099662003, 1.3989796725383112, 1.4027726912202048, 1.4065759938190154, 1.4103896082172707,
    1.4142135623730951, 1.4180478843204152, 1.4218926021691656, 1.4257477441054942, 1.42961333839197, 1.433489413367789, 1.4373759974489824, 1.4412731191286257,
    1.4451808069770467, 1.449099089642035, 1.4530279958490526, 1.4569675544014438, 1.460917794180647, 1.4648787441464057, 1.4688504333369818, 1.4728328908693675,
    1.4768261459394993, 1.4808302278224719, 1.4848451658727524, 1.488870989524397, 1.4929077282912648, 1.4969554117672355, 1.5010140696264256, 1.5050837316234065,
    1.5091644275934228, 1.5132561874526098, 1.5173590411982147, 1.5214730189088146, 1.5255981507445384, 1.529734466947287, 1.533881997840956, 1.5380407738316568,
    1.5422108254079407, 1.5463921831410214, 1.550584877685, 1.5547889397770887, 1.559004400237837, 1.5632312899713576, 1.567469639965553, 1.5717194812923414,
    1.5759808451078865, 1.5802537626528246, 1.5845382652524937, 1.588834384317164, 1.593142151342267, 1.597461597908627, 1.6017927556826934, 1.606135656416771,
    1.6104903319492543, 1.6148568142048607, 1.6192351351948637, 1.6236253270173289, 1.6280274218573478, 1.632441451987275, 1.6368674497669644, 1.6413054476440063,
    1.645755478153965, 1.6502175739206177, 1.6546917676561943, 1.6591780921616162, 1.6636765803267364, 1.6681872651305825, 1.6727101796415966, 1.6772453570178785,
    1.681792830507429, 1.6863526334483934, 1.6909247992693053, 1.6955093614893326, 1.7001063537185235, 1.7047158096580513, 1.709337763100463, 1.713972247929926,
    1.718619298122478, 1.723278947746274, 1.7279512309618377, 1.732636182022311, 1.7373338352737062, 1.7420442251551564, 1.746767386199169, 1.7515033530318782,
    1.7562521603732995, 1.761013843037584, 1.7657884359332727, 1.7705759740635547, 1.7753764925265212, 1.7801900265154245, 1.785016611318935, 1.789856282321401,
    1.7947090750031072, 1.7995750249405351, 1.804454167806624, 1.809346539371032, 1.8142521755003989, 1.8191711121586085, 1.8241033854070534, 1.8290490314048973,
    1.8340080864093424, 1.8389805867758937, 1.843966568958626, 1.8489660695104508, 1.8539791250833855, 1.8590057724288205, 1.864046048397789, 1.8690999899412386,
    1.8741676341103, 1.8792490180565602, 1.8843441790323345, 1.8894531543909392, 1.8945759815869656, 1.8997126981765553, 1.9048633418176741, 1.9100279502703899,
    1.9152065613971474, 1.9203992131630474, 1.925605943636125, 1.930826790987627, 1.9360617934922943, 1.9413109895286405, 1.9465744175792332, 1.9518521162309783,
    1.9571441241754002, 1.9624504802089273, 1.9677712232331759, 1.9731063922552343, 1.978456026387951, 1.9838201648502194, 1.9891988469672663, 1.9945921121709402};

// 2^(y / 256) for -256000 <= y <= 256000 as a product: the table's 2^(j / 256) with the whole part in its exponent, and the first four terms of the exponential's series
// for the rest, |rest| <= ln(2) / 512 (relative error 1.4e-13).  The nearest whole number of y stands in the low word of y + 1.5 * 2^52: conversions and
// rounding instructions of 64 bits take four times as long as sums.
struct sp_power {
    double power, p;
    __device__ __forceinline__ sp_power(const double *table, double y) {
        const double whole = y + 6755399441055744.0, r = y - (whole - 6755399441055744.0);
        const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, whole);
        p = __builtin_fma(3.3083026805413713e-09, r, 3.6655655969101062e-06);
        p = __builtin_fma(p, r, 0.0027076061740622863);
        p = __builtin_fma(p, r, 1.0);
        power = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, table[k & (SP_POWER_COUNT - 1)]) + ((uint64_t)((k << 12) & 0xfff00000u) << 32));
    }
};

// A number's key: its bits in the order of the numbers, +0 and -0 alike.  What has no weight lies outside of those that do: -inf and the NaNs with a sign at SP_NONE
// and below, the other NaNs above every largest key.
constexpr int SP_NONE = 0x3ff, SP_INFINITE = 0xfc00;       // (of +inf)
__device__ __forceinline__ ushort8_t sp_keys(half8_t v) {
    v += (half_t)0;                              // (-0 becomes +0)
    const ushort8_t bits = __builtin_bit_cast(ushort8_t, v), sign = __builtin_bit_cast(ushort8_t, __builtin_bit_cast(short8_t, v) >> 15);
    return bits ^ (sign | (uint16_t)0x8000);
}
__device__ __forceinline__ int sp_key(half_t x) {
    const half8_t v = {x, x, x, x, x, x, x, x};
    return sp_keys(v)[0];
}

// The row's values, piece p from index 8 p on, -inf behind the last one.  Rows start on any two bytes, and the hardware takes 16 bytes from there; the last piece is
// that of the last eight values, with -inf in the place of those that the one before it has.
struct sp_row {
    const half_t *x;
    int V;
    __device__ __forceinline__ sp_row(const half_t *row, int V) : x(row), V(V) {}
    __device__ __forceinline__ int first(int piece) const { return min(8 * piece, max(V - 8, 0)); }
    __device__ __forceinline__ half8_t values(int piece) const {
        half8_t v;
        const int at = first(piece), skip = 8 * piece - at;
        if (V >= 8) {
            __builtin_memcpy(&v, x + at, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = e < V ? x[e] : (half_t)-INFINITY;
        }
        if (skip > 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = e < skip ? (half_t)-INFINITY : v[e];
        }
        return v;
    }
};
__device__ __forceinline__ double sp_value(int key) {
    const uint16_t bits = key >= 0x8000 ? key - 0x8000 : (key - 0x8000) ^ 0x7fff;
    return (double)(float)__builtin_bit_cast(half_t, bits);
}

// smaller weights next to the largest are none
constexpr double SP_LEAST = 1e-300;

// from a number of the 1024 keys 1024 e .. to that of the next key
__device__ __forceinline__ double sp_step(int e) { return __builtin_ldexp(1.0, max(e >= 32 ? e - 32 : 31 - e, 1) - 25); }

// Weights next to the largest of some values.  Nothing branches: eight of them are computed side by side.
struct sp_weight {
    const double *table;
    double largest, scale;                       // scale: 256 log2(e) / T
    int top;
    // (next to +inf a finite number weighs nothing: 65536 stands for it)
    __device__ __forceinline__ sp_weight(const double *table, double factor, int top)
        : table(table), largest(top == SP_INFINITE ? 65536.0 : sp_value(top)), scale(top == SP_INFINITE ? 1e300 : factor), top(top) {}
    // of a value that is no larger: below 2^-1000 (and for -inf and NaN) 2^-1000, which no sum notices
    __device__ __forceinline__ sp_power of(double x) const { return sp_power(table, fmax((x - largest) * scale, -1000.0 * SP_POWER_COUNT)); }
    // of a key, 0 below SP_LEAST
    __device__ __forceinline__ double operator()(int key) const {
        const sp_power at = of(sp_value(key));
        const double w = at.power * at.p;
        return key == top ? 1.0 : w >= SP_LEAST ? w : 0.0;
    }
};

struct sp_args {
    const half_t *logits;
    const float *uniform, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int64_t *out;
    int64_t ld;
    int V, spans;
    double *sum;                                 // workspace, [rows, spans]
    uint2_t *largest;                            // of every 128 values of a span, four keys of 16 bits
};
// what a row has asked for
struct sp_rule {
    bool greedy, by_count, by_sum;
    int k;
    double scale, p, u;                          // u: the random number
    float least;                                 // min-p
    __device__ __forceinline__ sp_rule(const sp_args &a, int b) {
        const float T = a.temperature ? a.temperature[b] : 1.f;
        greedy = !(T > 0.f);
        scale = fmin(SP_POWER_COUNT * 1.4426950408889634074 / (double)T, 1e300);          // (finite: times 0 it is 0)
        const float random = a.uniform[b];
        u = (double)(random > 0.f ? fminf(random, 0.99999994f) : 0.f);
        k = a.top_k ? a.top_k[b] : 0;
        p = a.top_p ? (double)a.top_p[b] : 1.0;
        by_count = k > 0 && k < a.V;
        by_sum = p < 1.0;
        least = a.min_p && a.min_p[b] > 0.f ? fminf(a.min_p[b], 1.f) : 0.f;              // (the largest always stays)
    }
    __device__ __forceinline__ bool wants_sum() const { return !greedy && !by_count && (by_sum || least == 0.f); }
};
struct sp_plus {
    template <typename T>
    __device__ __forceinline__ T operator()(T a, T b) const { return a + b; }
};
struct sp_larger {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
};
template <int N>
struct sp_count {
    static constexpr int n = N;
};
// sum over the lanes up to this one
template <typename T>
__device__ __forceinline__ T sp_scan(T v) { return bs_scan(v, sp_plus()); }
template <typename T>
__device__ __forceinline__ T sp_wave_sum(T v) { return bs_read(sp_scan(v), 63); }
// sum over the lanes before this one
template <typename T>
__device__ __forceinline__ T sp_wave_before(T v) { return bs_lane_before(sp_scan(v)); }
// sum over the threads of 16 waves before this one, and the whole one; `to` is free again behind the next barrier
template <typename T>
__device__ __forceinline__ T sp_before(T v, T *to, T &total) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T s = sp_scan(v);
    if (lane == 63) to[wave] = s;
    __syncthreads();
    const T waves = bs_row_scan(to[lane & 15], sp_plus());
    total = bs_read(waves, 15);
    const T mine = bs_lane_before(s);
    return wave > 0 ? bs_read(waves, wave - 1) + mine : mine;
}
__device__ __forceinline__ uint32_t sp_wave_max(uint32_t v) { return bs_read(bs_scan(v, sp_larger()), 63); }       // (0 is the least)

constexpr int SP_SPAN_WAVES = 4;                 // spans of a workgroup of the first kernel

__global__ __launch_bounds__(SP_SPAN_WAVES * 64) void sample_spans_kernel(const sp_args a) {
    __shared__ double table[SP_POWER_COUNT];
    const int tid = threadIdx.x, lane = tid & 63, groups = (a.spans + SP_SPAN_WAVES - 1) / SP_SPAN_WAVES;
    const int b = blockIdx.x / groups, span = blockIdx.x % groups * SP_SPAN_WAVES + (tid >> 6);
    const sp_row row(a.logits + b * a.ld, a.V);
    const half8_t v = row.values(span * 64 + lane);          // (pieces behind the row: -inf)
    const double power = SP_POWERS[tid];
    static_assert(SP_POWER_COUNT == SP_SPAN_WAVES * 64, "one power per thread");
    const sp_rule rule(a, b);
    table[tid] = power;
    __syncthreads();
    float most = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; e++) most = fmaxf(most, (float)v[e]);             // (a NaN is no number's larger one)
    uint32_t quarter = (uint32_t)sp_key((half_t)most);                       // of the lanes of its row of 16 up to this one
    quarter = bs_row_scan(quarter, sp_larger());
    const uint32_t q0 = bs_read(quarter, 15), q1 = bs_read(quarter, 31), q2 = bs_read(quarter, 47), q3 = bs_read(quarter, 63);
    const int top = (int)max(max(q0, q1), max(q2, q3));
    double sum = 0.0;
    if (top > SP_NONE && rule.wants_sum()) {
        const sp_weight weight(table, rule.scale, top);
        double w[2] = {0.0, 0.0};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const sp_power at = weight.of(top == SP_INFINITE && v[e] == (half_t)INFINITY ? weight.largest : (double)(float)v[e]);
            w[e & 1] = __builtin_fma(at.power, at.p, w[e & 1]);
        }
        sum = w[0] + w[1];
        sum = sp_wave_sum(sum);
    }
    if (lane == 0 && span < a.spans) {
        a.largest[(int64_t)b * a.spans + span] = (uint2_t){q0 | q1 << 16, q2 | q3 << 16};
        a.sum[(int64_t)b * a.spans + span] = sum;
    }
}

// One wave: the lowest index of the span whose sum of kept weights up to it, and `before` in front of the span, is more than `goal`; `left` tokens with the border's key
// stay in this span, and no key below `from`.  Where the sum of the parts is a rounding short of it, the last one that is kept.
__device__ __forceinline__ int sp_draw(const sp_row &row, int span, int border, int from, const sp_weight &weight, uint32_t left, double before, double goal) {
    const int p = span * 64 + (threadIdx.x & 63), top = weight.top;
    const ushort8_t key = sp_keys(row.values(p));
    uint32_t ties = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) ties += key[e] == border;
    uint32_t seen = sp_wave_before(ties);
    double w[8], sum = 0.0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const bool tie = key[e] == border, kept = key[e] >= from && key[e] <= top && (key[e] > border || (tie && border > SP_NONE && seen < left));
        w[e] = kept ? weight(key[e]) : 0.0;
        seen += tie;
        sum += w[e];
    }
    double at = before + sp_wave_before(sum);
    int found = -1, last = -1;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        at += w[e];
        last = w[e] > 0.0 ? e : last;
        found = found < 0 && w[e] > 0.0 && at > goal ? e : found;
    }
    // (lanes hold their indexes in order)
    const uint64_t reach = __ballot(found >= 0), any = __ballot(last >= 0);
    const int l = reach ? __ffsll((unsigned long long)reach) - 1 : any ? 63 - __clzll((long long)any) : 0;
    return max(row.first(span * 64 + l) + __builtin_amdgcn_readlane(reach ? found : last, l), 0);
}

// The key of a number, or one to three below it (one is that of no number, between -0 and the largest number below); the lowest for what is below all numbers.
__device__ __forceinline__ int sp_key_below(float x) { return x > -65000.f ? max(SP_NONE + 1, sp_key((half_t)fminf(x, 65000.f)) - 3) : SP_NONE + 1; }

constexpr int SP_WAVES = SP_THREADS / 64, SP_LIST = SP_THREADS;      // (a token of the list per thread)

__global__ __launch_bounds__(SP_THREADS) void sample_rows_kernel(const sp_args a) {
    // tokens per key, from the highest key of the window down; then [wave][SP_LIST] keys and indexes
    extern __shared__ __attribute__((aligned(16))) uint32_t bins[];
    static_assert(SP_BINS >= 2 * SP_WAVES * SP_LIST && SP_BINS <= 64 * 4096 && SP_SPANS <= SP_THREADS && SP_SPANS <= 64 * SP_WAVES, "both fit; a span per thread; a wave's spans one per lane");
    __shared__ double table[SP_POWER_COUNT], part[SP_WAVES], chunk_sum[64], span_kept[SP_SPANS], span_before;
    __shared__ uint32_t part32[SP_WAVES], chunk_count[64], span_ties[SP_SPANS], span_left, wave_count[SP_WAVES], listed;
    __shared__ int keys[SP_SPANS], floor_key, at_first, at_last;
    __shared__ uint2_t quarter_keys[SP_SPANS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), b = blockIdx.x;
    const sp_row row(a.logits + b * a.ld, a.V);
    const uint2_t quarters = tid < a.spans ? a.largest[(int64_t)b * a.spans + tid] : (uint2_t)0u;        // (0: below all keys)
    const int mine = (int)max(max(quarters[0] & 0xffff, quarters[0] >> 16), max(quarters[1] & 0xffff, quarters[1] >> 16));
    const double my_sum = tid < a.spans ? a.sum[(int64_t)b * a.spans + tid] : 0.0;
    const double power = SP_POWERS[tid & (SP_POWER_COUNT - 1)];
    sp_rule rule(a, b);
    if (tid < a.spans) {
        keys[tid] = mine;
        quarter_keys[tid] = quarters;
    }
    if (tid < SP_POWER_COUNT) table[tid] = power;
    const uint32_t of_wave = sp_wave_max((uint32_t)mine);
    if (lane == 0) part32[wave] = of_wave;
    if (tid == 0) {
        floor_key = SP_NONE + 1;
        at_first = 0x7fffffff;
        at_last = -1;
    }
    __syncthreads();
    const int top = (int)sp_wave_max(part32[lane & 15]);
    __syncthreads();
    if (top <= SP_NONE) {                        // nothing but -inf and NaN
        if (tid == 0) a.out[b] = 0;
        return;
    }
    const sp_weight weight(table, rule.scale, top);
    // The wave's spans, one after another in the order of the row, that reach a key: f(span, values), the next one's values on their way.
    auto each_span = [&](int first, int end, int from, auto f) {
        const int per_wave = (end - first + SP_WAVES - 1) / SP_WAVES, span0 = first + wave * per_wave, at = span0 + lane;
        uint64_t left = __ballot(lane < per_wave && at < end && keys[min(at, a.spans - 1)] >= from);
        if (!left) return;
        int s = span0 + __ffsll((unsigned long long)left) - 1;
        half8_t v = row.values(s * 64 + lane);
#pragma unroll 1
        while (left) {
            const int now = s;
            left &= left - 1;
            if (left) s = span0 + __ffsll((unsigned long long)left) - 1;
            const half8_t ahead = row.values(s * 64 + lane);
            f(now, v);
            v = ahead;
        }
    };
    // the key of the value next to which others weigh w or more (or a little below it)
    auto key_of = [&](float log2_w) { return min(top, sp_key_below((float)weight.largest + (log2_w * 1.0001f - 0.0001f) * (float)(SP_POWER_COUNT / weight.scale))); };
    // the lowest key that weighs w or more
    auto key_from = [&](double w, float log2_w) {
        if (top == SP_INFINITE) return top;
        int key = key_of(log2_w);
        for (;;) {                               // (the first of 64 is it nearly always; the largest weighs 1)
            const uint64_t enough = __ballot(key + lane <= top && weight(key + lane) >= w);
            key += enough ? __ffsll((unsigned long long)enough) - 1 : 64;
            if (enough || key > top) return key;
        }
    };

    int border = SP_NONE;                        // the border's key (none), and how many tokens with that key stay
    uint32_t stay = 0;
    double kept = 0.0;                           // of this thread's span: the kept weights, but those of the border's key; its tokens
    uint32_t ties = 0;
    // The first of the threads whose part of a running sum reaches beyond the goal (sums are compared in one way only: a rounding leaves no gap), or the last one with a part.
    auto first_beyond = [&](double part, double before, double goal) {
        const uint64_t reach = __ballot(part > 0.0 && before + part > goal), any = __ballot(part > 0.0);
        if (reach && lane == __ffsll((unsigned long long)reach) - 1) atomicMin(&at_first, tid);
        if (any && lane == 63 - __clzll((long long)any)) atomicMax(&at_last, tid);
        __syncthreads();
        return at_first != 0x7fffffff ? at_first : max(at_last, 0);
    };
    bool sums_are_there = rule.greedy;
    if (rule.greedy) {                           // the first token with the largest key
        border = top;
        stay = 1;
        ties = mine == top;
        rule.u = 0.0;
    } else if (rule.wants_sum()) {
        kept = mine > SP_NONE ? my_sum * weight(mine) : 0.0;
        sums_are_there = !rule.by_sum;
    }
    // A small k is found in a list of the values from the k-th largest of some disjoint parts' largest on: the quarters of the spans, or, in short rows, what a thread reads.  At least
    // twice as many parts as k: then about 0.7 values per part are in the list.  (us, so / with as many parts as k, and counting where they are fewer: 11 rows of 3693, k to 100 with top-p, 15.1 / 33.0; 49 of 10338
    // 16.8 / 38.7; 49 of 3000, k alone, 14.8 / 20.9; 48 of 32000 with top-p 16.1 both.)
    const int pieces = (a.V + 7) / 8;
    const bool quarters_do = rule.k <= 2 * a.spans, few = rule.by_count && (quarters_do || rule.k <= min(256, min(pieces, SP_THREADS) / 2));
    uint32_t counted = 0, border_ties = 0;       // tokens down to the border and with its key, and the weights that stay, where they have been counted
    double counted_sum = 0.0;
    int from = SP_NONE + 1, first = 0, end = a.spans;          // no key below it is kept; the spans that are summed
    if (!sums_are_there) {
        // the lowest key that min-p leaves
        const int least = rule.least > 0.f ? key_from((double)rule.least, log2f(rule.least)) : top == SP_INFINITE ? top : SP_NONE + 1;
        if (few) {                               // the k-th largest of the largest keys of every 128 values, of the spans, or of the threads, bit by bit
            uint16_t *const thread_key = reinterpret_cast<uint16_t *>(bins);
            if (!quarters_do) {
                float most = -INFINITY;
#pragma unroll 1
                for (int i = tid; i < pieces; i += SP_THREADS) {
                    const half8_t v = row.values(i);
#pragma unroll
                    for (int e = 0; e < 8; e++) most = fmaxf(most, (float)v[e]);             // (a NaN is no number's larger one)
                }
                thread_key[tid] = (uint16_t)sp_key((half_t)most);
                __syncthreads();
            }
            if (wave == 0) {
                const uint16_t *all = reinterpret_cast<const uint16_t *>(quarter_keys);
                int kth = 0;
                auto search = [&](auto each, auto key_at) {              // (64 * each keys; 0 behind the last)
                    int key[each.n];
#pragma unroll
                    for (int j = 0; j < each.n; j++) key[j] = key_at(j * 64 + lane);
#pragma unroll 1
                    for (int bit = 0x8000; bit; bit >>= 1) {
                        int n = 0;
#pragma unroll
                        for (int j = 0; j < each.n; j++) n += __popcll(__ballot(key[j] >= (kth | bit)));
                        kth = n >= rule.k ? kth | bit : kth;
                    }
                };
                auto quarter_at = [&](int i) { return i < 4 * a.spans ? (int)all[i] : 0; };
                if (!quarters_do) search(sp_count<SP_WAVES>(), [&](int i) { return (int)thread_key[i]; });
                else if (4 * a.spans <= 256) search(sp_count<4>(), quarter_at);
                else if (2 * rule.k <= a.spans) search(sp_count<SP_SPANS / 64>(), [&](int i) { return i < a.spans ? keys[i] : 0; });
                else search(sp_count<4 * SP_SPANS / 64>(), quarter_at);
                floor_key = max(SP_NONE + 1, kth);
            }
            __syncthreads();
            from = floor_key;
        }
        // (what min-p drops still counts in the sum of which top-p is a part)
        if (!few || !rule.by_sum) from = max(from, least);

        // ---- the border of top-k and top-p by counting, where no list can be made: top-p leaves no bound on the tokens, nor does a large k
        auto count = [&]() {
            // no border is below the key at which all tokens together would have less than top-p leaves
            double total = 0.0;
            if (!rule.by_count) sp_before(kept, part, total);
            const int lowest = top == SP_INFINITE ? top : few ? floor_key : !rule.by_count ? key_of(log2f((float)((1.0 - rule.p) * total / a.V))) : SP_NONE + 1;
            int held = 0;                        // highest key of the window that the bins hold
            double limit = total, at_sum = 0.0;  // the sum that top-k leaves; up to what was found,
            int at_key = 0;                      // the key that was,
            uint32_t at_stay = 0, at_count = 0, at_ties = 0;     // how many tokens with it stay, how many there are down to it and with it
            // Twice: the first key at which the count reaches k, and the one at which the sum reaches the goal.  Every wave looks for them by itself.
#pragma unroll 1
            for (int turn = rule.by_count ? 0 : 1; turn < (rule.by_sum ? 2 : 1); turn++) {
                const bool by_count = turn == 0;
                const double goal = fmax(rule.p * limit, 1e-300);       // (the largest always stays)
                const uint32_t k = (uint32_t)rule.k;
                uint32_t seen = 0;
                double sum = 0.0;
                bool found = false;
#pragma unroll 1
                for (int hi = top; hi >= lowest && !found; hi -= SP_BINS) {
                    // up to 64 chunks of 64 keys or a multiple of that
                    const int lo = max(hi - SP_BINS + 1, lowest), n_bins = hi - lo + 1, chunk = (n_bins + 4095) / 4096 * 64, chunks = (n_bins + chunk - 1) / chunk;
                    if (held != hi) {
                        __syncthreads();         // (the last window's bins are read no more)
                        for (int i = tid; i < chunks * (chunk / 4); i += SP_THREADS) reinterpret_cast<uint4_t *>(bins)[i] = (uint4_t)0u;
                        __syncthreads();
                        each_span(0, a.spans, lo, [&](int, const half8_t v) {
                            const ushort8_t down = (uint16_t)hi - sp_keys(v);
#pragma unroll
                            for (int e = 0; e < 8; e++)
                                if (down[e] <= hi - lo) atomicAdd(&bins[down[e]], 1u);
                        });
                        __syncthreads();
                        // the chunks' counts and sums
#pragma unroll 1
                        for (int c = wave; c < chunks; c += SP_WAVES) {
                            uint32_t all = 0;
                            double w = 0.0;
#pragma unroll 1
                            for (int i = c * chunk + lane; i < (c + 1) * chunk; i += 64) {
                                const uint32_t in = bins[i];
                                all += in;
                                if (rule.by_sum && __any(in != 0)) w += in ? (double)in * weight(hi - i) : 0.0;
                            }
                            all = sp_wave_sum(all);
                            w = sp_wave_sum(w);
                            if (lane == 0) {
                                chunk_count[c] = all;
                                chunk_sum[c] = w;
                            }
                        }
                        __syncthreads();
                        held = hi;
                    }
                    const uint32_t n = lane < chunks ? chunk_count[lane] : 0, n_upto = sp_scan(n);
                    const double w = lane < chunks ? chunk_sum[lane] : 0.0, w_upto = sp_scan(w);
                    const uint64_t who = __ballot(n && (by_count ? seen + n_upto >= k : sum + w_upto >= goal));
                    const int c = who ? __ffsll((unsigned long long)who) - 1 : 64;
                    if (c > 0) {
                        seen += bs_read(n_upto, c - 1);
                        sum += bs_read(w_upto, c - 1);
                    }
                    found = who != 0;
                    if (!found) continue;
                    // the key within the chunk; a rounding short of the goal, the last one
#pragma unroll 1
                    for (int i = c * chunk + lane; i < (c + 1) * chunk; i += 64) {
                        const uint32_t in = bins[i];
                        const uint64_t any = __ballot(in != 0);
                        if (!any) continue;
                        const double each = rule.by_sum && in ? weight(hi - i) : 0.0;
                        const uint32_t upto = seen + sp_scan(in);
                        const double up = sum + sp_scan((double)in * each);
                        const uint64_t reach = __ballot(in && (by_count ? upto >= k : up >= goal));
                        const int l = reach ? __ffsll((unsigned long long)reach) - 1 : 63 - __clzll((long long)any);
                        const double in_front = up - (double)in * each, need = by_count ? (double)(k - (upto - in)) : ceil((goal - in_front) / each);
                        const uint32_t take = need < 1.0 ? 1 : need < (double)in ? (uint32_t)need : in;
                        at_key = __builtin_amdgcn_readlane(hi - i, l);
                        at_stay = bs_read(take, l);
                        at_count = bs_read(upto, l);
                        at_ties = bs_read(in, l);
                        at_sum = bs_read(in_front + (double)take * each, l);
                        if (reach) break;
                        seen = bs_read(upto, 63);
                        sum = bs_read(up, 63);
                    }
                }
                if (found && at_key >= border) {
                    stay = border > SP_NONE && at_key == border ? min(stay, at_stay) : at_stay;
                    border = at_key;
                    counted = at_count;
                    border_ties = at_ties;
                    counted_sum = at_sum;
                }
                limit = found ? at_sum : sum;    // (fewer than k: all stay)
            }
            from = max(max(from, border), least);
        };
        bool ranked = few;                       // whether the list is yet to be cut by top-k and top-p
        bool counting = (rule.by_count || rule.by_sum) && !few;

        // ---- the tokens that are left as a list, in the order of the row; twice at most (a list by the spans' largest keys that is too long)
        uint32_t n = 0, n_before = 0;
#pragma unroll 1
        for (;;) {
            if (counting) count();
            if (counted > SP_LIST) break;
            if (tid == 0) listed = 0;
            __syncthreads();                     // (the bins are read no more)
            uint32_t *const k_list = bins + wave * SP_LIST, *const i_list = bins + (SP_WAVES + wave) * SP_LIST;
            uint32_t have = 0;
            bool full = false;                   // (too many: then nobody goes on)
            each_span(0, a.spans, from, [&](int s, const half8_t v) {
                if (full) return;
                const ushort8_t key = sp_keys(v);
                uint32_t in = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) in += key[e] >= from && key[e] <= top;
                const uint32_t upto = sp_scan(in);
                uint32_t at = have + upto - in;
                if (in) {
                    const int first = row.first(s * 64 + lane);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (key[e] >= from && key[e] <= top) {
                            if (at < SP_LIST) {
                                k_list[at] = key[e];
                                i_list[at] = (uint32_t)(first + e);
                            }
                            at++;
                        }
                }
                const uint32_t more = bs_read(upto, 63);
                uint32_t all = 0;
                if (lane == 0) all = atomicAdd(&listed, more) + more;
                full = bs_read(all, 0) > SP_LIST;
                have += more;
            });
            if (lane == 0) wave_count[wave] = have;
            __syncthreads();
            const uint32_t upto = bs_row_scan(wave_count[lane & 15], sp_plus());
            n = listed;
            // thread t's token: the wave whose part of the list it lies in
            int of = 0;
            n_before = 0;
#pragma unroll
            for (int w = 0; w < SP_WAVES - 1; w++) {
                const uint32_t end = bs_read(upto, w);
                if ((uint32_t)tid >= end) {
                    of = w + 1;
                    n_before = end;
                }
            }
            if (n <= SP_LIST) {
                const bool in = (uint32_t)tid < n;
                const int key = in ? (int)bins[of * SP_LIST + tid - n_before] : 0, index = in ? (int)bins[(SP_WAVES + of) * SP_LIST + tid - n_before] : 0;
                const double w = in ? weight(key) : 0.0;
                bool stays = in;
                if (ranked) {                    // how many are ahead of it, and their sum: 1 to 16 threads per token, each takes a part of the others
                    double *const sums = reinterpret_cast<double *>(bins), *const list_w = sums + 2 * SP_LIST;
                    uint32_t *const ranks = bins + 2 * SP_LIST;
                    uint16_t *const list_key = reinterpret_cast<uint16_t *>(bins + 6 * SP_LIST);
                    __syncthreads();             // (the waves' lists are read no more)
                    list_w[tid] = w;
                    list_key[tid] = (uint16_t)key;
                    const int groups = n <= 64 ? 16 : n <= 128 ? 8 : n <= 256 ? 4 : n <= 512 ? 2 : 1, width = SP_LIST / groups, g = tid / width, i = tid % width;
                    const int each = ((int)n + groups - 1) / groups, j1 = min((g + 1) * each, (int)n);
                    __syncthreads();
                    const int my_key = list_key[i];
                    uint32_t rank = 0;
                    double sum = 0.0;
#pragma unroll 4
                    for (int j = g * each; j < j1; j++) {
                        const int other = list_key[j];
                        const bool ahead = other > my_key || (other == my_key && j < i);
                        rank += ahead;
                        sum += ahead ? list_w[j] : 0.0;
                    }
                    sums[tid] = sum;
                    ranks[tid] = rank;
                    __syncthreads();
                    rank = 0;
                    sum = 0.0;
                    if (in)
                        for (int q = 0; q < groups; q++) {
                            rank += ranks[q * width + tid];
                            sum += sums[q * width + tid];
                        }
                    stays = in && rank < (uint32_t)rule.k;
                    if (rule.by_sum) {
                        double limit;
                        sp_before(stays ? w : 0.0, part, limit);
                        stays = stays && (rank == 0 || sum < rule.p * limit);
                        __syncthreads();
                    }
                } else if (border > SP_NONE) {
                    uint32_t all;
                    const uint32_t before = sp_before((uint32_t)(key == border), part32, all);
                    stays = in && (key > border || before < stay);
                }
                const double mine = stays && key >= least ? w : 0.0;
                double total;
                const double before = sp_before(mine, part, total);
                if (tid == first_beyond(mine, before, rule.u * total)) a.out[b] = index;
                return;
            }
            if (!ranked) break;
            ranked = false;
            counting = true;
        }

        // ---- too many for a list: the spans' kept sums.  Where their total is known from the counting, the spans up to the one in which the random number will fall do, or those
        // from there on, if these are fewer: all of a span's weights (known) grow along the row nearly as the kept ones do.
        if (rule.by_sum && !rule.by_count && border > SP_NONE && least <= border) {
            double total;
            const double before = sp_before(kept, part, total);
            const int s = first_beyond(kept, before, rule.u * total), margin = a.spans / 16 + 2;
            if (2 * s < a.spans) end = min(a.spans, s + margin);
            else first = max(0, s - margin);
        }
    }
    // A weight of a token of these spans is a product of two from tables: of the lowest of the 32 keys next to its own, and of the steps above that, which are the same for
    // the 1024 keys next to it (one of 128256 values of which 0.95 of the sum stay: 16 us with the tables instead of 20, of 44; a row whose 2000 largest stay 28 instead of 34).
    // Where such steps are too large for that the weights are made one by one.
    double *const base = reinterpret_cast<double *>(bins), *const above = base + 2048;
    if (!sums_are_there && rule.least == 0.f) from = max(from, key_from(SP_LEAST, -996.6f));       // (the first token that weighs something may be the one)
    const bool by_products = top != SP_INFINITE && 31.0 * fmax(sp_step(top >> 10), sp_step(from >> 10)) * weight.scale < 500.0 * SP_POWER_COUNT;
    if (!sums_are_there && by_products) {
        __syncthreads();                         // (the bins and lists are read no more)
        for (int i = tid; i < 2048; i += SP_THREADS) {
            // (0 where no key has a weight; keys that are beyond the largest are not looked up)
            const bool in = i >= from >> 5 && i <= top >> 5, steps = i >> 5 >= from >> 10 && i >> 5 <= top >> 10;
            const sp_power at = weight.of(in ? sp_value(32 * i) : weight.largest), on(table, steps ? (double)(i & 31) * sp_step(i >> 5) * weight.scale : 0.0);
            base[i] = in ? at.power * at.p : 0.0;
            above[i] = on.power * on.p;
        }
    }
#pragma unroll 1
    for (;;) {
        const bool whole = first == 0 && end == a.spans;
        if (!sums_are_there) {
            __syncthreads();
            if (tid < a.spans) {
                span_kept[tid] = 0.0;
                span_ties[tid] = 0;
            }
            if (tid == 0) {
                at_first = 0x7fffffff;
                at_last = -1;
            }
            __syncthreads();
            each_span(first, end, from, [&](int s, const half8_t v) {
                const ushort8_t key = sp_keys(v);
                double w[2] = {0.0, 0.0};
                uint32_t n = 0;
                if (by_products) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int k = key[e] > border && key[e] >= from && key[e] <= top ? key[e] : 0, group = k >> 5;       // (base[0] is 0)
                        w[e & 1] = __builtin_fma(base[group], above[(group & ~31) | (k & 31)], w[e & 1]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) w[e & 1] += key[e] > border && key[e] >= from && key[e] <= top ? weight(key[e]) : 0.0;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) n += key[e] == border;
                double sum = w[0] + w[1];
                sum = sp_wave_sum(sum);
                n = sp_wave_sum(n);
                if (lane == 0) {
                    span_kept[s] = sum;
                    span_ties[s] = border > SP_NONE ? n : 0;
                }
            });
            __syncthreads();
            kept = tid < a.spans ? span_kept[tid] : 0.0;
            ties = tid < a.spans ? span_ties[tid] : 0;
        }
        // ---- the draw from the spans' sums: ties that stay are those of the first spans
        uint32_t ties_before = 0;
        if (border > SP_NONE) {
            uint32_t all;
            ties_before = sp_before(ties, part32, all);
            if (first > 0) ties_before += border_ties - all;
            kept += (double)(ties_before < stay ? min(ties, stay - ties_before) : 0) * (border >= from ? weight(border) : 0.0);
        }
        double total, before = sp_before(kept, part, total);
        if (!whole) {
            if (first > 0) before += counted_sum - total;
            total = counted_sum;
        }
        const double goal = rule.u * total;
        const int s = first_beyond(tid >= first && tid < end ? kept : 0.0, before, goal);
        if (tid == s) {
            span_before = before;
            span_left = ties_before < stay ? stay - ties_before : 0;
        }
        const bool reached = at_first != 0x7fffffff;
        __syncthreads();
        // (not in the spans that were summed, or in front of the first of them that has a kept token: then all)
        if (!whole && (!reached || (first > 0 && span_before > goal))) {
            first = 0;
            end = a.spans;
            continue;
        }
        if (wave == 0) {
            const int at = sp_draw(row, s, border, from, weight, span_left, span_before, goal);
            if (tid == 0) a.out[b] = at;
        }
        return;
    }
}

int sp_spans_of(int V) { return (V + 511) / 512; }

}  // namespace

int64_t bs_sample_scratch(int B, int V) { return (int64_t)B * sp_spans_of(V) * 16; }

int bs_launch_sample(const half_t *logits, int64_t ld, const float *uniform, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                     int64_t *out, int B, int V, void *workspace, hipStream_t s) {
    const int spans = sp_spans_of(V);
    const int64_t groups = bs_cdiv(spans, SP_SPAN_WAVES), all = (int64_t)B * spans;
    if (V > SP_MAX_V || groups * B > INT32_MAX) return BS_ERR_SHAPE;
    const sp_args a = {logits, uniform, temperature, top_p, min_p, top_k, out, ld, V, spans, (double *)workspace, (uint2_t *)((char *)workspace + all * 8)};
    static bs_lds_grant granted[BS_MAX_DEVICES];
    const int st = bs_allow_lds((const void *)sample_rows_kernel, SP_BINS * 4, granted);
    if (st != BS_OK) return st;
    sample_spans_kernel<<<(unsigned)(groups * B), SP_SPAN_WAVES * 64, 0, s>>>(a);
    BS_LAUNCH_CHECK();
    sample_rows_kernel<<<B, SP_THREADS, SP_BINS * 4, s>>>(a);
    BS_LAUNCH_CHECK();
    return BS_OK;
}
