// The next token of every row of logits, from given random numbers.
//
// With x the row, top its maximum and t the temperature, a token's weight is w = exp((x - top) / t).  Tokens in falling order of
// x, equal ones in rising order of index:
//   top-k   keeps the first k
//   top-p   of what is left, keeps the token while the weights before it sum to less than p times all that are left
//   min-p   keeps w >= min_p
// and the draw is in the vocabulary's order: the first kept token with (kept weights up to it) > u * (all kept weights).
// t <= 0 is the largest logit, the lowest index among equals.  Every filter keeps a prefix of the order, so a filter is one
// 64-bit number: the last kept token's (ordered logit, complement of the index), compared with every token's.
//
// Weights are whole numbers, 2^42 w rounded, from a 64-bit exponential: sums of up to 2^20 of them are exact in 64 bits, so the
// result depends neither on the order in which threads add nor on how the row is shared out, and a border between two
// tokens is off by 2^-42 of the largest weight (sums in f32 would be off by 2^-24, and with a vocabulary of 10^5 borders one row in
// some hundred would draw the neighbour).
//
// A CTA takes a row, or a cluster of them, a contiguous slice each (kept in shared memory where it fits).  The first one leads:
// it looks at what a pass over the row found, and says what the next pass is for:
//   the largest logit;
//   with top-k, a histogram over 1024 equal steps of (top - x) / t and the rest behind them, of the threads' own largest logits alone:
//   there are k tokens at least down to the step in which the k-th of those lies; then the tokens up to that step: where they are
//   few (2048), they are sorted, or counted out, and all filters and the draw are done among them;
//   with top-p alone, a histogram of rough weights, which says where the border is thought to be; then all weights once, those
//   above that place and those behind it, and the tokens around it (some dozens), among which the exact border is found;
//   where there are too many tokens, or the border is not where it was thought to be: a histogram of the tokens, or of their exact
//   weights, the tokens of the step that the filter ends in (split further by the next bits of their 64-bit order while they
//   are too many), which give the exact end;
//   the kept weights of every warp's stretch of the row, and the stretch that the draw falls into.
// Bound: the latency of the passes for few rows; for many, the instructions of the weights, the histogram's additions in shared
// memory and the reads.  Measured, all in us: one row of 32000 f32, all filters, 21 to 26; 24 rows of 50000 bf16 35; 64 rows of 128001
// f32, top-p, 75 (105 with the exact weights put into the histogram, which took two passes over them); no filter 48.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"

namespace xn {
namespace {
namespace cg = cooperative_groups;

typedef unsigned long long u64;
constexpr int SM_NT = 512, SM_WARPS = SM_NT / 32;  // as many registers a thread as the passes want: spilled ones would go to L2, see walk
constexpr int PER = 2, BINS = PER * SM_NT;  // steps of a histogram, a thread's of those; what is behind the last counts as one more
constexpr int EACH = 4, LIST = EACH * SM_NT;  // tokens that are sorted, and of those a thread's
constexpr int HANDFUL = 192;
constexpr int MAX_CLUSTER = 8;
constexpr float STEPS = 64.0f;          // histogram steps per unit of (top - x) / t
constexpr float MOST = 3.4028234663852886e38f;
constexpr int INDEX_BITS = 20;
constexpr double ONE = 4398046511104.0; // 2^42
constexpr int ROOTS = 64;
__constant__ double ROOT[ROOTS] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};

struct SampleArgs {
    const void *logits;
    size_t row_stride;
    int vocab;
    const float *uniform, *temperature, *top_p, *min_p;
    const int *top_k;
    int64_t *tokens;
};

enum Op { OP_TOPS, OP_STEPS, OP_BITS, OP_GATHER, OP_GUESS, OP_SPLIT, OP_SUMS, OP_PICK, OP_LEAVE };
struct Command {
    int op;
    int upto, step;      // OP_GATHER: tokens of the steps up to `upto`, and of `step`; OP_BITS: of `step`; OP_SUMS, OP_PICK: up to `upto`
    int base;            // OP_STEPS: the step that the histogram begins at
    int shift;           // OP_BITS, OP_GATHER: tokens whose place agrees with `prefix` above this bit
    int weights;         // a histogram of weights, not of tokens; OP_GATHER: the weights before `step` as OP_SUMS
    int warp;            // OP_PICK: stretch of the row
    u64 prefix, cut;     // tokens behind `cut` in the order do not count
    u64 target;          // OP_PICK: where in the stretch
    float floor;         // logits below need not be looked at
    float lo, hi;        // OP_SPLIT: in steps, where the top-p border is thought to lie
};

// A row as 16-byte groups, and a stretch of it, whose first groups are in shared memory too, as many as each warp has room for: a warp
// without any would be late for the others.
struct View {
    const void *row;             // its first logit
    int lead, vocab;             // logits of the first group that lie before the row, and of the row
    int cache_begin, cache_end;  // groups up to cache_end lie in cache()[g - cache_begin]
};
struct Row {
    float top;
    float pre, steps;  // (top - x) / t in steps: (top - x) * pre * steps; pre is 1, or for the smallest t what keeps steps finite
    double rate;       // (x - top) / t in 64ths of an octave: (x - top) * rate
    u64 least;         // weights below it do not stay (the largest always does)
};
struct Shared {
    Command cmd;
    Row row;
    u64 list[LIST], taken[LIST];     // the leader's, and what this CTA found
    unsigned low[2 * BINS];          // per step: tokens, or their weights as two words, the second ones BINS further on
    double root[ROOTS];              // 2^(42 + i / 64)
    u64 seg[MAX_CLUSTER * SM_WARPS];
    u64 scan[SM_WARPS];
    u64 best[MAX_CLUSTER];
    u64 far;                         // behind the histogram; OP_SPLIT: from `lo` on
    u64 ahead;                       // OP_SPLIT: above
    float lo, hi;
    bool few;
    unsigned listed, found, place;
    u64 found_q;
    int found_bin;
};


// A token's place in the falling order: its logit's bits, ordered, and the complement of its index.
__device__ __forceinline__ unsigned order_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);  // -0 as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ u64 place_of(float x, int index) {
    return (u64)order_of(x) << INDEX_BITS | (unsigned)(((1 << INDEX_BITS) - 1) - index);
}
__device__ __forceinline__ int index_of(u64 place) { return ((1 << INDEX_BITS) - 1) - (int)(place & ((1 << INDEX_BITS) - 1)); }
__device__ __forceinline__ float logit_of(u64 place) { return value_of((unsigned)(place >> INDEX_BITS)); }
constexpr int PLACE_BITS = 32 + INDEX_BITS;

struct Weigher : Row {
    const double *root;
    __device__ __forceinline__ Weigher(const Row &row, const double *root) : Row(row), root(root) {}
    __device__ __forceinline__ Weigher(const Shared &s) : Weigher(s.row, s.root) {}
    __device__ __forceinline__ float below(float x) const { return (top - x) * pre; }
    __device__ __forceinline__ int step(float x) const { return min(__float2int_rz(below(x) * steps), 2 * BINS); }  // beyond 32 t all is one
    // 2^42 exp((x - top) / t), rounded, where it is 2^-4 at least (2 BINS steps): 2^(42 + i / 64) from a table, the rest (less than a 128th
    // of an octave, y its logarithm) as 1 + y + y^2 / 2 + y^3 / 6 + y^4 / 24, off by y^5 / 120 = 4e-14.
    __device__ __forceinline__ u64 near_weight(float x) const {
        constexpr double C = 0.010830424696249145;  // ln 2 / 64
        constexpr double WHOLE = 6755399441055744.0, INT = 4503599627370496.0;  // 1.5 * 2^52, 2^52: a sum with them is rounded
        const double d = ((double)x - (double)top) * rate;
        const double k = d + WHOLE, y = d - (k - WHOLE);
        const int n = __double2loint(k);
        double p = fma(y, C * C * C * C / 24.0, C * C * C / 6.0);
        p = fma(p, y, C * C / 2.0);
        p = fma(p, y, C);
        p = fma(p, y, 1.0);
        p *= root[n & (ROOTS - 1)];
        p = __hiloint2double(__double2hiint(p) + (n & -ROOTS) * ((1 << 20) / ROOTS), __double2loint(p));
        return (u64)__double_as_longlong(p + INT) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ bool weighs(float y) const { return y < 2 * BINS; }  // y: (top - x) / t in steps; beyond, 0
    __device__ __forceinline__ u64 weight(float x) const { return weighs(below(x) * steps) ? near_weight(x) : 0; }
};

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// The values of the threads before this one, and of all.
__device__ __noinline__ ulonglong2 block_scan(Shared &s, u64 x) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    u64 inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) s.scan[warp] = inc;
    __syncthreads();
    u64 w = lane < SM_WARPS ? s.scan[lane] : 0;
#pragma unroll
    for (int o = 1; o < SM_WARPS; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    const u64 sum = __shfl_sync(0xffffffffu, w, SM_WARPS - 1), before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return make_ulonglong2((warp ? before : 0) + inc - x, sum);
}
// Sorts the first `count` values of the list, all different, in falling order.
__device__ __noinline__ void sort_list(Shared &s, int count) {
    const int tid = threadIdx.x;
    if (count <= SM_NT) {
        // One or two threads a value: how many are larger is its place.  The time goes with the square of their number; two sorts of 200 to
        // 250 values take 4 us less than by the steps below.
        const int parts = count <= SM_NT / 2 ? 2 : 1, i = tid / parts;
        if (tid == 0) s.list[count] = 0;  // two at a time are looked at
        __syncthreads();
        const u64 x = i < count ? s.list[i] : 0;
        int place = 0;
#pragma unroll 4
        for (int j = 2 * (tid % parts); j < count; j += 2 * parts) {
            place += (s.list[j] > x) + (s.list[j + 1] > x);
        }
        if (parts == 2) place += __shfl_xor_sync(0xffffffffu, place, 1);
        __syncthreads();
        if (i < count && tid % parts == 0) s.list[place] = x;
        __syncthreads();
        return;
    }
    // Value e of thread tid is the EACH * tid + e-th.  Exchanges within a thread, within a warp by shuffles, and beyond through `taken`;
    // only the warps that hold any take part.
    int size = 32 * EACH;
    while (size < count) size <<= 1;
    __syncthreads();
    if (tid < size / EACH) {
        u64 x[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) x[e] = EACH * tid + e < count ? s.list[EACH * tid + e] : 0;
#pragma unroll 1
        for (int run = 2; run <= size; run <<= 1)
#pragma unroll 1
            for (int d = run >> 1; d; d >>= 1) {
                u64 y[EACH];
                if (d >= 32 * EACH) {
                    asm volatile("bar.sync 1, %0;" ::"r"(size / EACH) : "memory");
#pragma unroll
                    for (int e = 0; e < EACH; ++e) s.taken[e * SM_NT + tid] = x[e];
                    asm volatile("bar.sync 1, %0;" ::"r"(size / EACH) : "memory");
#pragma unroll
                    for (int e = 0; e < EACH; ++e) y[e] = s.taken[e * SM_NT + (tid ^ (d / EACH))];
                } else if (d >= EACH) {
#pragma unroll
                    for (int e = 0; e < EACH; ++e) y[e] = __shfl_xor_sync(0xffffffffu, x[e], d / EACH);
                } else {
#pragma unroll
                    for (int e = 0; e < EACH; ++e) y[e] = d == 1 ? x[e ^ 1] : x[e ^ 2];
                }
#pragma unroll
                for (int e = 0; e < EACH; ++e) {
                    const int at = EACH * tid + e;
                    const bool falling = (at & run) == 0, lower = (at & d) == 0;
                    x[e] = (falling == lower) == (x[e] > y[e]) ? x[e] : y[e];
                }
            }
#pragma unroll
        for (int e = 0; e < EACH; ++e) s.list[EACH * tid + e] = x[e];
    }
    __syncthreads();
}

__device__ __forceinline__ Shared &shared() {
    extern __shared__ __align__(16) unsigned char raw[];
    return *reinterpret_cast<Shared *>(raw);
}
__device__ __forceinline__ uint4 *cache() {
    extern __shared__ __align__(16) unsigned char raw[];
    return reinterpret_cast<uint4 *>(raw + (sizeof(Shared) + 15) / 16 * 16);
}
__device__ __forceinline__ Shared &leader() { return *cg::this_cluster().map_shared_rank(&shared(), 0); }

// A group's logits, -inf outside the row.
template <typename T> __device__ __forceinline__ uint4 fetch(const View &v, int g) {
    constexpr int V = 16 / sizeof(T);
    const T *row = static_cast<const T *>(v.row);
    const int first = g * V - v.lead;
    if (first >= 0 && first + V <= v.vocab) return ld128(reinterpret_cast<const uint4 *>(row - v.lead) + g);
    T x[V];
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = first + e >= 0 && first + e < v.vocab ? row[first + e] : from_f32<T>(-INFINITY);
    uint4 q;
    memcpy(&q, x, 16);
    return q;
}
// NaN as -inf and inf as the largest number
__device__ __forceinline__ float tamed(float x) { return fminf(fmaxf(x, -INFINITY), MOST); }

// f(index, values) for fours of the logits of groups [g0, g1), with SOME for none that are below `floor`; the next loads are in flight
// meanwhile.  Values come tamed, but for FIRST.  Four at a time: eight would be twice the instructions to fetch, most of the time that a
// short row takes.  Spilled registers would go to L2, since shared memory takes L1's place (with 1024 threads of 64 registers
// instead of 512 of 128 they did, and the pass over 64000 weights took 67000 cycles).
enum Which { FIRST, EVERY, SOME };
template <typename T, int WHICH, typename F> __device__ __forceinline__ void walk(const View &v, int g0, int g1, float floor, F &&f) {
    constexpr int V = 16 / sizeof(T), AHEAD = WHICH == FIRST ? 6 : 3;
    auto load = [&](int g) { return WHICH != FIRST && g < v.cache_end ? cache()[g - v.cache_begin] : fetch<T>(v, g); };
    uint4 coming[AHEAD];
    int g = g0 + (int)(threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (g + 32 * i < g1) coming[i] = load(g + 32 * i);
#pragma unroll 1
    for (; g < g1; g += 32) {
        uint4 q = coming[0];
#pragma unroll
        for (int i = 0; i + 1 < AHEAD; ++i) coming[i] = coming[i + 1];
        if (g + 32 * AHEAD < g1) coming[AHEAD - 1] = load(g + 32 * AHEAD);
        if (WHICH == FIRST && g < v.cache_end) cache()[g - v.cache_begin] = q;
        const int index = g * V - v.lead;
#pragma unroll 1
        for (int part = 0; part < V; part += 4) {
            T x[4];
            memcpy(x, &q, sizeof(x));
            q.x = q.z, q.y = q.w;
            if (WHICH == SOME && fmaxf(fmaxf(to_f32(x[0]), to_f32(x[1])), fmaxf(to_f32(x[2]), to_f32(x[3]))) < floor) continue;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = WHICH == FIRST ? to_f32(x[e]) : tamed(to_f32(x[e]));
            f(index + part, y);
        }
    }
}

template <typename F> struct OneByOne {
    F f;
    __device__ __forceinline__ void operator()(int index, const float (&x)[4]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) f(index + e, x[e]);
    }
};
template <typename F> __device__ __forceinline__ OneByOne<F> one_by_one(F f) { return OneByOne<F>{f}; }

// ---- the passes, each in a function of its own: they need all registers, and hold what the leader keeps on the stack ----

// a 64-bit sum in two words, the carry by the lower one's old value
__device__ __forceinline__ void add_to(Shared &s, int bin, u64 w) {
    const unsigned lo = (unsigned)w, hi = (unsigned)(w >> 32) + (atomicAdd(&s.low[bin], lo) > ~lo);
    if (hi) atomicAdd(&s.low[BINS + bin], hi);
}
__device__ __forceinline__ void empty_bins(Shared &s) {
#pragma unroll
    for (int e = 0; e < 2 * PER; ++e) s.low[e * SM_NT + threadIdx.x] = 0;
    __syncthreads();
}
// What this CTA found goes to the leader's list.
__device__ __forceinline__ void hand_over(Shared &s) {
    Shared &to = leader();
    __syncthreads();
    if (threadIdx.x == 0) s.place = atomicAdd(&to.listed, s.found);
    __syncthreads();
    for (unsigned i = threadIdx.x; i < min(s.found, (unsigned)LIST) && s.place + i < LIST; i += SM_NT) to.list[s.place + i] = s.taken[i];
}
__device__ __forceinline__ void find(Shared &s, u64 place) {
    const unsigned at = atomicAdd(&s.found, 1u);
    if (at < LIST) s.taken[at] = place;
}

// The largest of a thread's logits and the first among equals, as a place; 0: none but -inf and NaN.
template <typename T> __device__ __noinline__ u64 first_pass(const View v, int g0, int g1) {
    float top = -INFINITY;
    int top_index = 0;
    walk<T, FIRST>(v, g0, g1, 0.0f, [&](int index, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            top_index = x[e] > top ? index + e : top_index;
            top = x[e] > top ? x[e] : top;  // neither -inf nor NaN
        }
    });
    return top > -INFINITY ? place_of(fminf(top, MOST), top_index) : 0;
}
// Weights by step in 12 bits of what the step's first token weighs: 4096 (1 - y / 64) for one y of a step behind it, all that 2^20 additions
// leave room for, and near enough to find where a border lies.
template <typename T> __device__ __noinline__ void guess_pass(const View v, int g0, int g1) {
    Shared &s = shared();
    const Weigher r(s);
    empty_bins(s);
    const float fine = 64.0f * r.steps;
    walk<T, EVERY>(v, g0, g1, 0.0f, [&](int, const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int z = __float2int_rz(r.below(x[e]) * fine);
            atomicAdd(&s.low[min(z >> 6, 2 * BINS - 1)], 4095u - (unsigned)(z & 63));
        }
    });
}
// All weights, above `lo` and from there on, and the tokens between `lo` and `hi`.
template <typename T, bool FILTER> __device__ __noinline__ void split_pass(const View v, int g0, int g1, int stretch) {
    Shared &s = shared();
    const Weigher r(s);
    const float lo = s.cmd.lo, hi = s.cmd.hi;
    if (threadIdx.x == 0) s.found = 0;
    __syncthreads();
    u64 ahead = 0, all = 0, slight = 0;
    walk<T, EVERY>(v, g0, g1, 0.0f, [&](int index, const float (&x)[4]) {
        float y[4];
        u64 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = r.below(x[e]) * r.steps;
            w[e] = r.near_weight(x[e]);
        }
        bool some = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (r.weighs(y[e])) all += w[e];
            if (y[e] < lo) ahead += w[e];
            if (FILTER && y[e] < lo && w[e] < r.least) slight += w[e];
            some |= y[e] >= lo && y[e] <= hi;
        }
        if (some)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (y[e] >= lo && y[e] <= hi) find(s, place_of(x[e], index + e));
    });
    ahead = warp_sum(ahead);
    all = warp_sum(all);
    if (FILTER) slight = warp_sum(slight);
    if ((threadIdx.x & 31) == 0) {
        Shared &to = leader();
        to.seg[stretch] = ahead - slight;
        atomicAdd(&to.ahead, ahead);
        atomicAdd(&to.far, all - ahead);
    }
    hand_over(s);
}
// A histogram of all weights; those behind the last step in one sum.
template <typename T> __device__ __noinline__ void weights_pass(const View v, int g0, int g1) {
    Shared &s = shared();
    const Weigher r(s);
    empty_bins(s);
    u64 far = 0;
    walk<T, EVERY>(v, g0, g1, 0.0f, [&](int, const float (&x)[4]) {
        u64 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = r.near_weight(x[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int bin = r.step(x[e]);
            if (bin < BINS) add_to(s, bin, w[e]);
            else if (bin < 2 * BINS) far += w[e];
        }
    });
    const u64 sum = warp_sum(far);
    if ((threadIdx.x & 31) == 0 && sum) atomicAdd(&leader().far, sum);
}
// A histogram of tokens or weights over the steps, or over the next bits of the tokens of one.
template <typename T> __device__ __noinline__ void histogram_pass(const View v, int g0, int g1) {
    Shared &s = shared();
    const Weigher r(s);
    const Command c = s.cmd;
    empty_bins(s);
    const int next = max(c.shift - 10, 0), top_bin = (1 << (c.shift - next)) - 1;
    walk<T, SOME>(v, g0, g1, c.floor, one_by_one([&](int index, float x) {
        int bin = r.step(x) - c.base;
        if (c.cut || c.op == OP_BITS) {
            const u64 place = place_of(x, index);
            if (place < c.cut) return;
            if (c.op == OP_BITS) {
                if (bin != c.step || (place >> c.shift) != c.prefix) return;
                bin = top_bin - (int)((place >> next) & (unsigned)top_bin);
            }
        }
        const u64 w = c.weights ? r.weight(x) : 1;
        if (bin >= 0 && bin < BINS) add_to(s, bin, w);
        else if (bin >= BINS && w) atomicAdd(&leader().far, w);
    }));
}
template <typename T> __device__ __noinline__ void gather_pass(const View v, int g0, int g1, int stretch) {
    Shared &s = shared();
    const Weigher r(s);
    const Command c = s.cmd;
    if (threadIdx.x == 0) s.found = 0;
    __syncthreads();
    u64 sum = 0;
    const int weighed_to = c.weights ? c.step : 0;
    walk<T, SOME>(v, g0, g1, c.floor, one_by_one([&](int index, float x) {
        const int step = r.step(x);
        if (step > c.upto && step != c.step) {
            if (step < weighed_to) {
                const u64 w = r.weight(x);
                if (w >= r.least) sum += w;
            }
            return;
        }
        const u64 place = place_of(x, index);
        if (place >= c.cut && (place >> c.shift) == c.prefix) find(s, place);
    }));
    if (c.weights) {
        sum = warp_sum(sum);
        if ((threadIdx.x & 31) == 0) leader().seg[stretch] = sum;
    }
    hand_over(s);
}
// Whether a token stays, but for its weight; most that do not are known by their step.
__device__ __forceinline__ bool stays(const Weigher &r, u64 cut, int upto, int index, float x) {
    return r.step(x) <= min(upto, 2 * BINS - 1) && !(cut && place_of(x, index) < cut);
}
__device__ __forceinline__ u64 kept(const Weigher &r, u64 cut, int upto, int index, float x) {
    const u64 w = stays(r, cut, upto, index, x) ? r.near_weight(x) : 0;
    return w >= r.least ? w : 0;
}
// The kept weights of a warp's groups.
template <typename T> __device__ __noinline__ u64 sums_pass(const View v, int g0, int g1) {
    Shared &s = shared();
    const Weigher r(s);
    const u64 cut = s.cmd.cut;
    const int upto = s.cmd.upto;
    u64 sum = 0;
    walk<T, SOME>(v, g0, g1, s.cmd.floor, [&](int index, const float (&x)[4]) {
        u64 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = r.near_weight(x[e]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (stays(r, cut, upto, index + e, x[e]) && w[e] >= r.least) sum += w[e];
    });
    return warp_sum(sum);
}
// The token among a warp's groups at which the running sum, `below` before them, exceeds the command's target.
template <typename T> __device__ __noinline__ int pick_pass(const View v, int g0, int g1, u64 below) {
    constexpr int V = 16 / sizeof(T);
    Shared &s = shared();
    const Weigher r(s);
    const u64 cut = s.cmd.cut, target = s.cmd.target;
    const int upto = s.cmd.upto, lane = threadIdx.x & 31;
#pragma unroll 1
    for (; g0 < g1; g0 += 32) {
        const int g = g0 + lane;
        T x[V];
        u64 own = 0;
        if (g < g1) {
            const uint4 q = g < v.cache_end ? cache()[g - v.cache_begin] : fetch<T>(v, g);
            memcpy(x, &q, 16);
#pragma unroll
            for (int e = 0; e < V; ++e) own += kept(r, cut, upto, g * V - v.lead + e, tamed(to_f32(x[e])));
        }
        u64 inc = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        const unsigned who = __ballot_sync(0xffffffffu, below + inc > target);
        if (who) {
            if (lane != __ffs(who) - 1) return -1;
            u64 up = below + inc - own;
            int at = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                up += kept(r, cut, upto, g * V - v.lead + e, tamed(to_f32(x[e])));
                if (up <= target) at = e + 1;
            }
            return g * V - v.lead + at;
        }
        below += __shfl_sync(0xffffffffu, inc, 31);
    }
    return -1;
}

template <typename T>
__global__ void __launch_bounds__(SM_NT, 1) sample_kernel(const SampleArgs a, const int cached) {  // groups of a warp's stretch in shared memory
    extern __shared__ __align__(16) unsigned char raw[];
    Shared &s = *reinterpret_cast<Shared *>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int row = blockIdx.x / ranks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto sync_all = [&]() {
        if (ranks == 1) __syncthreads();
        else cluster.sync();
    };
    // Completed by the wait ahead of the first store into another CTA's shared memory: by then every CTA of the cluster has started.
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (tid < ROOTS) s.root[tid] = ROOT[tid] * ONE;
    if (tid == 0) s.far = 0;
    dependent_begin();
    float t = a.temperature ? a.temperature[row] : 1.0f;
    t = t > 1e37f ? 1e37f : t;  // as good as infinite
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float mp = a.min_p ? a.min_p[row] : 0.0f, u = a.uniform[row];
    const int k = a.top_k ? a.top_k[row] : 0;

    constexpr int V = 16 / sizeof(T);
    const T *src = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
    asm volatile("" : "+l"(src));  // loads through it stay behind the wait above
    View view;
    view.row = src;
    view.lead = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    view.vocab = a.vocab;
    const int ngroups = (a.vocab + view.lead + V - 1) / V;
    const int stretches = ranks * SM_WARPS;
    auto stretch = [&](int w) { return (int)((unsigned)ngroups * (unsigned)w / (unsigned)stretches); };  // below 2^18 * 2^7
    const int mine = rank * SM_WARPS + warp, g_begin = stretch(mine), g_end = stretch(mine + 1);
    auto view_of = [&](int w) {
        view.cache_begin = stretch(w) - w % SM_WARPS * cached;
        view.cache_end = stretch(w) + cached;
    };
    view_of(mine);

    // ---- the largest ----
    const u64 own_top = first_pass<T>(view, g_begin, g_end);
    u64 best = own_top;
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) s.scan[warp] = best;
    __syncthreads();
    best = s.scan[lane % SM_WARPS];
#pragma unroll
    for (int o = SM_WARPS / 2; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (ranks > 1) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (tid < ranks) cluster.map_shared_rank(&s, tid)->best[rank] = best;
        cluster.sync();
        for (int q = 0; q < ranks; ++q) best = max(best, s.best[q]);
    }
    if (best == 0 || !(t > 0.0f)) {
        if (rank == 0 && tid == 0) a.tokens[row] = best == 0 ? -1 : index_of(best);
        return;  // every CTA of the cluster leaves here, and none reads another's memory any more
    }
    const bool by_count = k > 0 && k < a.vocab, by_weight = p < 1.0f;
    Row row_of;
    row_of.top = logit_of(best);
    row_of.pre = t < 0x1p-100f ? 0x1p64f : 1.0f;
    row_of.steps = STEPS / (t * row_of.pre);
    row_of.rate = 92.33248261893152 / (double)t;  // 64 / ln 2
    row_of.least = mp > 0.0f ? (u64)ceil(fmin((double)mp, 1.0) * ONE) : 0ull;
    const Weigher r(row_of, s.root);
    const u64 least = r.least;
    // tokens far below min_p or behind the cut are not weighed: two steps more than min_p's own, for the rounding of the step
    const int least_step = least ? (int)(STEPS * -__logf(fminf(mp, 1.0f)) + 2.0f) : 0x7fffffff;
    auto stretch_of = [&](int index) {
        const int g = (index + view.lead) / V;
        int to = (int)((unsigned)g * (unsigned)stretches / (unsigned)ngroups);
        while (stretch(to + 1) <= g) ++to;
        while (stretch(to) > g) --to;
        return to;
    };
    auto quota = [&](u64 sum) -> u64 {  // tokens stay while the weights before them are below this
        const double want = ceil((double)p * (double)sum);
        return want < 1.0 ? 1ull : (u64)want;
    };
    auto draw_at = [&](u64 sum) -> u64 {  // the token at which the running sum exceeds this
        const u64 x = u > 0.0f ? (u64)((double)u * (double)sum) : 0ull;
        return x < sum ? x : sum - 1;
    };
    // A logit below those of the steps up to this one, and one not below those from this one on.  A step is off by some 2^-22 of itself; the
    // rest is exact enough in 64 bits, down to the smallest t, and rounded outwards.
    const double width = (double)t / STEPS;
    auto edge = [&](int step) { return step < 2 * BINS ? __double2float_rd((double)r.top - (step + 1) * width * 1.00001) : -INFINITY; };
    auto upper_edge = [&](int step) { return step ? fminf(__double2float_ru((double)r.top - step * width * 0.99999), r.top) : r.top; };
    auto sums_command = [&](u64 cut) {
        Command c{};
        c.op = OP_SUMS; c.cut = cut;
        c.upto = least_step;
        if (cut) c.upto = min(c.upto, r.step(logit_of(cut)));
        c.floor = edge(c.upto);
        return c;
    };

    // The leader's progress: which filter is being cut, the histogram's first step, the quota that is left, whether seg is complete.
    bool weights = !by_count, tried = false, rough = by_count && k <= ranks * SM_NT / 2, summed = false;
    int base = 0;
    u64 rest = 0, cut = 0, whole = 0;
    if (tid == 0) {  // the first pass: nobody has to say so
        Command c{};
        c.shift = PLACE_BITS;
        c.weights = weights;
        c.op = rough ? OP_TOPS : by_count ? OP_STEPS : OP_GUESS;
        c.floor = edge(BINS - 1);
        s.cmd = by_count || by_weight ? c : sums_command(0);
        s.row = row_of;
    }
    __syncthreads();
    auto publish = [&](const Command &c) {  // what the next pass is for
        __syncthreads();  // everybody has read the word before
        if (tid == 0) {
            s.cmd = c;
            s.listed = 0;
            if (c.op == OP_STEPS || c.op == OP_BITS || c.op == OP_SPLIT) s.far = s.ahead = 0;
        }
        __syncthreads();
        constexpr int WORDS = sizeof(Command) / 4;
        for (int i = tid; i < WORDS * (ranks - 1); i += SM_NT)
            reinterpret_cast<unsigned *>(&cluster.map_shared_rank(&s, 1 + i / WORDS)->cmd)[i % WORDS] = reinterpret_cast<const unsigned *>(&s.cmd)[i % WORDS];
    };
    for (;;) {
        // ---- the pass ----
        const int op = s.cmd.op;
        const int shift = s.cmd.shift, next = max(shift - 10, 0), top_bin = (1 << (shift - next)) - 1;
        if (op == OP_TOPS) {
            empty_bins(s);
            const int bin = own_top ? r.step(logit_of(own_top)) : BINS;
            if (bin < BINS) atomicAdd(&s.low[bin], 1u);
        } else if (op == OP_GUESS) {
            guess_pass<T>(view, g_begin, g_end);
        } else if (op == OP_SPLIT) {
            if (least) split_pass<T, true>(view, g_begin, g_end, mine);
            else split_pass<T, false>(view, g_begin, g_end, mine);
        } else if (op == OP_STEPS && s.cmd.weights && s.cmd.base == 0 && s.cmd.cut == 0) {
            weights_pass<T>(view, g_begin, g_end);
        } else if (op == OP_STEPS || op == OP_BITS) {
            histogram_pass<T>(view, g_begin, g_end);
        } else if (op == OP_GATHER) {
            gather_pass<T>(view, g_begin, g_end, mine);
        } else if (op == OP_SUMS) {
            const u64 sum = sums_pass<T>(view, g_begin, g_end);
            if (lane == 0) leader().seg[mine] = sum;
        } else if (op == OP_PICK) {  // the kept weights of the parts of one stretch, and where among them the target is
            const int at = s.cmd.warp;
            const u64 target = s.cmd.target;
            if (at / SM_WARPS != rank) return;
            const int g0 = stretch(at), g1 = stretch(at + 1), part = (g1 - g0 + SM_WARPS - 1) / SM_WARPS;
            const int from = min(g0 + warp * part, g1), to = min(from + part, g1);
            view_of(at);
            const u64 sum = sums_pass<T>(view, from, to);
            if (lane == 0) s.scan[warp] = sum;
            __syncthreads();
            u64 below = 0;
            for (int w = 0; w < warp; ++w) below += s.scan[w];
            if (below > target || target >= below + sum) return;  // but one warp
            const int token = pick_pass<T>(view, from, to, below);
            if (token >= 0) a.tokens[row] = token;
            return;
        } else {
            return;
        }
        sync_all();

        // ---- the leader looks at what it found ----
        if (rank == 0 && op == OP_GUESS) {
            // Where the cumulated weights come to 2^-16 of all less than the quota, and where to 2^-16 more: rough weights are off by
            // 2^-13 each at most, to either side, and their sums by less.  The tokens of a step lie in it by chance, so that their number
            // up to a place is off by half the root of their number: four times that is looked at, and a few tokens more.  Of a step
            // with few tokens, or of values of 16 bits, which lie in clumps, all of them are.
            constexpr int MINE = 2 * PER;
            float n[MINE], tokens = 0.0f;
            u64 w[MINE], own = 0;
#pragma unroll
            for (int e = 0; e < MINE; ++e) {
                const int at = MINE * tid + e;
                u64 q = 0;
                for (int o = 0; o < ranks; ++o) q += cluster.map_shared_rank(&s, o)->low[at];
                if (at == 2 * BINS - 1) q = 0;  // the rest of the row
                n[e] = (float)q * (1.0f / 4096.0f);
                w[e] = (u64)((float)q * __expf(at * (-1.0f / STEPS)) * 1048576.0f);
                tokens += n[e];
                own += w[e];
            }
            ulonglong2 sum = block_scan(s, own);
            float before = (float)block_scan(s, (u64)(tokens + 0.5f)).x;
            const u64 want = (u64)((double)p * (double)sum.y), slack_of = sum.y >> 16;
            const u64 from = want > slack_of ? want - slack_of : 1, to = max(min(want + slack_of, sum.y), (u64)1);
#pragma unroll
            for (int e = 0; e < MINE; ++e) {
                const float about = fmaxf(n[e], 1.0f), reach = (2.0f * sqrtf(about) + 4.0f) / about;
                const int at = MINE * tid + e;
                const bool whole_step = sizeof(T) == 2 || about <= HANDFUL / 3;
                if (sum.x < from && from <= sum.x + w[e]) {
                    const float place = at + (float)(from - sum.x) / (float)w[e] - reach;
                    s.lo = whole_step ? fminf(place, (float)at) : place;
                }
                if (sum.x < to && to <= sum.x + w[e]) {
                    const float part = (float)(to - sum.x) / (float)w[e], place = at + part + reach;
                    s.hi = whole_step ? fmaxf(place, at + 1.0f) : place;
                    s.few = before + (whole_step ? 1.0f : part + reach) * about <= HANDFUL / 2;
                }
                sum.x += w[e];
                before += n[e];
            }
            __syncthreads();
            Command c{};
            c.op = OP_SPLIT;
            c.lo = s.few ? -INFINITY : s.lo;  // few tokens in all: all of them
            c.hi = s.hi;
            publish(c);
        } else if (rank == 0) {
            Command c = s.cmd;
            const int done = op;
            u64 m[PER] = {};  // this thread's steps of the whole row
            if (done == OP_TOPS || done == OP_STEPS || done == OP_BITS || (done == OP_GATHER && !tried))
                for (int q = 0; q < ranks; ++q) {
                    const Shared *o = cluster.map_shared_rank(&s, q);
#pragma unroll
                    for (int e = 0; e < PER; ++e) m[e] += (u64)o->low[BINS + PER * tid + e] << 32 | o->low[PER * tid + e];
                }
            // The bin in which the running sum of m reaches q, and q less what comes before it; BINS if it lies behind.
            int bin = 0;
            bool look = done == OP_TOPS || done == OP_STEPS || done == OP_BITS, cut_here = false, missed = false;
            const unsigned listed = s.listed;
            bool handful = false;
            if (done == OP_SPLIT) {
                whole = s.ahead + s.far;
                const u64 q = quota(whole);
                if (listed > LIST || s.ahead >= q) missed = true;
                else if (listed <= HANDFUL) handful = true;
                else {
                    rest = q - s.ahead;
                    cut_here = summed = true;
                }
            }
            if (done == OP_GATHER && !tried && listed <= HANDFUL) tried = handful = true;
            if (handful) {
                // A handful: everybody's place among the others, the weights before it and up to it in order of index are counted
                // out, by as many threads a token as there are; sorting takes longer, step after step.
                const int have = (int)listed;
                int parts = SM_NT / 32;
                while (SM_NT / parts < have) parts >>= 1;
                const int i = tid / parts;
                u64 *weight = s.taken, *stays = s.taken + HANDFUL;
                if (tid < have) weight[tid] = r.weight(logit_of(s.list[tid]));
                __syncthreads();
                const u64 place = i < have ? s.list[i] : 0, w = i < have ? weight[i] : 0;
                u64 before = 0;
                int rank_of = 0;
#pragma unroll 4
                for (int j = tid % parts; j < have; j += parts) {
                    const u64 other = weight[j];
                    const bool ahead = s.list[j] > place;
                    before += ahead ? other : 0;
                    rank_of += ahead;
                }
                for (int o = parts / 2; o; o >>= 1) {
                    before += __shfl_xor_sync(0xffffffffu, before, o);
                    rank_of += __shfl_xor_sync(0xffffffffu, rank_of, o);
                }
                const bool asks = i < have && tid % parts == 0;
                if (done == OP_SPLIT) before += s.ahead;
                if (asks && rank_of == (by_count ? min(k, have) : have) - 1) s.found_q = before + w;  // what top-k leaves, or all down to here
                __syncthreads();
                const u64 sum = s.found_q, q = quota(by_count ? sum : whole);
                missed = done == OP_SPLIT && (have == 0 || (sum < q && sum < whole));
                const bool kept_one = (!by_count || rank_of < k) && !(by_weight && before >= q) && w >= least;
                if (asks) stays[i] = kept_one ? w : 0;
                __syncthreads();
                if (done == OP_SPLIT && c.lo > -INFINITY) {  // those ahead are kept, too
                    cut_here = summed = !missed;
                    if (asks && (before < q && (before + w >= q || rank_of == have - 1))) s.found_q = place;
                    if (asks && kept_one && !missed) atomicAdd(&s.seg[stretch_of(index_of(place))], w);
                } else if (!missed) {
                    u64 up = 0, all = 0;
#pragma unroll 4
                    for (int j = tid % parts; j < have; j += parts) {
                        const u64 other = stays[j];
                        all += other;
                        up += index_of(s.list[j]) <= index_of(place) ? other : 0;
                    }
                    for (int o = parts / 2; o; o >>= 1) {
                        up += __shfl_xor_sync(0xffffffffu, up, o);
                        all += __shfl_xor_sync(0xffffffffu, all, o);
                    }
                    const u64 target = draw_at(all);
                    if (asks && kept_one && up - w <= target && target < up) a.tokens[row] = index_of(place);
                    c.op = OP_LEAVE;
                }
            } else if (done == OP_GATHER) {
                if (!tried) {  // all tokens up to the step that the first filter ends in
                    tried = true;
                    if (listed <= LIST) {
                        sort_list(s, (int)listed);
                        u64 place[EACH], w[EACH], own = 0;
#pragma unroll
                        for (int e = 0; e < EACH; ++e) {
                            const int at = EACH * tid + e;
                            place[e] = at < (int)listed ? s.list[at] : 0;
                            w[e] = at < (int)listed && (!by_count || at < k) ? r.weight(logit_of(place[e])) : 0;
                            own += w[e];
                        }
                        ulonglong2 sum = block_scan(s, own);
                        const u64 q = quota(by_count ? sum.y : whole);
                        u64 stay = 0;
#pragma unroll
                        for (int e = 0; e < EACH; ++e) {
                            const bool out = (by_weight && sum.x >= q) || w[e] < least;
                            sum.x += w[e];
                            if (out) w[e] = 0;
                            stay += w[e] != 0;
                        }
                        // the kept ones are the first: in order of index, then the running sum
                        const int kept_tokens = (int)block_scan(s, stay).y;
#pragma unroll
                        for (int e = 0; e < EACH; ++e)
                            s.list[EACH * tid + e] = w[e] ? (place[e] & ((1 << INDEX_BITS) - 1)) << 32 | (unsigned)(EACH * tid + e) : 0;
                        sort_list(s, kept_tokens);
#pragma unroll
                        for (int e = 0; e < EACH; ++e) s.taken[EACH * tid + e] = w[e];
                        __syncthreads();
                        own = 0;
#pragma unroll
                        for (int e = 0; e < EACH; ++e) {
                            const int at = EACH * tid + e;
                            place[e] = at < kept_tokens ? s.list[at] : 0;
                            w[e] = at < kept_tokens ? s.taken[(unsigned)place[e]] : 0;
                            own += w[e];
                        }
                        sum = block_scan(s, own);
                        const u64 target = draw_at(sum.y);
#pragma unroll
                        for (int e = 0; e < EACH; ++e) {
                            if (w[e] && sum.x <= target && target < sum.x + w[e]) a.tokens[row] = index_of(place[e] >> 32);
                            sum.x += w[e];
                        }
                        c.op = OP_LEAVE;
                    } else if (rough) {  // now the tokens themselves
                        tried = rough = false;
                        c = Command{};
                        c.op = OP_STEPS; c.shift = PLACE_BITS; c.floor = edge(BINS - 1);
                    } else {
                        look = true;
                    }
                } else if (listed <= LIST) {
                    cut_here = true;
                } else {
                    c.op = OP_BITS;
                    c.weights = weights;
                }
            }
            if (look) {
                u64 own = 0;
#pragma unroll
                for (int e = 0; e < PER; ++e) own += m[e];
                ulonglong2 sum = block_scan(s, own);
                if (done != OP_BITS && base == 0) {
                    whole = sum.y + s.far;
                    rest = weights ? quota(whole) : (u64)k;
                }
                if (tid == 0) { s.found_bin = BINS; s.found_q = rest - sum.y; }
                __syncthreads();
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    if (sum.x < rest && rest <= sum.x + m[e]) { s.found_bin = PER * tid + e; s.found_q = rest - sum.x; }
                    sum.x += m[e];
                }
                __syncthreads();
                bin = s.found_bin;
                if (done == OP_BITS) {
                    rest = s.found_q;
                    c.prefix = c.prefix << (c.shift - next) | (unsigned)(top_bin - bin);
                    c.shift = next;
                    c.op = OP_GATHER;
                    c.weights = 0;
                    summed = false;
                } else if (!tried) {
                    // How many tokens there are up to that step: their number, or what their weights come to at the least that a token
                    // of the step weighs (a few more, and the gathering sees for itself).
                    u64 up = 0;
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        const int at = PER * tid + e;
                        if (at <= bin) up += weights ? (u64)ceilf((float)m[e] * (float)(1.0 / ONE) * __expf((at + 1) / STEPS)) : m[e];
                    }
                    const u64 tokens = block_scan(s, up).y;
                    const bool few = bin < BINS && tokens <= (weights ? LIST + LIST / 2 : LIST);
                    if (rough && !few) {
                        rough = look = false;
                        c.op = OP_STEPS;
                    } else if (few) {
                        c.op = OP_GATHER; c.upto = bin; c.step = -1; c.weights = 0;
                        c.floor = edge(c.upto);
                        c.shift = PLACE_BITS; c.prefix = 0;
                        look = false;
                    } else {
                        tried = true;
                    }
                }
                if (look && done != OP_BITS) {
                    rest = s.found_q;
                    if (bin == BINS && base == 0) {
                        base = BINS;
                        c.op = OP_STEPS; c.base = base; c.weights = weights; c.floor = edge(2 * BINS - 1);
                    } else if (bin == BINS) {  // what is further below weighs nothing: nothing that can be drawn is cut
                        cut_here = true;
                        rest = 0;
                    } else {
                        // the tokens of that step: their places agree in the bits that the ends of the step have in common
                        c.step = base + bin;
                        c.upto = -1;
                        c.base = 0;
                        c.floor = edge(c.step);
                        const float above = upper_edge(c.step);
                        const unsigned high = order_of(above), low = order_of(c.floor);
                        const int same = c.floor <= above ? __clz(high ^ low) : 0;
                        c.shift = PLACE_BITS - same;
                        c.prefix = same ? (u64)high >> (32 - same) : 0;
                        c.op = OP_GATHER;
                        c.weights = summed = weights && cut == 0;  // the last filter
                    }
                }
            }
            if (cut_here && handful) {
                __syncthreads();
                cut = s.found_q;
            } else if (cut_here) {
                if (rest) {
                    const int have = (int)s.listed;
                    sort_list(s, have);
                    u64 w[EACH], own = 0;
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const int at = EACH * tid + e;
                        w[e] = at >= have ? 0 : weights ? r.weight(logit_of(s.list[at])) : 1;
                        own += w[e];
                    }
                    const ulonglong2 sum = block_scan(s, own);
                    missed = done == OP_SPLIT && sum.y < rest && (have == 0 || sum.y < s.far);
                    u64 before = sum.x;
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const int at = EACH * tid + e;
                        // the last kept one is where the next is not kept
                        if (at < have && before < rest && !missed) {
                            const u64 place = s.list[at];
                            if (at + 1 == have || before + w[e] >= rest) s.found_q = place;
                            if (summed && w[e] >= least) {  // to the stretch that it lies in
                                atomicAdd(&s.seg[stretch_of(index_of(place))], w[e]);
                            }
                        }
                        before += w[e];
                    }
                    __syncthreads();
                    cut = s.found_q;
                } else {
                    summed = false;
                }
                if (missed) {
                    cut_here = false;
                } else if (!weights && by_weight) {  // the other filter, among what is left
                    weights = true;
                    base = 0;
                    c = Command{};
                    c.op = OP_STEPS; c.shift = PLACE_BITS; c.weights = 1; c.cut = cut; c.floor = edge(r.step(logit_of(cut)));
                } else if (!summed) {
                    c = sums_command(cut);
                }
            }
            if (done == OP_SUMS || (cut_here && summed)) {
                __syncthreads();
                const u64 own = tid < stretches ? s.seg[tid] : 0;
                const ulonglong2 sum = block_scan(s, own);
                const u64 target = draw_at(sum.y);
                if (own && sum.x <= target && target < sum.x + own) {
                    s.found_bin = tid;
                    s.found_q = target - sum.x;
                }
                __syncthreads();
                c = sums_command(cut);
                c.op = OP_PICK; c.warp = s.found_bin; c.target = s.found_q;
            }
            if (missed) {  // the border is not where it was thought to be: step by step
                tried = summed = false;
                c = Command{};
                c.op = OP_STEPS; c.shift = PLACE_BITS; c.weights = 1; c.floor = edge(BINS - 1);
            }
            publish(c);
        }
        sync_all();
    }
}

template <typename T> int launch_sample(const SampleArgs &a, size_t rows, cudaStream_t st) {
    auto kern = sample_kernel<T>;
    // Ranks: as many as the machine has room for (a CTA fills an SM), a few thousand logits each at least
    unsigned ranks = 1;
    while (ranks < MAX_CLUSTER && rows * ranks * 2 <= (size_t)sm_count() && (size_t)a.vocab >= (size_t)ranks * 2 * 4096) ranks *= 2;
    // of every warp's stretch, as many groups as there is room for
    const size_t base = (sizeof(Shared) + 15) / 16 * 16, groups = ((size_t)a.vocab * sizeof(T) + 31) / 16 / (ranks * SM_WARPS) + 1;
    const size_t room = (227 * 1024 - base) / 16 / SM_WARPS, cached = groups < room ? groups : room;
    const size_t smem = base + cached * SM_WARPS * 16;
    XN_ENSURE_SMEM(kern, smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ranks));
    cfg.blockDim = dim3(SM_NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    XN_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a, (int)cached));
    return XN_OK;
}

}  // namespace
}  // namespace xn

using namespace xn;

extern "C" int xn_mm_sample(xn_dtype dtype, int64_t *tokens, const void *logits, size_t row_stride, size_t rows, size_t vocab,
                            const float *uniform, const float *temperature_or_null, const int32_t *top_k_or_null,
                            const float *top_p_or_null, const float *min_p_or_null, void *stream) {
    XN_API_RANGE("xn_mm_sample");
    XN_REQUIRE(valid_dtype(dtype), "sample: unknown dtype %d", (int)dtype);
    XN_REQUIRE(vocab <= (1u << 20), "sample: a vocabulary of %zu tokens (at most %u)", vocab, 1u << 20);
    if (rows == 0) return XN_OK;
    XN_REQUIRE(vocab > 0, "sample: an empty vocabulary");
    XN_REQUIRE(rows <= 0x0fffffffull, "sample: %zu rows are too many", rows);
    XN_REQUIRE(tokens && logits && uniform, "sample: null pointer");
    XN_REQUIRE(aligned(logits, dtype_size(dtype)), "sample: logits are not aligned to their type");
    SampleArgs a{logits, row_stride, (int)vocab, uniform, temperature_or_null, top_p_or_null, min_p_or_null, top_k_or_null, tokens};
    XN_DISPATCH_DTYPE(dtype, T, return launch_sample<T>(a, rows, (cudaStream_t)stream));
}

