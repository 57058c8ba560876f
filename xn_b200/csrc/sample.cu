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
// Weights are whole numbers, 2^42 w rounded, from a 64-bit exponential (an f32 one below e^-16, where it is as good): sums of up to 2^20 of them are exact in 64 bits, so the
// result depends neither on the order in which threads add nor on how the row is shared out, and a border between two
// tokens is off by 2^-42 of the largest weight (sums in f32 would be off by 2^-24, and with a vocabulary of 10^5 borders one row in
// some hundred would draw the neighbour).
//
// A CTA takes a row, or a cluster of them, a contiguous slice each (kept in shared memory where it fits).  The first one leads:
// it looks at what a pass over the row found, and says what the next pass is for:
//   the largest logit;
//   with top-k or top-p, a histogram over 1024 equal steps of (top - x) / t and the rest behind them, which finds the step that the filter
//   ends in -- for top-p of all weights, for top-k of the threads' own largest logits alone: there are k tokens at least down to the
//   step in which the k-th of those lies -- and then the tokens up to that step: where they are few (2048), they are sorted, and all
//   filters and the draw are done among them;
//   where they are many, the tokens of that step alone (split further by the next bits of their 64-bit order while they are too
//   many), which give the exact end;
//   the kept weights of every warp's stretch of the row, and the stretch that the draw falls into.
// Bound: the latency of the passes for few rows; for many, the 64-bit operations of the weights (eleven each), the histogram's
// additions and the reads.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"

namespace xn {
namespace {
namespace cg = cooperative_groups;

typedef unsigned long long u64;
constexpr int SM_NT = 1024, SM_WARPS = SM_NT / 32;
constexpr int BINS = SM_NT;             // steps of a histogram; what is behind the last counts as one more
constexpr int EACH = 2, LIST = EACH * SM_NT;  // tokens that are sorted, and of those a thread's
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

enum Op { OP_TOPS, OP_STEPS, OP_BITS, OP_GATHER, OP_SUMS, OP_PICK, OP_LEAVE };
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
};

struct Shared {
    Command cmd;
    u64 list[LIST], taken[LIST];     // the leader's, and what this CTA found
    unsigned low[BINS], high[BINS];  // per step: tokens, or their weights as two words
    double root[ROOTS];              // 2^(i / 64)
    u64 seg[MAX_CLUSTER * SM_WARPS];
    u64 scan[SM_WARPS];
    u64 best[MAX_CLUSTER];
    u64 far;                         // behind the histogram
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

struct Row {
    float top, steps;
    float fall;   // (top - x) / t in octaves, falling: (top - x) * fall
    double rate;  // (x - top) / t in 64ths of an octave: (x - top) * rate
    const double *root;
    __device__ __forceinline__ int step(float x) const {
        return min(__float2int_rz((top - x) * steps), 2 * BINS);  // beyond 32 all is one step; 0 for top itself, whatever t
    }
    // 2^42 exp((x - top) / t), rounded, of a token of the first BINS steps, 16 t: 2^(i / 64) from a table, the rest (less than a 128th of
    // an octave, y its logarithm) as 1 + y + y^2 / 2 + y^3 / 6 + y^4 / 24, off by y^5 / 120 = 4e-14.
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
        p = __hiloint2double(__double2hiint(p) + ((n >> 6) + 42) * (1 << 20), __double2loint(p));
        return (u64)__double_as_longlong(p + INT) & 0xfffffffffffffull;
    }
    // The same of one further below, less than 2^19: f32 is off by 1.5 at most.  With FAR_BITS added.
    static constexpr unsigned FAR_BITS = 0x4b000000u;  // 2^23: a sum with it is rounded to a whole number, which is its low bits
    __device__ __forceinline__ unsigned far_weight(float below) const {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaf(below, fall, 42.0f)));
        return __float_as_uint(w + 8388608.0f);
    }
    // by the step, as the histogram parts them
    __device__ __forceinline__ u64 weight(float x) const { return step(x) < BINS ? near_weight(x) : (u64)(far_weight(top - x) - FAR_BITS); }
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
// Sorts the first `count` values of the list in falling order: value e of thread tid is the EACH * tid + e-th.  Exchanges within a
// thread, within a warp by shuffles, and beyond through `taken`; only the warps that hold any take part.
__device__ __noinline__ void sort_list(Shared &s, int count) {
    const int tid = threadIdx.x;
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
                    for (int e = 0; e < EACH; ++e) y[e] = x[e ^ 1];
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

template <typename T>
__global__ void __launch_bounds__(SM_NT, 1) sample_kernel(const SampleArgs a, const int cached) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared &s = *reinterpret_cast<Shared *>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int row = blockIdx.x / ranks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    Shared *leader = cluster.map_shared_rank(&s, 0);
    auto sync_all = [&]() {
        if (ranks == 1) __syncthreads();
        else cluster.sync();
    };
    if (tid < ROOTS) s.root[tid] = ROOT[tid];
    if (tid == 0) s.far = 0;
    dependent_begin();
    float t = a.temperature ? a.temperature[row] : 1.0f;
    t = t > 1e37f ? 1e37f : t;  // as good as infinite
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float mp = a.min_p ? a.min_p[row] : 0.0f, u = a.uniform[row];
    const int k = a.top_k ? a.top_k[row] : 0;
    Row r;
    r.steps = STEPS / t;
    r.rate = 92.33248261893152 / (double)t;  // 64 / ln 2
    r.fall = fmaxf(-1.4426950408889634f / t, -MOST);
    r.root = s.root;

    constexpr int V = 16 / sizeof(T);
    const T *src = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
    const int lead = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));  // elements into a 16-byte group
    asm volatile("" : "+l"(src));  // loads through it stay behind the wait above
    const T *groups = src - lead;
    const int ngroups = (a.vocab + lead + V - 1) / V;
    const int stretches = ranks * SM_WARPS;
    auto stretch = [&](int w) { return (int)((unsigned)ngroups * (unsigned)w / (unsigned)stretches); };  // below 2^18 * 2^7
    const int mine = rank * SM_WARPS + warp, g_begin = stretch(mine), g_end = stretch(mine + 1);
    // the first groups of the CTA's slice stay in shared memory, as many as there is room for
    uint4 *cache = reinterpret_cast<uint4 *>(raw + (sizeof(Shared) + 15) / 16 * 16) - stretch(rank * SM_WARPS);
    const int cache_end = stretch(rank * SM_WARPS) + cached;
    // a group's logits, -inf outside the row
    auto fetch = [&](int g) -> uint4 {
        const int first = g * V - lead;
        if (first >= 0 && first + V <= a.vocab) return ld128(reinterpret_cast<const uint4 *>(groups) + g);
        T x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = first + e >= 0 && first + e < a.vocab ? src[first + e] : from_f32<T>(-INFINITY);
        uint4 v;
        memcpy(&v, x, 16);
        return v;
    };
    // f(index, value) for the logits of groups [g0, g1) (of a group that is below `floor`, none), the next loads in flight meanwhile.  NaN comes as -inf and inf as the
    // largest number (the first pass gets both as they are).
    auto walk = [&](int g0, int g1, float floor, auto first_pass, auto &&f) __attribute__((always_inline)) {
        constexpr bool FIRST = decltype(first_pass)::value;
        constexpr int AHEAD = 3;
        auto load = [&](int g) { return !FIRST && g < cache_end ? cache[g] : fetch(g); };
        uint4 coming[AHEAD];
        int g = g0 + lane;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (g + 32 * i < g1) coming[i] = load(g + 32 * i);
#pragma unroll 1
        for (; g < g1; g += 32) {
            const uint4 v = coming[0];
#pragma unroll
            for (int i = 0; i + 1 < AHEAD; ++i) coming[i] = coming[i + 1];
            if (g + 32 * AHEAD < g1) coming[AHEAD - 1] = load(g + 32 * AHEAD);
            if (FIRST && g < cache_end) cache[g] = v;
            T x[V];
            memcpy(x, &v, 16);
            float y[V], most = -INFINITY;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                y[e] = to_f32(x[e]);
                most = fmaxf(most, y[e]);
            }
            if (FIRST || floor == -INFINITY || most >= floor) {
#pragma unroll
                for (int e = 0; e < V; ++e) f(g * V - lead + e, FIRST ? y[e] : fminf(fmaxf(y[e], -INFINITY), MOST));
            }
        }
    };

    // ---- the largest ----
    float top = -INFINITY;
    int top_index = 0;
    walk(g_begin, g_end, 0.0f, std::true_type(), [&](int index, float x) {
        top_index = x > top ? index : top_index;
        top = x > top ? x : top;  // neither -inf nor NaN
    });
    u64 best = top > -INFINITY ? place_of(fminf(top, MOST), top_index) : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) s.scan[warp] = best;
    __syncthreads();
    best = s.scan[lane % SM_WARPS];
#pragma unroll
    for (int o = SM_WARPS / 2; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (ranks > 1) {
        if (tid < ranks) cluster.map_shared_rank(&s, tid)->best[rank] = best;
        cluster.sync();
        for (int q = 0; q < ranks; ++q) best = max(best, s.best[q]);
    }
    if (best == 0 || !(t > 0.0f)) {
        if (rank == 0 && tid == 0) a.tokens[row] = best == 0 ? -1 : index_of(best);
        return;  // every CTA of the cluster leaves here, and none reads another's memory any more
    }
    r.top = logit_of(best);

    const bool by_count = k > 0 && k < a.vocab, by_weight = p < 1.0f;
    const u64 least = mp > 0.0f ? (u64)ceil(fmin((double)mp, 1.0) * ONE) : 0ull;  // the largest logit always stays
    // tokens far below min_p or behind the cut are not weighed: two steps more than min_p's own, for the rounding of the step
    const int least_step = least ? (int)(STEPS * -__logf(fminf(mp, 1.0f)) + 2.0f) : 0x7fffffff;
    auto quota = [&](u64 sum) -> u64 {  // tokens stay while the weights before them are below this
        const double want = ceil((double)p * (double)sum);
        return want < 1.0 ? 1ull : (u64)want;
    };
    auto draw_at = [&](u64 sum) -> u64 {  // the token at which the running sum exceeds this
        const u64 x = u > 0.0f ? (u64)((double)u * (double)sum) : 0ull;
        return x < sum ? x : sum - 1;
    };
    // a token's weight if it stays; most that do not are known by their step
    auto kept = [&](u64 cut, int upto, int index, float x) -> u64 {
        if (r.step(x) > upto || (cut && place_of(x, index) < cut)) return 0;
        const u64 w = r.weight(x);
        return w >= least ? w : 0;
    };
    // a logit below those of the steps up to this one, and one above those from this one on, whatever was rounded
    const float width = t / STEPS, slack = 0.01f * width + 1e-6f * fabsf(r.top);
    auto edge = [&](int step) { return step < 2 * BINS ? r.top - (step + 1) * width * 1.00001f - slack : -INFINITY; };
    auto upper_edge = [&](int step) { return step ? fminf(r.top - step * width * 0.99999f + slack, r.top) : r.top; };
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
        c.op = rough ? OP_TOPS : OP_STEPS;
        c.floor = edge(BINS - 1);
        s.cmd = by_count || by_weight ? c : sums_command(0);
    }
    __syncthreads();
    for (;;) {
        // ---- the pass ----
        const Command &c = s.cmd;
        const int next = max(c.shift - 10, 0), top_bin = (1 << (c.shift - next)) - 1;
        const float floor = c.floor;
        if (c.op == OP_TOPS || c.op == OP_STEPS || c.op == OP_BITS) {
            // a histogram over the steps, or over the next bits of the tokens of one
            s.low[tid] = s.high[tid] = 0;
            __syncthreads();
            const int from = c.base;
            // a 64-bit sum in two words, the carry by the lower one's old value
            auto add = [&](int bin, u64 w) {
                const unsigned lo = (unsigned)w, hi = (unsigned)(w >> 32) + (atomicAdd(&s.low[bin], lo) > ~lo);
                if (hi) atomicAdd(&s.high[bin], hi);
            };
            if (c.op == OP_TOPS) {
                const int bin = top > -INFINITY ? r.step(fminf(top, MOST)) : BINS;
                if (bin < BINS) atomicAdd(&s.low[bin], 1u);
            } else if (c.weights && c.op == OP_STEPS && from == 0 && c.cut == 0) {
                // all weights; those behind the last step in one sum
                unsigned far = 0, n = 0;
                walk(g_begin, g_end, -INFINITY, std::false_type(), [&](int index, float x) {
                    const int bin = r.step(x);
                    far += bin < BINS ? Row::FAR_BITS : r.far_weight(r.top - x);
                    ++n;
                    if (bin < BINS) add(bin, r.near_weight(x));
                });
                const u64 sum = warp_sum(far - n * Row::FAR_BITS);
                if (lane == 0 && sum) atomicAdd(&leader->far, sum);
            } else {
                walk(g_begin, g_end, floor, std::false_type(), [&](int index, float x) {
                    int bin = r.step(x) - from;
                    if (c.cut || c.op == OP_BITS) {
                        const u64 place = place_of(x, index);
                        if (place < c.cut) return;
                        if (c.op == OP_BITS) {
                            if (bin != c.step || (place >> c.shift) != c.prefix) return;
                            bin = top_bin - (int)((place >> next) & (unsigned)top_bin);
                        }
                    }
                    const u64 w = c.weights ? r.weight(x) : 1;
                    if (bin >= 0 && bin < BINS) add(bin, w);
                    else if (bin >= BINS && w) atomicAdd(&leader->far, w);
                });
            }
        } else if (c.op == OP_GATHER) {
            if (tid == 0) s.found = 0;
            __syncthreads();
            u64 sum = 0;
            const int all_to = c.upto, only = c.step, weighed_to = c.weights ? c.step : 0;
            walk(g_begin, g_end, floor, std::false_type(), [&](int index, float x) {
                const int step = r.step(x);
                if (step > all_to && step != only) {
                    if (step < weighed_to) {
                        const u64 w = r.weight(x);
                        if (w >= least) sum += w;
                    }
                    return;
                }
                const u64 place = place_of(x, index);
                if (place < c.cut || (place >> c.shift) != c.prefix) return;
                const unsigned at = atomicAdd(&s.found, 1u);
                if (at < LIST) s.taken[at] = place;
            });
            if (c.weights) {
                sum = warp_sum(sum);
                if (lane == 0) leader->seg[mine] = sum;
            }
            __syncthreads();
            if (tid == 0) s.place = atomicAdd(&leader->listed, s.found);
            __syncthreads();
            for (unsigned i = tid; i < min(s.found, (unsigned)LIST) && s.place + i < LIST; i += SM_NT) leader->list[s.place + i] = s.taken[i];
        } else if (c.op == OP_SUMS || c.op == OP_PICK) {
            // the kept weights of the warps' stretches; to draw, of the parts of one stretch
            int from = g_begin, to = g_end;
            if (c.op == OP_PICK) {
                if (c.warp / SM_WARPS != rank) return;
                const int g0 = stretch(c.warp), g1 = stretch(c.warp + 1), part = (g1 - g0 + SM_WARPS - 1) / SM_WARPS;
                from = min(g0 + warp * part, g1);
                to = min(from + part, g1);
            }
            u64 sum = 0;
            const u64 end = c.cut;
            const int upto = c.upto;
            walk(from, to, floor, std::false_type(), [&](int index, float x) { sum += kept(end, upto, index, x); });
            sum = warp_sum(sum);
            if (c.op == OP_SUMS) {
                if (lane == 0) leader->seg[mine] = sum;
            } else {
                if (lane == 0) s.scan[warp] = sum;
                __syncthreads();
                u64 below = 0;
                for (int w = 0; w < warp; ++w) below += s.scan[w];
                if (below > c.target || c.target >= below + sum) return;  // but one warp
#pragma unroll 1
                for (int g0 = from; g0 < to; g0 += 32) {
                    const int g = g0 + lane;
                    u64 w[V], own = 0;
                    T x[V];
                    if (g < to) {
                        const uint4 v = g < cache_end ? cache[g] : fetch(g);
                        memcpy(x, &v, 16);
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        w[e] = g < to ? kept(end, upto, g * V - lead + e, fminf(fmaxf(to_f32(x[e]), -INFINITY), MOST)) : 0;
                        own += w[e];
                    }
                    u64 inc = own;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
                        if (lane >= o) inc += y;
                    }
                    const unsigned who = __ballot_sync(0xffffffffu, below + inc > c.target);
                    if (who) {
                        if (lane == __ffs(who) - 1) {
                            u64 up = below + inc - own;
                            int at = 0;
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                up += w[e];
                                if (up <= c.target) at = e + 1;
                            }
                            a.tokens[row] = g * V - lead + at;
                        }
                        return;
                    }
                    below += __shfl_sync(0xffffffffu, inc, 31);
                }
                return;
            }
        } else {
            return;
        }
        sync_all();

        // ---- the leader looks at what it found ----
        if (rank == 0) {
            Command c = s.cmd;
            const int done = c.op;
            u64 m = 0;  // this thread's step of the whole row
            if (done == OP_TOPS || done == OP_STEPS || done == OP_BITS || (done == OP_GATHER && !tried))
                for (int q = 0; q < ranks; ++q) {
                    const Shared *o = cluster.map_shared_rank(&s, q);
                    m += (u64)o->high[tid] << 32 | o->low[tid];
                }
            // The bin in which the running sum of m reaches q, and q less what comes before it; BINS if it lies behind.
            int bin = 0;
            bool look = done == OP_TOPS || done == OP_STEPS || done == OP_BITS, cut_here = false;
            if (done == OP_GATHER) {
                const unsigned listed = s.listed;
                if (!tried) {  // all tokens up to the step that the first filter ends in
                    tried = true;
                    if (listed <= HANDFUL) {
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
                        for (int j = tid % parts; j < have; j += parts)
                            if (s.list[j] > place) {
                                before += weight[j];
                                ++rank_of;
                            }
                        for (int o = parts / 2; o; o >>= 1) {
                            before += __shfl_xor_sync(0xffffffffu, before, o);
                            rank_of += __shfl_xor_sync(0xffffffffu, rank_of, o);
                        }
                        const bool asks = i < have && tid % parts == 0;
                        if (asks && by_count && rank_of == min(k, have) - 1) s.found_q = before + w;  // what top-k leaves
                        __syncthreads();
                        const u64 q = quota(by_count ? s.found_q : whole);
                        const bool kept_one = (!by_count || rank_of < k) && !(by_weight && before >= q) && w >= least;
                        if (asks) stays[i] = kept_one ? w : 0;
                        __syncthreads();
                        u64 up = 0, all = 0;
                        for (int j = tid % parts; j < have; j += parts) {
                            const u64 other = stays[j];
                            all += other;
                            if (index_of(s.list[j]) <= index_of(place)) up += other;
                        }
                        for (int o = parts / 2; o; o >>= 1) {
                            up += __shfl_xor_sync(0xffffffffu, up, o);
                            all += __shfl_xor_sync(0xffffffffu, all, o);
                        }
                        const u64 target = draw_at(all);
                        if (asks && kept_one && up - w <= target && target < up) a.tokens[row] = index_of(place);
                        c.op = OP_LEAVE;
                    } else if (listed <= LIST) {
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
                const ulonglong2 sum = block_scan(s, m);
                if (done != OP_BITS && base == 0) {
                    whole = sum.y + s.far;
                    rest = weights ? quota(whole) : (u64)k;
                }
                if (tid == 0) { s.found_bin = BINS; s.found_q = rest - sum.y; }
                __syncthreads();
                if (sum.x < rest && rest <= sum.x + m) { s.found_bin = tid; s.found_q = rest - sum.x; }
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
                    const float up = tid > bin ? 0.0f : weights ? (float)m * (float)(1.0 / ONE) * __expf((tid + 1) / STEPS) : (float)m;
                    const u64 tokens = block_scan(s, (u64)ceilf(up)).y;
                    const bool few = bin < BINS && tokens <= (weights ? LIST + SM_NT : LIST);
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
            if (cut_here) {
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
                    u64 before = block_scan(s, own).x;
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const int at = EACH * tid + e;
                        // the last kept one is where the next is not kept
                        if (at < have && before < rest) {
                            const u64 place = s.list[at];
                            if (at + 1 == have || before + w[e] >= rest) s.found_q = place;
                            if (summed && w[e] >= least) {  // to the stretch that it lies in
                                const int g = (index_of(place) + lead) / V;
                                int to = (int)((unsigned)g * (unsigned)stretches / (unsigned)ngroups);
                                while (stretch(to + 1) <= g) ++to;
                                while (stretch(to) > g) --to;
                                atomicAdd(&s.seg[to], w[e]);
                            }
                        }
                        before += w[e];
                    }
                    __syncthreads();
                    cut = s.found_q;
                } else {
                    summed = false;
                }
                if (!weights && by_weight) {  // the other filter, among what is left
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
            __syncthreads();  // everybody has read the word before
            if (tid == 0) {
                s.cmd = c;
                s.listed = 0;
                if (c.op == OP_STEPS || c.op == OP_BITS) s.far = 0;
            }
            __syncthreads();
            constexpr int WORDS = sizeof(Command) / 4;
            for (int i = tid; i < WORDS * (ranks - 1); i += SM_NT)
                reinterpret_cast<unsigned *>(&cluster.map_shared_rank(&s, 1 + i / WORDS)->cmd)[i % WORDS] = reinterpret_cast<const unsigned *>(&s.cmd)[i % WORDS];
        }
        sync_all();
    }
}

template <typename T> int launch_sample(const SampleArgs &a, size_t rows, cudaStream_t st) {
    auto kern = sample_kernel<T>;
    // Ranks: as many as the machine has room for (a CTA fills an SM), a few thousand logits each at least
    unsigned ranks = 1;
    while (ranks < MAX_CLUSTER && rows * ranks * 2 <= (size_t)sm_count() && (size_t)a.vocab >= (size_t)ranks * 2 * 4096) ranks *= 2;
    const size_t base = (sizeof(Shared) + 15) / 16 * 16, groups = ((size_t)a.vocab * sizeof(T) + 31) / 16 / ranks + 1;
    const size_t room = (227 * 1024 - base) / 16 - 64, cached = groups < room ? groups : room;
    const size_t smem = base + cached * 16;
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

