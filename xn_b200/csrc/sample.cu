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
// Weights are whole numbers, round(2^42 w) from a 64-bit exponential: sums of up to 2^20 of them are exact in 64 bits, so the
// result depends neither on the order in which threads add nor on how the row is shared out, and a border between two
// tokens is off by 2^-43 of the largest weight at most (sums in f32 would be off by 2^-24, and with a vocabulary of 10^5 borders
// one row in some hundred would draw the neighbour).
//
// A cluster of CTAs shares a row, a contiguous slice each.  The first CTA leads: it looks at what a pass over the row
// found, and says what the next pass is for.
//   maximum, then a histogram over 2048 equal steps of (x - top) / t (counts and weights), which finds the step that a filter ends in;
//   the few tokens of that step, sorted and summed in order, give the exact end (too many for that: they are split further by the
//   next bits of their 64-bit order first);
//   kept weights per warp's stretch of the row, then the stretch in which the draw falls.
// The row comes from memory once and from L2 in the later passes.  Bound: latency of the passes for few rows, memory for many.
#include <cooperative_groups.h>

#include "common.cuh"

namespace xn {
namespace {
namespace cg = cooperative_groups;

typedef unsigned long long u64;
constexpr int SM_NT = 1024, SM_WARPS = SM_NT / 32;
constexpr int BINS = 2048, LIST = 2048;
constexpr int MAX_CLUSTER = 8;
constexpr float STEPS = 64.0f;          // histogram steps per unit of (top - x) / t
constexpr double ONE = 4398046511104.0; // 2^42

struct SampleArgs {
    const void *logits;
    size_t row_stride;
    int vocab;
    const float *uniform, *temperature, *top_p, *min_p;
    const int *top_k;
    int64_t *tokens;
};

enum Op { OP_STEPS, OP_BITS, OP_GATHER, OP_SUMS, OP_PICK };
struct Command {
    int op;
    int step;            // OP_BITS, OP_GATHER: tokens of this step
    int shift;           // ... whose order agrees with `prefix` above this bit
    int weights;         // whether weights are summed too
    u64 prefix, cut;     // tokens before `cut` in the order do not count any more
    int warp;            // OP_PICK: stretch of the row
    u64 target;
    u64 least;           // OP_SUMS, OP_PICK: smaller weights do not count
};

struct Shared {
    Command cmd;
    u64 weight[BINS];
    u64 list[LIST];
    unsigned count[BINS];
    u64 seg[MAX_CLUSTER * SM_WARPS];
    u64 scan[SM_WARPS];
    u64 best[MAX_CLUSTER];
    unsigned listed, members;
    u64 found_q, found_before;
    int found_bin;
};

// NaN counts as -inf, -0 as 0
__device__ __forceinline__ unsigned order_of(float x) {
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ u64 place_of(float x, int index) { return (u64)order_of(x) << 32 | (unsigned)~index; }

struct Row {
    float top, steps;
    double inv_t;
    __device__ __forceinline__ int step(float x) const {
        const int s = __float2int_rz((top - x) * steps);  // 0 for top itself, also where it is infinite
        return x == top ? 0 : min(max(s, 0), BINS - 1);
    }
    __device__ __forceinline__ u64 weight(float x) const {
        if (x == top) return (u64)ONE;
        const double d = ((double)x - (double)top) * inv_t;
        return d >= -31.0 ? __double2ull_rn(exp(d) * ONE) : 0ull;  // below half of 2^-42 (and where top is infinite): nothing
    }
};

template <typename T>
__global__ void __launch_bounds__(SM_NT, 1) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared &s = *reinterpret_cast<Shared *>(raw);
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), ranks = cluster.num_blocks();
    const int row = blockIdx.x / ranks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    dependent_begin();

    constexpr int V = 16 / sizeof(T);
    const T *src = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
    const int lead = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));  // elements into a 16-byte group
    asm volatile("" : "+l"(src));  // loads through it stay behind the wait above
    const T *groups = src - lead;
    const int ngroups = (a.vocab + lead + V - 1) / V;
    const int stretches = (int)ranks * SM_WARPS;
    auto stretch = [&](int w) { return (int)((long long)ngroups * w / stretches); };
    const int mine = (int)rank * SM_WARPS + warp;
    // f(first index of the group, values): values outside the row are -inf
    auto walk = [&](int g0, int g1, auto &&f) {
        for (int g = g0 + lane; g - lane < g1; g += 32) {
            float x[V];
            const int first = g * V - lead;
            if (g < g1 && first >= 0 && first + V <= a.vocab) {
                const uint4 u = ld128(reinterpret_cast<const uint4 *>(groups) + g);
                const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = to_f32(t[e]);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = g < g1 && first + e >= 0 && first + e < a.vocab ? to_f32(src[first + e]) : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = x[e] == x[e] ? x[e] + 0.0f : -INFINITY;
            f(first, x);
        }
    };
    auto block_scan = [&](u64 x, u64 &sum) {  // exclusive
        u64 inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        __syncthreads();
        if (lane == 31) s.scan[warp] = inc;
        __syncthreads();
        u64 w = s.scan[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        sum = __shfl_sync(0xffffffffu, w, 31);
        const u64 before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
        return (warp ? before : 0) + inc - x;
    };

    // ---- the largest ----
    Shared *leader = cluster.map_shared_rank(&s, 0);
    {
        u64 best = 0;
        walk(stretch(mine), stretch(mine + 1), [&](int first, const float (&x)[V]) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (x[e] != -INFINITY) best = max(best, place_of(x[e], first + e));
        });
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) s.scan[warp] = best;
        __syncthreads();
        if (warp == 0) {
            best = s.scan[lane];
#pragma unroll
            for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            if (lane < (int)ranks) cluster.map_shared_rank(&s, lane)->best[rank] = best;
        }
        cluster.sync();
    }
    u64 best = 0;
    for (unsigned r = 0; r < ranks; ++r) best = max(best, s.best[r]);
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    if (best == 0 || !(t > 0.0f)) {
        if (rank == 0 && tid == 0) a.tokens[row] = best == 0 ? -1 : (int64_t)(unsigned)~(unsigned)best;
        return;  // every CTA of the cluster leaves here, and none reads another's memory any more
    }
    Row r;
    r.top = value_of((unsigned)(best >> 32));
    r.steps = STEPS / t;
    r.inv_t = 1.0 / (double)t;

    // ---- the passes ----
    auto kept = [&](const Command &c, float x, int index) -> u64 {
        if (x == -INFINITY || place_of(x, index) < c.cut) return 0;
        const u64 w = r.weight(x);
        return w >= c.least ? w : 0;
    };
    auto run_pass = [&](const Command c) {
        if (c.op == OP_STEPS || c.op == OP_BITS) {
            for (int i = tid; i < BINS; i += SM_NT) { s.count[i] = 0; s.weight[i] = 0; }
            __syncthreads();
            const int next = max(c.shift - 11, 0), top_bin = (1 << (c.shift - next)) - 1;
            walk(stretch(mine), stretch(mine + 1), [&](int first, const float (&x)[V]) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (x[e] == -INFINITY) continue;
                    int bin = r.step(x[e]);
                    if (c.op == OP_BITS) {
                        if (bin != c.step) continue;
                        const u64 p = place_of(x[e], first + e);
                        if (p < c.cut || (c.shift < 64 && (p >> c.shift) != c.prefix)) continue;
                        bin = top_bin - (int)((p >> next) & (unsigned)top_bin);
                    }
                    atomicAdd(&s.count[bin], 1u);
                    if (c.weights) {
                        const u64 w = r.weight(x[e]);
                        if (w) atomicAdd(&s.weight[bin], w);
                    }
                }
            });
            cluster.sync();
            if (ranks > 1) {
                const int per = BINS / (int)ranks;
                for (int i = (int)rank * per + tid; i < ((int)rank + 1) * per; i += SM_NT) {
                    unsigned n = 0;
                    u64 w = 0;
                    for (unsigned q = 0; q < ranks; ++q) {
                        const Shared *o = cluster.map_shared_rank(&s, q);
                        n += o->count[i];
                        w += o->weight[i];
                    }
                    leader->count[i] = n;
                    leader->weight[i] = w;
                }
                cluster.sync();
            }
        } else if (c.op == OP_GATHER) {
            walk(stretch(mine), stretch(mine + 1), [&](int first, const float (&x)[V]) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (x[e] == -INFINITY || r.step(x[e]) != c.step) continue;
                    const u64 p = place_of(x[e], first + e);
                    if (p < c.cut || (c.shift < 64 && (p >> c.shift) != c.prefix)) continue;
                    const unsigned at = atomicAdd(&leader->listed, 1u);
                    if (at < LIST) leader->list[at] = p;
                }
            });
            cluster.sync();
        } else if (c.op == OP_SUMS) {
            u64 sum = 0;
            walk(stretch(mine), stretch(mine + 1), [&](int first, const float (&x)[V]) {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    sum += kept(c, x[e], first + e);
            });
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) leader->seg[mine] = sum;
            cluster.sync();
        } else if (c.op == OP_PICK && mine == c.warp) {
            u64 below = 0;
            bool done = false;
            walk(stretch(mine), stretch(mine + 1), [&](int first, const float (&x)[V]) {
                u64 w[V], sum = 0;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    w[e] = kept(c, x[e], first + e);
                    sum += w[e];
                }
                u64 inc = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 y = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += y;
                }
                const bool past = !done && below + inc > c.target;
                const unsigned who = __ballot_sync(0xffffffffu, past);
                if (who) {
                    if (lane == __ffs(who) - 1) {
                        u64 up = below + inc - sum;
                        int e = 0;
#pragma unroll
                        for (int k = 0; k < V; ++k) {
                            up += w[k];
                            if (up <= c.target) e = k + 1;
                        }
                        a.tokens[row] = first + e;
                    }
                    done = true;
                }
                below += __shfl_sync(0xffffffffu, inc, 31);
            });
        }
    };
    if (rank != 0) {  // the leader says what comes
        for (;;) {
            cluster.sync();
            const Command c = leader->cmd;
            if (c.op == OP_PICK) cluster.sync();  // the leader may leave once everybody has read its word
            run_pass(c);
            if (c.op == OP_PICK) return;
        }
    }
    auto say = [&](Command c) {
        __syncthreads();
        if (tid == 0) s.cmd = c;
        if (c.op == OP_GATHER && tid == 0) s.listed = 0;
        cluster.sync();
        if (c.op == OP_PICK) cluster.sync();
        run_pass(c);
    };

    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const bool by_count = k > 0 && k < a.vocab, by_weight = p < 1.0f;
    u64 cut = 0, all = 0;  // all: the weights of what is left
    if (by_count || by_weight) {
        Command c{};
        c.op = OP_STEPS; c.shift = 64; c.weights = by_weight;
        say(c);
        // the histogram of the steps outlives the passes behind it in registers: two bins a thread
        static_assert(BINS == 2 * SM_NT, "two bins per thread");
        unsigned n0 = s.count[2 * tid], n1 = s.count[2 * tid + 1];
        u64 w0 = s.weight[2 * tid], w1 = s.weight[2 * tid + 1];
        __syncthreads();
        // keeps, in order, while the measure of what came before is below q; `whole`: the measure of everything
        auto cut_at = [&](bool weights, u64 q, u64 &kept_weight) {
            u64 m0 = weights ? w0 : n0, m1 = weights ? w1 : n1, v0 = w0, v1 = w1;
            u64 kept_before = 0;  // weights before the bin that is split
            Command g{};
            g.shift = 64; g.cut = cut; g.weights = by_weight;
            bool level0 = true;
            for (;;) {
                u64 sum, wsum;
                const u64 before = block_scan(m0 + m1, sum);
                const u64 wbefore = block_scan(v0 + v1, wsum);
                if (tid == 0) s.found_bin = -1;
                __syncthreads();
                if (before < q && q <= before + m0) { s.found_bin = 2 * tid; s.found_q = q - before; s.found_before = wbefore; }
                else if (before + m0 < q && q <= before + m0 + m1) {
                    s.found_bin = 2 * tid + 1; s.found_q = q - before - m0; s.found_before = wbefore + v0;
                }
                __syncthreads();
                const int bin = s.found_bin;
                if (bin < 0) { kept_weight = kept_before + wsum; return; }  // fewer than q: nothing is cut
                q = s.found_q;
                kept_before += s.found_before;
                if (level0 && tid == bin / 2) s.members = (bin & 1) ? n1 : n0;
                __syncthreads();
                const unsigned members = level0 ? s.members : s.count[bin];
                if (level0) g.step = bin;
                else {
                    const int next = max(g.shift - 11, 0), top_bin = (1 << (g.shift - next)) - 1;
                    g.prefix = (g.shift < 64 ? g.prefix << (g.shift - next) : 0) | (unsigned)(top_bin - bin);
                    g.shift = next;
                }
                level0 = false;
                if (members <= LIST) break;
                g.op = OP_BITS;
                say(g);
                m0 = weights ? s.weight[2 * tid] : s.count[2 * tid];
                m1 = weights ? s.weight[2 * tid + 1] : s.count[2 * tid + 1];
                v0 = s.weight[2 * tid]; v1 = s.weight[2 * tid + 1];
                __syncthreads();
            }
            g.op = OP_GATHER;
            say(g);
            const int n = (int)min(s.listed, (unsigned)LIST);
            int size = 2;
            while (size < n) size <<= 1;
            for (int i = n + tid; i < size; i += SM_NT) s.list[i] = 0;
            __syncthreads();
            for (int run = 2; run <= size; run <<= 1)  // bitonic, falling
                for (int d = run >> 1; d; d >>= 1) {
                    for (int i = tid; i < size / 2; i += SM_NT) {
                        const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
                        const u64 x = s.list[lo], y = s.list[hi];
                        if ((x < y) == ((lo & run) == 0)) { s.list[lo] = y; s.list[hi] = x; }
                    }
                    __syncthreads();
                }
            const int i0 = 2 * tid, i1 = i0 + 1;
            const u64 p0 = i0 < n ? s.list[i0] : 0, p1 = i1 < n ? s.list[i1] : 0;
            const u64 x0 = i0 < n ? r.weight(value_of((unsigned)(p0 >> 32))) : 0, x1 = i1 < n ? r.weight(value_of((unsigned)(p1 >> 32))) : 0;
            u64 sum, wsum;
            const u64 c0 = weights ? x0 : (u64)(i0 < n), c1 = weights ? x1 : (u64)(i1 < n);
            const u64 before = block_scan(c0 + c1, sum);
            const u64 wbefore = block_scan(x0 + x1, wsum);
            const bool k0 = i0 < n && before < q, k1 = i1 < n && before + c0 < q;
            // the last kept one is where the next is not kept
            if (k0 && !k1) { s.found_q = p0; s.found_before = wbefore + x0; }
            if (k1 && (i1 + 1 >= n || before + c0 + c1 >= q)) { s.found_q = p1; s.found_before = wbefore + x0 + x1; }
            __syncthreads();
            cut = s.found_q;
            kept_weight = kept_before + s.found_before;
            __syncthreads();
        };
        u64 left = 0;
        if (by_count) cut_at(false, (u64)k, left);
        else {
            block_scan(w0 + w1, left);
        }
        if (by_weight) {
            double want = ceil((double)p * (double)left);
            u64 q = want < 1.0 ? 1ull : (u64)want;
            u64 unused;
            cut_at(true, q, unused);
        }
    }
    const float mp = a.min_p ? a.min_p[row] : 0.0f;
    Command c{};
    c.op = OP_SUMS; c.cut = cut;
    c.least = mp > 0.0f ? (u64)ceil(fmin((double)mp, 1.0) * ONE) : 0ull;  // the largest logit always stays
    say(c);
    {
        u64 x = tid < stretches ? s.seg[tid] : 0;
        const u64 before = block_scan(x, all);
        const float u = a.uniform[row];
        u64 target = u > 0.0f ? (u64)((double)u * (double)all) : 0ull;
        if (target >= all) target = all - 1;
        if (x && before <= target && target < before + x) {
            s.found_bin = tid;
            s.found_q = target - before;
        }
        __syncthreads();
        c.op = OP_PICK; c.warp = s.found_bin; c.target = s.found_q;
    }
    say(c);
}

template <typename T> int launch_sample(const SampleArgs &a, size_t rows, cudaStream_t st) {
    auto kern = sample_kernel<T>;
    XN_ENSURE_SMEM(kern, sizeof(Shared));
    // A row's share of the machine: a CTA of 1024 threads fills an SM, and wants a few thousand logits at least
    unsigned ranks = 1;
    while (ranks < MAX_CLUSTER && rows * ranks * 2 <= (size_t)sm_count() && (size_t)a.vocab >= (size_t)ranks * 2 * 2048) ranks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * ranks));
    cfg.blockDim = dim3(SM_NT);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    XN_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
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
