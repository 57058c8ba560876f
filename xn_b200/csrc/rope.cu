// Rotary positions, alone and on the way into a paged cache.
//
// Pair j of a head turns by the angle a = position * freqs[j]:
//   (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
// with x0, x1 side by side (elements 2 j, 2 j + 1) or half the rotated part apart (j, j + pairs); what lies behind the rotated
// part of the head is copied.  Products and sums in f32, one rounding to the element type.
//
// The angle is formed as half turns, t = position * (freqs[j] / pi), less the nearest even number, and only the rest, at most one
// half turn, is rounded to f32 for the sine and cosine.  A product in f32 would be off by position * 2^-24 radians: 0.06 at
// position 10^6; one in 64 bits by position * 2^-53.  Here freqs[j] / pi and t are held in two numbers of 64 bits each, the second what
// the first one's rounding left (products with fma), so that the rest is off by 2^-25 half turns whatever the position, as long as t
// is below 2^52 and the position a whole number that 64-bit floats hold (2^53).  It needs no table of a length that somebody
// has to know beforehand, and one thread's pairs keep their sine and cosine for all the heads that the thread turns.
//
// Bound: latency.  A thread reads its position and its frequencies and takes sines before it asks for its heads (caches cold, DRAM is busy
// for a fifth of the time and the issue slots for less than a half).  It moves a chunk of 2 x 16 bytes per head (16-bit elements: 8 pairs, f32: 4) where the sizes and the
// alignment allow it, single pairs otherwise; several heads share its sines and cosines.  Measured: 4001 tokens x 16 heads of 64 in
// f32, 16 elements turned, 7.8 us (4.2 TB/s); append of 4096 tokens x (16 + 16 + 16) heads of 64 in f16 11.9 us (4.2 TB/s).
#include "common.cuh"

namespace xn {
namespace {

constexpr int ROPE_NT = 128;  // 256: 13.2 us instead of 11.2 for the f16 append above (before its angles were kept whole), whose last blocks run alone for longer

// One tensor [tokens, heads, head_dim] of the call: where it is read and where it goes.  dst == null marks an unused one.
struct RopePart {
    const void *src;
    void *dst;
    long long src_token, src_head;  // strides in elements
    long long dst_token, dst_head;  // paged: strides of a page's row and of a head
    int heads;
    int rotate;
    int paged;  // dst is a pool of pages, the token's row is its slot
};

struct RopeArgs {
    RopePart part[3];
    const int64_t *positions;
    const int64_t *slots;
    const double *freqs;
    long long page_stride;
    int64_t num_slots;
    int page_size;
    int tokens, head_dim, pairs;
    int interleaved;
    int rotated_chunks, chunks;  // per head
    int head_groups;             // a thread takes heads g, g + head_groups, ...
};

template <typename T, int V> struct Chunk { T v[V]; };

template <typename T, int V> __device__ __forceinline__ Chunk<T, V> load_chunk(const T *p) {
    Chunk<T, V> c;
    if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(&c) = ld_act128(p);
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) c.v[i] = ld_act(p + i);
    }
    return c;
}
template <typename T, int V> __device__ __forceinline__ void store_chunk(T *p, const Chunk<T, V> &c) {
    if constexpr (V * sizeof(T) == 16) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&c);
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = c.v[i];
    }
}

// V pairs per chunk: a chunk is two runs of V elements, `gap` elements apart.
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(ROPE_NT) rope_kernel(const RopeArgs a) {
    dependent_begin();
    const unsigned i = blockIdx.x * ROPE_NT + threadIdx.x;
    const unsigned per_token = (unsigned)(a.chunks * a.head_groups);
    const unsigned token = i / per_token, rest = i % per_token;
    if (token >= (unsigned)a.tokens) return;
    const int chunk = (int)(rest % (unsigned)a.chunks), group = (int)(rest / (unsigned)a.chunks);
    const bool turned = chunk < a.rotated_chunks;

    float cs[V], sn[V];
    if (turned) {
        const double pos = (double)a.positions[token];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            constexpr double INV_PI = 0.3183098861837907, REST = -1.9678676675182486e-17;  // 1 / pi in two numbers
            const double f = a.freqs[chunk * V + j], c = f * INV_PI, c_rest = fma(f, REST, fma(f, INV_PI, -c));
            const double t = pos * c, t_rest = fma(pos, c_rest, fma(pos, c, -t));
            const double k = t + 13510798882111488.0;  // a sum with 1.5 * 2^53 is rounded to an even number
            sincospif((float)(t - (k - 13510798882111488.0) + t_rest), &sn[j], &cs[j]);
        }
    }
    // the two runs of the chunk within its head, with and without rotation
    const int tail = 2 * a.pairs + (chunk - a.rotated_chunks) * 2 * V;
    const int turn0 = turned ? (INTER ? 2 * V * chunk : V * chunk) : tail;
    const int turn1 = turned ? (INTER ? turn0 + V : turn0 + a.pairs) : tail + V;
    const int plain0 = 2 * V * chunk, plain1 = plain0 + V;
    long long slot = 0;
    bool stored = true;
    if (a.slots) {
        const int64_t s = a.slots[token];
        stored = s >= 0 && s < a.num_slots;  // a slot outside the pool stores nothing
        if (stored) {
            const unsigned long long page = (unsigned long long)s / (unsigned)a.page_size;
            slot = (long long)page * a.page_stride;
            // the row within the page is added with the part's row stride below
            const int row = (int)((unsigned long long)s - page * (unsigned)a.page_size);
            slot += (long long)row * a.part[1].dst_token;
        }
    }
    auto turn = [&](Chunk<T, V> &x0, Chunk<T, V> &x1) {
        T u[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) { u[j] = x0.v[j]; u[V + j] = x1.v[j]; }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : V + j;
            const float xa = to_f32(u[ia]), xb = to_f32(u[ib]);
            u[ia] = from_f32<T>(xa * cs[j] - xb * sn[j]);
            u[ib] = from_f32<T>(xa * sn[j] + xb * cs[j]);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) { x0.v[j] = u[j]; x1.v[j] = u[V + j]; }
    };
    int head = group;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        const RopePart &part = a.part[p];
        const bool turns = part.rotate && turned;
        const int e0 = part.rotate ? turn0 : plain0, e1 = part.rotate ? turn1 : plain1;
        const T *src = static_cast<const T *>(part.src) + (long long)token * part.src_token;
        T *dst = static_cast<T *>(part.dst) + (part.paged ? slot : (long long)token * part.dst_token);
        if (part.paged && !stored) break;  // nor is the part behind
        const int first = head;
        constexpr int AT = 2;  // heads whose loads are in flight together
        for (; head < part.heads; head += AT * a.head_groups) {
            Chunk<T, V> x0[AT], x1[AT];
#pragma unroll
            for (int i = 0; i < AT; ++i) {
                const int h = head + i * a.head_groups;
                if (h < part.heads) {
                    x0[i] = load_chunk<T, V>(src + (long long)h * part.src_head + e0);
                    x1[i] = load_chunk<T, V>(src + (long long)h * part.src_head + e1);
                }
            }
#pragma unroll
            for (int i = 0; i < AT; ++i) {
                const int h = head + i * a.head_groups;
                if (h < part.heads) {
                    if (turns) turn(x0[i], x1[i]);
                    store_chunk<T, V>(dst + (long long)h * part.dst_head + e0, x0[i]);
                    store_chunk<T, V>(dst + (long long)h * part.dst_head + e1, x1[i]);
                }
            }
        }
        // the first of this thread's heads in the next part: they go on in steps of head_groups
        head = first - part.heads + (first < part.heads ? (part.heads - first + a.head_groups - 1) / a.head_groups * a.head_groups : 0);
    }
}

template <typename T, int V>
int launch_chunks(RopeArgs &a, cudaStream_t st) {
    a.rotated_chunks = a.pairs / V;
    a.chunks = a.head_dim / (2 * V);
    const int heads = a.part[0].heads + a.part[1].heads + a.part[2].heads;
    // Heads per thread: one as long as that leaves the machine with threads to spare; up to eight share a sine and cosine beyond.
    const size_t one_each = (size_t)a.tokens * a.chunks * heads, room = (size_t)sm_count() * 1024;
    int per = (int)(one_each / room);
    per = per < 1 ? 1 : (per > 8 ? 8 : per);
    a.head_groups = (heads + per - 1) / per;
    const size_t threads = (size_t)a.tokens * a.chunks * a.head_groups, blocks = (threads + ROPE_NT - 1) / ROPE_NT;
    if (threads > 0xffffff00ull) return fail(XN_ERR_UNSUPPORTED, "rope: too many elements for one call");
    return launch_dependent(a.interleaved ? rope_kernel<T, V, true> : rope_kernel<T, V, false>, dim3((unsigned)blocks), dim3(ROPE_NT), 0,
                            st, a);
}

template <typename T> int launch_typed(RopeArgs &a, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool vec = a.head_dim % (2 * V) == 0 && a.pairs % V == 0 && a.page_stride % V == 0;
    for (const RopePart &p : a.part)
        if (p.heads)
            vec = vec && aligned(p.src, 16) && aligned(p.dst, 16) && p.src_token % V == 0 && p.src_head % V == 0 && p.dst_token % V == 0 &&
                  p.dst_head % V == 0;
    return vec ? launch_chunks<T, V>(a, st) : launch_chunks<T, 1>(a, st);
}

int check_turn(const char *name, xn_dtype dtype, size_t tokens, size_t heads, size_t head_dim, size_t rotated) {
    XN_REQUIRE(valid_dtype(dtype), "%s: unknown dtype %d", name, (int)dtype);
    XN_REQUIRE(head_dim % 2 == 0 && head_dim <= 65536, "%s: head_dim %zu must be even and at most 65536", name, head_dim);
    XN_REQUIRE(rotated % 2 == 0 && rotated <= head_dim, "%s: %zu rotated elements of a head of %zu", name, rotated, head_dim);
    XN_REQUIRE(tokens <= 0x7fffffffull && heads <= 0x1fffffffull, "%s: %zu tokens x %zu heads is too large", name, tokens, heads);
    return XN_OK;
}

}  // namespace
}  // namespace xn

using namespace xn;

extern "C" int xn_mm_rope(xn_dtype dtype, void *dst, size_t dst_token_stride, size_t dst_head_stride, const void *src,
                          size_t src_token_stride, size_t src_head_stride, const int64_t *positions, const double *freqs, size_t tokens,
                          size_t heads, size_t head_dim, size_t rotated, int interleaved, void *stream) {
    XN_API_RANGE("xn_mm_rope");
    if (int rc = check_turn("rope", dtype, tokens, heads, head_dim, rotated)) return rc;
    if (tokens == 0 || heads == 0 || head_dim == 0) return XN_OK;
    XN_REQUIRE(dst && src && (rotated == 0 || (positions && freqs)), "rope: null pointer");
    RopeArgs a{};
    a.part[0] = RopePart{src, dst, (long long)src_token_stride, (long long)src_head_stride, (long long)dst_token_stride,
                         (long long)dst_head_stride, (int)heads, 1, 0};
    a.positions = positions; a.freqs = freqs;
    a.page_size = 1;
    a.tokens = (int)tokens; a.head_dim = (int)head_dim; a.pairs = (int)(rotated / 2); a.interleaved = interleaved != 0;
    XN_DISPATCH_DTYPE(dtype, T, return launch_typed<T>(a, (cudaStream_t)stream));
}

extern "C" int xn_mm_paged_append(xn_dtype dtype, void *k_pages, void *v_pages, size_t page_stride, size_t head_stride, size_t row_stride,
                                  size_t num_pages, size_t page_size, const void *k, size_t k_token_stride, size_t k_head_stride,
                                  const void *v, size_t v_token_stride, size_t v_head_stride, const int64_t *slots, size_t tokens,
                                  size_t kv_heads, size_t head_dim, void *q_dst_or_null, const void *q, size_t q_token_stride,
                                  size_t q_head_stride, size_t heads, const int64_t *positions, const double *freqs_or_null,
                                  size_t rotated, int interleaved, void *stream) {
    XN_API_RANGE("xn_mm_paged_append");
    const size_t q_heads = q_dst_or_null ? heads : 0;
    if (!freqs_or_null) rotated = 0;
    if (int rc = check_turn("paged_append", dtype, tokens, kv_heads > q_heads ? kv_heads : q_heads, head_dim, rotated)) return rc;
    XN_REQUIRE(page_size > 0 && page_size <= 0x7fffffffull, "paged_append: a page of %zu tokens", page_size);
    XN_REQUIRE(num_pages <= 0x7fffffffull, "paged_append: %zu pages are too many", num_pages);
    if (tokens == 0 || head_dim == 0 || kv_heads + q_heads == 0) return XN_OK;
    XN_REQUIRE(slots && (kv_heads == 0 || num_pages == 0 || (k_pages && v_pages)) && (kv_heads == 0 || (k && v)) && (q_heads == 0 || q) &&
                   (rotated == 0 || positions), "paged_append: null pointer");
    RopeArgs a{};
    a.part[0] = RopePart{q, q_dst_or_null, (long long)q_token_stride, (long long)q_head_stride, (long long)(heads * head_dim),
                         (long long)head_dim, (int)q_heads, 1, 0};
    a.part[1] = RopePart{k, k_pages, (long long)k_token_stride, (long long)k_head_stride, (long long)row_stride, (long long)head_stride,
                         (int)kv_heads, 1, 1};
    a.part[2] = RopePart{v, v_pages, (long long)v_token_stride, (long long)v_head_stride, (long long)row_stride, (long long)head_stride,
                         (int)kv_heads, 0, 1};
    a.positions = positions; a.slots = slots; a.freqs = freqs_or_null;
    a.page_stride = (long long)page_stride; a.page_size = (int)page_size; a.num_slots = (int64_t)(num_pages * page_size);
    a.tokens = (int)tokens; a.head_dim = (int)head_dim; a.pairs = (int)(rotated / 2); a.interleaved = interleaved != 0;
    XN_DISPATCH_DTYPE(dtype, T, return launch_typed<T>(a, (cudaStream_t)stream));
}
